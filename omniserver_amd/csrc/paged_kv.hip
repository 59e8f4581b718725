// Pages of a paged KV cache: who holds which, where new tokens go, and beams that take over their
// parents' pages.
//
// Sequence r holds lengths[r] tokens; token t is in page tables[r][t / page_size], place t %
// page_size.  Nothing else is kept: a page is free where no sequence's table names it within its
// length, so sequences may share pages, and a page that is held no longer is free by itself.  New
// pages are the lowest free ones, in the order of the requests: the same inputs give the same tables.
#include "common.h"

#define PG_THREADS 1024
#define PG_WAVES (PG_THREADS / 64)
#define PG_MAX_PAGES (1 << 20)     // a bit each in LDS: 128 KB
#define PG_MAX_SEQS 2048

struct PageTables {
  int* tables;             // [seqs][width]
  int64_t* lengths;        // [seqs]
  int seqs, width, pages, shift, max_len;
};

__device__ __forceinline__ int pg_length(const PageTables& t, int64_t row) {
  const int64_t v = t.lengths[row];
  return (int)(v < 0 ? 0 : v > t.max_len ? t.max_len : v);
}
// pages of that many tokens
__device__ __forceinline__ int pg_pages(const PageTables& t, int64_t tokens) {
  return (int)((tokens + (1 << t.shift) - 1) >> t.shift);
}

// Sums of non-negative numbers up to 2^30, which they stay at.
__device__ __forceinline__ int pg_add(int a, int b) { return min(a + b, 1 << 30); }

// Inclusive prefix sum over the workgroup; total in all threads.  lds: PG_WAVES ints.
__device__ __forceinline__ int pg_scan(int v, int* lds, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int x = __shfl_up(v, o);
    if (lane >= o) v = pg_add(v, x);
  }
  __syncthreads();                                 // the last call's sums are read
  if (lane == 63) lds[wave] = v;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < PG_WAVES; ++w) {
    if (w == wave) before = total;
    total = pg_add(total, lds[w]);
  }
  return pg_add(v, before);
}

// First i in [0, n) with ends[i] > x (ends ascends), n if there is none.
__device__ __forceinline__ int pg_find(const int* ends, int n, int x) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (ends[mid] > x) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

// Set the bits of the pages that sequences hold; held(row) gives how many of a row's entries count
// and which one of them does not.  2^group lanes a row, four entries a lane.
template <typename Held>
__device__ __forceinline__ void pg_mark(const PageTables& t, uint32_t* used, int group, Held held) {
  const int lanes = 1 << group, l = threadIdx.x & (lanes - 1);
  for (int row = threadIdx.x >> group; row < t.seqs; row += PG_THREADS >> group) {
    int but;
    const int count = held(row, but);
    const int* entry = t.tables + (int64_t)row * t.width;
#pragma unroll 4
    for (int j = l; j < count; j += lanes) {
      const int p = entry[j];
      if (j != but && p >= 0 && p < t.pages) atomicOr(&used[p >> 5], 1u << (p & 31));
    }
  }
}

// The free pages counted in order: first[t] of them are below thread t's words; returns how many
// there are.  Bits past the pool count as used.
__device__ __forceinline__ int pg_count_free(const PageTables& t, uint32_t* used, int* first, int* lds) {
  const int words = (t.pages + 31) >> 5, per = ceil_div(words, PG_THREADS);
  int mine = 0;
  for (int w = threadIdx.x * per; w < min((int)(threadIdx.x + 1) * per, words); ++w) {
    if (w == words - 1 && (t.pages & 31)) used[w] |= ~0u << (t.pages & 31);
    mine += 32 - __popc(used[w]);
  }
  int total;
  const int upto = pg_scan(mine, lds, total);
  first[threadIdx.x] = upto - mine;
  __syncthreads();
  return total;
}

// give(rank, page) for the `want` lowest free pages; half a wave a word, a lane a bit.
template <typename Give>
__device__ __forceinline__ void pg_deal(const PageTables& t, const uint32_t* used, const int* first,
                                        int want, Give give) {
  const int words = (t.pages + 31) >> 5, per = ceil_div(words, PG_THREADS);
  const int bit = threadIdx.x & 31;
  for (int w = threadIdx.x >> 5; w < words; w += PG_THREADS / 32) {
    int rank = first[w / per];
    if (rank >= want) break;
    for (int x = w / per * per; x < w; ++x) rank += 32 - __popc(used[x]);
    const uint32_t free = ~used[w];
    rank += __popc(free & ((1u << bit) - 1));
    if ((free >> bit & 1) && rank < want) give(rank, w * 32 + bit);
  }
}

// ---------------------------------------------------------------------------
// Pages and slots for the tokens that n requests bring: request i brings counts[i] tokens to
// sequence rows[i].  It is granted where they fit max_len, its token rows fit T, and its pages are
// there: the requests' new pages are counted in order, those of a request that goes without too, so
// that one that needs none is never turned down for another.
//
// One workgroup: bits of the held pages, how many are free below each, then every free page of
// low enough rank looks up the request that it goes to.  And the attention's schedule for single
// tokens (paged_attn.hip): the sequences' keys in units of PG_UNIT stand in one line that is cut into
// at most ncols equal stretches, one a column of workgroups; a row of the schedule is
//   (keys, first column, last column, 0)
// and a column (sequence, first unit there, units in all, 0).
// ---------------------------------------------------------------------------
#define PG_UNIT 128

struct ReserveArgs {
  const int* counts;           // null: one each
  const int64_t* rows;         // null: sequence i
  const int64_t* rope_delta;   // per sequence, or null
  int n, T, dense;             // dense: request i's token is row i, counts at most one
  int axes;                    // copies of the positions
  int64_t* starts;             // [n]
  int64_t* after;              // [n]
  int64_t* token_page;         // [T]
  int64_t* token_pos;          // [T]
  int64_t* positions;          // [axes][T]
  int* granted;                // [n]
  int* cu;                     // [n + 1]
  int* schedule;               // [n][4] then [ncols][4], or null
  int ncols;
  int group, slots_here;
};

__device__ __forceinline__ void pg_slot(const PageTables& t, const ReserveArgs& r, int tok, int i,
                                        int row, int L, int at, bool ok) {
  int64_t page = -1, place = -1, pos = -1;
  if (ok) {
    const int p = L + at;
    page = t.tables[(int64_t)row * t.width + (p >> t.shift)];
    place = p & ((1 << t.shift) - 1);
    pos = p + (r.rope_delta ? r.rope_delta[row] : 0);
  }
  r.token_page[tok] = page;
  r.token_pos[tok] = place;
  for (int a = 0; a < r.axes; ++a) r.positions[(int64_t)a * r.T + tok] = pos;
}

__global__ __launch_bounds__(PG_THREADS) void page_reserve_kernel(PageTables t, ReserveArgs r) {
  extern __shared__ uint32_t pg_smem[];
  __shared__ int first[PG_THREADS], lds[PG_WAVES];
  const int tid = threadIdx.x, words = (t.pages + 31) >> 5;
  uint32_t* used = pg_smem;
  int* ends = (int*)pg_smem + words;                // new pages up to and with request i
  int* last = ends + r.n;                           // token rows up to and with request i
  for (int w = tid; w < words; w += PG_THREADS) used[w] = 0;
  auto row_of = [&](int i) { return r.rows ? r.rows[i] : (int64_t)i; };
  // tokens of request i: none where they do not fit
  auto ask = [&](int i, int& L, int& asked) {
    const int64_t row = row_of(i);
    const bool in = row >= 0 && row < t.seqs;
    L = in ? pg_length(t, row) : 0;
    asked = max(r.counts ? r.counts[i] : 1, 0);
    if (r.dense) asked = min(asked, 1);
    return in && asked <= t.max_len - L ? asked : 0;
  };
  int wanted = 0, rows_sum = 0;
  for (int base = 0; base < r.n; base += PG_THREADS) {
    const int i = base + tid;
    int need = 0, asked = 0, L;
    if (i < r.n) {
      const int c = ask(i, L, asked);
      need = pg_pages(t, L + c) - pg_pages(t, L);
    }
    // a request whose token rows run past T needs nothing: sums of token rows first
    int total;
    const int upto = pg_add(pg_scan(min(asked, 1 << 30), lds, total), rows_sum);
    rows_sum = pg_add(rows_sum, total);
    if (!r.dense && upto > r.T) need = 0;
    const int pages = pg_add(pg_scan(need, lds, total), wanted);
    wanted = pg_add(wanted, total);
    if (i < r.n) {
      ends[i] = pages;
      last[i] = r.dense ? i + 1 : upto;
    }
  }
  __syncthreads();
  pg_mark(t, used, r.group, [&](int row, int& but) {
    but = -1;
    return pg_pages(t, pg_length(t, row));
  });
  __syncthreads();
  const int left = pg_count_free(t, used, first, lds);
  pg_deal(t, used, first, min(left, wanted), [&](int rank, int page) {
    const int i = pg_find(ends, r.n, rank);
    if (i >= r.n || ends[i] > left) return;
    const int64_t row = row_of(i);
    const int j = pg_pages(t, pg_length(t, row)) + rank - (i ? ends[i - 1] : 0);
    t.tables[row * t.width + j] = page;
  });
  auto grant = [&](int i, int& L) {
    int asked;
    const int c = ask(i, L, asked);
    const bool fits = r.dense || last[i] <= r.T;
    const bool paid = ends[i] == (i ? ends[i - 1] : 0) || ends[i] <= left;
    return fits && paid ? c : 0;
  };
  __syncthreads();                                  // the tables are written
  for (int i = tid; i < r.n; i += PG_THREADS) {
    int L;
    const int c = grant(i, L);
    r.granted[i] = c;
    r.starts[i] = L;
    r.after[i] = L + c;
    r.cu[i + 1] = last[i];
    if (i == 0) r.cu[0] = 0;
    if (r.dense) pg_slot(t, r, i, i, (int)row_of(i), L, 0, c > 0);
  }
  if (!r.dense && r.slots_here) {
    for (int tok = tid; tok < r.T; tok += PG_THREADS) {
      const int i = pg_find(last, r.n, tok);
      int L = 0, c = 0;
      if (i < r.n) c = grant(i, L);
      pg_slot(t, r, tok, i, c ? (int)row_of(i) : 0, L, c ? tok - (i ? last[i - 1] : 0) : 0, c > 0);
    }
  }
  if (!r.schedule) return;
  // the schedule, over the sums of units (in place of the sums of token rows)
  int units = 0;
  __syncthreads();
  for (int base = 0; base < r.n; base += PG_THREADS) {
    const int i = base + tid;
    int L, c = 0, mine = 0, total;
    if (i < r.n && (c = grant(i, L)) > 0) mine = ceil_div(L + c, PG_UNIT);
    const int upto = pg_scan(mine, lds, total) + units;
    units += total;
    if (i < r.n) last[i] = upto;
  }
  __syncthreads();
  const int cols = min(r.ncols, units);
  auto cut = [&](int c) { return (int)((int64_t)c * units / cols); };
  auto column_of = [&](int x) { return (int)((((int64_t)x + 1) * cols - 1) / units); };
  for (int i = tid; i < r.n; i += PG_THREADS) {
    int L;
    const int c = grant(i, L), lo = i ? last[i - 1] : 0, hi = last[i];
    i32x4 v = {c ? L + c : 0, 0, 0, 0};
    if (hi > lo) {
      v[1] = column_of(lo);
      v[2] = column_of(hi - 1);
    }
    *(i32x4*)(r.schedule + 4 * i) = v;
  }
  for (int c = tid; c < r.ncols; c += PG_THREADS) {
    i32x4 v = {0, 0, 0, 0};
    if (c < cols) {
      const int lo = cut(c), i = pg_find(last, r.n, lo);
      v = (i32x4){i, lo - (i ? last[i - 1] : 0), cut(c + 1) - lo, 0};
    }
    *(i32x4*)(r.schedule + 4 * r.n + 4 * c) = v;
  }
}

// Slots of many tokens, a token a thread: the request is looked up in the sums of token rows.
__global__ __launch_bounds__(256) void page_slots_kernel(PageTables t, ReserveArgs r) {
  __shared__ int last[PG_MAX_SEQS];
  for (int i = threadIdx.x; i < r.n; i += 256) last[i] = r.cu[i + 1];
  __syncthreads();
  const int tok = blockIdx.x * 256 + threadIdx.x;
  if (tok >= r.T) return;
  const int i = pg_find(last, r.n, tok);
  const int c = i < r.n ? r.granted[i] : 0;
  const int L = c ? (int)r.starts[i] : 0;
  pg_slot(t, r, tok, i, c ? (int)(r.rows ? r.rows[i] : i) : 0, L, c ? tok - (i ? last[i - 1] : 0) : 0,
          c > 0);
}

__global__ void page_gather_kernel(PageTables t, const int* __restrict__ parents, int rows, int W);
struct CopyItem {
  int from, to, rows, pad;       // pages, token rows
};
__global__ void page_fork_kernel(PageTables t, const int* __restrict__ parents, int rows, int W,
                                 CopyItem* __restrict__ items, int group);

static int pg_shift(int page_size) {
  int s = 4;
  while (s < 10 && (1 << s) != page_size) ++s;
  return (1 << s) == page_size ? s : -1;
}

// Lanes that mark one row: as many as leave no more than one round of rows.
static int pg_group(int seqs) {
  int g = 0;
  while (g < 10 && (PG_THREADS >> (g + 1)) >= seqs) ++g;
  return g;
}

static int pg_tables_ok(const int* tables, const int64_t* lengths, int seqs, int width, int pages,
                        int page_size, int max_len) {
  if (seqs <= 0 || width <= 0 || pages <= 0 || max_len <= 0 || page_size <= 0) return OMNI_EINVAL;
  if (pg_shift(page_size) < 0 || pages > PG_MAX_PAGES || seqs > PG_MAX_SEQS) return OMNI_EUNSUPPORTED;
  if (max_len > (1 << 30) || (int64_t)pages * page_size > (1ll << 40)) return OMNI_EUNSUPPORTED;
  if ((int64_t)seqs * width > (1 << 30)) return OMNI_EUNSUPPORTED;
  if ((int64_t)width * page_size < max_len) return OMNI_EINVAL;
  if (!tables || !lengths) return OMNI_EINVAL;
  return OMNI_OK;
}

// Workgroups of these kernels may take more dynamic LDS than a launch allows by default.
static int pg_allow_lds() {
  static const int rc = [] {
    hipError_t e = hipSuccess;
    for (const void* k : {(const void*)page_reserve_kernel, (const void*)page_fork_kernel,
                          (const void*)page_gather_kernel})
      if (e == hipSuccess)
        e = hipFuncSetAttribute(k, hipFuncAttributeMaxDynamicSharedMemorySize, 152 << 10);
    return (int)e;
  }();
  return rc;
}

// How many tokens the slots are written for by the workgroup that deals the pages.
#define PG_SLOTS_HERE 2048

extern "C" int omni_page_reserve(int* tables, int64_t* lengths, int seqs, int width, int pages,
                                 int page_size, int max_len, const int* counts, const int64_t* rows,
                                 const int64_t* rope_delta, int n, int tokens, int dense, int axes,
                                 int64_t* starts, int64_t* after, int64_t* token_page,
                                 int64_t* token_pos, int64_t* positions, int* granted, int* cu,
                                 int* schedule, int columns, void* stream) {
  if (n < 0 || tokens < 0 || axes < 1) return OMNI_EINVAL;
  const int rc = pg_tables_ok(tables, lengths, seqs, width, pages, page_size, max_len);
  if (rc) return rc;
  if (n > seqs || (dense && tokens != n)) return OMNI_EINVAL;
  if (axes > 3 || tokens > (1 << 28)) return OMNI_EUNSUPPORTED;
  if (n == 0) return OMNI_OK;
  if (!starts || !after || !granted || !cu) return OMNI_EINVAL;
  if (tokens && (!token_page || !token_pos || !positions)) return OMNI_EINVAL;
  if (schedule && (!dense || columns <= 0 || ((uintptr_t)schedule & 15))) return OMNI_EINVAL;
  if (schedule && (columns > 65535 || (int64_t)n * ceil_div(max_len, PG_UNIT) > (1 << 30)))
    return OMNI_EUNSUPPORTED;
  const PageTables t = {tables, lengths, seqs, width, pages, pg_shift(page_size), max_len};
  ReserveArgs r = {counts, rows, rope_delta, n, tokens, dense, axes, starts, after, token_page,
                   token_pos, positions, granted, cu, schedule, columns, pg_group(seqs),
                   tokens <= PG_SLOTS_HERE};
  const size_t smem = 4 * ((size_t)(pages + 31) / 32 + 2 * (size_t)n);
  if (smem > (32 << 10) && pg_allow_lds()) return pg_allow_lds();
  hipLaunchKernelGGL(page_reserve_kernel, dim3(1), dim3(PG_THREADS), smem, (hipStream_t)stream, t, r);
  OMNI_CHECK_LAUNCH();
  if (!dense && !r.slots_here) {
    hipLaunchKernelGGL(page_slots_kernel, dim3(ceil_div(tokens, 256)), dim3(256), 0,
                       (hipStream_t)stream, t, r);
    OMNI_CHECK_LAUNCH();
  }
  return OMNI_OK;
}

// ---------------------------------------------------------------------------
// Beams after a choice: row s W + w of the first n W rows goes on from row s W + parents[s][w].  Its
// table and length are that row's; whole pages are shared.  A page that is not full has one holder:
// a parent's first child keeps it, every other child gets a page of its own with a copy of the rows
// that hold tokens, in all layers (a child for which there is none is left empty, as are rows
// without a parent).  Launches: the tables' columns, 16 a workgroup, through LDS (in place); lengths
// and new pages, one workgroup; the copies.
// ---------------------------------------------------------------------------
#define PG_COLS 16

__global__ __launch_bounds__(256) void page_gather_kernel(PageTables t, const int* __restrict__ parents,
                                                          int rows, int W) {
  extern __shared__ int pg_tile[];                  // [rows][PG_COLS]
  const int c = blockIdx.x * PG_COLS + (threadIdx.x & (PG_COLS - 1));
  for (int r = threadIdx.x / PG_COLS; r < rows; r += 256 / PG_COLS)
    pg_tile[r * PG_COLS + (threadIdx.x & (PG_COLS - 1))] = c < t.width ? t.tables[(int64_t)r * t.width + c] : 0;
  __syncthreads();
  if (c >= t.width) return;
  for (int r = threadIdx.x / PG_COLS; r < rows; r += 256 / PG_COLS) {
    const int p = parents[r], w = r % W;
    if (p >= 0 && p < W && p != w)
      t.tables[(int64_t)r * t.width + c] = pg_tile[(r - w + p) * PG_COLS + (threadIdx.x & (PG_COLS - 1))];
  }
}

__global__ __launch_bounds__(PG_THREADS) void page_fork_kernel(PageTables t, const int* __restrict__ parents,
                                                               int rows, int W, CopyItem* __restrict__ items,
                                                               int group) {
  extern __shared__ uint32_t pg_smem[];
  __shared__ int first[PG_THREADS], lds[PG_WAVES];
  const int tid = threadIdx.x, words = (t.pages + 31) >> 5, page = 1 << t.shift;
  uint32_t* used = pg_smem;
  int* len = (int*)pg_smem + words;                 // lengths after; ~length: with a page of its own
  int* ends = len + rows;                           // pages up to and with row r
  for (int w = tid; w < words; w += PG_THREADS) used[w] = 0;
  int wanted = 0;
  for (int base = 0; base < rows; base += PG_THREADS) {
    const int r = base + tid;
    int L = 0, total;
    bool later = false;
    if (r < rows) {
      const int w = r % W, p = parents[r];
      if (p >= 0 && p < W) {
        L = pg_length(t, r - w + p);
        for (int x = 0; x < w; ++x) later |= parents[r - w + x] == p;
        later &= (L & (page - 1)) != 0;
      }
      len[r] = later ? ~L : L;
    }
    const int upto = pg_scan(later ? 1 : 0, lds, total) + wanted;
    wanted += total;
    if (r < rows) ends[r] = upto;
  }
  __syncthreads();
  pg_mark(t, used, group, [&](int row, int& but) {
    but = -1;
    if (row >= rows) return pg_pages(t, pg_length(t, row));
    const int v = len[row], L = v < 0 ? ~v : v;
    if (v < 0) but = L >> t.shift;
    return pg_pages(t, L);
  });
  __syncthreads();
  const int left = pg_count_free(t, used, first, lds);
  for (int r = tid; r < rows; r += PG_THREADS) {
    const int v = len[r];
    if (v >= 0 || ends[r] > left) {
      t.lengths[r] = v >= 0 ? v : 0;
      items[r] = {0, 0, 0, 0};
    }
  }
  pg_deal(t, used, first, min(left, wanted), [&](int rank, int to) {
    const int r = pg_find(ends, rows, rank);
    if (r >= rows) return;
    const int L = ~len[r];
    int* entry = t.tables + (int64_t)r * t.width + (L >> t.shift);
    const int from = *entry;
    *entry = to;
    t.lengths[r] = L;
    const bool in = from >= 0 && from < t.pages;
    items[r] = {in ? from : 0, to, in ? L & (page - 1) : 0, 0};
  });
}

__global__ __launch_bounds__(256) void page_copy_kernel(half_t* __restrict__ pool, int64_t seg_stride,
                                                        int64_t page_halfs, int row_halfs,
                                                        const CopyItem* __restrict__ items) {
  const CopyItem it = items[blockIdx.y];
  if (!it.rows) return;
  half_t* seg = pool + blockIdx.x * seg_stride;
  const half8_t* from = (const half8_t*)(seg + it.from * page_halfs);
  half8_t* to = (half8_t*)(seg + it.to * page_halfs);
  const int chunks = it.rows * (row_halfs >> 3);
#pragma unroll 4
  for (int c = threadIdx.x; c < chunks; c += 256) to[c] = from[c];
}

extern "C" int omni_page_reorder(void* pool, int n_layers, int row_halfs, int* tables,
                                 int64_t* lengths, int seqs, int width, int pages, int page_size,
                                 int max_len, const int* parents, int n, int beams, int* work,
                                 int64_t work_ints, void* stream) {
  if (n_layers <= 0 || row_halfs <= 0 || n < 0 || beams <= 0) return OMNI_EINVAL;
  const int rc = pg_tables_ok(tables, lengths, seqs, width, pages, page_size, max_len);
  if (rc) return rc;
  if ((row_halfs & 7) || n_layers > (1 << 20)) return OMNI_EUNSUPPORTED;
  if ((int64_t)page_size * row_halfs > (1 << 28)) return OMNI_EUNSUPPORTED;
  if ((int64_t)n * beams > seqs) return OMNI_EINVAL;
  if (n == 0) return OMNI_OK;
  const int rows = n * beams;
  if (!pool || !parents || !work || work_ints < 4ll * rows) return OMNI_EINVAL;
  if (((uintptr_t)pool & 15) || ((uintptr_t)work & 15)) return OMNI_EINVAL;
  const PageTables t = {tables, lengths, seqs, width, pages, pg_shift(page_size), max_len};
  hipStream_t st = (hipStream_t)stream;
  if (const int e = pg_allow_lds()) return e;
  hipLaunchKernelGGL(page_gather_kernel, dim3(ceil_div(width, PG_COLS)), dim3(256),
                     (size_t)rows * PG_COLS * 4, st, t, parents, rows, beams);
  OMNI_CHECK_LAUNCH();
  const size_t smem = 4 * ((size_t)(pages + 31) / 32 + 2 * (size_t)rows);
  hipLaunchKernelGGL(page_fork_kernel, dim3(1), dim3(PG_THREADS), smem, st, t, parents, rows, beams,
                     (CopyItem*)work, pg_group(seqs));
  OMNI_CHECK_LAUNCH();
  const int64_t page_halfs = (int64_t)page_size * row_halfs;
  hipLaunchKernelGGL(page_copy_kernel, dim3(2 * n_layers, rows), dim3(256), 0, st, (half_t*)pool,
                     page_halfs * pages, page_halfs, row_halfs, (const CopyItem*)work);
  OMNI_CHECK_LAUNCH();
  return OMNI_OK;
}
