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
#define PG_MAX_PAGES (1 << 19)     // a bit each in LDS: 64 KB
#define PG_MAX_SEQS 2048
// Table entries that the dealing workgroup moves itself, against a launch that does it before: 4 rows of
// 32 entries 6.3 us a call and 9.5, 128 of 38 12.6 and 16.5, 256 of 63 19.6 and 25.3.
#define PG_TILE 16384
#define PG_LDS (152 << 10)

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

// Sums of non-negative numbers up to 2^30, which they stay at (two of those add up to 2^31, which is
// no int).
__device__ __forceinline__ int pg_add(int a, int b) {
  return (int)min((uint32_t)a + (uint32_t)b, (uint32_t)1 << 30);
}
template <bool MAX>
__device__ __forceinline__ int pg_join(int a, int b) { return MAX ? max(a, b) : pg_add(a, b); }
// v with what the lane CTRL moves here holds, in the rows of 16 lanes that ROWS names.
template <bool MAX, int CTRL, int ROWS = 0xf>
__device__ __forceinline__ int pg_step(int v) {
  return pg_join<MAX>(v, __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false));
}

// Inclusive prefix sum (or maximum) of non-negative numbers over the workgroup; total in all
// threads.  lds: PG_WAVES ints, free for a new call after the caller's next barrier.
template <bool MAX = false>
__device__ __forceinline__ int pg_scan(int v, int* lds, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  v = pg_step<MAX, 0x111>(v);                      // from 1, 2, 4, 8 lanes below
  v = pg_step<MAX, 0x112>(v);
  v = pg_step<MAX, 0x114>(v);
  v = pg_step<MAX, 0x118>(v);
  v = pg_step<MAX, 0x142, 0xa>(v);                 // a row's total into the next row
  v = pg_step<MAX, 0x143, 0xc>(v);                 // the lower half's into the upper
  if (lane == 63) lds[wave] = v;
  __syncthreads();
  // a wave's sum a lane, the same way
  int sums = lane < PG_WAVES ? lds[lane] : 0;
  sums = pg_step<MAX, 0x111>(sums);
  sums = pg_step<MAX, 0x112>(sums);
  sums = pg_step<MAX, 0x114>(sums);
  sums = pg_step<MAX, 0x118>(sums);
  total = __builtin_amdgcn_readlane(sums, PG_WAVES - 1);
  const int w = __builtin_amdgcn_readfirstlane(wave);
  return pg_join<MAX>(v, w ? __builtin_amdgcn_readlane(sums, w - 1) : 0);
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

// Set the bits of the pages that sequences hold; held(row, but) gives how many of a row's entries
// count and, for FORK, which one of them does not.  2^group lanes a row, four entries a lane at a
// time.  For COMMON, common[row] of the first n rows becomes the number of entries before the first
// one that the row above has otherwise, of those that both hold (it comes as that many or more).
template <bool FORK, bool COMMON, typename Held>
__device__ __forceinline__ void pg_mark(const PageTables& t, uint32_t* used, int group, Held held,
                                        int* common = nullptr, int n = 0) {
  constexpr int DEEP = 4;                           // loads of a lane under way; 8 took no less
  const int lanes = 1 << group, l = threadIdx.x & (lanes - 1);
#pragma unroll 1
  for (int row = threadIdx.x >> group; row < t.seqs; row += PG_THREADS >> group) {
    int but = -1;
    const int count = held(row, but);
    const int* entry = t.tables + (int64_t)row * t.width;
    int both = 0;
    if (COMMON && row && row < n) {
      int x;
      both = min(count, held(row - 1, x));
    }
    auto take = [&](int j, int x, int above) {
      bool in = j < count && (unsigned)x < (unsigned)t.pages;
      if (FORK) in &= j != but;
      if (in) atomicOr(&used[x >> 5], 1u << (x & 31));
      return COMMON && j < both && x != above;
    };
    if (t.width < 4) {
      for (int j = l; j < count; j += lanes)
        if (take(j, entry[j], j < both ? entry[j - t.width] : 0)) atomicMin(&common[row], j);
      continue;
    }
    // whole pieces of the row, the last ones moved back into it: an entry may come twice
#pragma unroll 1
    for (int j0 = 4 * l; j0 < count; j0 += 4 * DEEP * lanes) {
      i32x4 p[DEEP], above[DEEP];
#pragma unroll
      for (int u = 0; u < DEEP; ++u) {
        const int j = min(j0 + 4 * lanes * u, t.width - 4);
        __builtin_memcpy(&p[u], entry + j, 16);
        if (COMMON) __builtin_memcpy(&above[u], entry - (row ? t.width : 0) + j, 16);
      }
      int other = both;
#pragma unroll
      for (int u = DEEP - 1; u >= 0; --u) {
        const int from = j0 + 4 * lanes * u, j = min(from, t.width - 4);
        if (from >= count) continue;
#pragma unroll
        for (int e = 3; e >= 0; --e)
          if (take(j + e, p[u][e], COMMON ? above[u][e] : 0)) other = min(other, j + e);
      }
      if (COMMON && other < both) atomicMin(&common[row], other);
    }
  }
}

// A thread's share of the pages: 2^k of one word's bits, or whole words where they are many.
struct PgShare {
  int word, end, shift;
  uint32_t mask;
  __device__ __forceinline__ explicit PgShare(const PageTables& t) {
    const int words = (t.pages + 31) >> 5, per = ceil_div(words, PG_THREADS);
    int bits = 32;
    while (bits > 1 && (bits / 2) * PG_THREADS >= t.pages) bits /= 2;
    const int at = threadIdx.x * (bits < 32 ? bits : 32 * per);
    word = at >> 5;
    end = min(bits < 32 ? word + 1 : word + per, words);
    shift = at & 31;
    mask = bits < 32 ? (1u << bits) - 1 : ~0u;
  }
  __device__ __forceinline__ uint32_t free(const uint32_t* used, int w) const {
    return ~used[w] >> shift & mask;
  }
};

// The free pages counted in order: `first` of them are below this thread's; returns how many there
// are.
__device__ __forceinline__ int pg_count_free(const PgShare& own, const uint32_t* used, int& first, int* lds) {
  int mine = 0, total;
#pragma unroll 1
  for (int w = own.word; w < own.end; ++w) mine += __popc(own.free(used, w));
  first = pg_scan(mine, lds, total) - mine;
  return total;
}

// Bits to start with: none held, those past the pool not there.
__device__ __forceinline__ void pg_clear(const PageTables& t, uint32_t* used) {
  const int words = (t.pages + 31) >> 5;
#pragma unroll 1
  for (int w = threadIdx.x; w < words; w += PG_THREADS)
    used[w] = w == words - 1 && (t.pages & 31) ? ~0u << (t.pages & 31) : 0u;
}

// give(rank, page) for the `want` lowest free pages, by the threads that counted them, in order.
template <typename Give>
__device__ __forceinline__ void pg_deal(const PgShare& own, const uint32_t* used, int first, int want,
                                        Give give) {
#pragma unroll 1
  for (int w = own.word; w < own.end && first < want; ++w)
#pragma unroll 1
    for (uint32_t free = own.free(used, w); free && first < want; free &= free - 1, ++first)
      give(first, w * 32 + own.shift + __ffs(free) - 1);
}

// ---------------------------------------------------------------------------
// Pages and slots for the tokens that n requests bring: request i brings counts[i] tokens to
// sequence rows[i].  It is granted where they fit max_len, its token rows fit T, and its pages are
// there: the requests' new pages are counted in order, those of a request that goes without too, so
// that one that needs none is never turned down for another.
//
// One workgroup: bits of the held pages, how many are free below each, then every free page of
// low enough rank goes to the request whose sum of new pages it falls into.  What it takes is a chain:
// fetched code, loads of lengths and tables (1 us each from other XCDs' stores), sums over the
// workgroup.  32 tokens behind 2048 5.8 us (half of it before the pages are counted); 384 requests among
// 512 sequences of up to 4096 tokens 16.5, most of it the marks of 65000 entries in LDS.  Bits in LDS
// rather than counts kept in memory: nothing has to be given back, and a captured step can be repeated.
//
// And the attention's schedule for single tokens (paged_attn.hip).  Neighbouring sequences whose
// tables begin with the same pages, for half of the shorter one's length or more, form groups of up to
// `most`: what they all share, in whole units of PG_UNIT keys, is one item, read once for all of them,
// and the rest of each is another.  Runs are cut at multiples of `most` whatever they share, and the least
// that two neighbours of a group share is what counts for it: beams of two requests in a group share the
// requests' common prompt and no more.  The items stand in one line, every group's shared one before its
// rows', that is cut into at most ncols equal stretches, one a column of workgroups:
//   row     (keys, shared units, the group's first row, its rows,
//            first and last column of the shared item, of the row's own)
//   column  (2 row + (1: its own, 0: its group's shared item), first unit there, units in all, 0)
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
  int* schedule;               // [n][8] then [ncols][4], or null
  int ncols, most;
  int group, slots_here;
};

// Token row tok is position p of the sequence, in that page (-1: it has no slot).
__device__ __forceinline__ void pg_slot(const PageTables& t, const ReserveArgs& r, int tok, int page,
                                        int p, int64_t delta) {
  const bool ok = page >= 0 && page < t.pages;
  r.token_page[tok] = ok ? page : -1;
  r.token_pos[tok] = ok ? p & ((1 << t.shift) - 1) : -1;
  for (int a = 0; a < r.axes; ++a) r.positions[(int64_t)a * r.T + tok] = ok ? p + delta : -1;
}

__global__ __launch_bounds__(PG_THREADS) void page_reserve_kernel(PageTables t, ReserveArgs r) {
  extern __shared__ uint32_t pg_smem[];
  __shared__ int lds[4][PG_WAVES];
  const int tid = threadIdx.x, words = (t.pages + 31) >> 5;
  uint32_t* used = pg_smem;
  int* ends = (int*)pg_smem + words;                // new pages up to and with request i
  int* last = ends + r.n;                           // token rows up to and with request i, then units
  int* len = last + r.n;                            // length, and tokens that it may be granted
  int* ask = len + r.n;
  int* at = ask + r.n;                              // dense: the token's page, then the group
  int* common = at + r.n;                           // dense: pages, then units, as the row above
  int* share = common + r.n;                        // dense: a group's shared units
  int* size = share + r.n;                          // dense: its rows
  pg_clear(t, used);
  int wanted = 0, rows_sum = 0;
#pragma unroll 1
  for (int base = 0; base < r.n; base += PG_THREADS) {
    const int i = base + tid;
    int need = 0, asked = 0, total;
    if (i < r.n) {
      const int64_t row = r.rows ? r.rows[i] : (int64_t)i;
      const bool in = row >= 0 && row < t.seqs;
      const int L = in ? pg_length(t, row) : 0;
      asked = max(r.counts ? r.counts[i] : 1, 0);
      if (r.dense) asked = min(asked, 1);
      const int c = in && asked <= t.max_len - L ? asked : 0;
      need = pg_pages(t, L + c) - pg_pages(t, L);
      if (r.dense) at[i] = c && !need ? t.tables[row * t.width + (L >> t.shift)] : -1;
      len[i] = L;
      ask[i] = c;
      last[i] = i + 1;
      if (r.dense) {
        common[i] = pg_pages(t, L);
        share[i] = 1 << 30;
        size[i] = 0;
      }
    }
    if (!r.dense) {
      // a request whose token rows run past T gets none
      const int upto = pg_add(pg_scan(min(asked, 1 << 30), lds[0], total), rows_sum);
      rows_sum = pg_add(rows_sum, total);
      if (i < r.n) {
        last[i] = upto;
        if (upto > r.T) need = ask[i] = 0;
      }
    }
    const int pages = pg_add(pg_scan(need, lds[1], total), wanted);
    wanted = pg_add(wanted, total);
    if (i < r.n) ends[i] = pages;
    __syncthreads();                                // the sums are read
  }
  auto held = [&](int row, int& but) { return pg_pages(t, pg_length(t, row)); };
  if (r.schedule && r.most > 1 && r.n > 1) pg_mark<false, true>(t, used, r.group, held, common, r.n);
  else pg_mark<false, false>(t, used, r.group, held);
  __syncthreads();
  const PgShare own(t);
  int first;
  const int left = pg_count_free(own, used, first, lds[2]);
  int to = -1, low = 0, high = 0;                   // the request of this thread's next page
  pg_deal(own, used, first, min(left, wanted), [&](int rank, int page) {
    if (rank >= high) {
      to = to < 0 ? pg_find(ends, r.n, rank) : to + 1;
      while (to < r.n && ends[to] <= rank) ++to;
      if (to >= r.n) return;
      low = to ? ends[to - 1] : 0;
      high = ends[to];
    }
    if (to >= r.n || high > left) return;
    const int64_t row = r.rows ? r.rows[to] : (int64_t)to;
    t.tables[row * t.width + pg_pages(t, len[to]) + rank - low] = page;
    if (r.dense) at[to] = page;
  });
  __syncthreads();                                  // the tables are written
#pragma unroll 1
  for (int i = tid; i < r.n; i += PG_THREADS) {
    const int L = len[i], low_i = i ? ends[i - 1] : 0;
    const int c = ends[i] == low_i || ends[i] <= left ? ask[i] : 0;
    r.granted[i] = c;
    r.starts[i] = L;
    r.after[i] = L + c;
    r.cu[i + 1] = last[i];
    if (i == 0) r.cu[0] = 0;
    ask[i] = c;
    if (r.dense) {
      const int64_t row = r.rows ? r.rows[i] : (int64_t)i;
      pg_slot(t, r, i, c ? at[i] : -1, L, c && r.rope_delta ? r.rope_delta[row] : 0);
    }
  }
  __syncthreads();
  if (!r.dense && r.slots_here) {
#pragma unroll 1
    for (int tok = tid; tok < r.T; tok += PG_THREADS) {
      const int i = pg_find(last, r.n, tok), in = tok - (i ? last[i - 1] : 0);
      int page = -1, p = 0;
      int64_t row = 0;
      if (i < r.n && in < ask[i]) {
        row = r.rows ? r.rows[i] : (int64_t)i;
        p = len[i] + in;
        page = t.tables[row * t.width + (p >> t.shift)];
      }
      pg_slot(t, r, tok, page, p, page >= 0 && r.rope_delta ? r.rope_delta[row] : 0);
    }
  }
  if (!r.schedule) return;
  // groups: a row that goes on from its neighbour, and the places in such a run cut at `most`
  int units = 0, start = 0;
  const bool groups = r.most > 1 && r.n > 1;
#pragma unroll 1
  for (int base = 0; base < r.n && groups; base += PG_THREADS) {
    const int i = base + tid;
    int total, shared = 0;
    if (i && i < r.n && ask[i] && ask[i - 1]) {
      const int least = min(len[i], len[i - 1]);
      shared = min(least, (int)min((int64_t)common[i] << t.shift, (int64_t)1 << 30)) / PG_UNIT;
      if (shared * PG_UNIT < least - shared * PG_UNIT) shared = 0;
    }
    const int run = max(pg_scan<true>(shared ? 0 : i, lds[3], total), start);
    start = max(start, total);
    if (i < r.n) {
      const int group = i - (i - run) % r.most;
      at[i] = group;
      atomicAdd(&size[group], 1);
      if (group != i) atomicMin(&share[group], shared);
    }
    __syncthreads();
  }
#pragma unroll 1
  for (int base = 0; base < r.n; base += PG_THREADS) {
    const int i = base + tid;
    int mine = 0, total;
    if (i < r.n) {
      const int group = groups ? at[i] : i, S = groups && size[group] > 1 ? share[group] : 0;
      if (!groups) {
        at[i] = i;
        size[i] = 1;
      }
      common[i] = S;
      mine = ask[i] ? ceil_div(len[i] + ask[i], PG_UNIT) - (group == i ? 0 : S) : 0;
    }
    const int upto = pg_scan(mine, lds[0], total) + units;
    units += total;
    if (i < r.n) last[i] = upto;
    __syncthreads();
  }
  const int cols = min(r.ncols, units);
  auto column_of = [&](int x) { return (int)((((int64_t)x + 1) * cols - 1) / units); };
#pragma unroll 1
  for (int i = tid; i < r.n; i += PG_THREADS) {
    const int group = at[i], S = common[i], first_i = i ? last[i - 1] : 0, first_g = group ? last[group - 1] : 0;
    i32x4 v = {0, 0, group, size[group]}, w = {0, 0, 0, 0};
    if (last[i] > first_i) {
      v[0] = len[i] + ask[i];
      v[1] = S;
      if (S) {
        w[0] = column_of(first_g);
        w[1] = column_of(first_g + S - 1);
      }
      w[2] = column_of(first_i + (group == i ? S : 0));
      w[3] = column_of(last[i] - 1);
    }
    *(i32x4*)(r.schedule + 8 * i) = v;
    *(i32x4*)(r.schedule + 8 * i + 4) = w;
  }
#pragma unroll 1
  for (int c = tid; c < r.ncols; c += PG_THREADS) {
    i32x4 v = {0, 0, 0, 0};
    if (c < cols) {
      const int lo = (int)((int64_t)c * units / cols), hi = (int)(((int64_t)c + 1) * units / cols);
      const int i = pg_find(last, r.n, lo), in = lo - (i ? last[i - 1] : 0);
      const int S = at[i] == i ? common[i] : 0;
      v = in < S ? (i32x4){2 * i, in, hi - lo, 0} : (i32x4){2 * i + 1, in - S, hi - lo, 0};
    }
    *(i32x4*)(r.schedule + 8 * r.n + 4 * c) = v;
  }
}

// Slots of many tokens, a token a thread: the request is looked up in the sums of token rows.  49000
// tokens 4.0 us, a search of nine steps and two dependent loads.
__global__ __launch_bounds__(256) void page_slots_kernel(PageTables t, ReserveArgs r) {
  __shared__ int last[PG_MAX_SEQS];
  for (int i = threadIdx.x; i < r.n; i += 256) last[i] = r.cu[i + 1];
  __syncthreads();
  const int tok = blockIdx.x * 256 + threadIdx.x;
  if (tok >= r.T) return;
  const int i = pg_find(last, r.n, tok), in = tok - (i ? last[i - 1] : 0);
  int page = -1, p = 0;
  int64_t row = 0;
  if (i < r.n && in < r.granted[i]) {
    row = r.rows ? r.rows[i] : (int64_t)i;
    p = (int)r.starts[i] + in;
    page = t.tables[row * t.width + (p >> t.shift)];
  }
  pg_slot(t, r, tok, page, p, page >= 0 && r.rope_delta ? r.rope_delta[row] : 0);
}

__global__ void page_gather_kernel(PageTables t, const int* __restrict__ parents, int rows, int W);
struct CopyItem {
  int from, to, rows, pad;       // pages, token rows
};
template <bool HERE>
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

// Workgroups of these kernels may take more dynamic LDS than a launch allows by default; said once
// per device.
static int pg_allow_lds() {
  static bool said[64];
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return (int)e;
  if (dev >= 0 && dev < 64 && said[dev]) return OMNI_OK;
  for (const void* k : {(const void*)page_reserve_kernel, (const void*)page_fork_kernel<false>,
                        (const void*)page_fork_kernel<true>, (const void*)page_gather_kernel})
    if (e == hipSuccess) e = hipFuncSetAttribute(k, hipFuncAttributeMaxDynamicSharedMemorySize, PG_LDS);
  if (e == hipSuccess && dev >= 0 && dev < 64) said[dev] = true;
  return (int)e;
}

// How many tokens the slots are written for by the workgroup that deals the pages: 512 tokens 7.5 us a
// call, with a launch of their own 9.4; 2048 8.2 and 9.4; 4096 9.8 and 9.1; 8192 14.1 and 9.8.
#define PG_SLOTS_HERE 2048

extern "C" int omni_page_reserve(int* tables, int64_t* lengths, int seqs, int width, int pages,
                                 int page_size, int max_len, const int* counts, const int64_t* rows,
                                 const int64_t* rope_delta, int n, int tokens, int dense, int axes,
                                 int64_t* starts, int64_t* after, int64_t* token_page,
                                 int64_t* token_pos, int64_t* positions, int* granted, int* cu,
                                 int* schedule, int columns, int most, void* stream) {
  if (n < 0 || tokens < 0 || axes < 1) return OMNI_EINVAL;
  const int rc = pg_tables_ok(tables, lengths, seqs, width, pages, page_size, max_len);
  if (rc) return rc;
  if (n > seqs || (dense && tokens != n)) return OMNI_EINVAL;
  if (axes > 3 || tokens > (1 << 28)) return OMNI_EUNSUPPORTED;
  if (n == 0) return OMNI_OK;
  if (!starts || !after || !granted || !cu) return OMNI_EINVAL;
  if (tokens && (!token_page || !token_pos || !positions)) return OMNI_EINVAL;
  if (schedule && (!dense || rows || columns <= 0 || most <= 0 || ((uintptr_t)schedule & 15)))
    return OMNI_EINVAL;
  if (schedule && (columns > 65535 || (int64_t)n * ceil_div(max_len, PG_UNIT) > (1 << 30)))
    return OMNI_EUNSUPPORTED;
  const PageTables t = {tables, lengths, seqs, width, pages, pg_shift(page_size), max_len};
  ReserveArgs r = {counts, rows, rope_delta, n, tokens, dense, axes, starts, after, token_page,
                   token_pos, positions, granted, cu, schedule, columns, most, pg_group(seqs),
                   tokens <= PG_SLOTS_HERE};
  const size_t smem = 4 * ((size_t)(pages + 31) / 32 + (dense ? 8 : 4) * (size_t)n);
  if (smem > (32 << 10))
    if (const int e = pg_allow_lds()) return e;
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
// without a parent).  Launches: where the tables are large their columns, 16 a workgroup, through LDS (in
// place); lengths, new pages and small tables, one workgroup (4 rows of 500 tokens 3.9 us, 128 of 400
// 7.5: the chain of omni_page_reserve); the copies, a workgroup a row, layer and K or V (128 rows in 28
// layers, 11 MB each way, 4.2-5.1 us).
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

// HERE: the tables are few enough for this workgroup's LDS, and it moves them itself.
template <bool HERE>
__global__ __launch_bounds__(PG_THREADS) void page_fork_kernel(PageTables t, const int* __restrict__ parents,
                                                               int rows, int W, CopyItem* __restrict__ items,
                                                               int group) {
  extern __shared__ uint32_t pg_smem[];
  __shared__ int lds[2][PG_WAVES];
  const int tid = threadIdx.x, words = (t.pages + 31) >> 5, page = 1 << t.shift;
  uint32_t* used = pg_smem;
  int* len = (int*)pg_smem + words;                 // lengths after; ~length: with a page of its own
  int* ends = len + rows;                           // pages up to and with row r
  int* from = ends + rows;                          // the page that is filled in part
  int* up = from + rows;                            // the row that row r goes on from, or -1
  int* tile = up + rows;                            // HERE: [rows][width], the tables before
  pg_clear(t, used);
  if (HERE) {
#pragma unroll 4
    for (int e = tid; e < rows * t.width; e += PG_THREADS) tile[e] = t.tables[e];
  }
  int wanted = 0;
#pragma unroll 1
  for (int base = 0; base < rows; base += PG_THREADS) {
    const int r = base + tid;
    int L = 0, total;
    bool later = false;
    if (r < rows) {
      const int w = r % W, p = parents[r];
      up[r] = -1;
      if (p >= 0 && p < W) {
        up[r] = r - w + p;
        L = pg_length(t, r - w + p);
        for (int x = 0; x < w; ++x) later |= parents[r - w + x] == p;
        later &= (L & (page - 1)) != 0;
        // moved tables are this row's own by now
        if (later && !HERE) from[r] = t.tables[(int64_t)r * t.width + (L >> t.shift)];
      }
      len[r] = later ? ~L : L;
    }
    const int upto = pg_scan(later ? 1 : 0, lds[0], total) + wanted;
    wanted += total;
    if (r < rows) ends[r] = upto;
    __syncthreads();                                // the sums are read
  }
  if (HERE) {
    // a wave a row: its new table, and the pages in it
#pragma unroll 1
    for (int r = tid >> 6; r < rows; r += PG_WAVES) {
      const int v = len[r], L = v < 0 ? ~v : v, source = up[r];
      if (source < 0) continue;
      const int held = pg_pages(t, L), but = v < 0 ? L >> t.shift : -1;
#pragma unroll 2
      for (int c = tid & 63; c < held; c += 64) {
        const int p = tile[source * t.width + c];
        if (source != r) t.tables[r * t.width + c] = p;
        if (c == but) from[r] = p;
        else if (p >= 0 && p < t.pages) atomicOr(&used[p >> 5], 1u << (p & 31));
      }
    }
  }
  pg_mark<true, false>(t, used, group, [&](int row, int& but) {
    if (row >= rows) return pg_pages(t, pg_length(t, row));
    if (HERE) return 0;
    const int v = len[row], L = v < 0 ? ~v : v;
    if (v < 0) but = L >> t.shift;
    return pg_pages(t, L);
  });
  __syncthreads();
  const PgShare share(t);
  int first;
  const int left = pg_count_free(share, used, first, lds[1]);
#pragma unroll 1
  for (int r = tid; r < rows; r += PG_THREADS) {
    const int v = len[r];
    const bool copies = v < 0 && ends[r] <= left;
    t.lengths[r] = v >= 0 ? v : copies ? ~v : 0;
    if (!copies) items[r] = {0, 0, 0, 0};
  }
  int to = -1;
  pg_deal(share, used, first, min(left, wanted), [&](int rank, int own) {
    to = to < 0 ? pg_find(ends, rows, rank) : to + 1;
    while (len[to] >= 0) ++to;                      // the next row with a page of its own
    const int L = ~len[to], p = from[to];
    t.tables[(int64_t)to * t.width + (L >> t.shift)] = own;
    const bool in = p >= 0 && p < t.pages;
    items[to] = {in ? p : 0, own, in ? L & (page - 1) : 0, 0};
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
  const size_t base = 4 * ((size_t)(pages + 31) / 32 + 4 * (size_t)rows), tile = 4 * (size_t)rows * width;
  const bool here = tile <= 4 * PG_TILE && base + tile <= PG_LDS;
  const size_t smem = here ? base + tile : base;
  const int group = pg_group(seqs);
  if (here) {
    hipLaunchKernelGGL(page_fork_kernel<true>, dim3(1), dim3(PG_THREADS), smem, st, t, parents, rows,
                       beams, (CopyItem*)work, group);
  } else {
    hipLaunchKernelGGL(page_gather_kernel, dim3(ceil_div(width, PG_COLS)), dim3(256),
                       (size_t)rows * PG_COLS * 4, st, t, parents, rows, beams);
    OMNI_CHECK_LAUNCH();
    hipLaunchKernelGGL(page_fork_kernel<false>, dim3(1), dim3(PG_THREADS), smem, st, t, parents, rows,
                       beams, (CopyItem*)work, group);
  }
  OMNI_CHECK_LAUNCH();
  const int64_t page_halfs = (int64_t)page_size * row_halfs;
  hipLaunchKernelGGL(page_copy_kernel, dim3(2 * n_layers, rows), dim3(256), 0, st, (half_t*)pool,
                     page_halfs * pages, page_halfs, row_halfs, (const CopyItem*)work);
  OMNI_CHECK_LAUNCH();
  return OMNI_OK;
}
