// Attention for trees of drafted tokens over the KV pool, and the tree's plan.
//
// Sequence s has a valid prefix of starts[s] tokens in its pool row; node i of its tree (n_nodes
// <= 64 of them, parents before children) has its K/V at position starts[s] + i and attends to
// the prefix, itself and its ancestors.  The ancestors of a node are one 64-bit word.
#include "attn_rows.h"

#define TREE_HD 128
#define TREE_MAX 64

// ---------------------------------------------------------------------------
// The plan of a step, once for all layers.
//
// Per node its ancestors (itself included; bit j = node j), its pool row and position (row -1: not
// in use, or past the pool), its rotary position starts + depth + rope_delta on all three axes; per
// sequence the prefix length, a copy, so that the plan stays what it was when the lengths move on.
// A node whose parent does not precede it is a root of its own.
//
// And the attention's schedule.  A sequence's keys count in units of `unit` (what a workgroup takes
// in a step), once per KV head.  Every (sequence, KV head) item gets one of the ncols columns of
// workgroups and a share of the others by its length, and is cut into as many equal pieces: none
// of a batch of one length runs over an item's end.  Where that would leave some column more than
// three units above the mean, the units of all items stand in one line instead, cut into equal
// stretches: as even for one long and many short contexts, whatever the lengths on the device
// are, but a stretch that runs over an item's end costs its workgroup another start and merge, some
// 4 us.  No piece is under `least` units; least 0: a column for each item.
//   seqs[s]     (prefix length, nodes in use, units, pool row)
//   columns[c]  (s, g, first unit there, units in all, then of s: length, nodes, pool row)
//   heads[s][g] (first column | 1 << 30 where the item is not the first that column sees, last)
// One wave a sequence: lane i walks up from node i; every wave sums all sequences' units and
// writes the columns that start in its own sequence.  A chain of dependent loads: 4-6.5 us, once
// per step.
// ---------------------------------------------------------------------------
struct TreeCols {
  int* seqs;       // [n][4]
  int* columns;    // [ncols][8]
  int* heads;      // [n][nkv][2]
  int ncols, nkv, unit, least;
};

__global__ __launch_bounds__(64) void tree_plan_kernel(
    const int* __restrict__ parents, const int* __restrict__ counts,
    const int64_t* __restrict__ slots, const int64_t* __restrict__ lengths,
    const int64_t* __restrict__ rope_delta, int n, int T, int pool_rows, int max_len,
    int64_t* __restrict__ starts, uint64_t* __restrict__ ancestors,
    int64_t* __restrict__ positions, int64_t* __restrict__ token_slot,
    int64_t* __restrict__ token_pos, TreeCols tc) {
  __shared__ int up[TREE_MAX];
  const int s = blockIdx.x, i = threadIdx.x;
  if (i < T) up[i] = parents[(int64_t)s * T + i];
  auto prefix = [&](int r) {
    const int64_t row = slots ? slots[r] : r;
    const int64_t v = row >= 0 && row < pool_rows ? lengths[row] : 0;
    return (int)(v < 0 ? 0 : v > max_len ? max_len : v);
  };
  auto in_use = [&](int r) { return counts ? min(max(counts[r], 0), T) : T; };
  const int64_t slot = slots ? slots[s] : s;
  const bool row_ok = slot >= 0 && slot < pool_rows;
  const int L = prefix(s), used = in_use(s);
  const int64_t delta = row_ok && rope_delta ? rope_delta[slot] : 0;

  auto units_of = [&](int r) {
    const int64_t row = slots ? slots[r] : r;
    const int m = in_use(r);
    return m && row >= 0 && row < pool_rows ? ceil_div(min(prefix(r) + m, max_len), tc.unit) : 0;
  };
  // units of the sequences before this one, its own, and all
  int before = 0, all = 0;
  for (int r0 = 0; r0 < n; r0 += 64) {
    int w = r0 + i < n ? units_of(r0 + i) : 0, lo = r0 + i < s ? w : 0;
    for (int o = 32; o; o >>= 1) {
      w += __shfl_xor(w, o);
      lo += __shfl_xor(lo, o);
    }
    all += w;
    before += lo;
  }
  const int units = units_of(s);
  all *= tc.nkv;
  before *= tc.nkv;
  const int items = n * tc.nkv;
  auto column = [&](int c, int g, int first, int count) {
    int* col = tc.columns + 8 * c;
    *(i32x4*)col = (i32x4){s, g, first, count};
    *(i32x4*)(col + 4) = (i32x4){L, used, (int)slot, 0};
  };
  // pieces of an item; the columns before this sequence's, and all; the longest piece
  auto pieces_of = [&](int w) {
    if (!w || !tc.least) return w ? 1 : 0;
    const int more = (int)((uint64_t)w * (uint64_t)(tc.ncols - items) / (uint64_t)all);
    return min(1 + more, max(1, w / tc.least));
  };
  bool apart = !tc.least;
  int first = 0, taken = 0;
  if (items <= tc.ncols) {
    int most = 0;
    for (int r0 = 0; r0 < n; r0 += 64) {
      const int w = r0 + i < n ? units_of(r0 + i) : 0;
      int c = pieces_of(w), lo = r0 + i < s ? c : 0, hi = c ? ceil_div(w, c) : 0;
      for (int o = 32; o; o >>= 1) {
        c += __shfl_xor(c, o);
        lo += __shfl_xor(lo, o);
        hi = max(hi, __shfl_xor(hi, o));
      }
      taken += c;
      first += lo;
      most = max(most, hi);
    }
    apart |= most <= all / tc.ncols + 3;
    taken *= tc.nkv;
    first *= tc.nkv;
  }
  if (apart) {
    const int pieces = pieces_of(units);
    for (int k = i; k < tc.nkv * pieces; k += 64) {
      const int g = k / pieces, j = k - g * pieces;
      const int lo = j * units / pieces;
      column(first + k, g, lo, (j + 1) * units / pieces - lo);
    }
    for (int c = taken + i; c < tc.ncols && s == 0; c += 64) column(c, 0, 0, 0);
    for (int g = i; g < tc.nkv; g += 64)
      *(int2*)(tc.heads + 2 * (s * tc.nkv + g)) =
          make_int2(first + g * pieces, first + max(g * pieces + pieces - 1, 0));
  } else {
    // column c starts at unit c all / cols (in two parts: all < 2^30, cols < 2^15)
    const unsigned cols = min(tc.ncols, max(1, all / tc.least));
    const unsigned per = (unsigned)all / cols, over = (unsigned)all - per * cols;
    auto cut = [&](unsigned c) { return (int)(c * per + c * over / cols); };
    for (int c = i; c < tc.ncols; c += 64) {
      const int lo = c < cols ? cut(c) : all, cnt = c < cols ? cut(c + 1) - lo : 0;
      if (cnt > 0 && lo >= before && lo < before + units * tc.nkv) {
        const int g = (lo - before) / units;
        column(c, g, lo - before - g * units, cnt);
      } else if (cnt <= 0 && s == 0) {
        column(c, 0, 0, 0);
      }
    }
    for (int g = i; g < tc.nkv; g += 64) {
      int2 at = make_int2(0, 0);
      if (units) {
        const int lo = before + g * units, hi = lo + units - 1;
        // the last column that starts at or before a unit: a guess and its neighbours
        auto column_of = [&](int x) {
          unsigned c = min(cols - 1, (unsigned)((float)x * (float)cols / (float)all));
          while (c + 1 < cols && cut(c + 1) <= x) ++c;
          while (cut(c) > x) --c;
          return (int)c;
        };
        at.x = column_of(lo);
        at.y = column_of(hi);
        if (cut(at.x) < lo) at.x |= 1 << 30;
      }
      *(int2*)(tc.heads + 2 * (s * tc.nkv + g)) = at;
    }
  }
  if (i == 0) {
    starts[s] = L;
    *(i32x4*)(tc.seqs + 4 * s) = (i32x4){L, used, units, (int)slot};
  }
  __syncthreads();
  if (i >= T) return;
  uint64_t m = 0;
  if (i < used) {
    int at = i;
    while (true) {                       // parents precede their children: at most 64 steps
      m |= 1ull << at;
      const int p = up[at];
      if (p < 0 || p >= at) break;
      at = p;
    }
  }
  const int64_t t = (int64_t)s * T + i, NT = (int64_t)n * T;
  const int64_t rot = m ? L + __popcll(m) - 1 + delta : 0;
  ancestors[t] = m;
  positions[t] = positions[NT + t] = positions[2 * NT + t] = rot;
  token_slot[t] = m && row_ok && L + i < max_len ? slot : -1;
  token_pos[t] = L + i;
}

// K/V rows of packed tokens to the pool at (slots, positions); rows outside it are skipped.  8
// tokens 3.1 us, a launch's own time.
__global__ __launch_bounds__(256) void kv_rows_kernel(const half_t* __restrict__ k, int64_t k_stride,
                                                      const half_t* __restrict__ v, int64_t v_stride,
                                                      half_t* __restrict__ k_cache,
                                                      half_t* __restrict__ v_cache,
                                                      const int64_t* __restrict__ slots,
                                                      const int64_t* __restrict__ pos, int pool_rows,
                                                      int max_len, int row_halfs) {
  const int t = blockIdx.x;
  const int64_t slot = slots[t], p = pos[t];
  if (slot < 0 || slot >= pool_rows || p < 0 || p >= max_len) return;
  const int64_t to = (slot * max_len + p) * row_halfs;
  const int chunks = row_halfs >> 3;
  for (int c = threadIdx.x; c < 2 * chunks; c += 256) {
    if (c < chunks) *(half8_t*)(k_cache + to + 8 * c) = *(const half8_t*)(k + t * k_stride + 8 * c);
    else *(half8_t*)(v_cache + to + 8 * (c - chunks)) = *(const half8_t*)(v + t * v_stride + 8 * (c - chunks));
  }
}

// ---------------------------------------------------------------------------
// The tile structure and what bounds it are in attn_rows.h.  A workgroup takes 32 R (node, query
// head) rows, node-major, of the sequences and KV heads that its column of the schedule runs
// through, one stretch of keys after another; the S groups of R waves take contiguous runs of a
// stretch's KT-key tiles (each group has its own LDS tiles, as in attn_rows.hip).  A K / V byte
// staged in LDS serves all query heads of the group and up to 32 R / G nodes.  A stretch that is
// an item's whole gives outputs, a part of one a softmax state for the merging launch: only a
// column's first and last can be parts.
//
// The keys are the prefix and, behind it, the nodes.  Only tiles that reach past the prefix are
// masked, with the row's ancestor word shifted to the tile.  A node that a row does not attend to
// has probability 0 there, and 0 times an infinity or NaN in its V row is NaN: rows whose merged
// outputs are not all finite are taken again, key by key and without the keys they do not
// attend to (tree_row).  That costs the others the check and a barrier.
//
// P is rounded to fp16 for the second product: outputs are off by 2.6e-4 of their size, 2.1e-4 of it
// their own rounding.  The next bits of P would take the product's matrix instructions once more.
//
// MI355X, 12 / 2 heads.  A launch has some 8 us of its own (column and Q loads, first tile, LDS
// merge).  128 rows: a step of 128 keys 1.84 us on up to 144 workgroups, 2.03 on 192, 2.53 on 240,
// whether K and V come from memory or cache.  A workgroup takes the same cycles at any of them
// (300000 at 8128 tokens, matrix busy 44 % of them, vector issue 48 %), but the clock falls: 2.50 GHz at
// 48 workgroups, 2.39 at 144, 2.27 at 192, 2.10 at 240, with idle times between the launches.
// 64 rows: a step 1.2 us on 2 workgroups, 3.15 on 256 = 5.3 TB/s, memory's.  32 x 64 nodes at 4000
// tokens 74 + 4.8 of merge, 32 x 8 at 2048 18 + 4.1, 1 x 26 at 4000 10.7 + 4.3.
// ---------------------------------------------------------------------------
struct TreeArgs {
  const half_t* q;
  int64_t q_stride;
  const half_t* k_cache;
  const half_t* v_cache;
  int max_len, nkv, G, T, n;
  unsigned magic;              // row / G = high word of row * magic (G > 1)
  int ncols, rblocks;          // columns of the schedule, row blocks (workgroups) of each
  const uint64_t* ancestors;   // [n][T]
  const int* seqs;
  const int* columns;
  half_t* out;
  int out_stride;
  float scale_log2;
  float* states;               // [ncols][rblocks][2][32 R][ATT_REC]
};

// One row over keys [k0, k1) by one wave: 64 keys a step, a key a lane for the scores, then two
// dims a lane for the output, hidden keys left out.
// rec: the row's state, or null for its output.
__device__ __forceinline__ void tree_row(const TreeArgs& a, int slot, int s, int g, int row, int L,
                                         int k0, int k1, float* rec) {
  const int lane = threadIdx.x & 63;
  const int node = row / a.G, head = g * a.G + row - node * a.G;
  const int64_t tok = (int64_t)s * a.T + node;
  const uint64_t mask = a.ancestors[tok];
  const int64_t tstride = (int64_t)a.nkv * TREE_HD;
  const int64_t base = (int64_t)slot * a.max_len * tstride + g * TREE_HD;
  const half_t* qp = a.q + tok * a.q_stride + head * TREE_HD;
  float mr = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
#pragma unroll 1
  for (int tb = k0; tb < k1; tb += 64) {
    const int key = tb + lane;
    const bool seen = key < k1 && (key < L || ((mask >> (key - L)) & 1));
    float sc = -INFINITY;
    if (seen) {
      const half_t* kp = a.k_cache + base + key * tstride;
      sc = 0.f;
#pragma unroll 1
      for (int c = 0; c < TREE_HD; ++c) sc = fmaf((float)kp[c], (float)qp[c], sc);
      sc *= a.scale_log2;
    }
    const uint64_t all = __ballot(seen);
    if (!all) continue;
    const float mn = fmaxf(mr, wave_max(sc)), ref = mn == -INFINITY ? 0.f : mn;
    const float alpha = exp2f(mr - ref), p = seen ? exp2f(sc - ref) : 0.f;
    mr = mn;
    l = l * alpha + wave_sum(p);
    o0 *= alpha;
    o1 *= alpha;
#pragma unroll 1
    for (int j = 0; j < 64; ++j) {
      const float pj = __shfl(p, j);
      if (!((all >> j) & 1)) continue;
      const half2_t vv = *(const half2_t*)(a.v_cache + base + (tb + j) * tstride + 2 * lane);
      o0 = fmaf(pj, (float)vv[0], o0);
      o1 = fmaf(pj, (float)vv[1], o1);
    }
  }
  if (rec) {
    *(float2*)(rec + 2 * lane) = make_float2(o0, o1);
    if (lane == 0) *(float2*)(rec + 128) = make_float2(mr, l);
  } else {
    const half2_t r = {(half_t)(l == 0.f ? 0.f : o0 / l), (half_t)(l == 0.f ? 0.f : o1 / l)};
    *(half2_t*)(a.out + tok * a.out_stride + head * TREE_HD + 2 * lane) = r;
  }
}

template <int R, int S, int KT>
__global__ __launch_bounds__(64 * R * S, 2) void tree_attn_kernel(TreeArgs a) {
  constexpr int NBUF = R == 1 ? 1 : 2;
  constexpr int TB = KT * TREE_HD * 2;              // bytes of a K (or V) tile
  constexpr int NL = TB / 1024;                     // 1 KB (4-row) pieces of a tile
  constexpr int NB = KT / 32;
  constexpr int MB = R * S * 64 * 64 * 4;           // the merge's outputs
  constexpr int SB = S * NBUF * 2 * TB > MB ? S * NBUF * 2 * TB : MB;
  __shared__ __attribute__((aligned(16))) char smem[SB];
  __shared__ float ml_lds[S][R][2][32];
  __shared__ uint32_t bad_rows[R][S];
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int grp = wave / R;                          // key group
  const int rt = wave - grp * R;                     // row tile
  const int l32 = lane & 31, h = lane >> 5;
  // the row blocks of a column, which read the same keys, on one XCD (workgroup b on XCD b % 8)
  const int y = blockIdx.x >> 3;
  const int rb = y % a.rblocks;
  const int col = (y / a.rblocks) * 8 + (blockIdx.x & 7);
  if (col >= a.ncols) return;
  // through the scalar cache: the plan wrote it in an earlier launch
  typedef const __attribute__((address_space(4))) int plan_int;
  const plan_int* column = (const plan_int*)a.columns + 8 * col;
  const plan_int* seqs = (const plan_int*)a.seqs;
  int s = column[0], g = column[1], u0 = column[2], left = column[3];
  int L = column[4], used = column[5], slot = column[6];
  constexpr int UNIT = S * KT;
  const int cr = lane >> 4, cc = lane & 15;
  const int64_t tstride = (int64_t)a.nkv * TREE_HD;  // halfs per token
  const uint32_t kv_row = (uint32_t)tstride * 2;     // bytes
  for (int part = 0; left > 0; part = 1) {
  const int end = min(L + used, a.max_len);
  const int ntiles = ceil_div(end, KT), units = ceil_div(end, UNIT);
  const int steps = min(left, units - u0);
  const bool whole = u0 == 0 && steps == units;
  const int nrows = used * a.G - 32 * R * rb;        // this block's
  if (nrows > 0) {
  const int tbeg = u0 * S + grp * steps;
  const int nt = min(steps, ntiles - tbeg);          // may be <= 0
  const int64_t base = (int64_t)slot * a.max_len * tstride + g * TREE_HD;
  const half_t* kb0 = a.k_cache + base;
  const half_t* vb0 = a.v_cache + base;

  // R = 1 stages through registers (its one buffer is free only once the tile is used): chunk
  // lane + 64 j of a tile is row cr + 4 j, 16-byte chunk cc.
  half8_t kr[NL], vr[NL];
  auto load_tile = [&](int tb) {
    const char* kp = (const char*)kb0 + (int64_t)tb * kv_row;
    const char* vp = (const char*)vb0 + (int64_t)tb * kv_row;
    if (tb + KT <= end) {
      const uint32_t at = cr * kv_row + cc * 16;
#pragma unroll
      for (int j = 0; j < NL; ++j) {
        kr[j] = *(const half8_t*)(kp + 4 * j * (int64_t)kv_row + at);
        vr[j] = *(const half8_t*)(vp + 4 * j * (int64_t)kv_row + at);
      }
    } else {                                         // past the end: the last key again
#pragma unroll
      for (int j = 0; j < NL; ++j) {
        const uint32_t at = (uint32_t)min(cr + 4 * j, end - 1 - tb) * kv_row + cc * 16;
        kr[j] = *(const half8_t*)(kp + at);
        vr[j] = *(const half8_t*)(vp + at);
      }
    }
  };
  auto store_tile = [&](char* kt) {
    char* vt = kt + TB;
#pragma unroll
    for (int j = 0; j < NL; ++j) {
      const int r = cr + 4 * j;
      *(half8_t*)(kt + r * 256 + ((cc ^ (r & 15)) << 4)) = kr[j];
      *(half8_t*)(vt + r * 256 + ((cc << 4) ^ ((r & 3) << 6))) = vr[j];
    }
  };

  char* gbuf = smem + grp * NBUF * 2 * TB;
  // R > 1 stages straight to LDS, 1 KB (4 rows) per instruction, the swizzle in the source
  // addresses: they are a lane's constant, for R = 2 but for one bit, off uniform bases.
  const uint32_t koffs = cr * kv_row + ((cc ^ (4 * rt + cr)) << 4);
  const uint32_t voffs = cr * kv_row + ((cc ^ (cr << 2)) << 4);
  auto dma_tile = [&](int tb, char* kt) {
    const uint32_t l0 = __builtin_amdgcn_readfirstlane(lds_offset(kt)) + rt * 1024;
    if (tb + KT <= end) {
      const int64_t first = (int64_t)(tb + 4 * rt) * kv_row;
      const char* kp = (const char*)kb0 + first;
      const char* vp = (const char*)vb0 + first;
#pragma unroll
      for (int j = 0; j < NL / R; ++j) {
        const uint32_t flip = (4 * R * j & 15) << 4;     // of the rows' swizzle
        dma16(kp + (int64_t)(4 * R * j) * kv_row, koffs ^ flip, l0 + R * j * 1024);
        dma16(vp + (int64_t)(4 * R * j) * kv_row, voffs, l0 + TB + R * j * 1024);
      }
    } else {                                             // past the end: the last key again
      const char* kp = (const char*)kb0 + (int64_t)tb * kv_row;
      const char* vp = (const char*)vb0 + (int64_t)tb * kv_row;
#pragma unroll
      for (int j = 0; j < NL / R; ++j) {
        const int r = 4 * (rt + R * j) + cr;
        const uint32_t at = (uint32_t)min(r, end - 1 - tb) * kv_row;
        dma16(kp, at + ((cc ^ (r & 15)) << 4), l0 + R * j * 1024);
        dma16(vp, at + ((cc ^ ((r & 3) << 2)) << 4), l0 + TB + R * j * 1024);
      }
    }
  };
  // the first tile's transfers go out before anything else is asked for
  if (nt > 0) {
    if constexpr (R > 1) dma_tile(tbeg * KT, gbuf);
    else load_tile(tbeg * KT);
  }

  const int row = min(32 * rt + l32, nrows - 1);
  const int node = a.G == 1 ? 32 * R * rb + row : (int)__umulhi(32 * R * rb + row, a.magic);
  const int u = 32 * R * rb + row - node * a.G;
  const int64_t tok = (int64_t)s * a.T + node;
  const bool rows_here = 32 * rt < nrows;
  uint64_t mask = a.ancestors[tok];
  half8_t qf[8];
  {
    const half_t* qp = a.q + tok * a.q_stride + (int64_t)(g * a.G + u) * TREE_HD + 8 * h;
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) qf[ks] = *(const half8_t*)(qp + 16 * ks);
  }
  if (end - L < 64) mask &= (1ull << (end - L)) - 1;   // nodes behind the pool's end

  float m_run = -INFINITY, l_run = 0.f;
  f32x16 o[4];
#pragma unroll
  for (int d = 0; d < 4; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
  const int koff = l32 * 256 + ((h ^ (l32 & 15)) << 4);
  const int i16 = lane & 15;
  const int voff = (4 * h + (i16 >> 2)) * 256 + ((i16 >> 2) << 6) + ((lane >> 4) & 1) * 32 +
                   (i16 & 3) * 8;
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
  f32x16 sc[NB];
  half8_t p[2 * NB];
  auto scores = [&](const char* kt) {
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) sc[b][i] = 0.f;
#pragma unroll
    for (int ks = 0; ks < 8; ++ks)
#pragma unroll
      for (int b = 0; b < NB; ++b)
        sc[b] = mfma32x32x16(*(const half8_t*)(kt + 8192 * b + (koff ^ (ks << 5))), qf[ks], sc[b]);
    // the first reads ahead, then one step's reads beside each step's MFMAs
    __builtin_amdgcn_sched_group_barrier(0x100, 3 * NB, 0);
#pragma unroll
    for (int ks = 0; ks < 5; ++ks) {
      __builtin_amdgcn_sched_group_barrier(0x008, NB, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, NB, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, 3 * NB, 0);
  };
  // bit j: the row attends to key tb + j
  auto tile_word = [&](int tb) {
    const int off = tb - L;
    return off >= 0 ? mask >> off : (mask << -off) | ((1ull << -off) - 1);
  };
  auto hide = [&](int tb) {
    if (tb + KT > L) {
      const uint64_t w = tile_word(tb) >> (4 * h);
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (!((w >> (32 * b + 8 * (i >> 2) + (i & 3))) & 1)) sc[b][i] = -INFINITY;
    }
  };
  auto output = [&](const char* vt) {
#pragma unroll
    for (int t = 0; t < 2 * NB; ++t)
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        const char* vp = vt + 4096 * t + (voff ^ (d << 6));
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)vp);
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(vp + 2048));
        const half4_t a0 = __builtin_bit_cast(half4_t, lo), a1 = __builtin_bit_cast(half4_t, hi);
        o[d] = mfma32x32x16((half8_t){a0[0], a0[1], a0[2], a0[3], a1[0], a1[1], a1[2], a1[3]},
                            p[t], o[d]);
      }
    // V of the first 16 keys ahead, then each 16 keys' MFMAs beside the next 16's exponentials
    __builtin_amdgcn_sched_group_barrier(0x100, 8, 0);
    __builtin_amdgcn_sched_group_barrier(0x002, 28, 0);
#pragma unroll
    for (int t = 0; t < 2 * NB - 1; ++t)
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, 7, 0);
      }
    __builtin_amdgcn_sched_group_barrier(0x008, 4, 0);
  };
  // Q has landed: without this the compiler counts the Q loads as outstanding inside the loop
  // and makes every tile's first MFMAs wait for the transfers just requested
  __builtin_amdgcn_s_waitcnt(0x0f70);
  // Eight waves' transfers take the CU's load path some 1100 cycles to accept, and a wave waits
  // there.  One wave of every SIMD issues its own at the start of a step, the other (wave + 4)
  // behind its softmax: so one is at its products while the other waits.
  const bool late = R > 1 && wave >= 4;
  auto next_tile = [&](int it) {
    if constexpr (R > 1) {
      if (it + 1 < nt) dma_tile((tbeg + it + 1) * KT, gbuf + ((it + 1) & 1) * 2 * TB);
    }
  };
  for (int it = 0; it < steps; ++it) {
    char* kt = gbuf + (NBUF == 2 ? (it & 1) * 2 * TB : 0);
    const int tb = (tbeg + it) * KT;
    if constexpr (R > 1) {
      vm_wait();             // this wave's part of tile it has landed; so, past the barrier,
      lds_barrier();         // have the others', and tile it - 1's buffer is free
      if (!late) next_tile(it);
    } else {
      if (it < nt) store_tile(kt);
      if (it + 1 < nt) load_tile(tb + KT);
    }
    if (it < nt && rows_here) {
      scores(kt);
      hide(tb);
      softmax32<NB, 4>(sc, a.scale_log2, m_run, l_run, o, p);
      if (late) next_tile(it);
      output(kt + TB);
    } else if (late) {
      next_tile(it);
    }
  }

  // Every group's unnormalised output and (max, sum) per row go to LDS; wave (rt, grp)
  // merges its share of the 16 output quads (4 dims) of row tile rt over the S groups.
  {
    float x, y2;
    half_pair(l_run, x, y2);
    l_run = x + y2;
  }
  __syncthreads();
  float* om = (float*)smem;
  if (rows_here) {
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
      for (int b = 0; b < 4; ++b)
        *(float4*)(om + (((grp * R + rt) * 16 + 4 * d + b) * 64 + lane) * 4) =
            make_float4(o[d][4 * b], o[d][4 * b + 1], o[d][4 * b + 2], o[d][4 * b + 3]);
    if (h == 0) {
      ml_lds[grp][rt][0][l32] = m_run;
      ml_lds[grp][rt][1][l32] = l_run;
    }
  }
  __syncthreads();
  const int64_t head = g * a.G + u;
  float* state = a.states + ((int64_t)(col * a.rblocks + rb) * 2 + part) * (32 * R * ATT_REC);
  if (rows_here) {
    float M = ml_lds[0][rt][0][l32];
#pragma unroll
    for (int k = 1; k < S; ++k) M = fmaxf(M, ml_lds[k][rt][0][l32]);
    const float ref = M == -INFINITY ? 0.f : M;        // no key at all: factors 0
    float f[S], den = 0.f;
#pragma unroll
    for (int k = 0; k < S; ++k) {
      f[k] = __builtin_amdgcn_exp2f(ml_lds[k][rt][0][l32] - ref);
      den += ml_lds[k][rt][1][l32] * f[k];
    }
    const float inv = den == 0.f ? 0.f : 1.0f / den;
    const bool mine = 32 * rt + l32 < nrows;
    float* rec = state + (32 * rt + l32) * ATT_REC;
    half_t* op = a.out + tok * a.out_stride + head * TREE_HD;
    constexpr int NQ = 16 / S;
    float bad = den * 0.f;                             // NaN where an output is not finite
#pragma unroll
    for (int k = 0; k < NQ; k += 2) {
      unsigned w[2][2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int quad = grp * NQ + k + e;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int m = 0; m < S; ++m) {
          const float4 v = *(const float4*)(om + (((m * R + rt) * 16 + quad) * 64 + lane) * 4);
          acc.x = fmaf(v.x, f[m], acc.x);
          acc.y = fmaf(v.y, f[m], acc.y);
          acc.z = fmaf(v.z, f[m], acc.z);
          acc.w = fmaf(v.w, f[m], acc.w);
        }
        bad = fmaf(acc.x, 0.f, fmaf(acc.y, 0.f, fmaf(acc.z, 0.f, fmaf(acc.w, 0.f, bad))));
        if (!whole) {                                  // the state, for the merging launch
          if (mine) *(float4*)(rec + 8 * quad + 4 * h) = acc;
        } else {
          const half2_t c0 = {(half_t)(acc.x * inv), (half_t)(acc.y * inv)};
          const half2_t c1 = {(half_t)(acc.z * inv), (half_t)(acc.w * inv)};
          w[e][0] = __builtin_bit_cast(unsigned, c0);
          w[e][1] = __builtin_bit_cast(unsigned, c1);
        }
      }
      if (whole) {
        // lane half h holds dims 8 quad + 4 h .. + 3 of quads k and k + 1: exchanged, half 0 has
        // all 8 dims of quad k and half 1 those of quad k + 1
        const auto r0 = __builtin_amdgcn_permlane32_swap(w[0][0], w[1][0], false, false);
        const auto r1 = __builtin_amdgcn_permlane32_swap(w[0][1], w[1][1], false, false);
        const u32x4 st = {r0[0], r1[0], r0[1], r1[1]};
        if (mine) *(u32x4*)(op + 8 * (grp * NQ + k + h)) = st;
      }
    }
    if (!whole && mine && grp == 0 && h == 0) *(float2*)(rec + 128) = make_float2(M, den);
    const uint64_t lanes = __ballot(bad != bad && mine);
    if (lane == 0) bad_rows[rt][grp] = (uint32_t)lanes | (uint32_t)(lanes >> 32);
  }
  if (!rows_here && lane == 0) bad_rows[rt][grp] = 0;
  __syncthreads();
  uint32_t again = 0;
  for (int k = 0; k < S; ++k) again |= bad_rows[rt][k];
  for (int i = 0; again; ++i, again &= again - 1) {
    if (i % S != grp) continue;
    const int r = 32 * rt + __ffs(again) - 1;
    tree_row(a, slot, s, g, 32 * R * rb + r, L, u0 * UNIT, min((u0 + steps) * UNIT, end),
             whole ? nullptr : state + r * ATT_REC);
  }
  __syncthreads();                                     // the LDS is the next stretch's
  }
  // on to the next item
  left -= steps;
  u0 = 0;
  if (left > 0 && ++g == a.nkv) {
    g = 0;
    while (++s < a.n - 1 && seqs[4 * s + 2] == 0) {}
    L = seqs[4 * s];
    used = seqs[4 * s + 1];
    slot = seqs[4 * s + 3];
  }
  }
}

// The states of a (node, query head) row to its output, for items that more than one column has
// parts of.  Half a wave takes a part's state, four dims a lane; a row's parts go round GROUPS
// half waves, four in flight in each, and the groups meet in LDS.  One group a row for a handful
// of parts, eight (a workgroup a row) for many: 32 at 4000 keys 7.2 us in one wave.
template <int GROUPS>
__global__ __launch_bounds__(256) void tree_merge_kernel(TreeArgs a, const int* __restrict__ heads,
                                                         int block_rows, int64_t rows) {
  __shared__ __attribute__((aligned(16))) float acc[GROUPS][TREE_HD];
  __shared__ float ml[GROUPS][2];
  const int half = threadIdx.x >> 5, l = threadIdx.x & 31;
  const int grp = half % GROUPS;
  const int64_t r = (int64_t)blockIdx.x * (8 / GROUPS) + half / GROUPS;
  if (r >= rows) return;
  const int nh = a.nkv * a.G;
  const int tok = (int)(r / nh), head = (int)(r - (int64_t)tok * nh);
  const int s = tok / a.T, node = tok - s * a.T, g = head / a.G;
  const i32x4 seq = *(const i32x4*)(a.seqs + 4 * s);
  const int2 at = *(const int2*)(heads + 2 * (s * a.nkv + g));
  const int first = at.x & ~(1 << 30), splits = at.y - first + 1;
  if (node >= seq[1] || seq[2] == 0 || splits == 1) return;
  const int row = node * a.G + head - g * a.G, rb = row / block_rows;
  const int64_t block = (int64_t)block_rows * ATT_REC, step = a.rblocks * 2 * block;
  const float* rec = a.states + (int64_t)first * step + rb * 2 * block + (row - rb * block_rows) * ATT_REC;
  const int64_t skip = at.x >> 30 ? block : 0;       // in its first column the item is the second
  float M = -INFINITY, den = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int k0 = grp; k0 < splits; k0 += 4 * GROUPS) {
    float2 st[4];
    float4 v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int k = k0 + j * GROUPS;
      st[j] = make_float2(-INFINITY, 0.f);
      v[j] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (k < splits) {
        const float* from = rec + k * step + (k ? 0 : skip);
        st[j] = *(const float2*)(from + 128);
        v[j] = *(const float4*)(from + 4 * l);
      }
    }
    const float mn = fmaxf(fmaxf(fmaxf(st[0].x, st[1].x), fmaxf(st[2].x, st[3].x)), M);
    const float ref = mn == -INFINITY ? 0.f : mn;
    const float f = exp2f(M - ref);
    M = mn;
    den *= f;
    o = make_float4(o.x * f, o.y * f, o.z * f, o.w * f);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float e = exp2f(st[j].x - ref);
      den = fmaf(e, st[j].y, den);
      o.x = fmaf(e, v[j].x, o.x);
      o.y = fmaf(e, v[j].y, o.y);
      o.z = fmaf(e, v[j].z, o.z);
      o.w = fmaf(e, v[j].w, o.w);
    }
  }
  if (GROUPS > 1) {
    *(float4*)&acc[grp][4 * l] = o;
    if (l == 0) {
      ml[grp][0] = M;
      ml[grp][1] = den;
    }
    __syncthreads();
    if (grp) return;
#pragma unroll
    for (int k = 1; k < GROUPS; ++k) M = fmaxf(M, ml[k][0]);
    const float ref = M == -INFINITY ? 0.f : M;
    den = 0.f;
    o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int k = 0; k < GROUPS; ++k) {
      const float e = exp2f(ml[k][0] - ref);
      const float4 v = *(const float4*)&acc[k][4 * l];
      den = fmaf(e, ml[k][1], den);
      o.x = fmaf(e, v.x, o.x);
      o.y = fmaf(e, v.y, o.y);
      o.z = fmaf(e, v.z, o.z);
      o.w = fmaf(e, v.w, o.w);
    }
  }
  const float inv = den == 0.f ? 0.f : 1.0f / den;
  const half4_t h4 = {(half_t)(o.x * inv), (half_t)(o.y * inv), (half_t)(o.z * inv), (half_t)(o.w * inv)};
  *(half4_t*)(a.out + (int64_t)tok * a.out_stride + head * TREE_HD + 4 * l) = h4;
}

// The workgroup forms, (rows, groups): 32 R rows, S key groups of KT-key tiles.
static int tree_form(int rows, int groups, int* unit) {
  *unit = groups * (groups == 2 ? 64 : 32);
  return rows * groups == 256 && (groups == 2 || groups == 4 || groups == 8) ? groups : 0;
}

// 32-bit positions, indexes into the schedule, products of a column and an item's units hold.
static bool tree_size_ok(int64_t n, int64_t nkv, int64_t columns, int max_len, int unit, int least) {
  const int64_t units = ((int64_t)max_len + unit - 1) / unit;
  return max_len <= 1 << 30 && n * nkv <= 1 << 24 && columns <= 1 << 24 && n * nkv * units <= 0x3fffffff &&
         (!least || (columns <= 32767 && columns * units <= 0x7fffffff));
}

// A workgroup divides its (node, query head) rows by the heads' ratio through a 32-bit reciprocal.
static bool tree_heads_ok(int n_nodes, int64_t ratio) {
  return n_nodes * ratio * ratio <= (int64_t)1 << 32;
}

// schedule: [n][4] seqs, [ncols][8] columns, [n][nkv][2] heads
static int64_t tree_schedule_ints(int n, int nkv, int ncols) {
  return 4 * (int64_t)n + 8 * (int64_t)ncols + 2 * (int64_t)n * nkv;
}

extern "C" int omni_tree_plan(const int* parents, const int* counts, const int64_t* slots,
                              const int64_t* lengths, const int64_t* rope_delta, int n, int n_nodes,
                              int pool_rows, int max_len, int64_t* starts, void* ancestors,
                              int64_t* positions, int64_t* token_slot, int64_t* token_pos,
                              int n_kv_heads, int rows, int groups, int columns, int least,
                              int* schedule, int64_t schedule_ints, void* stream) {
  if (n < 0 || n_nodes < 1 || pool_rows <= 0 || max_len <= 0 || n_kv_heads <= 0) return OMNI_EINVAL;
  if (n_nodes > TREE_MAX) return OMNI_EUNSUPPORTED;
  if (!slots && n > pool_rows) return OMNI_EINVAL;
  int unit;
  if (!tree_form(rows, groups, &unit) || columns < 1 || least < 0) return OMNI_EINVAL;
  if (!least && columns != (int64_t)n * n_kv_heads && n) return OMNI_EINVAL;
  if (!tree_size_ok(n, n_kv_heads, columns, max_len, unit, least)) return OMNI_EUNSUPPORTED;
  if (n == 0) return OMNI_OK;
  if (!parents || !lengths || !starts || !ancestors || !positions || !token_slot || !token_pos ||
      !schedule || ((uintptr_t)schedule & 15))
    return OMNI_EINVAL;
  if (schedule_ints < tree_schedule_ints(n, n_kv_heads, columns)) return OMNI_EINVAL;
  TreeCols tc = {schedule, schedule + 4 * (int64_t)n, schedule + 4 * (int64_t)n + 8 * (int64_t)columns,
                 columns, n_kv_heads, unit, least};
  hipLaunchKernelGGL(tree_plan_kernel, dim3(n), dim3(64), 0, (hipStream_t)stream, parents, counts,
                     slots, lengths, rope_delta, n, n_nodes, pool_rows, max_len, starts,
                     (uint64_t*)ancestors, positions, token_slot, token_pos, tc);
  OMNI_CHECK_LAUNCH();
  return OMNI_OK;
}

extern "C" int omni_kv_write_rows(const void* k, int64_t k_stride, const void* v, int64_t v_stride,
                                  void* k_cache, void* v_cache, const int64_t* slots,
                                  const int64_t* positions, int pool_rows, int max_len,
                                  int row_halfs, int tokens, void* stream) {
  if (tokens < 0 || pool_rows <= 0 || max_len <= 0 || row_halfs <= 0) return OMNI_EINVAL;
  if ((row_halfs & 7) || (k_stride & 7) || (v_stride & 7) || tokens > 0xffffff) return OMNI_EUNSUPPORTED;
  if (k_stride < row_halfs || v_stride < row_halfs) return OMNI_EINVAL;
  if (tokens == 0) return OMNI_OK;
  if (!k || !v || !k_cache || !v_cache || !slots || !positions) return OMNI_EINVAL;
  if (((uintptr_t)k | (uintptr_t)v | (uintptr_t)k_cache | (uintptr_t)v_cache) & 15) return OMNI_EINVAL;
  hipLaunchKernelGGL(kv_rows_kernel, dim3(tokens), dim3(256), 0, (hipStream_t)stream,
                     (const half_t*)k, k_stride, (const half_t*)v, v_stride, (half_t*)k_cache,
                     (half_t*)v_cache, slots, positions, pool_rows, max_len, row_halfs);
  OMNI_CHECK_LAUNCH();
  return OMNI_OK;
}

extern "C" int omni_tree_attention(const void* q, int64_t q_stride, const void* k_cache,
                                   const void* v_cache, int pool_rows, int max_len,
                                   const void* ancestors, int n, int n_nodes, void* out,
                                   int out_stride, int n_heads, int n_kv_heads,
                                   int head_dim, float scale, int rows, int groups, int columns,
                                   int least, const int* schedule, float* workspace,
                                   int64_t workspace_floats, void* stream) {
  if (n < 0 || n_nodes < 1 || n_heads <= 0 || n_kv_heads <= 0 || pool_rows <= 0 || max_len <= 0)
    return OMNI_EINVAL;
  if (head_dim != TREE_HD || n_heads % n_kv_heads || n_heads > 65536 || n_nodes > TREE_MAX)
    return OMNI_EUNSUPPORTED;
  if (!(scale >= 0x1p-126f) || scale > 0x1p126f) return OMNI_EUNSUPPORTED;
  int unit;
  const int form = tree_form(rows, groups, &unit);
  if (!form || columns < 1 || least < 0) return OMNI_EINVAL;
  if (!least && columns != (int64_t)n * n_kv_heads && n) return OMNI_EINVAL;
  if (!tree_size_ok(n, n_kv_heads, columns, max_len, unit, least)) return OMNI_EUNSUPPORTED;
  if (!tree_heads_ok(n_nodes, n_heads / n_kv_heads)) return OMNI_EUNSUPPORTED;
  const int64_t rblocks = ((int64_t)n_nodes * (n_heads / n_kv_heads) + rows - 1) / rows;
  const int64_t grid = (columns + 7) / 8 * 8 * rblocks, out_rows = (int64_t)n * n_nodes * n_heads;
  // the merge: parts of an item are at least one, some columns / items
  const bool wide = columns > 8 * (int64_t)n * n_kv_heads;
  const int64_t merges = !least ? 0 : wide ? out_rows : (out_rows + 7) / 8;
  // a launch counts its threads in 32 bits
  if (512 * grid > 0xffffffff || 256 * merges > 0xffffffff || out_rows > 0x7fffffff)
    return OMNI_EUNSUPPORTED;
  if (q_stride < n_heads * TREE_HD || (q_stride & 7)) return OMNI_EINVAL;
  if (out_stride < n_heads * TREE_HD || (out_stride & 7)) return OMNI_EINVAL;
  if (n == 0) return OMNI_OK;
  if (!q || !k_cache || !v_cache || !ancestors || !schedule || !out) return OMNI_EINVAL;
  if (((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)out | (uintptr_t)schedule) & 15)
    return OMNI_EINVAL;
  TreeArgs a;
  a.G = n_heads / n_kv_heads;
  a.magic = 0xffffffffu / a.G + 1;                     // exact for rows below 2^32 / G: tree_heads_ok
  if (least && (!workspace || ((uintptr_t)workspace & 15) ||
                workspace_floats < columns * rblocks * 2 * rows * ATT_REC))
    return OMNI_EINVAL;
  a.q = (const half_t*)q;
  a.q_stride = q_stride;
  a.k_cache = (const half_t*)k_cache;
  a.v_cache = (const half_t*)v_cache;
  a.max_len = max_len;
  a.nkv = n_kv_heads;
  a.T = n_nodes;
  a.n = n;
  a.ncols = columns;
  a.rblocks = (int)rblocks;
  a.ancestors = (const uint64_t*)ancestors;
  a.seqs = schedule;
  a.columns = schedule + 4 * (int64_t)n;
  a.out = (half_t*)out;
  a.out_stride = out_stride;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.states = workspace;
  const dim3 gd((unsigned)grid);
  hipStream_t st = (hipStream_t)stream;
  if (form == 2)
    hipLaunchKernelGGL((tree_attn_kernel<4, 2, 64>), gd, dim3(512), 0, st, a);
  else if (form == 4)
    hipLaunchKernelGGL((tree_attn_kernel<2, 4, 32>), gd, dim3(512), 0, st, a);
  else
    hipLaunchKernelGGL((tree_attn_kernel<1, 8, 32>), gd, dim3(512), 0, st, a);
  OMNI_CHECK_LAUNCH();
  if (least) {
    const int* heads = a.columns + 8 * (int64_t)columns;
    if (wide)
      hipLaunchKernelGGL((tree_merge_kernel<8>), dim3((unsigned)merges), dim3(256), 0, st, a, heads,
                         rows, out_rows);
    else
      hipLaunchKernelGGL((tree_merge_kernel<1>), dim3((unsigned)merges), dim3(256), 0, st, a, heads,
                         rows, out_rows);
    OMNI_CHECK_LAUNCH();
  }
  return OMNI_OK;
}
