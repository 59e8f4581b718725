// Attention of one new token per sequence over a paged KV cache, split over the cache's length.
//
// Row i of the schedule (omni_page_reserve) attends to keys [0, keys_i) of the sequence whose block
// table is tables[i]: softmax(scale q K^T) V, heads grouped.  What the tables of a group of neighbours
// share is read once for all of them.
#include "common.h"

#include <type_traits>

#define PA_WAVES 4
#define PA_UNIT 128                // keys of a workgroup's step: 32 a wave
// KV heads from which on a column's heads are neighbouring workgroups, on XCDs of their own, and not
// its columns: 32 x 2048 tokens of 16 heads 97.6 us, the other way 105; 32 x 4096 of 8 heads 103 and
// 107; 200 x 1000 of 4 heads 88.7 and 87.0; 32 x 2048 of 2 heads 19.5 and 18.6.
#define PA_BY_HEAD 8

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));

template <bool BF>
__device__ __forceinline__ f32x4 pa_mfma(u32x4 a, u32x4 b, f32x4 c) {
  if (BF)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                   __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  return mfma16x16x32(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c);
}
// The lower and upper half of a packed pair as fp32.
template <bool BF>
__device__ __forceinline__ float pa_half(uint32_t v, bool upper) {
  if (BF) return __builtin_bit_cast(float, upper ? v & 0xffff0000u : v << 16);
  return (float)__builtin_bit_cast(half2_t, v)[upper ? 1 : 0];
}
template <bool BF>
__device__ __forceinline__ uint32_t pa_pack(float lo, float hi) {
  if (BF) {
    typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
    const bf16x2_t v = {(__bf16)lo, (__bf16)hi};
    return __builtin_bit_cast(uint32_t, v);
  }
  const half2_t v = {(half_t)lo, (half_t)hi};
  return __builtin_bit_cast(uint32_t, v);
}

struct PagedArgs {
  const unsigned short* q;
  int64_t q_stride;
  const unsigned short* k_cache;
  const unsigned short* v_cache;
  int pages, shift, nkv, G, n, ncols, width, most;
  const int* tables;
  const int* schedule;
  unsigned short* out;
  int64_t out_stride;
  float scale_log2;
  float* states;                 // [nkv][shared_recs] then [nkv][own_recs] records of HD + 4
  int shared_recs, own_recs;
  int by_head;                   // workgroups in the order of KV heads, not of columns
};

// The record of a row's head in a column: the columns and rows of an item ascend together, so that
// column times the most records of a column, plus those of the rows before, is a place of its own.
__device__ __forceinline__ int pa_shared_rec(const PagedArgs& a, int g, int col, int row, int h) {
  return g * a.shared_recs + (col * a.most + row) * a.G + h;
}
__device__ __forceinline__ int pa_own_rec(const PagedArgs& a, int g, int col, int row, int h) {
  return a.nkv * a.shared_recs + g * a.own_recs + (col + row) * a.G + h;
}

typedef const __attribute__((address_space(4))) int plan_int;

// Queries of an item, 16 a tile: query c is row c / G of its rows, head c % G.
struct PaItem {
  int row, rows, heads, keys0, end, h0, g;
  const plan_int* table;
};

// Where 32 keys are: two runs of 16, each in one page, and how many of each there are.
struct PaPlace {
  int64_t at[2];
  int there[2];
  __device__ __forceinline__ PaPlace(const PagedArgs& a, const PaItem& it, int kb, int HD) {
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const int k0 = min(kb, it.end - 1) + 16 * b;
      there[b] = min(it.end - k0, 16);
      int page = it.table[min(min(k0, it.end - 1) >> a.shift, a.width - 1)];
      if (page < 0 || page >= a.pages) {
        page = 0;
        there[b] = 0;
      }
      at[b] = (((int64_t)page << a.shift) + (k0 & ((1 << a.shift) - 1))) * a.nkv * HD + it.g * HD;
    }
  }
};

// ---------------------------------------------------------------------------
// A wave takes 32 keys a step: S^T = K Q^T as two 16x16 tiles of keys by up to 16 queries, K rows
// straight from memory in the matrix operand's layout.  In S^T a lane holds, of its query, the keys
// 4 g4 .. + 3 of each tile; taken as the k index of the second product that is the operand P^T as it
// stands, if V^T's k index names the same keys.  V rows are read whole, 16 lanes a row, a lane HD /
// 16 columns of each of its eight keys, and its operand for output tile t is column t of these: two
// halves a v_perm.  Output row m of tile t is then column m HD / 16 + t.  Nothing goes through LDS
// before the waves' states are merged.
//
// Keys that are not there (of a page outside the pool, or past the item) have probability 0 and
// their V taken as 0, whatever the memory holds.
//
// P goes into the second product in 16-bit parts that hold its 24 bits (bf16: three) or 22 (fp16: two),
// rounded, rest, and the rest's rest: the matrix cores are idle otherwise, and the outputs are off by
// their own rounding alone (2.1e-4 of their size in fp16, 1.7e-3 in bf16; with the rounded part alone
// 2.6e-4 and 2.1e-3).  The second part costs 3 % (32 x 2048 tokens 15.1 -> 15.7 us), which the next
// step's loads, issued as soon as this one's K and V are used up, give back.  bf16's third costs up to 3 %
// (32 x 4096 tokens of 8 KV heads 101.5 -> 103.6 us, 128 x 4096 in groups of 4 beams 32.9 -> 33.7, 64 x
// 20-4000 of 16 97.1 both): of 65536 outputs 13 are rounded to the other neighbour instead of 128, and
// where terms cancel an output is no longer off by 2^-18 of them, many of its own steps.
//
// In fp16 all of them, and the sums with them, are 2^15 times as large: its steps end at 2^-24, and of a
// largest probability of 1 the keys below 2^-25 that a wave has beside it would be gone from the product
// though not from the sum (60 keys of 2^-20 to 2^-35 beside one of 1: an output 2.5 times as far off as
// fp32's would be).  Of 2^15 a step is 2^-39.
//
// The bound is the K/V bytes.  MI355X: a kernel that only reads takes 10.4 us for 64 MB, 19.3 for 128 MB
// (which the cache holds), 88 for 512 MB (6.1 TB/s).  Here, us with the merge, launches in a row over one
// layer's K/V (of which the cache holds 256 MB): 32 x 2048 tokens of 2 KV heads 18.8 (67 MB; 15.5 + 3.9),
// 32 x 2048 of 16 96 (538 MB, 5.5 TB/s), 32 x 4096 of 8 102, 200 x 1000 of 4 83, 128 x 4096 of 2 in groups
// of 4 beams 32 (131 MB; each row for itself 79).  Over 28 layers one after another, as a step has it: 32 x
// 2048 22, the groups 38, one row of 32000 tokens of 4 heads 20 (66 MB; 18 from the cache).
// What is left of the small ones is start and end: schedule, table and Q loads behind each other (3 us),
// the waves' merge through LDS, the merging launch.
// ---------------------------------------------------------------------------
template <bool BF, int HD, int NT>
struct PaState {
  static constexpr int CV = HD / 16;                // columns of a V row a lane reads
  static constexpr int KC = HD / 32;                // matrix operands of a K row
  static constexpr int PARTS = BF ? 3 : 2;          // of a probability
  static constexpr float UNIT_P = BF ? 1.f : 0x1p15f;   // the largest probability, and what l counts in
  u32x4 qf[NT][KC];
  f32x4 o[NT][CV];
  float m[NT], l[NT];

  __device__ __forceinline__ void load(const PagedArgs& a, const PaItem& it, int l16, int g4) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int c = n * 16 + l16;
      // c / G by a product, for several rows (c < 32, G <= 16)
      const int r = it.rows > 1 ? c * (65536 / it.heads + 1) >> 16 : 0, h = c - r * it.heads;
      const bool in = c < it.rows * it.heads;
      const unsigned short* qp = a.q + (it.row + r) * a.q_stride +
                                 (int64_t)(it.g * a.G + it.h0 + h) * HD + g4 * 8;
#pragma unroll
      for (int j = 0; j < KC; ++j) qf[n][j] = in ? *(const u32x4*)(qp + j * 32) : (u32x4){0, 0, 0, 0};
#pragma unroll
      for (int t = 0; t < CV; ++t) o[n][t] = (f32x4){0.f, 0.f, 0.f, 0.f};
      m[n] = -INFINITY;
      l[n] = 0.f;
    }
  }

  u32x4 kf[2][KC];
  uint32_t vf[8][CV / 2];

  __device__ __forceinline__ void load_k(const PagedArgs& a, const PaPlace& at, int l16, int g4) {
    const int tstride = a.nkv * HD;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int j = 0; j < KC; ++j)
        kf[b][j] = *(const u32x4*)(a.k_cache + at.at[b] + l16 * tstride + j * 32 + g4 * 8);
  }
  __device__ __forceinline__ void load_v(const PagedArgs& a, const PaPlace& at, int l16, int g4) {
    const int tstride = a.nkv * HD;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      __builtin_memcpy(vf[e], a.v_cache + at.at[e >> 2] + (4 * g4 + (e & 3)) * tstride + l16 * CV, 2 * CV);
  }

  // The keys at kb; the next step's K goes out once this one's is used up, and V likewise.
  __device__ __forceinline__ void step(const PagedArgs& a, const PaPlace& at, const PaPlace& then, bool more,
                                       int l16, int g4) {
    const bool part = at.there[0] < 16 || at.there[1] < 16;
    f32x4 s[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        s[n][b] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < KC; ++j) s[n][b] = pa_mfma<BF>(kf[b][j], qf[n][j], s[n][b]);
      }
    if (more) load_k(a, then, l16, g4);
    u32x4 pf[NT][PARTS];
    float alpha[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      if (part) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (4 * g4 + (e & 3) >= at.there[e >> 2]) s[n][e >> 2][e & 3] = -INFINITY;
      }
      float top = -INFINITY;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        s[n][e >> 2][e & 3] *= a.scale_log2;
        top = fmaxf(top, s[n][e >> 2][e & 3]);
      }
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      const float mn = fmaxf(m[n], top), ref = mn == -INFINITY ? 0.f : mn;
      alpha[n] = exp2f(m[n] - ref);
      m[n] = mn;
      l[n] *= alpha[n];
      float p[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        p[e] = __builtin_amdgcn_exp2f(s[n][e >> 2][e & 3] - ref) * UNIT_P;   // 0 below 2^-126
        l[n] += p[e];
      }
#pragma unroll
      for (int d = 0; d < 4; ++d) {
#pragma unroll
        for (int i = 0; i < PARTS; ++i) {
          const uint32_t w = pa_pack<BF>(p[2 * d], p[2 * d + 1]);
          pf[n][i][d] = w;
          p[2 * d] -= pa_half<BF>(w, false);
          p[2 * d + 1] -= pa_half<BF>(w, true);
        }
      }
    }
    if (part) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const bool off = 4 * g4 + (e & 3) >= at.there[e >> 2];
#pragma unroll
        for (int d = 0; d < CV / 2; ++d) vf[e][d] = off ? 0 : vf[e][d];
      }
    }
#pragma unroll
    for (int t = 0; t < CV; ++t) {
      u32x4 vt;
#pragma unroll
      for (int d = 0; d < 4; ++d)
        vt[d] = __builtin_amdgcn_perm(vf[2 * d + 1][t / 2], vf[2 * d][t / 2],
                                      t & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        o[n][t] *= alpha[n];
#pragma unroll
        for (int i = 0; i < PARTS; ++i) o[n][t] = pa_mfma<BF>(vt, pf[n][i], o[n][t]);
      }
    }
    if (more) load_v(a, then, l16, g4);
  }
};

template <bool BF, int HD>
__global__ __launch_bounds__(64 * PA_WAVES, 2) void paged_attn_kernel(PagedArgs a) {
  constexpr int CV = HD / 16, OS = HD + 4;
  __shared__ __attribute__((aligned(16))) float o_lds[PA_WAVES][16][OS];
  __shared__ float ml_lds[PA_WAVES][2][16];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, g4 = lane >> 4;
  const int col = a.by_head ? blockIdx.y : blockIdx.x;
  const plan_int* schedule = (const plan_int*)a.schedule;
  const plan_int* column = schedule + 8 * a.n + 4 * col;
  int item = column[0], u0 = column[1], left = column[2];
  PaItem it;
  it.g = a.by_head ? blockIdx.x : blockIdx.y;
  it.h0 = blockIdx.z * 32;
  it.heads = min(32, a.G - it.h0);
  while (left > 0) {
    const int i = item >> 1;
    const plan_int* row = schedule + 8 * i;
    const int keys = row[0], S = row[1], own = item & 1;
    it.row = i;
    it.rows = own ? 1 : row[3];
    it.keys0 = own ? S * PA_UNIT : 0;
    it.end = own ? keys : S * PA_UNIT;
    it.table = (const plan_int*)(a.tables + (int64_t)i * a.width);
    const int units = ceil_div(it.end - it.keys0, PA_UNIT), steps = min(left, units - u0);
    if (steps <= 0) break;                          // no schedule of omni_page_reserve's
    const int from = it.keys0 + u0 * PA_UNIT, to = min(from + steps * PA_UNIT, it.end);
    const int queries = it.rows * it.heads;
    const bool whole = own && !S && u0 == 0 && steps == units;
    auto run = [&](auto tiles) {
      constexpr int NT = decltype(tiles)::value;
      PaState<BF, HD, NT> st;
      st.load(a, it, l16, g4);
      int kb = from + wave * 32;
      if (kb < to) {
        PaPlace at(a, it, kb, HD);
        st.load_k(a, at, l16, g4);
        st.load_v(a, at, l16, g4);
        for (; kb < to; kb += PA_UNIT) {
          const bool more = kb + PA_UNIT < to;
          const PaPlace then(a, it, more ? kb + PA_UNIT : kb, HD);
          st.step(a, at, then, more, l16, g4);
          at = then;
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float l = st.l[n];
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
        if (g4 == 0) {
          ml_lds[wave][0][l16] = st.m[n];
          ml_lds[wave][1][l16] = l;
        }
        // lane (g4, l16): query l16, columns (4 g4 + r) CV + t
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int t = 0; t < CV; t += 4) {
            const f32x4 v = {st.o[n][t][r], st.o[n][t + 1][r], st.o[n][t + 2][r], st.o[n][t + 3][r]};
            *(f32x4*)&o_lds[wave][l16][(4 * g4 + r) * CV + t] = v;
          }
        __syncthreads();
        // 16 threads a query
        const int q = tid >> 4, c = (tid & 15) * CV, query = n * 16 + q;
        if (query < queries) {
          float M = -INFINITY, L = 0.f, v[CV];
#pragma unroll
          for (int t = 0; t < CV; ++t) v[t] = 0.f;
#pragma unroll
          for (int w = 0; w < PA_WAVES; ++w) M = fmaxf(M, ml_lds[w][0][q]);
#pragma unroll
          for (int w = 0; w < PA_WAVES; ++w) {
            const float f = M == -INFINITY ? 0.f : exp2f(ml_lds[w][0][q] - M);
            L = fmaf(f, ml_lds[w][1][q], L);
#pragma unroll
            for (int t = 0; t < CV; ++t) v[t] = fmaf(f, o_lds[w][q][c + t], v[t]);
          }
          if (whole) {
            const int head = it.g * a.G + it.h0 + query;
            unsigned short* op = a.out + i * a.out_stride + (int64_t)head * HD + c;
            const float inv = L == 0.f ? 0.f : 1.f / L;
            uint32_t w[CV / 2];
#pragma unroll
            for (int t = 0; t < CV; t += 2) w[t / 2] = pa_pack<BF>(v[t] * inv, v[t + 1] * inv);
            __builtin_memcpy(op, w, 2 * CV);
          } else {
            float* rec = a.states + (own ? pa_own_rec(a, it.g, col, i, it.h0 + query)
                                         : pa_shared_rec(a, it.g, col, i, query)) * OS;
#pragma unroll
            for (int t = 0; t < CV; t += 4)
              *(float4*)(rec + c + t) = make_float4(v[t], v[t + 1], v[t + 2], v[t + 3]);
            if (c == 0) *(float2*)(rec + HD) = make_float2(M, L);
          }
        }
        __syncthreads();
      }
    };
    if (queries <= 16) run(std::integral_constant<int, 1>());
    else run(std::integral_constant<int, 2>());
    left -= steps;
    u0 = 0;
    if (left > 0) {
      if (own) {
        int next = i;
        do ++next;
        while (next < a.n - 1 && schedule[8 * next] == 0);
        if (next >= a.n) break;
        const plan_int* after = schedule + 8 * next;
        item = 2 * next + (after[1] && after[2] == next ? 0 : 1);
      } else {
        ++item;
      }
    }
  }
}

// The states of a row that several columns share, merged: one workgroup a row, head and DIMS of its
// columns, DIMS / 4 lanes a state.  All maxima first, a state a thread, then every state's outputs
// once, by its factor: no load waits for another state's.  Rows without keys are zero.  28 heads of 128
// states 4.2 us, a state after another 7.8.
#define PA_PARTS 256               // states in a round
template <bool BF, int HD, int DIMS>
__global__ __launch_bounds__(256) void paged_merge_kernel(PagedArgs a) {
  constexpr int OS = HD + 4, LANES = DIMS / 4, SETS = 256 / LANES, DEEP = 4;
  __shared__ float factor[PA_PARTS], wred[2][4];
  __shared__ __attribute__((aligned(16))) float part[SETS][DIMS];
  const int i = blockIdx.y, h = blockIdx.x, tid = threadIdx.x, g = blockIdx.z / (HD / DIMS);
  const int head = g * a.G + h, d0 = blockIdx.z % (HD / DIMS) * DIMS;
  const plan_int* row = (const plan_int*)a.schedule + 8 * i;
  const int keys = row[0], S = row[1];
  const int shared = S ? row[5] - row[4] + 1 : 0, n = keys ? shared + row[7] - row[6] + 1 : 0;
  if (n == 1) return;                               // written where it was made
  const int set = tid / LANES, c = (tid % LANES) * 4;
  const int rec0 = pa_shared_rec(a, g, row[4], i, h) * OS, next0 = a.most * a.G * OS;
  const int rec1 = pa_own_rec(a, g, row[6] - shared, i, h) * OS, next1 = a.G * OS;
  auto rec = [&](int p) { return a.states + (p < shared ? rec0 + p * next0 : rec1 + p * next1); };
  float M = -INFINITY, L = 0.f;
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
  for (int base = 0; base < n; base += PA_PARTS) {
    const int here = min(n - base, PA_PARTS);
    float2 s = make_float2(-INFINITY, 0.f);
    if (tid < here) s = *(const float2*)(rec(base + tid) + HD);
    // the first states' outputs are on their way meanwhile
    f32x4 x[DEEP];
#pragma unroll
    for (int u = 0; u < DEEP; ++u)
      if (set + u * SETS < here) x[u] = *(const f32x4*)(rec(base + set + u * SETS) + d0 + c);
    const float top = wave_max(s.x);
    if ((tid & 63) == 0) wred[0][tid >> 6] = top;
    __syncthreads();
    const float mn = fmaxf(M, fmaxf(fmaxf(wred[0][0], wred[0][1]), fmaxf(wred[0][2], wred[0][3])));
    const float ref = mn == -INFINITY ? 0.f : mn, old = exp2f(M - ref), f = exp2f(s.x - ref);
    factor[tid] = f;
    const float sum = wave_sum(f * s.y);
    if ((tid & 63) == 0) wred[1][tid >> 6] = sum;
    __syncthreads();
    L = L * old + ((wred[1][0] + wred[1][1]) + (wred[1][2] + wred[1][3]));
    M = mn;
    v *= old;
#pragma unroll
    for (int u = 0; u < DEEP; ++u)
      if (set + u * SETS < here) v += x[u] * factor[set + u * SETS];
#pragma unroll 4
    for (int p = set + DEEP * SETS; p < here; p += SETS)
      v += *(const f32x4*)(rec(base + p) + d0 + c) * factor[p];
  }
  *(f32x4*)&part[set][c] = v;
  __syncthreads();
  if (tid >= DIMS / 2) return;
  float y0 = 0.f, y1 = 0.f;
#pragma unroll
  for (int k = 0; k < SETS; ++k) {
    const float2 y = *(const float2*)&part[k][2 * tid];
    y0 += y.x;
    y1 += y.y;
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  *(uint32_t*)(a.out + i * a.out_stride + (int64_t)head * HD + d0 + 2 * tid) = pa_pack<BF>(y0 * inv, y1 * inv);
}

// The same where rows have few states: one wave a row and head, two columns a lane, sixteen states at
// a time.  128 rows of 12 heads 4.5 us.
template <bool BF, int HD>
__global__ __launch_bounds__(256) void paged_merge_few_kernel(PagedArgs a) {
  constexpr int OS = HD + 4;
  const int lane = threadIdx.x & 63, heads = a.nkv * a.G, c = 2 * (lane & (HD / 2 - 1));
  const int i = blockIdx.y, head = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
  if (head >= heads) return;
  const plan_int* row = (const plan_int*)a.schedule + 8 * i;
  const int keys = row[0], S = row[1];
  const int shared = S ? row[5] - row[4] + 1 : 0, n = keys ? shared + row[7] - row[6] + 1 : 0;
  if (n == 1) return;                               // written where it was made
  const int g = head / a.G, h = head - g * a.G;
  const int rec0 = pa_shared_rec(a, g, row[4], i, h) * OS, next0 = a.most * a.G * OS;
  const int rec1 = pa_own_rec(a, g, row[6] - shared, i, h) * OS, next1 = a.G * OS;
  auto rec = [&](int p) { return a.states + (p < shared ? rec0 + p * next0 : rec1 + p * next1); };
  float M = -INFINITY, L = 0.f, y0 = 0.f, y1 = 0.f;
#pragma unroll 1
  for (int base = 0; base < n; base += 16) {
    float2 x[16], s = make_float2(-INFINITY, 0.f);
#pragma unroll
    for (int u = 0; u < 16; ++u)
      if (base + u < n) x[u] = *(const float2*)(rec(base + u) + c);
    if (base + (lane & 15) < n) s = *(const float2*)(rec(base + (lane & 15)) + HD);
    const float mn = fmaxf(M, wave_max(s.x)), ref = mn == -INFINITY ? 0.f : mn;
    const float old = exp2f(M - ref), f = exp2f(s.x - ref), fl = f * s.y;
    M = mn;
    L *= old;
    y0 *= old;
    y1 *= old;
#pragma unroll
    for (int u = 0; u < 16; ++u)
      if (base + u < n) {
        const float fu = __shfl(f, u);
        L += __shfl(fl, u);
        y0 = fmaf(fu, x[u].x, y0);
        y1 = fmaf(fu, x[u].y, y1);
      }
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  if (lane < HD / 2)
    *(uint32_t*)(a.out + i * a.out_stride + (int64_t)head * HD + c) = pa_pack<BF>(y0 * inv, y1 * inv);
}

template <bool BF, int HD>
static int pa_launch(const PagedArgs& a, hipStream_t st) {
  const int groups = ceil_div(a.G, 32);
  const dim3 grid = a.by_head ? dim3(a.nkv, a.ncols, groups) : dim3(a.ncols, a.nkv, groups);
  hipLaunchKernelGGL((paged_attn_kernel<BF, HD>), grid, dim3(64 * PA_WAVES), 0, st, a);
  OMNI_CHECK_LAUNCH();
  // few rows have many states each
  const int heads = a.nkv * a.G;
  // us of both launches, few / many: 4 rows of 64 columns 10.6 / 8.7, 8 of 32 13.4 / 11.5, 16 of 16 17.5 /
  // 17.3, 32 of 8 19.0 / 19.7, 128 of 2 (and their shared ones) 32.4 / 37.2
  if (a.ncols <= 16 * a.n)
    hipLaunchKernelGGL((paged_merge_few_kernel<BF, HD>), dim3(ceil_div(heads, 4), a.n), dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((paged_merge_kernel<BF, HD, 32>), dim3(a.G, a.n, a.nkv * (HD / 32)), dim3(256), 0, st, a);
  OMNI_CHECK_LAUNCH();
  return OMNI_OK;
}

extern "C" int omni_paged_attention(const void* q, int64_t q_stride, const void* k_cache,
                                    const void* v_cache, int dtype, int pages, int page_size,
                                    const int* tables, int width, int n, const int* schedule,
                                    int columns, int most, void* out, int64_t out_stride, int n_heads,
                                    int n_kv_heads, int head_dim, float scale, float* workspace,
                                    int64_t workspace_floats, void* stream) {
  if (n < 0 || most <= 0 || pages <= 0 || page_size <= 0 || width <= 0 || columns <= 0 || n_heads <= 0 ||
      n_kv_heads <= 0)
    return OMNI_EINVAL;
  if ((dtype != 0 && dtype != 1) || (head_dim != 64 && head_dim != 128) || n_heads % n_kv_heads)
    return OMNI_EUNSUPPORTED;
  int shift = 4;
  while (shift < 10 && (1 << shift) != page_size) ++shift;
  if ((1 << shift) != page_size || columns > 65535 || n > 65535 || n_kv_heads > 1024 ||
      n_heads > 65536)
    return OMNI_EUNSUPPORTED;
  if (!(scale >= 0x1p-126f && scale <= 0x1p126f)) return OMNI_EUNSUPPORTED;
  const int64_t width_q = (int64_t)n_heads * head_dim;
  if (q_stride < width_q || (q_stride & 7) || out_stride < width_q || (out_stride & 7))
    return OMNI_EINVAL;
  if (n == 0) return OMNI_OK;
  if (!q || !k_cache || !v_cache || !tables || !schedule || !out || !workspace) return OMNI_EINVAL;
  if (((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)out | (uintptr_t)workspace |
       (uintptr_t)schedule) & 15)
    return OMNI_EINVAL;
  const int G = n_heads / n_kv_heads;
  if (most > 1 && most * G > 32) return OMNI_EUNSUPPORTED;
  const int64_t shared_recs = most > 1 ? ((int64_t)columns * most + n) * G : 0;
  const int64_t own_recs = ((int64_t)columns + n) * G;
  const int64_t floats = n_kv_heads * (shared_recs + own_recs) * (head_dim + 4);
  if (floats > 0x7fffffff) return OMNI_EUNSUPPORTED;
  if (workspace_floats < floats) return OMNI_EINVAL;
  const PagedArgs a = {(const unsigned short*)q, q_stride, (const unsigned short*)k_cache,
                       (const unsigned short*)v_cache, pages, shift, n_kv_heads, G, n, columns, width,
                       most, tables, schedule, (unsigned short*)out, out_stride,
                       scale * 1.4426950408889634f, workspace, (int)shared_recs, (int)own_recs,
                       n_kv_heads >= PA_BY_HEAD};
  hipStream_t st = (hipStream_t)stream;
  if (dtype) return head_dim == 64 ? pa_launch<true, 64>(a, st) : pa_launch<true, 128>(a, st);
  return head_dim == 64 ? pa_launch<false, 64>(a, st) : pa_launch<false, 128>(a, st);
}
