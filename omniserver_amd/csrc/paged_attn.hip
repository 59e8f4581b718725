// Attention of one new token per sequence over a paged KV cache, split over the cache's length.
//
// Row i of the schedule (omni_page_reserve) attends to keys [0, keys_i) of the sequence whose block
// table is tables[i]: softmax(scale q K^T) V, heads grouped.
#include "common.h"

#define PA_WAVES 4
#define PA_UNIT 128                // keys of a workgroup's step: 32 a wave

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));

template <bool BF>
__device__ __forceinline__ f32x4 pa_mfma(u32x4 a, u32x4 b, f32x4 c) {
  if (BF)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                   __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  return mfma16x16x32(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c);
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
  int pages, shift, nkv, G, n, ncols, width;
  const int* tables;
  const int* schedule;
  unsigned short* out;
  int64_t out_stride;
  float scale_log2;
  float* states;                 // [ncols + n][nkv G][HD + 4]
};

// ---------------------------------------------------------------------------
// A wave takes 32 keys a step: S^T = K Q^T as two 16x16 tiles of keys by up to 16 query heads, K
// rows straight from memory in the matrix operand's layout.  In S^T a lane holds, of its query head,
// the keys 4 g4 .. + 3 of each tile; taken as the k index of the second product that is the operand
// P^T as it stands, if V^T's k index names the same keys.  V rows are read whole, 16 lanes a row, a
// lane HD / 16 columns of each of its eight keys, and its operand for output tile t is column t of
// these: two halves a v_perm.  Output row m of tile t is then column m HD / 16 + t.  Nothing goes
// through LDS before the waves' states are merged.
//
// Keys that are not there (past the length, or of a page outside the pool) have probability 0 and
// their V taken as 0, whatever the memory holds.
// ---------------------------------------------------------------------------
template <bool BF, int HD>
__global__ __launch_bounds__(64 * PA_WAVES) void paged_attn_kernel(PagedArgs a) {
  constexpr int CV = HD / 16;                       // columns of a V row a lane reads
  constexpr int KC = HD / 32;                       // matrix operands of a K row
  constexpr int OS = HD + 4;
  __shared__ __attribute__((aligned(16))) float o_lds[PA_WAVES][16][OS];
  __shared__ float ml_lds[PA_WAVES][2][16];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, g4 = lane >> 4;
  const int col = blockIdx.x, g = blockIdx.y, h0 = blockIdx.z * 16;
  const int heads = min(16, a.G - h0);
  typedef const __attribute__((address_space(4))) int plan_int;
  const plan_int* rows = (const plan_int*)a.schedule;
  const plan_int* column = rows + 4 * (a.n + col);
  int i = column[0], u0 = column[1], left = column[2];
  const int64_t tstride = (int64_t)a.nkv * HD;
  while (left > 0) {
    const int keys = rows[4 * i];
    const int units = ceil_div(keys, PA_UNIT), steps = min(left, units - u0);
    const int end = min((u0 + steps) * PA_UNIT, keys);
    const plan_int* table = (const plan_int*)(a.tables + (int64_t)i * a.width);
    u32x4 qf[KC];
    {
      const unsigned short* qp = a.q + i * a.q_stride + (int64_t)(g * a.G + h0 + l16) * HD + g4 * 8;
#pragma unroll
      for (int j = 0; j < KC; ++j)
        qf[j] = l16 < heads ? *(const u32x4*)(qp + j * 32) : (u32x4){0, 0, 0, 0};
    }
    f32x4 o[CV];
#pragma unroll
    for (int t = 0; t < CV; ++t) o[t] = (f32x4){0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    for (int kb = u0 * PA_UNIT + wave * 32; kb < end; kb += PA_UNIT) {
      const unsigned short *kp[2], *vp[2];
      int there[2];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const int k0 = kb + 16 * b;
        there[b] = min(keys - k0, 16);
        int page = table[min(k0, keys - 1) >> a.shift];
        if (page < 0 || page >= a.pages) {
          page = 0;
          there[b] = 0;
        }
        const int64_t at = (((int64_t)page << a.shift) + (k0 & ((1 << a.shift) - 1))) * tstride + g * HD;
        kp[b] = a.k_cache + at;
        vp[b] = a.v_cache + at;
      }
      u32x4 kf[2][KC];
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int j = 0; j < KC; ++j)
          kf[b][j] = *(const u32x4*)(kp[b] + l16 * tstride + j * 32 + g4 * 8);
      uint32_t vf[8][CV / 2];
#pragma unroll
      for (int e = 0; e < 8; ++e)
        __builtin_memcpy(vf[e], vp[e >> 2] + (4 * g4 + (e & 3)) * tstride + l16 * CV, 2 * CV);
      f32x4 s[2];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        s[b] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < KC; ++j) s[b] = pa_mfma<BF>(kf[b][j], qf[j], s[b]);
      }
      if (there[0] < 16 || there[1] < 16) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const bool off = 4 * g4 + (e & 3) >= there[e >> 2];
          if (off) s[e >> 2][e & 3] = -INFINITY;
#pragma unroll
          for (int d = 0; d < CV / 2; ++d) vf[e][d] = off ? 0 : vf[e][d];
        }
      }
      float top = -INFINITY;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        s[e >> 2][e & 3] *= a.scale_log2;
        top = fmaxf(top, s[e >> 2][e & 3]);
      }
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      const float mn = fmaxf(m, top), ref = mn == -INFINITY ? 0.f : mn;
      const float alpha = exp2f(m - ref);
      m = mn;
      l *= alpha;
      float p[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        p[e] = exp2f(s[e >> 2][e & 3] - ref);
        l += p[e];
      }
      const u32x4 pf = {pa_pack<BF>(p[0], p[1]), pa_pack<BF>(p[2], p[3]), pa_pack<BF>(p[4], p[5]),
                        pa_pack<BF>(p[6], p[7])};
#pragma unroll
      for (int t = 0; t < CV; ++t) {
        u32x4 vt;
#pragma unroll
        for (int d = 0; d < 4; ++d)
          vt[d] = __builtin_amdgcn_perm(vf[2 * d + 1][t / 2], vf[2 * d][t / 2],
                                        t & 1 ? 0x07060302u : 0x05040100u);
        o[t] *= alpha;
        o[t] = pa_mfma<BF>(vt, pf, o[t]);
      }
    }
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (g4 == 0) {
      ml_lds[wave][0][l16] = m;
      ml_lds[wave][1][l16] = l;
    }
    // lane (g4, l16): head l16, columns (4 g4 + r) CV + t
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int t = 0; t < CV; t += 4) {
        const f32x4 v = {o[t][r], o[t + 1][r], o[t + 2][r], o[t + 3][r]};
        *(f32x4*)&o_lds[wave][l16][(4 * g4 + r) * CV + t] = v;
      }
    __syncthreads();
    // 16 threads a head
    const int h = tid >> 4, c = (tid & 15) * CV;
    if (h < heads) {
      float M = -INFINITY, L = 0.f, v[CV];
#pragma unroll
      for (int t = 0; t < CV; ++t) v[t] = 0.f;
#pragma unroll
      for (int w = 0; w < PA_WAVES; ++w) M = fmaxf(M, ml_lds[w][0][h]);
#pragma unroll
      for (int w = 0; w < PA_WAVES; ++w) {
        const float f = M == -INFINITY ? 0.f : exp2f(ml_lds[w][0][h] - M);
        L = fmaf(f, ml_lds[w][1][h], L);
#pragma unroll
        for (int t = 0; t < CV; ++t) v[t] = fmaf(f, o_lds[w][h][c + t], v[t]);
      }
      const int head = g * a.G + h0 + h;
      if (u0 == 0 && steps == units) {
        unsigned short* op = a.out + i * a.out_stride + (int64_t)head * HD + c;
        const float inv = L == 0.f ? 0.f : 1.f / L;
        uint32_t w[CV / 2];
#pragma unroll
        for (int t = 0; t < CV; t += 2) w[t / 2] = pa_pack<BF>(v[t] * inv, v[t + 1] * inv);
        __builtin_memcpy(op, w, 2 * CV);
      } else {
        float* rec = a.states + ((int64_t)(col + i) * a.nkv * a.G + head) * OS;
#pragma unroll
        for (int t = 0; t < CV; t += 4) *(float4*)(rec + c + t) = make_float4(v[t], v[t + 1], v[t + 2], v[t + 3]);
        if (c == 0) *(float2*)(rec + HD) = make_float2(M, L);
      }
    }
    left -= steps;
    u0 = 0;
    if (left > 0)
      do ++i;
      while (i < a.n && rows[4 * i] == 0);
    __syncthreads();
  }
}

// The states of a row that several columns share, merged: one workgroup a row, head and DIMS of its
// columns, DIMS / 4 lanes a state.  All maxima first, a state a thread, then every state's outputs
// once, by its factor: no load waits for another state's.  Rows without keys are zero.
#define PA_PARTS 256               // states in a round
template <bool BF, int HD, int DIMS>
__global__ __launch_bounds__(256) void paged_merge_kernel(PagedArgs a) {
  constexpr int OS = HD + 4, LANES = DIMS / 4, SETS = 256 / LANES, DEEP = 4;
  __shared__ float factor[PA_PARTS], wred[2][4];
  __shared__ __attribute__((aligned(16))) float part[SETS][DIMS];
  const int i = blockIdx.y, head = blockIdx.x, heads = a.nkv * a.G, tid = threadIdx.x;
  const int d0 = blockIdx.z * DIMS;
  typedef const __attribute__((address_space(4))) int plan_int;
  const plan_int* row = (const plan_int*)a.schedule + 4 * i;
  const int keys = row[0], first = row[1], last = row[2];
  if (keys && first == last) return;
  const int n = keys ? last - first + 1 : 0, set = tid / LANES, c = (tid % LANES) * 4;
  const float* rec = a.states + ((int64_t)(first + i) * heads + head) * OS;
  const int64_t next = (int64_t)heads * OS;
  float M = -INFINITY, L = 0.f;
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
  for (int base = 0; base < n; base += PA_PARTS) {
    const int here = min(n - base, PA_PARTS);
    float2 s = make_float2(-INFINITY, 0.f);
    if (tid < here) s = *(const float2*)(rec + (base + tid) * next + HD);
    // the first states' outputs are on their way meanwhile
    f32x4 x[DEEP];
#pragma unroll
    for (int u = 0; u < DEEP; ++u)
      if (set + u * SETS < here) x[u] = *(const f32x4*)(rec + (base + set + u * SETS) * next + d0 + c);
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
      v += *(const f32x4*)(rec + (base + p) * next + d0 + c) * factor[p];
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

template <bool BF, int HD>
static int pa_launch(const PagedArgs& a, hipStream_t st) {
  const int groups = ceil_div(a.G, 16);
  hipLaunchKernelGGL((paged_attn_kernel<BF, HD>), dim3(a.ncols, a.nkv, groups), dim3(64 * PA_WAVES), 0,
                     st, a);
  OMNI_CHECK_LAUNCH();
  // few rows have many states each
  const dim3 rows(a.nkv * a.G, a.n, a.n * a.nkv * a.G < 256 && a.ncols >= 64 ? HD / 32 : 1);
  if (rows.z > 1) hipLaunchKernelGGL((paged_merge_kernel<BF, HD, 32>), rows, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((paged_merge_kernel<BF, HD, HD>), rows, dim3(256), 0, st, a);
  OMNI_CHECK_LAUNCH();
  return OMNI_OK;
}

extern "C" int omni_paged_attention(const void* q, int64_t q_stride, const void* k_cache,
                                    const void* v_cache, int dtype, int pages, int page_size,
                                    const int* tables, int width, int n, const int* schedule,
                                    int columns, void* out, int64_t out_stride, int n_heads,
                                    int n_kv_heads, int head_dim, float scale, float* workspace,
                                    int64_t workspace_floats, void* stream) {
  if (n < 0 || pages <= 0 || page_size <= 0 || width <= 0 || columns <= 0 || n_heads <= 0 ||
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
  if (workspace_floats < (int64_t)(columns + n) * n_heads * (head_dim + 4)) return OMNI_EINVAL;
  const PagedArgs a = {(const unsigned short*)q, q_stride, (const unsigned short*)k_cache,
                       (const unsigned short*)v_cache, pages, shift, n_kv_heads,
                       n_heads / n_kv_heads, n, columns, width, tables, schedule,
                       (unsigned short*)out, out_stride, scale * 1.4426950408889634f, workspace};
  hipStream_t st = (hipStream_t)stream;
  if (dtype) return head_dim == 64 ? pa_launch<true, 64>(a, st) : pa_launch<true, 128>(a, st);
  return head_dim == 64 ? pa_launch<false, 64>(a, st) : pa_launch<false, 128>(a, st);
}
