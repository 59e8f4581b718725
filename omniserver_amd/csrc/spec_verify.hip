// Verification of drafted tokens against the target's probabilities, from given random numbers.
//
// Sequence s has n_nodes drafted nodes, node 0 its last emitted token; logits row (s, i) is the
// target's after node i, and the drafted tokens at i's children are tested against it:
//   p = softmax(logits / temperature)   (temperature <= 0: all mass on the first maximum)
//   trees   child k of a node (index order), token x_k, random number u_k: accepted if
//             u_k (1 - p(x_1) - .. - p(x_{k-1})) < p(x_k)
//           - a token drawn from p, one child at a time; if no child is accepted the next token
//           comes from p without the tried tokens.
//   chains  node i + 1 is node i's only child, drawn from q = softmax(draft logits / temperature):
//           accepted if u q(x) < p(x); at the first rejection the next token comes from
//           max(p - q, 0), after the last node from p.
// Both leave the emitted tokens distributed as if sampled from p one by one.  A next token is the
// first v whose running sum of weights exceeds u_0 times their total.  A NaN logit counts as
// -inf; a row without a token above -inf accepts nothing and gives -1.
//
// Every row is read once, in 32 bits: largest logit and sum of weights per 8192 tokens (the bound
// is the rows' bytes).  A test that these sums leave open - they are good to 2^-17, so one in some
// 10^5 - is decided by a 64-bit sum of its row.  Where a random number falls among 151936 tokens
// is a matter of borders 1e-6 apart and closer, which 32-bit sums would move across one draw in a
// few hundred: the one row per sequence that the next token comes from is summed and searched in
// 64 bits.  Launches: row statistics; the walk, with the drawn row's 64-bit chunk sums; the draw.
//
// max(p - q, 0) is summed without knowing both rows' 64-bit totals first: with weights p, q not yet
// normalised it is max(p - r q, 0), r = the totals' ratio.  From the 32-bit ratio r0 the walk sums
// max(p - r0 q, 0) and the q of its positive terms, and the draw moves the sums by (r0 - r) times
// the latter: exact but for terms that change sign between r0 and r.  The walk also sums the q of
// the terms within 2^-20 r0 q of zero (what r0 is good to): a chunk where |r - r0| times these is
// more than 2^-48 of the residual's total is summed anew by the draw, at r, and so are all where r
// is further off.  151936 tokens have one such chunk in some 4 draws.  Where a draft is next to its
// target the residual is hardly more than those terms and all chunks are: a call of 32 such
// sequences takes 160-190 us, of others like them 43-46.
#include "common.h"

#define SV_MAX_NODES 64
#define SV_WAVES 4                 // waves of a workgroup
#define SV_BLOCK 8192              // tokens of a workgroup in 32 bits: 32 a lane
#define SV_CHUNK 1024              // tokens a wave sums in 64 bits: 16 a lane
#define SV_PARTS 768              // workgroups of the walk in all: more walk again what others walk
// Relative error of a row's 32-bit sum.  A weight 2^t is off by |t| ln 2 of the roundings of its
// exponent (difference, scale and its quotient, product: 1.9e-7), 1.2e-7 by its exponential and some
// 14 additions by 6e-8 each; 2^30 tokens that together weigh against the largest have t = -30:
// 5e-6 at worst.
#define SV_ERR 0x1p-17
#define SV_BAND 0x1p-20            // of r0: what two 32-bit sums' ratio is mostly good to
#define SV_SUMS 5                  // 64-bit sums of a chunk

enum { SV_DONE = 0, SV_TARGET = 1, SV_RESIDUAL = 2 };   // where the next token comes from

struct SvArgs {
  const void* logits;
  int64_t seq_stride, row_stride;
  const void* draft;
  int64_t dseq_stride, drow_stride;
  const int64_t* tokens;
  const int* parents;      // null: a chain
  const int* counts;
  const float* uniforms;
  const float* temperature;
  float temp;
  int n, T, V, chunks, blocks;
  int parts;               // workgroups of the walk for a sequence
  int* path;
  int64_t* out_tokens;
  int* emitted;
  float2* rec;             // [n T target rows, n (T - 1) draft rows][blocks] (largest, sum or index)
  double* sums;            // [SV_SUMS][n][chunks]: target, draft, residual at r0, its draft weights,
                           // draft weights of the terms about zero
  struct SvSeq* seqs;      // [n]
};

struct SvSeq {             // what the walk leaves for the draw
  int mode, last, len;
  float m, mq;             // largest logits of the drawn row and of the draft's
  uint32_t tried[2];       // children tried at the last node
  uint32_t pad;
  double r0;               // the drawn rows' ratio of 32-bit sums, target / draft
};

template <int DT>
__device__ __forceinline__ constexpr int sv_size() { return DT == 2 ? 4 : 2; }

template <int DT>   // 0 fp16, 1 bf16, 2 fp32; NaN as -inf
__device__ __forceinline__ float sv_logit(const void* row, int64_t v) {
  float x;
  if (DT == 2) x = ((const float*)row)[v];
  else x = ld16f<DT == 1>(((const unsigned short*)row)[v]);
  return x == x ? x : -INFINITY;
}

template <int DT>
__device__ __forceinline__ const void* sv_row(const SvArgs& a, int s, int i) {
  return (const char*)a.logits + (s * a.seq_stride + i * a.row_stride) * sv_size<DT>();
}
template <int DT>
__device__ __forceinline__ const void* sv_draft_row(const SvArgs& a, int s, int i) {
  return (const char*)a.draft + (s * a.dseq_stride + i * a.drow_stride) * sv_size<DT>();
}

__device__ __forceinline__ float sv_temp(const SvArgs& a, int s) {
  return a.temperature ? a.temperature[s] : a.temp;
}
__device__ __forceinline__ int sv_used(const SvArgs& a, int s) {
  return a.counts ? min(max(a.counts[s], 0), a.T) : a.T;
}

// 2^t for -2100 <= t <= 0: t = n + f, |f| <= 1/2, n from the low word of t + 1.5 2^52, 2^f by the
// polynomial through its values at the eleven Chebyshev points of [-1/2, 1/2] (relative error 4e-16,
// its roundings included), 2^n by the exponent (0 far below).  Nine points are off by 1.1e-12: a
// random number that near to a border between two tokens would draw the other one.
__device__ __forceinline__ double sv_exp2(double t) {
#pragma clang fp contract(off)          // the same wherever it is inlined
  const double a = t + 0x1.8p52, f = t - (a - 0x1.8p52);
  double r = 0x1.e6063f7217bc6p-28;
  r = fma(r, f, 0x1.b675bca4eeebbp-24);
  r = fma(r, f, 0x1.62bfd47773353p-20);
  r = fma(r, f, 0x1.ffcb54062e698p-17);
  r = fma(r, f, 0x1.430913096fd9fp-13);
  r = fma(r, f, 0x1.5d87fe9d7a584p-10);
  r = fma(r, f, 0x1.3b2ab6fba1ddap-7);
  r = fma(r, f, 0x1.c6b08d703ce49p-5);
  r = fma(r, f, 0x1.ebfbdff82c598p-3);
  r = fma(r, f, 0x1.62e42fefa3a19p-1);
  r = fma(r, f, 1.0);
  return ldexp(r, (int)(uint32_t)__builtin_bit_cast(uint64_t, a));
}

// log2(e) / temperature, and 2000 / that: so far below the largest logit every weight is 0.
struct SvScale {
  double c, span;
  __device__ __forceinline__ explicit SvScale(float temp)
      : c(1.4426950408889634073599 / (double)temp), span(1386.2943611198906 * (double)temp) {}
};

// The weights of a row whose largest logit is m: 1 at m, infinite or not, 0 at -inf and NaN.  Where m
// and the scale are ordinary, whatever lies `span` below m is as good as a finite logit there.
struct SvRow {
  float m, low;
  double c, mc;
  bool plain;
  __device__ __forceinline__ SvRow(float m_, const SvScale& t) : m(m_), c(t.c), mc(m_ * t.c) {
    low = (float)((double)m - t.span);
    plain = fabsf(m) < 1e30f && c > 1e-25 && c < 1e25 && ((double)m - (double)low) * c > 1100.0;
  }
  __device__ __forceinline__ double weight(float x) const {
#pragma clang fp contract(off)
    if (plain) return sv_exp2(fma((double)fmaxf(x, low), c, -mc));
    if (!(x > -INFINITY)) return 0.0;
    if (x == m) return 1.0;
    return m == INFINITY ? 0.0 : sv_exp2(fmax(((double)x - (double)m) * c, -2000.0));
  }
};

// Reductions and prefix sums by data-parallel moves within rows of 16 lanes (a move is a VALU
// operation; through LDS, as wave_sum does it, a step takes some 100 cycles and these kernels are
// chains of such steps).  SHR + k: lane l gets lane l - k of its row, or 0; ROR + k: rotated.
enum { DPP_SHR = 0x110, DPP_ROR = 0x120, DPP_BCAST15 = 0x142, DPP_BCAST31 = 0x143 };

template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ float dpp(float v, float other = 0.f) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(
      __builtin_bit_cast(int, other), __builtin_bit_cast(int, v), CTRL, ROWS, 0xf, false));
}
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ double dpp(double v, double other = 0.0) {
  const int2 x = __builtin_bit_cast(int2, v), o = __builtin_bit_cast(int2, other);
  return __builtin_bit_cast(double,
                            make_int2(__builtin_amdgcn_update_dpp(o.x, x.x, CTRL, ROWS, 0xf, false),
                                      __builtin_amdgcn_update_dpp(o.y, x.y, CTRL, ROWS, 0xf, false)));
}
__device__ __forceinline__ float lane_of(float v, int lane) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}
__device__ __forceinline__ double lane_of(double v, int lane) {
  const int2 x = __builtin_bit_cast(int2, v);
  return __builtin_bit_cast(double, make_int2(__builtin_amdgcn_readlane(x.x, lane),
                                              __builtin_amdgcn_readlane(x.y, lane)));
}

// Inclusive prefix sums over the wave.
template <typename T>
__device__ __forceinline__ T wave_scan(T v) {
  v += dpp<DPP_SHR + 1>(v);
  v += dpp<DPP_SHR + 2>(v);
  v += dpp<DPP_SHR + 4>(v);
  v += dpp<DPP_SHR + 8>(v);
  v += dpp<DPP_BCAST15, 0xa>(v);       // a row's total into the next row
  v += dpp<DPP_BCAST31, 0xc>(v);       // the lower half's into the upper
  return v;
}
template <typename T>
__device__ __forceinline__ T wave_total(T v) {
  return lane_of(wave_scan(v), 63);
}
__device__ __forceinline__ float row_max(float v) {         // over 16 lanes, in all of them
  v = fmaxf(v, dpp<DPP_ROR + 1>(v));
  v = fmaxf(v, dpp<DPP_ROR + 2>(v));
  v = fmaxf(v, dpp<DPP_ROR + 4>(v));
  return fmaxf(v, dpp<DPP_ROR + 8>(v));
}
__device__ __forceinline__ float wave_top(float v) {
  v = row_max(v);
  return fmaxf(fmaxf(lane_of(v, 0), lane_of(v, 16)), fmaxf(lane_of(v, 32), lane_of(v, 48)));
}

// A lane's logits as they are stored, N in a 16-byte piece; element e of piece j is token v0 +
// at(lane, j) + e.
template <int DT>
struct SvPiece {
  static constexpr int N = DT == 2 ? 4 : 8;
  u32x4 w;
  static __device__ __forceinline__ int at(int lane, int j) { return j * 64 * N + lane * N; }
  __device__ __forceinline__ float get(int e) const {      // may be NaN
    if (DT == 2) return __builtin_bit_cast(float, (uint32_t)w[e % N]);
    return ld16f<DT == 1>((unsigned short)(w[e % N / 2] >> (16 * (e & 1))));
  }
  // tokens past the vocabulary: -inf
  __device__ __forceinline__ void load(const void* row, int v0, int V, int lane, int j) {
    const int v1 = v0 + at(lane, j);
    if (v0 + (j + 1) * 64 * N <= V) {    // rows of an odd width are off every alignment
      __builtin_memcpy(&w, (const char*)row + (int64_t)v1 * sv_size<DT>(), 16);
      return;
    }
    constexpr uint32_t NONE = DT == 0 ? 0xfc00fc00u : DT == 1 ? 0xff80ff80u : 0xff800000u;
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      const int v = v1 + d * N / 4;
      uint32_t x = NONE;
      if (DT == 2) {
        if (v < V) x = ((const uint32_t*)row)[v];
      } else {
        const unsigned short* r = (const unsigned short*)row;
        if (v < V) x = (x & 0xffff0000u) | r[v];
        if (v + 1 < V) x = (x & 0xffffu) | (uint32_t)r[v + 1] << 16;
      }
      w[d] = x;
    }
  }
};

// ---------------------------------------------------------------------------
// Row statistics: one workgroup 8192 tokens of a row, rec = (largest logit, sum of weights
// relative to it), for greedy rows (largest logit, its first index).  32 x 16 nodes, half of them
// in use, 80 MB: 21 us = 3.8 TB/s (a large copy's rate is 4.7-5.2).  The whole call there 40 us; with
// 4096 or 16384 tokens a workgroup 5 and 2 more, with one round of workgroups that go over all rows,
// loads one piece ahead, 5-12 more.
// ---------------------------------------------------------------------------
template <int DT>
__global__ __launch_bounds__(64 * SV_WAVES) void sv_stats_kernel(SvArgs a) {
  __shared__ float wm[SV_WAVES], wz[SV_WAVES];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = blockIdx.x / a.blocks, block = blockIdx.x - r * a.blocks;
  const int target_rows = a.n * a.T;
  const bool is_draft = r >= target_rows;
  const int T = is_draft ? a.T - 1 : a.T, rr = is_draft ? r - target_rows : r;
  const int s = rr / T, i = rr - s * T;
  const float temp = sv_temp(a, s);
  const bool greedy = !(temp > 0.f);
  const int used = sv_used(a, s);
  if (is_draft ? (greedy || i + 1 >= used) : i >= used) return;
  const void* row = is_draft ? sv_draft_row<DT>(a, s, i) : sv_row<DT>(a, s, i);
  constexpr int PER = SV_BLOCK / SV_WAVES;
  const int v0 = block * SV_BLOCK + wave * PER;
  typedef SvPiece<DT> P;
  P x[32 / P::N];
#pragma unroll
  for (int j = 0; j < 32 / P::N; ++j) x[j].load(row, v0, a.V, lane, j);
  float m = -INFINITY;
#pragma unroll
  for (int e = 0; e < 32; ++e) m = fmaxf(m, x[e / P::N].get(e));       // leaves a NaN out
  m = wave_top(m);
  // (x - m) c in two steps: c may be as large as fp32 goes, and an infinite m stays in order
  const float c = greedy ? 0.f : fminf(1.4426950408889634f / temp, 1e38f);
  float sum;
  if (greedy) {
    int at = 0x7fffffff;
#pragma unroll
    for (int e = 31; e >= 0; --e)
      if (x[e / P::N].get(e) == m) at = v0 + P::at(lane, e / P::N) + e % P::N;
    for (int o = 32; o; o >>= 1) at = min(at, __shfl_xor(at, o));
    sum = __builtin_bit_cast(float, at);
  } else {
    float z[4] = {0.f, 0.f, 0.f, 0.f};
    if (fabsf(m) < INFINITY) {
#pragma unroll
      for (int e = 0; e < 32; ++e) {
        const float w = __builtin_amdgcn_exp2f((x[e / P::N].get(e) - m) * c);
        z[e & 3] += w == w ? w : 0.f;
      }
    } else if (m == INFINITY) {
#pragma unroll
      for (int e = 0; e < 32; ++e) z[e & 3] += x[e / P::N].get(e) == m ? 1.f : 0.f;
    }
    sum = wave_total((z[0] + z[1]) + (z[2] + z[3]));
  }
  if (lane == 0) {
    wm[wave] = m;
    wz[wave] = sum;
  }
  __syncthreads();
  if (threadIdx.x) return;
  float M = wm[0];
  for (int w = 1; w < SV_WAVES; ++w) M = fmaxf(M, wm[w]);
  if (greedy) {
    int at = 0x7fffffff;
    for (int w = 0; w < SV_WAVES; ++w)
      if (wm[w] == M) at = min(at, __builtin_bit_cast(int, wz[w]));
    sum = __builtin_bit_cast(float, at);
  } else {
    sum = 0.f;
    for (int w = 0; w < SV_WAVES; ++w)
      if (wz[w] > 0.f) sum += wz[w] * (wm[w] == M ? 1.f : __builtin_amdgcn_exp2f((wm[w] - M) * c));
  }
  a.rec[(int64_t)r * a.blocks + block] = make_float2(M, sum);
}

// A row's blocks together, by half a wave: largest logit and 64-bit sum of their 32-bit sums
// (greedy: first index).
__device__ __forceinline__ void sv_combine(const float2* rec, int blocks, int lane, const SvScale& t,
                                           bool greedy, float& m, double& z, int& best) {
  const int l = lane & 31;
  const float2 own = l < blocks ? rec[l] : make_float2(-INFINITY, 0.f);
  m = own.x;
  for (int k = l + 32; k < blocks; k += 32) m = fmaxf(m, rec[k].x);
  m = row_max(m);
  m = fmaxf(m, __shfl_xor(m, 16));
  const SvRow row(m, t);
  z = 0.0;
  best = 0x7fffffff;
  for (int k = l; k < blocks; k += 32) {
    const float2 v = k < 32 ? own : rec[k];
    if (greedy) {
      if (v.x == m) best = min(best, __builtin_bit_cast(int, v.y));
    } else if (v.y > 0.f) {
      z += (double)v.y * row.weight(v.x);
    }
  }
  if (greedy) {
#pragma unroll
    for (int o = 16; o; o >>= 1) best = min(best, __shfl_xor(best, o));
    return;
  }
  z += dpp<DPP_ROR + 1>(z);
  z += dpp<DPP_ROR + 2>(z);
  z += dpp<DPP_ROR + 4>(z);
  z += dpp<DPP_ROR + 8>(z);
  z += __shfl_xor(z, 16);
}

// 64-bit sum of a chunk's weights, the tried tokens left out; by one wave.
template <int DT>
__device__ __forceinline__ double sv_chunk_sum(const void* row, int chunk, int V, int lane,
                                               const SvRow& w, const int64_t* tok, uint64_t tried) {
  typedef SvPiece<DT> P;
  const int v0 = chunk * SV_CHUNK;
  double z[2] = {0.0, 0.0};
  P next;
  next.load(row, v0, V, lane, 0);
#pragma unroll 1
  for (int j = 0; j < 16 / P::N; ++j) {
    const P x = next;
    if (j + 1 < 16 / P::N) next.load(row, v0, V, lane, j + 1);
    uint32_t gone = 0;                                  // elements that hold a tried token
    for (uint64_t b = tried; b; b &= b - 1) {
      const int64_t t = tok[__ffsll((unsigned long long)b) - 1] - (v0 + P::at(lane, j));
      if (t >= 0 && t < P::N) gone |= 1u << t;
    }
#pragma unroll
    for (int e = 0; e < P::N; ++e) z[e & 1] += w.weight(gone >> e & 1 ? -INFINITY : x.get(e));
  }
  return wave_total(z[0] + z[1]);
}

// A chunk's 64-bit sums of p, of q, of max(p - r0 q, 0), of the q of its positive terms and of the
// q of those about zero.
template <int DT>
__device__ __forceinline__ void sv_residual_sums(const void* row, const void* drow, int chunk, int V,
                                                 int lane, const SvRow& wp, const SvRow& wq, double r0,
                                                 double (&z)[SV_SUMS]) {
#pragma clang fp contract(off)          // equal rows leave exactly nothing
  typedef SvPiece<DT> P;
  const int v0 = chunk * SV_CHUNK;
  for (int k = 0; k < SV_SUMS; ++k) z[k] = 0.0;
  P nx, ny;
  nx.load(row, v0, V, lane, 0);
  ny.load(drow, v0, V, lane, 0);
#pragma unroll 1
  for (int j = 0; j < 16 / P::N; ++j) {
    const P x = nx, y = ny;
    if (j + 1 < 16 / P::N) {
      nx.load(row, v0, V, lane, j + 1);
      ny.load(drow, v0, V, lane, j + 1);
    }
#pragma unroll
    for (int e = 0; e < P::N; ++e) {
      const double p = wp.weight(x.get(e)), q = wq.weight(y.get(e)), rq = r0 * q, d = p - rq;
      z[0] += p;
      z[1] += q;
      z[2] += d > 0.0 ? d : 0.0;
      z[3] += d > 0.0 ? q : 0.0;
      z[4] += fabs(d) <= SV_BAND * rq ? q : 0.0;
    }
  }
#pragma unroll
  for (int k = 0; k < SV_SUMS; ++k) z[k] = wave_total(z[k]);
}

// ---------------------------------------------------------------------------
// The walk, by every workgroup of a sequence (part 0 writes it down), then this part's share of
// the drawn row's chunk sums.  A lane a node: all nodes' weights at their parents' rows at once; then
// one wave goes from the root, children in index order.
// ---------------------------------------------------------------------------
template <int DT>
__global__ __launch_bounds__(64 * SV_WAVES) void sv_walk_kernel(SvArgs a) {
  __shared__ float ms[2][SV_MAX_NODES];
  __shared__ double zs[2][SV_MAX_NODES];
  __shared__ int best[SV_MAX_NODES];
  __shared__ int64_t tok[SV_MAX_NODES];
  __shared__ double part[SV_WAVES];
  __shared__ uint64_t tried_s;
  __shared__ int open_s, last_s, len_s;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int s = blockIdx.x / a.parts, mine = blockIdx.x - s * a.parts;
  const int T = a.T, used = sv_used(a, s);
  const float temp = sv_temp(a, s);
  const bool greedy = !(temp > 0.f), chain_q = a.draft && !greedy;
  int* path = a.path + (int64_t)s * T;
  int64_t* out = a.out_tokens + (int64_t)s * T;
  if (used == 0) {
    if (mine) return;
    if (tid < T) {
      path[tid] = -1;
      out[tid] = -1;
    }
    if (tid == 0) {
      a.emitted[s] = 0;
      a.seqs[s].mode = SV_DONE;
    }
    return;
  }
  // a lane a node: its parent, token and random number, its logits at the parent's rows
  int up = -1, id = -1;
  int64_t x = 0;
  double u = 0.0;
  float lp = -INFINITY, lq = -INFINITY;
  if (lane < T) {
    up = lane == 0 ? -1 : a.parents ? a.parents[(int64_t)s * T + lane] : lane - 1;
    x = a.tokens[(int64_t)s * T + lane];
    if (a.uniforms) u = (double)a.uniforms[(int64_t)s * T + lane];
    if (up < 0 || up >= lane || lane >= used) up = -1;
    if (x >= 0 && x < a.V) id = (int)x;
    if (up >= 0 && id >= 0) {
      lp = sv_logit<DT>(sv_row<DT>(a, s, up), id);
      if (chain_q) lq = sv_logit<DT>(sv_draft_row<DT>(a, s, up), id);
    }
  }
  const SvScale scale(greedy ? 1.f : temp);
  const int nrows = chain_q ? 2 * used - 1 : used;        // the target's rows, then the draft's
  for (int r0 = 2 * wave; r0 < nrows; r0 += 2 * SV_WAVES) {
    const int r = min(r0 + (lane >> 5), nrows - 1), d = r >= used, i = d ? r - used : r;
    const int64_t at = d ? (int64_t)a.n * T + (int64_t)s * (T - 1) + i : (int64_t)s * T + i;
    float m;
    double z;
    int b;
    sv_combine(a.rec + at * a.blocks, a.blocks, lane, scale, greedy, m, z, b);
    if ((lane & 31) == 0) {
      ms[d][i] = m;
      zs[d][i] = z;
      if (!d) best[i] = b;
    }
  }
  if (wave == 0) tok[lane] = x;
  __syncthreads();

  uint64_t exact = 0;                                     // rows whose sums are 64-bit by now
  while (true) {
    if (wave == 0) {
      double w = 0.0;
      if (up >= 0 && id >= 0)
        w = greedy ? (ms[0][up] > -INFINITY && id == best[up] ? 1.0 : 0.0)
                   : SvRow(ms[0][up], scale).weight(lp);
      int here = 0, len = 1, doubt = -1;
      uint64_t tried = 0;
      if (greedy || chain_q) {
        bool stands = w > 0.0, open = false;
        if (chain_q && stands && zs[1][up] > 0.0) {       // else the draft's row is empty: q = 0
          // u q / Zq < w / Z, both sides times Z Zq
          const double a0 = u * SvRow(ms[1][up], scale).weight(lq) * zs[0][up], a1 = w * zs[1][up];
          stands = a0 < a1;
          open = fabs(a0 - a1) <= 2.0 * SV_ERR * a1 && !(exact >> up & 1);
        }
        const uint64_t ok = __ballot(stands), unsure = __ballot(open);
        while (true) {
          tried = __ballot(up == here);
          const uint64_t next = tried & (ok | unsure);
          if (!next) break;
          const int i = __ffsll((unsigned long long)next) - 1;
          if (unsure >> i & 1) {
            doubt = here;
            break;
          }
          here = i;
          if (mine == 0 && lane == 0) {
            path[len] = here;
            out[len - 1] = tok[here];
          }
          ++len;
        }
      } else {
        for (int taken = 0; taken >= 0;) {
          taken = -1;
          tried = 0;
          const double z = zs[0][here];
          const bool sure = exact >> here & 1;
          double left = z;
          for (uint64_t kids = __ballot(up == here); kids; kids &= kids - 1) {
            const int i = __ffsll((unsigned long long)kids) - 1;
            const double ui = lane_of(u, i);
            // a token that a sibling has tried has no mass left
            const bool twice = __ballot(id == __builtin_amdgcn_readlane(id, i)) & tried;
            const double wi = twice ? 0.0 : lane_of(w, i), by = ui * left - wi;
            tried |= 1ull << i;
            if (wi > 0.0) {
              if (!sure && fabs(by) <= ui * z * SV_ERR) {
                doubt = here;
                break;
              }
              if (by < 0.0) {
                taken = i;
                break;
              }
            }
            left -= wi;
          }
          if (doubt >= 0) break;
          if (taken >= 0) {
            here = taken;
            if (mine == 0 && lane == 0) {
              path[len] = here;
              out[len - 1] = tok[here];
            }
            ++len;
          }
        }
      }
      if (lane == 0) {
        open_s = doubt;
        last_s = here;
        len_s = len;
        tried_s = tried;
      }
    }
    __syncthreads();
    const int i = open_s;
    if (i < 0) break;
    // the open row's sums in 64 bits, by the whole workgroup
    for (int d = 0; d < (chain_q ? 2 : 1); ++d) {
      const void* row = d ? sv_draft_row<DT>(a, s, i) : sv_row<DT>(a, s, i);
      const SvRow w(ms[d][i], scale);
      double z = 0.0;
      for (int k = wave; k < a.chunks; k += SV_WAVES)
        z += sv_chunk_sum<DT>(row, k, a.V, lane, w, tok, 0);
      if (lane == 0) part[wave] = z;
      __syncthreads();
      if (tid == 0) {
        double t = 0.0;
        for (int k = 0; k < SV_WAVES; ++k) t += part[k];
        zs[d][i] = t;
      }
      __syncthreads();
    }
    exact |= 1ull << i;
  }
  const int last = last_s, len = len_s;
  const uint64_t tried = tried_s;
  const float m = ms[0][last];
  const bool residual = chain_q && tried != 0;
  // a draft row without a token: q is nowhere
  const double r0 = residual && zs[1][last] > 0.0 ? zs[0][last] / zs[1][last] : 0.0;
  const int mode = greedy || m == -INFINITY ? SV_DONE : residual ? SV_RESIDUAL : SV_TARGET;
  if (mine == 0) {
    if (tid == 0) {
      path[0] = 0;
      a.emitted[s] = len;
      if (mode == SV_DONE) out[len - 1] = m == -INFINITY ? -1 : best[last];
      SvSeq* q = a.seqs + s;
      q->mode = mode;
      q->last = last;
      q->len = len;
      q->m = m;
      q->mq = residual ? ms[1][last] : 0.f;
      q->r0 = r0;
      q->tried[0] = (uint32_t)tried;
      q->tried[1] = (uint32_t)(tried >> 32);
    }
    if (tid >= len && tid < T) {
      path[tid] = -1;
      out[tid] = -1;
    }
  }
  if (mode == SV_DONE) return;
  const SvRow wp(m, scale), wq(residual ? ms[1][last] : 0.f, scale);
  double* sums = a.sums + (int64_t)s * a.chunks;
  const int64_t next = (int64_t)a.n * a.chunks;
  for (int k = mine * SV_WAVES + wave; k < a.chunks; k += a.parts * SV_WAVES) {
    if (residual) {
      double z[SV_SUMS];
      sv_residual_sums<DT>(sv_row<DT>(a, s, last), sv_draft_row<DT>(a, s, last), k, a.V, lane, wp, wq,
                           r0, z);
      if (lane == 0)
        for (int d = 0; d < SV_SUMS; ++d) sums[d * next + k] = z[d];
    } else {
      const double z = sv_chunk_sum<DT>(sv_row<DT>(a, s, last), k, a.V, lane, wp, tok, tried);
      if (lane == 0) sums[k] = z;
    }
  }
}

// ---------------------------------------------------------------------------
// The draw, one workgroup a sequence: the chunk that u_0 times the total falls into, then the token
// within it, four a thread.  Where nothing is left of p, from p itself (the second turn).
// ---------------------------------------------------------------------------
template <int DT>
__global__ __launch_bounds__(256) void sv_draw_kernel(SvArgs a) {
  static_assert(SV_CHUNK == 4 * 256, "four tokens a thread");
  __shared__ double wsum[4];
  __shared__ double base_s, want_s;
  __shared__ int chunk_s, pick[4], tail[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int s = blockIdx.x;
  const SvSeq q = a.seqs[s];
  if (q.mode == SV_DONE) return;
  const SvScale scale(sv_temp(a, s));
  const double u0 = (double)a.uniforms[(int64_t)s * a.T];
  const int64_t* tok = a.tokens + (int64_t)s * a.T;
  const void* row = sv_row<DT>(a, s, q.last);
  const SvRow wp(q.m, scale), wq(q.mq, scale);
  double* sums = a.sums + (int64_t)s * a.chunks;
  const int64_t next = (int64_t)a.n * a.chunks;
  for (int turn = 0; turn < 2; ++turn) {
    const bool residual = turn == 0 && q.mode == SV_RESIDUAL;
    const uint64_t tried = turn || residual ? 0 : (uint64_t)q.tried[1] << 32 | q.tried[0];
    const void* drow = residual ? sv_draft_row<DT>(a, s, q.last) : nullptr;
    if (turn) {
      for (int k = wave; k < a.chunks; k += 4) {
        const double z = sv_chunk_sum<DT>(row, k, a.V, lane, wp, tok, 0);
        if (lane == 0) sums[k] = z;
      }
      __syncthreads();                                  // both turns' sums are this workgroup's
    }
    const double r0 = q.r0;
    double ratio = 0.0;
    if (residual) {
      double z[SV_SUMS] = {};
      for (int k = lane; k < a.chunks; k += 64)
#pragma unroll
        for (int d = 0; d < SV_SUMS; ++d) z[d] += sums[d * next + k];
#pragma unroll
      for (int d = 0; d < SV_SUMS; ++d) z[d] = wave_total(z[d]);
      ratio = z[1] > 0.0 ? z[0] / z[1] : 0.0;
      const double off = fabs(r0 - ratio), least = 0x1p-48 * (z[2] + (r0 - ratio) * z[3]);
      const bool all = off > SV_BAND * r0;
      if (all || off * z[4] > least) {                  // the same in every wave
        __syncthreads();                                // all have read the sums
        int turn_of = 0;
        for (int k0 = 0; k0 < a.chunks; k0 += 64) {
          const int k = k0 + lane;
          uint64_t open = __ballot(k < a.chunks && (all || off * sums[4 * next + k] > least));
          for (; open; open &= open - 1, ++turn_of) {
            if ((turn_of & 3) != wave) continue;
            const int c = k0 + __ffsll((unsigned long long)open) - 1;
            sv_residual_sums<DT>(row, drow, c, a.V, lane, wp, wq, ratio, z);
            if (lane == 0) {
              sums[2 * next + c] = z[2];
              sums[3 * next + c] = 0.0;                 // at the 64-bit ratio already
            }
          }
        }
        __syncthreads();
      }
    }
    auto chunk_sum = [&](int k) {
#pragma clang fp contract(off)
      if (k >= a.chunks) return 0.0;
      if (!residual) return sums[k];
      return fmax(sums[2 * next + k] + (r0 - ratio) * sums[3 * next + k], 0.0);
    };
    if (wave == 0) {
      // 256 chunks at a time: their sums' loads together
      double own[4], total = 0.0, base = 0.0, at = 0.0;
      int full = -1;
      for (int k0 = 0; k0 < a.chunks; k0 += 256) {
#pragma unroll
        for (int j = 0; j < 4; ++j) own[j] = chunk_sum(k0 + 64 * j + lane);
#pragma unroll
        for (int j = 0; j < 4; ++j) total += wave_total(own[j]);
      }
      const double want = u0 * total;
      bool found = false;
      for (int k0 = 0; k0 < a.chunks && !found; k0 += 256) {
        if (a.chunks > 256) {
#pragma unroll
          for (int j = 0; j < 4; ++j) own[j] = chunk_sum(k0 + 64 * j + lane);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const double v = wave_scan(own[j]) + base;
          const uint64_t hit = __ballot(own[j] > 0.0 && v > want), some = __ballot(own[j] > 0.0);
          const int l = hit ? __ffsll((unsigned long long)hit) - 1
                        : some ? 63 - __clzll((long long)some) : -1;
          if (!found && l >= 0) {                       // so far the last chunk with weight
            full = k0 + 64 * j + l;
            at = l ? lane_of(v, l - 1) : base;
          }
          found |= hit != 0;
          base = lane_of(v, 63);
        }
      }
      if (lane == 0) {
        chunk_s = full;
        base_s = at;
        want_s = want;
      }
    }
    __syncthreads();
    int mine = 0x7fffffff, heavy = -1;
    if (chunk_s >= 0) {
      const int v0 = chunk_s * SV_CHUNK + tid * 4;
      float x[4], y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] = v0 + e < a.V ? sv_logit<DT>(row, v0 + e) : -INFINITY;
        y[e] = drow && v0 + e < a.V ? sv_logit<DT>(drow, v0 + e) : -INFINITY;
      }
      for (uint64_t b = tried; b; b &= b - 1) {
        const int64_t t = tok[__ffsll((unsigned long long)b) - 1] - v0;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (t == e) x[e] = -INFINITY;
      }
      double w[4], sum = 0.0;
      {
#pragma clang fp contract(off)          // equal rows leave exactly nothing
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          w[e] = wp.weight(x[e]);
          if (residual) w[e] = fmax(w[e] - ratio * wq.weight(y[e]), 0.0);
          sum += w[e];
        }
      }
      double run = wave_scan(sum);
      if (lane == 63) wsum[wave] = run;
      __syncthreads();
      run -= sum;
      for (int k = 0; k < wave; ++k) run += wsum[k];
      run += base_s;
      const double want = want_s;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        run += w[e];
        if (w[e] > 0.0) {
          heavy = v0 + e;
          if (mine == 0x7fffffff && run > want) mine = v0 + e;
        }
      }
      for (int o = 32; o; o >>= 1) {
        mine = min(mine, __shfl_xor(mine, o));
        heavy = max(heavy, __shfl_xor(heavy, o));
      }
      if (lane == 0) {
        pick[wave] = mine;
        tail[wave] = heavy;
      }
      __syncthreads();
      for (int k = 0; k < 4; ++k) {
        mine = min(mine, pick[k]);
        heavy = max(heavy, tail[k]);
      }
    }
    // rounding, or u_0 >= 1: the chunk's last token with weight
    const int token = mine != 0x7fffffff ? mine : heavy;
    if (token >= 0) {
      if (tid == 0) a.out_tokens[(int64_t)s * a.T + q.len - 1] = token;
      return;
    }
    __syncthreads();
  }
}

static_assert(sizeof(SvSeq) == 40, "five doubles");

static int64_t sv_rows(int64_t n, int64_t T, bool drafted) {
  return n * T + (drafted ? n * (T - 1) : 0);
}

// Doubles of workspace, -1 where they do not count in 32 bits or the statistics' threads do not.
static int64_t sv_work(int64_t n, int64_t T, int64_t V, bool drafted) {
  const int64_t chunks = (V + SV_CHUNK - 1) / SV_CHUNK;
  const int64_t records = sv_rows(n, T, drafted) * ((V + SV_BLOCK - 1) / SV_BLOCK);
  const int64_t work = records + SV_SUMS * n * chunks + 5 * n;  // records, sums, sequences
  return work > 0x7fffffff || records * 64 * SV_WAVES > 0xffffffff ? -1 : work;
}

extern "C" int omni_spec_verify_work(int n, int n_nodes, int vocab, int drafted) {
  if (n < 0 || n_nodes < 1 || vocab < 1) return OMNI_EINVAL;
  if (n_nodes > SV_MAX_NODES || vocab > 1 << 30) return OMNI_EUNSUPPORTED;
  const int64_t work = sv_work(n, n_nodes, vocab, drafted);
  return work < 0 ? OMNI_EUNSUPPORTED : (int)work;
}

// Every workgroup of a sequence walks its tree while the first one writes the outcome.
static bool sv_apart(const void* out, int64_t out_bytes, const void* in, int64_t in_bytes) {
  const uintptr_t o = (uintptr_t)out, i = (uintptr_t)in;
  return !in || o + out_bytes <= i || i + in_bytes <= o;
}

template <int DT>
static void sv_launch(const SvArgs& a, hipStream_t st) {
  const int rows = (int)sv_rows(a.n, a.T, a.draft);
  hipLaunchKernelGGL((sv_stats_kernel<DT>), dim3(rows * a.blocks), dim3(64 * SV_WAVES), 0, st, a);
  hipLaunchKernelGGL((sv_walk_kernel<DT>), dim3(a.n * a.parts), dim3(64 * SV_WAVES), 0, st, a);
  if (a.uniforms)                                       // else every row is greedy
    hipLaunchKernelGGL((sv_draw_kernel<DT>), dim3(a.n), dim3(256), 0, st, a);
}

extern "C" int omni_spec_verify(const void* logits, int dtype, int64_t seq_stride, int64_t row_stride,
                                const void* draft, int64_t draft_seq_stride, int64_t draft_row_stride,
                                const int64_t* tokens, const int* parents, const int* counts,
                                const float* uniforms, const float* temperature, float temp, int n,
                                int n_nodes, int vocab, int* path, int64_t* out_tokens,
                                int* emitted, void* workspace, int64_t workspace_doubles,
                                void* stream) {
  if (n < 0 || n_nodes < 1 || vocab < 1 || dtype < 0 || dtype > 2) return OMNI_EINVAL;
  if (n_nodes > SV_MAX_NODES || vocab > 1 << 30) return OMNI_EUNSUPPORTED;
  if (seq_stride < 0 || row_stride < 0 || draft_seq_stride < 0 || draft_row_stride < 0) return OMNI_EINVAL;
  if (draft && parents) return OMNI_EUNSUPPORTED;
  if (!temperature && !(temp >= 0.f)) return OMNI_EINVAL;
  if (!uniforms && (temperature || temp > 0.f)) return OMNI_EINVAL;
  if (n == 0) return OMNI_OK;
  if (!logits || !tokens || !path || !out_tokens || !emitted) return OMNI_EINVAL;
  if (n_nodes == 1) draft = nullptr;
  const int64_t work = sv_work(n, n_nodes, vocab, draft != nullptr);
  if (work < 0) return OMNI_EUNSUPPORTED;
  if (!workspace || ((uintptr_t)workspace & 7) || workspace_doubles < work) return OMNI_EINVAL;
  const int64_t nodes = (int64_t)n * n_nodes;
  const void* outs[3] = {path, out_tokens, emitted};
  const int64_t out_bytes[3] = {4 * nodes, 8 * nodes, 4 * (int64_t)n};
  for (int k = 0; k < 3; ++k)
    if (!sv_apart(outs[k], out_bytes[k], tokens, 8 * nodes) ||
        !sv_apart(outs[k], out_bytes[k], parents, 4 * nodes) ||
        !sv_apart(outs[k], out_bytes[k], counts, 4 * (int64_t)n) ||
        !sv_apart(outs[k], out_bytes[k], uniforms, 4 * nodes) ||
        !sv_apart(outs[k], out_bytes[k], temperature, 4 * (int64_t)n))
      return OMNI_EINVAL;
  SvArgs a;
  a.logits = logits;
  a.seq_stride = seq_stride;
  a.row_stride = row_stride;
  a.draft = draft;
  a.dseq_stride = draft_seq_stride;
  a.drow_stride = draft_row_stride;
  a.tokens = tokens;
  a.parents = parents;
  a.counts = counts;
  a.uniforms = uniforms;
  a.temperature = temperature;
  a.temp = temp;
  a.n = n;
  a.T = n_nodes;
  a.V = vocab;
  a.chunks = ceil_div(vocab, SV_CHUNK);
  a.blocks = ceil_div(vocab, SV_BLOCK);
  a.parts = max(1, min(ceil_div(a.chunks, SV_WAVES), SV_PARTS / max(n, 1)));
  a.path = path;
  a.out_tokens = out_tokens;
  a.emitted = emitted;
  a.rec = (float2*)workspace;
  a.sums = (double*)workspace + sv_rows(n, n_nodes, draft) * a.blocks;
  a.seqs = (SvSeq*)(a.sums + SV_SUMS * (int64_t)n * a.chunks);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == 0) sv_launch<0>(a, st);
  else if (dtype == 1) sv_launch<1>(a, st);
  else sv_launch<2>(a, st);
  OMNI_CHECK_LAUNCH();
  return OMNI_OK;
}
