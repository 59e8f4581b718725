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
// Which token a random number falls on is decided by sums over the whole vocabulary, so all
// weights and sums are 64-bit: the borders between 151936 tokens lie 1e-6 apart and closer, and
// 32-bit sums would move one in a few hundred draws to a neighbour.
#include "common.h"

#define SV_MAX_NODES 64
#define SV_THREADS 1024

template <int DT>   // 0 fp16, 1 bf16, 2 fp32
__device__ __forceinline__ float sv_logit(const void* row, int64_t v) {
  float x;
  if (DT == 2) x = ((const float*)row)[v];
  else x = ld16f<DT == 1>(((const unsigned short*)row)[v]);
  return x == x ? x : -INFINITY;
}

// weight of logit x where m is the row's largest (1 there, infinite or not)
__device__ __forceinline__ double sv_weight(float x, float m, double inv_t) {
  return x == -INFINITY ? 0.0 : x == m ? 1.0 : exp(((double)x - (double)m) * inv_t);
}

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
  int n, T, V;
  int* path;
  int64_t* out_tokens;
  int* emitted;
};

struct SvRow {
  const void* row;
  float m;        // largest logit
  int best;       // its first index
  double z;       // sum of weights
};

template <int DT>
__device__ SvRow sv_stats(const void* row, int V, double inv_t, bool greedy) {
  __shared__ float wm[16];
  __shared__ int wi[16];
  __shared__ double wz[16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  float m = -INFINITY;
  int at = 0x7fffffff;
  for (int v = tid; v < V; v += SV_THREADS) {
    const float x = sv_logit<DT>(row, v);
    if (x > m) {
      m = x;
      at = v;
    }
  }
  for (int o = 32; o; o >>= 1) {
    const float xm = __shfl_xor(m, o);
    const int xi = __shfl_xor(at, o);
    if (xm > m || (xm == m && xi < at)) {
      m = xm;
      at = xi;
    }
  }
  __syncthreads();
  if (lane == 0) {
    wm[wave] = m;
    wi[wave] = at;
  }
  __syncthreads();
  for (int w = 0; w < 16; ++w)
    if (wm[w] > m || (wm[w] == m && wi[w] < at)) {
      m = wm[w];
      at = wi[w];
    }
  SvRow r = {row, m, at, 1.0};
  if (greedy) return r;
  double z = 0.0;
  for (int v = tid; v < V; v += SV_THREADS) z += sv_weight(sv_logit<DT>(row, v), m, inv_t);
  for (int o = 32; o; o >>= 1) z += __shfl_xor(z, o);
  if (lane == 0) wz[wave] = z;
  __syncthreads();
  r.z = 0.0;
  for (int w = 0; w < 16; ++w) r.z += wz[w];
  if (r.z == 0.0) r.z = 1.0;      // no token above -inf: every probability is 0
  return r;
}

// One workgroup a sequence, walking from the root.
template <int DT>
__global__ __launch_bounds__(SV_THREADS) void spec_verify_kernel(SvArgs a) {
  constexpr int SIZE = DT == 2 ? 4 : 2;
  __shared__ double part[SV_THREADS];
  __shared__ int64_t found;
  const int tid = threadIdx.x;
  const int s = blockIdx.x;
  const int used = a.counts ? min(max(a.counts[s], 0), a.T) : a.T;
  const int64_t* tok = a.tokens + (int64_t)s * a.T;
  const int* par = a.parents ? a.parents + (int64_t)s * a.T : nullptr;
  const float* u = a.uniforms ? a.uniforms + (int64_t)s * a.T : nullptr;
  int* path = a.path + (int64_t)s * a.T;
  int64_t* out = a.out_tokens + (int64_t)s * a.T;
  const float temp = a.temperature ? a.temperature[s] : a.temp;
  const bool greedy = !(temp > 0.f);
  const double inv_t = greedy ? 1.0 : 1.0 / (double)temp;
  if (used == 0) {
    for (int i = tid; i < a.T; i += SV_THREADS) {
      path[i] = -1;
      out[i] = -1;
    }
    if (tid == 0) a.emitted[s] = 0;
    return;
  }
  int here = 0, len = 1;
  uint64_t tried = 0;
  SvRow p, q;
  while (true) {
    p = sv_stats<DT>((const char*)a.logits + (s * a.seq_stride + here * a.row_stride) * SIZE, a.V,
                     inv_t, greedy);
    const bool chain_q = a.draft && here + 1 < used && !greedy;
    q.row = nullptr;
    if (chain_q)
      q = sv_stats<DT>((const char*)a.draft + (s * a.dseq_stride + here * a.drow_stride) * SIZE,
                       a.V, inv_t, false);
    tried = 0;
    int taken = -1;
    double left = p.z;
    for (int i = here + 1; i < used && taken < 0 && p.m > -INFINITY; ++i) {
      if ((par ? par[i] : i - 1) != here) continue;
      const int64_t x = tok[i];
      double w = 0.0;
      bool twice = x < 0 || x >= a.V;
      for (int j = here + 1; j < i; ++j) twice |= ((tried >> j) & 1) && tok[j] == x;
      if (!twice) w = greedy ? (x == p.best ? 1.0 : 0.0) : sv_weight(sv_logit<DT>(p.row, x), p.m, inv_t);
      bool ok;
      if (greedy) ok = w > 0.0;
      else if (chain_q)
        ok = !twice && (double)u[i] * (sv_weight(sv_logit<DT>(q.row, x), q.m, inv_t) / q.z) < w / p.z;
      else ok = (double)u[i] * left < w;
      if (ok) taken = i;
      tried |= 1ull << i;
      left -= w;
    }
    if (taken < 0) break;
    if (tid == 0) {
      path[len] = taken;
      out[len - 1] = tok[taken];
    }
    here = taken;
    ++len;
  }
  // the next token
  int64_t next = -1;
  if (greedy || p.m == -INFINITY) {
    next = p.m == -INFINITY ? -1 : p.best;
  } else {
    const int seg = (a.V + SV_THREADS - 1) / SV_THREADS;
    const int lo = min(a.V, tid * seg), hi = min(a.V, lo + seg);
    for (int full = 0; full < 2 && next < 0; ++full) {   // second: an empty residual, p itself
      auto weight = [&](int v) {
        const double w = sv_weight(sv_logit<DT>(p.row, v), p.m, inv_t);
        if (full) return w;
        if (q.row) {
          const double d = w / p.z - sv_weight(sv_logit<DT>(q.row, v), q.m, inv_t) / q.z;
          return d > 0.0 ? d : 0.0;
        }
        for (uint64_t b = tried; b; b &= b - 1)
          if (tok[__ffsll((unsigned long long)b) - 1] == v) return 0.0;
        return w;
      };
      double sum = 0.0;
      for (int v = lo; v < hi; ++v) sum += weight(v);
      __syncthreads();
      part[tid] = sum;
      if (tid == 0) found = 0x7fffffff;
      __syncthreads();
      double before = 0.0, total = 0.0;
      for (int i = 0; i < SV_THREADS; ++i) {
        if (i == tid) before = total;
        total += part[i];
      }
      const double want = (double)u[0] * total;
      int mine = 0x7fffffff, last = -1;
      double run = before;
      if (total > 0.0)
        for (int v = lo; v < hi; ++v) {
          const double w = weight(v);
          if (w > 0.0) last = v;
          run += w;
          if (w > 0.0 && run > want) {
            mine = v;
            break;
          }
        }
      if (mine != 0x7fffffff) atomicMin((unsigned long long*)&found, (unsigned long long)mine);
      __syncthreads();
      if (found != 0x7fffffff) {
        next = found;
      } else if (total > 0.0) {            // rounding, or u >= 1: the last token with weight
        __syncthreads();
        if (tid == 0) found = -1;
        __syncthreads();
        if (last >= 0) atomicMax((long long*)&found, (long long)last);
        __syncthreads();
        next = found;
      }
      __syncthreads();
    }
  }
  if (tid == 0) {
    path[0] = 0;
    out[len - 1] = next;
    a.emitted[s] = len;
  }
  for (int i = len + tid; i < a.T; i += SV_THREADS) {
    path[i] = -1;
    out[i] = -1;
  }
}

extern "C" int omni_spec_verify_work(int n, int n_nodes, int vocab, int drafted) {
  if (n < 0 || n_nodes < 1 || vocab < 1) return OMNI_EINVAL;
  if (n_nodes > SV_MAX_NODES) return OMNI_EUNSUPPORTED;
  return 0;
}

extern "C" int omni_spec_verify(const void* logits, int dtype, int64_t seq_stride, int64_t row_stride,
                                const void* draft, int64_t draft_seq_stride, int64_t draft_row_stride,
                                const int64_t* tokens, const int* parents, const int* counts,
                                const float* uniforms, const float* temperature, float temp, int n,
                                int n_nodes, int vocab, int* path, int64_t* out_tokens,
                                int* emitted, void* workspace, int64_t workspace_doubles,
                                void* stream) {
  if (n < 0 || n_nodes < 1 || vocab < 1 || dtype < 0 || dtype > 2) return OMNI_EINVAL;
  if (n_nodes > SV_MAX_NODES) return OMNI_EUNSUPPORTED;
  if (seq_stride < 0 || row_stride < 0 || draft_seq_stride < 0 || draft_row_stride < 0) return OMNI_EINVAL;
  if (draft && parents) return OMNI_EUNSUPPORTED;
  if (!temperature && !(temp >= 0.f)) return OMNI_EINVAL;
  if (!uniforms && (temperature || temp > 0.f)) return OMNI_EINVAL;
  if (n == 0) return OMNI_OK;
  if (!logits || !tokens || !path || !out_tokens || !emitted) return OMNI_EINVAL;
  const SvArgs a = {logits, seq_stride, row_stride, draft, draft_seq_stride, draft_row_stride, tokens,
                    parents, counts, uniforms, temperature, temp, n, n_nodes, vocab, path, out_tokens,
                    emitted};
  hipStream_t st = (hipStream_t)stream;
  if (dtype == 0) hipLaunchKernelGGL((spec_verify_kernel<0>), dim3(n), dim3(SV_THREADS), 0, st, a);
  else if (dtype == 1) hipLaunchKernelGGL((spec_verify_kernel<1>), dim3(n), dim3(SV_THREADS), 0, st, a);
  else hipLaunchKernelGGL((spec_verify_kernel<2>), dim3(n), dim3(SV_THREADS), 0, st, a);
  OMNI_CHECK_LAUNCH();
  return OMNI_OK;
}
