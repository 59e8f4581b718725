// Attention for trees of drafted tokens over the KV pool, and the tree's plan.
//
// Sequence s has a valid prefix of starts[s] tokens in its pool row; node i of its tree (n_nodes
// <= 64 of them, parents before children) has its K/V at position starts[s] + i and attends to
// the prefix, itself and its ancestors.  The ancestors of a node are one 64-bit word.
#include "common.h"

#define TREE_HD 128
#define TREE_MAX 64

// ---------------------------------------------------------------------------
// The plan of a step, once for all layers: per node its ancestors (itself included; bit j =
// node j), its pool row and position (row -1: not in use, or past the pool), its rotary
// position starts + depth + rope_delta on all three axes; per sequence the prefix length, a
// copy, so that the plan stays what it was when the lengths move on.  A node whose parent does
// not precede it is a root of its own.  One wave a sequence: lane i walks up from node i.
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(64) void tree_plan_kernel(
    const int* __restrict__ parents, const int* __restrict__ counts,
    const int64_t* __restrict__ slots, const int64_t* __restrict__ lengths,
    const int64_t* __restrict__ rope_delta, int n, int T, int pool_rows, int max_len,
    int64_t* __restrict__ starts, uint64_t* __restrict__ ancestors,
    int64_t* __restrict__ positions, int64_t* __restrict__ token_slot,
    int64_t* __restrict__ token_pos) {
  __shared__ int up[TREE_MAX];
  const int s = blockIdx.x, i = threadIdx.x;
  const int64_t slot = slots ? slots[s] : s;
  const bool row_ok = slot >= 0 && slot < pool_rows;
  int64_t L = row_ok ? lengths[slot] : 0;
  L = L < 0 ? 0 : L > max_len ? max_len : L;
  const int64_t delta = row_ok && rope_delta ? rope_delta[slot] : 0;
  const int used = counts ? min(max(counts[s], 0), T) : T;
  if (i < T) up[i] = parents[(int64_t)s * T + i];
  __syncthreads();
  if (i == 0) starts[s] = L;
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

// K/V rows of packed tokens to the pool at (slots, positions); rows outside it are skipped.
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
// One wave a (node, query head): 64 keys a step, one a lane for the scores, then two dims a lane
// for the output, with the running maximum and sum of a softmax.
// ---------------------------------------------------------------------------
struct TreeArgs {
  const half_t* q;
  int q_stride;
  const half_t* k_cache;
  const half_t* v_cache;
  int pool_rows, max_len, nkv, G, T;
  const int64_t* slots;        // [n] or null
  const int64_t* starts;       // [n]
  const uint64_t* ancestors;   // [n][T]
  half_t* out;
  int out_stride;
  float scale_log2;
};

__global__ __launch_bounds__(64) void tree_attn_kernel(TreeArgs a) {
  const int lane = threadIdx.x;
  const int t = blockIdx.x, head = blockIdx.y;
  const int s = t / a.T;
  const int64_t slot = a.slots ? a.slots[s] : s;
  const uint64_t m = a.ancestors[t];
  if (slot < 0 || slot >= a.pool_rows || !m) return;
  const int64_t L = a.starts[s];
  const int64_t end = min(L + a.T, (int64_t)a.max_len);
  const int64_t tstride = (int64_t)a.nkv * TREE_HD;
  const int64_t base = slot * a.max_len * tstride + (head / a.G) * TREE_HD;
  const half_t* qp = a.q + (int64_t)t * a.q_stride + head * TREE_HD;
  float mr = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
  for (int64_t tb = 0; tb < end; tb += 64) {
    const int64_t key = tb + lane;
    const bool seen = key < end && (key < L || ((m >> (key - L)) & 1));
    float sc = -INFINITY;
    if (seen) {
      const half_t* kp = a.k_cache + base + key * tstride;
      sc = 0.f;
      for (int c = 0; c < 16; ++c) {
        const half8_t kv = *(const half8_t*)(kp + 8 * c), qv = *(const half8_t*)(qp + 8 * c);
#pragma unroll
        for (int e = 0; e < 8; ++e) sc = fmaf((float)kv[e], (float)qv[e], sc);
      }
      sc *= a.scale_log2;
    }
    const float mn = fmaxf(mr, wave_max(sc));
    if (mn == -INFINITY) continue;
    const float alpha = exp2f(mr - mn), p = seen ? exp2f(sc - mn) : 0.f;
    mr = mn;
    l = l * alpha + wave_sum(p);
    o0 *= alpha;
    o1 *= alpha;
    const uint64_t all = __ballot(seen);
    for (int j = 0; j < 64; ++j) {
      if (!((all >> j) & 1)) continue;
      const float pj = __shfl(p, j);
      const half2_t vv = *(const half2_t*)(a.v_cache + base + (tb + j) * tstride + 2 * lane);
      o0 = fmaf(pj, (float)vv[0], o0);
      o1 = fmaf(pj, (float)vv[1], o1);
    }
  }
  const half2_t r = {(half_t)(l == 0.f ? 0.f : o0 / l), (half_t)(l == 0.f ? 0.f : o1 / l)};
  *(half2_t*)(a.out + (int64_t)t * a.out_stride + head * TREE_HD + 2 * lane) = r;
}

extern "C" int omni_tree_plan(const int* parents, const int* counts, const int64_t* slots,
                              const int64_t* lengths, const int64_t* rope_delta, int n, int n_nodes,
                              int pool_rows, int max_len, int64_t* starts, void* ancestors,
                              int64_t* positions, int64_t* token_slot, int64_t* token_pos,
                              void* stream) {
  if (n < 0 || n_nodes < 1 || pool_rows <= 0 || max_len <= 0) return OMNI_EINVAL;
  if (n_nodes > TREE_MAX) return OMNI_EUNSUPPORTED;
  if (!slots && n > pool_rows) return OMNI_EINVAL;
  if (n == 0) return OMNI_OK;
  if (!parents || !lengths || !starts || !ancestors || !positions || !token_slot || !token_pos)
    return OMNI_EINVAL;
  hipLaunchKernelGGL(tree_plan_kernel, dim3(n), dim3(64), 0, (hipStream_t)stream, parents, counts,
                     slots, lengths, rope_delta, n, n_nodes, pool_rows, max_len, starts,
                     (uint64_t*)ancestors, positions, token_slot, token_pos);
  OMNI_CHECK_LAUNCH();
  return OMNI_OK;
}

extern "C" int omni_kv_write_rows(const void* k, int64_t k_stride, const void* v, int64_t v_stride,
                                  void* k_cache, void* v_cache, const int64_t* slots,
                                  const int64_t* positions, int pool_rows, int max_len,
                                  int row_halfs, int tokens, void* stream) {
  if (tokens < 0 || pool_rows <= 0 || max_len <= 0 || row_halfs <= 0) return OMNI_EINVAL;
  if ((row_halfs & 7) || (k_stride & 7) || (v_stride & 7)) return OMNI_EUNSUPPORTED;
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

extern "C" int omni_tree_attention(const void* q, int q_stride, const void* k_cache,
                                   const void* v_cache, int pool_rows, int max_len,
                                   const int64_t* slots, const int64_t* starts,
                                   const void* ancestors, int n, int n_nodes, void* out,
                                   int out_stride, int n_heads, int n_kv_heads, int head_dim,
                                   float scale, int splits, float* workspace,
                                   int64_t workspace_floats, void* stream) {
  if (n < 0 || n_nodes < 1 || n_heads <= 0 || n_kv_heads <= 0 || pool_rows <= 0 || max_len <= 0)
    return OMNI_EINVAL;
  if (head_dim != TREE_HD || n_heads % n_kv_heads || n_nodes > TREE_MAX) return OMNI_EUNSUPPORTED;
  if (!(scale >= 0x1p-126f) || scale > 3e38f) return OMNI_EUNSUPPORTED;
  if (q_stride < n_heads * TREE_HD || (q_stride & 7)) return OMNI_EINVAL;
  if (out_stride < n_heads * TREE_HD || (out_stride & 7)) return OMNI_EINVAL;
  if (splits < 1 || splits > 256 || (!slots && n > pool_rows)) return OMNI_EINVAL;
  if (n == 0) return OMNI_OK;
  if (!q || !k_cache || !v_cache || !starts || !ancestors || !out) return OMNI_EINVAL;
  if (((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)out) & 15) return OMNI_EINVAL;
  if (splits > 1 &&
      (!workspace || workspace_floats < (int64_t)n * n_nodes * n_heads * splits * ATT_REC))
    return OMNI_EINVAL;
  if ((int64_t)n * n_nodes > 0x7fffffff || n_heads > 65535) return OMNI_EUNSUPPORTED;
  TreeArgs a;
  a.q = (const half_t*)q;
  a.q_stride = q_stride;
  a.k_cache = (const half_t*)k_cache;
  a.v_cache = (const half_t*)v_cache;
  a.pool_rows = pool_rows;
  a.max_len = max_len;
  a.nkv = n_kv_heads;
  a.G = n_heads / n_kv_heads;
  a.T = n_nodes;
  a.slots = slots;
  a.starts = starts;
  a.ancestors = (const uint64_t*)ancestors;
  a.out = (half_t*)out;
  a.out_stride = out_stride;
  a.scale_log2 = scale * 1.4426950408889634f;
  hipLaunchKernelGGL(tree_attn_kernel, dim3(n * n_nodes, n_heads), dim3(64), 0, (hipStream_t)stream, a);
  OMNI_CHECK_LAUNCH();
  return OMNI_OK;
}
