// Beam search's choice: the k best continuations of each request over its beams and the vocabulary.
//
// Beam b of request s has the score scores[s][b] (a sum of log-probabilities) and the logits
// x = logits[s][b]; its continuation by token v is worth scores[s][b] + x_v - log sum exp x.  A
// finished beam has one continuation, itself.  Ties go to the lower beam, then to the lower token.
//
// Within a beam the order of the continuations is that of its logits, so the first launch, over
// blocks of a row, lists each block's k best logits and its sum of weights; the second, a request a
// workgroup, merges a row's lists, then the rows', whose values need the sums.
#include "logit_rows.h"

#define BM_WAVES 4
#define BM_MAX_BEAMS 32
#define BM_MAX_K 64
#define BM_MAX_BLOCKS 64           // of a row: a lane of the merging wave each

struct BeamArgs {
  const void* logits;
  int64_t req_stride, row_stride;
  const float* scores;       // [n][W]
  const uint8_t* done;       // [n][W] or null
  const int64_t* stop;       // [n or 1][stops] or null
  int64_t stop_stride;
  int stops, n, W, V, k, blocks;
  int64_t pad;
  float2* lists;             // [n W][blocks][k] (logit, token), best first, -inf behind them
  double2* sums;             // [n W][blocks] (largest logit, sum of weights relative to it)
  float* out_scores;
  int* parents;
  int64_t* tokens;
  uint8_t* out_done;
};

__device__ __forceinline__ bool bm_done(const BeamArgs& a, int r) { return a.done && a.done[r]; }

// Weight of a logit in a row whose largest is m: 1 at m, infinite or not, 0 at -inf.
__device__ __forceinline__ double bm_weight(float x, float m) {
#pragma clang fp contract(off)
  if (x == m) return 1.0;
  if (!(x > -INFINITY) || m == INFINITY) return 0.0;
  return sv_exp2(fmax(((double)x - (double)m) * 1.4426950408889634073599, -2000.0));
}

// The lane that holds the largest v, of the lowest token among equals.
__device__ __forceinline__ int bm_winner(float v, int token) {
  const float top = wave_top(v);
  uint64_t best = __ballot(v == top);
  if (best & (best - 1)) {
    int t = v == top ? token : 0x7fffffff;
#pragma unroll
    for (int o = 32; o; o >>= 1) t = min(t, __shfl_xor(t, o));
    best = __ballot(v == top && token == t);
  }
  return __ffsll((unsigned long long)best) - 1;
}

template <int DT, int EPT>
__global__ __launch_bounds__(64 * BM_WAVES) void beam_scan_kernel(BeamArgs a) {
  typedef SvPiece<DT> P;
  __shared__ float2 list[BM_WAVES][BM_MAX_K];
  __shared__ float wm[BM_WAVES];
  __shared__ double wz[BM_WAVES];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = blockIdx.x / a.blocks, block = blockIdx.x - r * a.blocks;
  if (bm_done(a, r) || !(fabsf(a.scores[r]) < INFINITY)) return;
  const int s = r / a.W, b = r - s * a.W;
  const void* row = (const char*)a.logits + (s * a.req_stride + b * a.row_stride) * sv_size<DT>();
  const int v0 = (block * BM_WAVES + wave) * 64 * EPT;
  float x[EPT];
#pragma unroll
  for (int j = 0; j < EPT / P::N; ++j) {
    P p;
    p.load(row, v0, a.V, lane, j);
#pragma unroll
    for (int e = 0; e < P::N; ++e) {
      const float y = p.get(e);
      x[j * P::N + e] = y == y ? y : -INFINITY;
    }
  }
  auto token = [&](int e) { return v0 + P::at(lane, e / P::N) + e % P::N; };
  float m = x[0];
#pragma unroll
  for (int e = 1; e < EPT; ++e) m = fmaxf(m, x[e]);
  m = wave_top(m);
  double z = 0.0;
#pragma unroll 4
  for (int e = 0; e < EPT; ++e) z += bm_weight(x[e], m);
  z = wave_total(m > -INFINITY ? z : 0.0);
  if (lane == 0) {
    wm[wave] = m;
    wz[wave] = z;
  }
  // the wave's k best, one after another: every lane's best behind the last one taken
  float lastv = INFINITY;
  int lastt = -1;
  float bv;
  int bt;
  auto next = [&]() {
    bv = -INFINITY;
    bt = 0x7fffffff;
#pragma unroll
    for (int e = 0; e < EPT; ++e) {
      const bool behind = x[e] < lastv || (x[e] == lastv && token(e) > lastt);
      if (behind && x[e] > bv) {
        bv = x[e];
        bt = token(e);
      }
    }
  };
  next();
  for (int j = 0; j < a.k; ++j) {
    const int w = bm_winner(bv, bt);
    lastv = lane_of(bv, w);
    lastt = __builtin_amdgcn_readlane(bt, w);
    if (lane == 0) list[wave][j] = make_float2(lastv, __builtin_bit_cast(float, lastt));
    if (!(lastv > -INFINITY)) {
      for (int i = j + lane; i < a.k; i += 64) list[wave][i] = make_float2(-INFINITY, 0.f);
      break;
    }
    if (lane == w) next();
  }
  __syncthreads();
  if (wave) return;
  float2* out = a.lists + (int64_t)blockIdx.x * a.k;
  int at = 0;
  float2 head = lane < BM_WAVES ? list[lane][0] : make_float2(-INFINITY, 0.f);
  for (int j = 0; j < a.k; ++j) {
    const int w = bm_winner(head.x, __builtin_bit_cast(int, head.y));
    if (lane == w) {
      out[j] = head;
      ++at;
      head = at < a.k && lane < BM_WAVES ? list[lane][at] : make_float2(-INFINITY, 0.f);
    }
  }
  if (lane == 0) {
    float M = wm[0];
#pragma unroll
    for (int w = 1; w < BM_WAVES; ++w) M = fmaxf(M, wm[w]);
    double Z = 0.0;
#pragma unroll
    for (int w = 0; w < BM_WAVES; ++w) Z += wz[w] * bm_weight(wm[w], M);
    a.sums[blockIdx.x] = make_double2((double)M, Z);
  }
}

#define BM_PICK_WAVES 8

__global__ __launch_bounds__(64 * BM_PICK_WAVES) void beam_pick_kernel(BeamArgs a) {
  __shared__ double value[BM_MAX_BEAMS][BM_MAX_K];
  __shared__ int token[BM_MAX_BEAMS][BM_MAX_K], count[BM_MAX_BEAMS];
  __shared__ int pick_b[BM_MAX_K];
  __shared__ int64_t pick_t[BM_MAX_K];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, s = blockIdx.x;
  for (int b = wave; b < a.W; b += BM_PICK_WAVES) {
    const int r = s * a.W + b;
    const float score = a.scores[r];
    const bool in = fabsf(score) < INFINITY, over = bm_done(a, r);
    if (!in || over) {
      if (lane == 0) {
        value[b][0] = (double)score;
        count[b] = in ? 1 : 0;
      }
      continue;
    }
    const int64_t first = (int64_t)r * a.blocks;
    const double2 own = lane < a.blocks ? a.sums[first + lane] : make_double2(-INFINITY, 0.0);
    const float M = wave_top((float)own.x);
    const double Z = wave_total(M > -INFINITY ? own.y * bm_weight((float)own.x, M) : 0.0);
    const double base = log(Z);
    const float2* list = a.lists + (first + lane) * a.k;
    int at = 0, got = 0;
    float2 head = lane < a.blocks ? list[0] : make_float2(-INFINITY, 0.f);
    for (; got < a.k; ++got) {
      const int w = bm_winner(head.x, __builtin_bit_cast(int, head.y));
      const float x = lane_of(head.x, w);
      if (!(x > -INFINITY) || (M == INFINITY && x < M)) break;
      if (lane == w) {
        value[b][got] = (double)score + ((x == M ? 0.0 : (double)x - (double)M) - base);
        token[b][got] = __builtin_bit_cast(int, head.y);
        ++at;
        head = at < a.k ? list[at] : make_float2(-INFINITY, 0.f);
      }
    }
    if (lane == 0) count[b] = got;
  }
  __syncthreads();
  if (wave == 0) {
    int at = 0;
    const int have = lane < a.W ? count[lane] : 0;
    double head = have ? value[lane][0] : -INFINITY;
    for (int j = 0; j < a.k; ++j) {
      double top = head;
#pragma unroll
      for (int o = 32; o; o >>= 1) top = fmax(top, __shfl_xor(top, o));
      const uint64_t best = __ballot(head == top);
      const int w = __ffsll((unsigned long long)best) - 1;
      if (lane == w) {
        const bool found = top > -INFINITY;
        const int64_t t = !found ? -1 : bm_done(a, s * a.W + lane) ? a.pad : token[lane][at];
        pick_b[j] = found ? lane : -1;
        pick_t[j] = t;
        a.out_scores[s * a.k + j] = (float)top;
        if (found) {
          ++at;
          head = at < have ? value[lane][at] : -INFINITY;
        }
      }
    }
  }
  __syncthreads();
  for (int j = threadIdx.x; j < a.k; j += 64 * BM_PICK_WAVES) {
    const int b = pick_b[j];
    const int64_t t = pick_t[j];
    bool over = b < 0 || bm_done(a, s * a.W + b);
    for (int i = 0; i < a.stops; ++i) over |= a.stop[s * a.stop_stride + i] == t;
    const int64_t o = (int64_t)s * a.k + j;
    a.parents[o] = b;
    a.tokens[o] = t;
    a.out_done[o] = over;
  }
}

// Tokens of a block: 4096 where rows are few, 8192 else.
static int bm_ept(int64_t rows, int V) {
  return rows * ceil_div(V, 8192) < 512 && V <= 4096 * BM_MAX_BLOCKS ? 16 : 32;
}

static int64_t bm_work(int n, int W, int V, int k) {
  if (n < 0 || W < 1 || V < 1 || k < 1) return OMNI_EINVAL;
  if (W > BM_MAX_BEAMS || k > BM_MAX_K || V > 8192 * BM_MAX_BLOCKS) return OMNI_EUNSUPPORTED;
  const int64_t rows = (int64_t)n * W;
  const int64_t blocks = ceil_div(V, 64 * BM_WAVES * bm_ept(rows, V));
  const int64_t work = rows * blocks * (k + 2);
  return rows * blocks > 0x7fffffff || work > 0x7fffffff ? OMNI_EUNSUPPORTED : work;
}

// 8-byte words of workspace.
extern "C" int omni_beam_select_work(int n, int beams, int vocab, int k) {
  return (int)bm_work(n, beams, vocab, k);
}

extern "C" int omni_beam_select(const void* logits, int dtype, int64_t req_stride, int64_t row_stride,
                                const float* scores, const void* done, const int64_t* stop, int stops,
                                int64_t stop_stride, int64_t pad, int n, int beams, int vocab, int k,
                                float* out_scores, int* parents, int64_t* tokens, void* out_done,
                                void* workspace, int64_t workspace_words, void* stream) {
  const int64_t work = bm_work(n, beams, vocab, k);
  if (work < 0) return (int)work;
  if (dtype < 0 || dtype > 2) return OMNI_EUNSUPPORTED;
  if (req_stride < 0 || row_stride < 0 || stops < 0 || stop_stride < 0) return OMNI_EINVAL;
  if (n == 0) return OMNI_OK;
  if (!logits || !scores || !out_scores || !parents || !tokens || !out_done || !workspace ||
      (stops && !stop) || workspace_words < work || ((uintptr_t)workspace & 15))
    return OMNI_EINVAL;
  const int64_t rows = (int64_t)n * beams;
  const int ept = bm_ept(rows, vocab), blocks = ceil_div(vocab, 64 * BM_WAVES * ept);
  double2* sums = (double2*)workspace;
  const BeamArgs a = {logits, req_stride, row_stride, scores, (const uint8_t*)done, stop, stop_stride,
                      stops, n, beams, vocab, k, blocks, pad, (float2*)(sums + rows * blocks), sums,
                      out_scores, parents, tokens, (uint8_t*)out_done};
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid((unsigned)(rows * blocks)), block(64 * BM_WAVES);
  if (ept == 16) {
    if (dtype == 0) hipLaunchKernelGGL((beam_scan_kernel<0, 16>), grid, block, 0, st, a);
    else if (dtype == 1) hipLaunchKernelGGL((beam_scan_kernel<1, 16>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((beam_scan_kernel<2, 16>), grid, block, 0, st, a);
  } else {
    if (dtype == 0) hipLaunchKernelGGL((beam_scan_kernel<0, 32>), grid, block, 0, st, a);
    else if (dtype == 1) hipLaunchKernelGGL((beam_scan_kernel<1, 32>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((beam_scan_kernel<2, 32>), grid, block, 0, st, a);
  }
  OMNI_CHECK_LAUNCH();
  hipLaunchKernelGGL(beam_pick_kernel, dim3(n), dim3(64 * BM_PICK_WAVES), 0, st, a);
  OMNI_CHECK_LAUNCH();
  return OMNI_OK;
}
