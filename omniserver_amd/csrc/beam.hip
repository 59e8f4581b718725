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
  float2* sums;              // [n W][blocks] (largest logit, sum of weights relative to it)
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

// Whether (logit, token) stands before another.
__device__ __forceinline__ bool bm_before(float2 x, float2 y) {
  return x.x > y.x || (x.x == y.x && __builtin_bit_cast(int, x.y) < __builtin_bit_cast(int, y.y));
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

#define BM_LOG2E 1.4426950216f     // log2 e in 32 bits

// Sum of a lane's N weights exp(x - m) in 32 bits, m finite.  Near zero one fma gives the exponent,
// relative to the rounded product R = m log2 e instead of m: the caller's sum is then to be taken
// times bm_shift(m).
__device__ __forceinline__ bool bm_direct(float m) { return fabsf(m) <= 256.f; }
__device__ __forceinline__ double bm_shift(float m) {
  return bm_direct(m) ? 1.0 + 0.6931471805599453 * ((double)(m * BM_LOG2E) - (double)m * BM_LOG2E) : 1.0;
}
template <int N>
__device__ __forceinline__ float bm_weights(const float (&x)[N], float m) {
  float z[4] = {0.f, 0.f, 0.f, 0.f};
  if (bm_direct(m)) {
    const float R = m * BM_LOG2E;
#pragma unroll
    for (int e = 0; e < N; ++e) z[e & 3] += __builtin_amdgcn_exp2f(fmaf(x[e], BM_LOG2E, -R));
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) z[e & 3] += __builtin_amdgcn_exp2f((x[e] - m) * BM_LOG2E);
  }
  return (z[0] + z[1]) + (z[2] + z[3]);
}

// ---------------------------------------------------------------------------
// A block of a row, EPT tokens a lane in registers.  Its k best: every wave finds the largest value
// that at least k / 4 of its lanes reach; the smallest of the four waves' is reached by k tokens or
// more, and mostly by few more.  Those go to LDS, where each counts the ones before it.
// Where they are too many (equal logits, all of the best in a few lanes) the waves take out their k
// best one after another, and the four lists are merged.
//
// 128 rows of 151936 fp16 logits, 39 MB, 13.5 us where a copy's rate is 8.  A workgroup is a chain (loads,
// largest, thresholds, sum, list, with two barriers), and eight waves a SIMD hide it from one another:
// with five 15, and fewer vector operations (maxima and fma of fp16 pairs as they are) change nothing.
// With weights in 64 bits and the lists taken out one after another it was 59.  4 rows 6.1 us.
// ---------------------------------------------------------------------------
#define BM_CAP 512                 // tokens that are ranked

template <int DT, int EPT>
__global__ __launch_bounds__(64 * BM_WAVES, 8) void beam_scan_kernel(BeamArgs a) {
  typedef SvPiece<DT> P;
  __shared__ float2 list[BM_CAP];
  static_assert(BM_CAP >= BM_WAVES * BM_MAX_K, "the waves' lists");
  __shared__ float wm[BM_WAVES], wz[BM_WAVES], wt[BM_WAVES];
  __shared__ int found;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int block = blockIdx.x, b = blockIdx.y, s = blockIdx.z, r = s * a.W + b;
  const int64_t place = (int64_t)r * a.blocks + block;
  const bool off = bm_done(a, r) || !(fabsf(a.scores[r]) < INFINITY);
  const void* row = (const char*)a.logits + (s * a.req_stride + b * a.row_stride) * sv_size<DT>();
  constexpr int PIECE = 64 * P::N;                  // tokens of a wave's load; waves take turns
  const int v0 = block * BM_WAVES * 64 * EPT + wave * PIECE;
  if (threadIdx.x == 0) found = 0;
  P p[EPT / P::N];
#pragma unroll
  for (int j = 0; j < EPT / P::N; ++j) p[j].load(row, v0 + j * BM_WAVES * PIECE, a.V, lane, 0);
  float x[EPT];
#pragma unroll
  for (int e = 0; e < EPT; ++e)
    x[e] = fmaxf(p[e / P::N].get(e % P::N), -INFINITY);       // leaves a NaN out
  float best[EPT / P::N], own = -INFINITY;          // of a piece, of all
#pragma unroll
  for (int j = 0; j < EPT / P::N; ++j) {
    best[j] = x[j * P::N];
#pragma unroll
    for (int e = 1; e < P::N; ++e) best[j] = fmaxf(best[j], x[j * P::N + e]);
    own = fmaxf(own, best[j]);
  }
  if (off) return;                                  // looked at once the logits are under way
  const float m = wave_top(own);
  // what k / nw lanes reach, of the nw waves with a token for every lane
  const int nw = min(max((a.V - block * BM_WAVES * 64 * EPT) / PIECE, 1), BM_WAVES);
  float least = wave < nw ? m : INFINITY;
  if (wave < nw) {
    float v = own;
    for (int left = (a.k + nw - 1) / nw; least > -INFINITY;) {
      const bool top = v == least;
      left -= __popcll(__ballot(top));
      if (left <= 0) break;
      v = top ? -INFINITY : v;
      least = wave_top(v);
    }
  }
  if (lane == 0) {
    wm[wave] = m;
    wt[wave] = least;
  }
  __syncthreads();
  const float M = fmaxf(fmaxf(wm[0], wm[1]), fmaxf(wm[2], wm[3]));
  // the lowest finite number where -inf would do
  const float from = fmaxf(fminf(fminf(wt[0], wt[1]), fminf(wt[2], wt[3])), -3.402823466e38f);
  // a lane's pieces with such a token are read again, the first while the sum is made: registers
  // have no index, and unrolled code is slow to fetch
  uint32_t mine = 0;
#pragma unroll
  for (int j = 0; j < EPT / P::N; ++j) mine |= best[j] >= from ? 1u << j : 0u;
  P again;
  int piece = 0;
  auto take = [&]() {
    if (!mine) return;
    piece = __ffs(mine) - 1;
    again.load(row, v0 + piece * BM_WAVES * PIECE, a.V, lane, 0);
  };
  take();
  float sum = 0.f;
  if (fabsf(M) < INFINITY) {
    sum = bm_weights(x, M);
  } else if (M == INFINITY) {
#pragma unroll
    for (int e = 0; e < EPT; ++e) sum += x[e] == M ? 1.f : 0.f;
  }
  sum = wave_total(sum);
  if (lane == 0) wz[wave] = sum;
  while (mine) {
    const int t = v0 + piece * BM_WAVES * PIECE + lane * P::N;
#pragma unroll
    for (int e = 0; e < P::N; ++e) {
      const float v = again.get(e);
      if (v >= from) {
        const int at = atomicAdd(&found, 1);
        if (at < BM_CAP) list[at] = make_float2(v, __builtin_bit_cast(float, t + e));
      }
    }
    mine &= mine - 1;
    take();
  }
  __syncthreads();
  const int count = found;
  float2* out = a.lists + place * a.k;
  if (threadIdx.x == 0) a.sums[place] = make_float2(M, (wz[0] + wz[1]) + (wz[2] + wz[3]));
  if (count <= BM_CAP) {
#pragma unroll 1
    for (int t = threadIdx.x; t < count; t += 64 * BM_WAVES) {
      const float2 own_t = list[t];
      int rank = 0;
#pragma unroll 8
      for (int i = 0; i < count; ++i) rank += bm_before(list[i], own_t);
      if (rank < a.k) out[rank] = own_t;
    }
    if (threadIdx.x >= count && threadIdx.x < a.k) out[threadIdx.x] = make_float2(-INFINITY, 0.f);
    return;
  }
  __syncthreads();                                  // the list is read, and used again
  // the wave's k best, one after another: every lane's best behind the last one taken
  float lastv = INFINITY;
  int lastt = -1;
  float bv;
  int bt;
  auto next = [&]() {
    const int first = v0 + lane * P::N, taken = lastt - first;
    bv = -INFINITY;
    bt = 0;
#pragma unroll
    for (int e = 0; e < EPT; ++e) {
      const int t = e / P::N * BM_WAVES * PIECE + e % P::N;
      const bool behind = x[e] < lastv || (x[e] == lastv && t > taken);
      if (behind && x[e] > bv) {
        bv = x[e];
        bt = t;
      }
    }
    bt += first;
  };
  next();
  for (int j = 0; j < a.k; ++j) {
    const int w = bm_winner(bv, bt);
    lastv = lane_of(bv, w);
    lastt = __builtin_amdgcn_readlane(bt, w);
    if (lane == 0) list[wave * BM_MAX_K + j] = make_float2(lastv, __builtin_bit_cast(float, lastt));
    if (!(lastv > -INFINITY)) {
      for (int i = j + lane; i < a.k; i += 64) list[wave * BM_MAX_K + i] = make_float2(-INFINITY, 0.f);
      break;
    }
    if (lane == w) next();
  }
  __syncthreads();
  if (wave) return;
  int at = 0;
  float2 head = lane < BM_WAVES ? list[lane * BM_MAX_K] : make_float2(-INFINITY, 0.f);
  for (int j = 0; j < a.k; ++j) {
    const int w = bm_winner(head.x, __builtin_bit_cast(int, head.y));
    if (lane == w) {
      out[j] = head;
      ++at;
      head = at < a.k && lane < BM_WAVES ? list[lane * BM_MAX_K + at] : make_float2(-INFINITY, 0.f);
    }
  }
}

// ---------------------------------------------------------------------------
// The choice, one workgroup a request.  A wave merges the lists of a row (a list a lane, the next
// four of it in registers) and makes values of their logits; then every value counts the ones before
// it: among all, where these are 64 at most, a value a lane; else among those that reach the k-th best
// of the rows' first few values, or stand close below it.
//
// The rows' 32-bit sums are good to BM_ERR, and so are the values.  Where two rows' values stand
// closer than twice that and one of them is among the k, the sums of those rows are made again in 64
// bits, and the order with them.  The scores of rows that are not stay as they are, 4e-6 off at most
// (3e-8 on a language model's rows, which is fp32's rounding).
//
// A chain of waits: 4 beams, k = 4, 5.9 us; 5 beams, k = 10, 7.8.  Loads of the lists and sums (1 us),
// sums and logarithm in 64 bits (1), k entries (0.2 each), the count (1.3).  Sixteen waves where the beams
// are more than eight: 12 beams, k = 12 21.2 us a call, with eight 24.4; 8 x 16, k = 32 48 and 52.
// ---------------------------------------------------------------------------
#define BM_AHEAD 4
// Of a sum, relative: a weight 2^t is off by |t| ln 2 2^-24 of its exponent's rounding (and as
// much of the difference's, or log2 e's), 2^-23 of its exponential; |t| up to 30 counts (2^19 tokens
// 2^-30 weigh 2^-11), and EPT / 4 + 9 additions are off by 2^-24 each: 4e-6.
#define BM_ERR 0x1p-17

struct BmRow {
  float m;
  double z;
};

__device__ __forceinline__ double bm_value(float score, float x, const BmRow& r, double log_z) {
#pragma clang fp contract(off)
  return (double)score + ((x == r.m ? 0.0 : (double)x - (double)r.m) - log_z);
}

// A row's weights in 64 bits, by the whole workgroup.
template <int DT, int WAVES>
__device__ double bm_exact_sum(const BeamArgs& a, int s, int b, float m, double* lds) {
  typedef SvPiece<DT> P;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const void* row = (const char*)a.logits + (s * a.req_stride + b * a.row_stride) * sv_size<DT>();
  double z[2] = {0.0, 0.0};
  for (int64_t v0 = wave * 64 * P::N; v0 < a.V; v0 += WAVES * 64 * P::N) {
    P p;
    p.load(row, (int)v0, a.V, lane, 0);
#pragma unroll
    for (int e = 0; e < P::N; ++e) {
      const float y = p.get(e);
      z[e & 1] += bm_weight(y == y ? y : -INFINITY, m);
    }
  }
  __syncthreads();
  const double mine = wave_total(z[0] + z[1]);
  if (lane == 0) lds[wave] = mine;
  __syncthreads();
  double total = 0.0;
  for (int w = 0; w < WAVES; ++w) total += lds[w];
  return total;
}

// LDS that lanes of one wave hand each other: operations of a wave are in order.
__device__ __forceinline__ void bm_wave_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// The k best of a row's lists, a list a lane with its first entries in head, one after another; how
// many there are.  (Counting, among the entries that reach the k-th best of the lists' first ones, those
// before each, costs more fetched code than it saves: 1 x 4 beams, k = 4 13.1 us a call, this 11.5; 1 x 8,
// k = 16 23.4 and 22.2; only 8 x 16, k = 32 47.3 and 49.5.)
__device__ __forceinline__ int bm_merge(const BeamArgs& a, const float2* list, float2 (&head)[BM_AHEAD],
                                        float2* out, float M) {
  const int lane = threadIdx.x & 63;
  const float2 none = make_float2(-INFINITY, 0.f);
  int at = 0, got = 0;
  for (; got < a.k; ++got) {
    const int w = bm_winner(head[0].x, __builtin_bit_cast(int, head[0].y));
    const float x = lane_of(head[0].x, w);
    if (!(x > -INFINITY) || (M == INFINITY && x < M)) break;
    if (lane == w) {
      out[got] = head[0];
      ++at;
#pragma unroll
      for (int j = 0; j + 1 < BM_AHEAD; ++j) head[j] = head[j + 1];
      head[BM_AHEAD - 1] = none;
      if (at % BM_AHEAD == 0) {
#pragma unroll
        for (int j = 0; j < BM_AHEAD; ++j)
          if (at + j < a.k) head[j] = list[at + j];
      }
    }
  }
  bm_wave_lds();
  return got;
}

template <int DT, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void beam_pick_kernel(BeamArgs a) {
  __shared__ double value[BM_MAX_BEAMS][BM_MAX_K];
  __shared__ float2 cand[BM_MAX_BEAMS][BM_MAX_K];
  __shared__ int count[BM_MAX_BEAMS];
  __shared__ BmRow rows[BM_MAX_BEAMS];
  __shared__ double lds[WAVES];
  __shared__ int pick_b[BM_MAX_K], pick_t[BM_MAX_K];
  __shared__ int64_t stops[BM_MAX_K];
  __shared__ bool ended[BM_MAX_BEAMS];
  __shared__ double flat[64];                       // all values in a row, where they are few
  __shared__ int ranks[64], order[64];
  __shared__ uint16_t line[BM_MAX_BEAMS * BM_MAX_K], place[BM_MAX_BEAMS * BM_MAX_K];    // where they are many
  __shared__ double reach[BM_MAX_BEAMS * BM_MAX_K], least;
  __shared__ int asked;
  __shared__ uint32_t near;                         // a bit a beam
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, s = blockIdx.x;
  if (tid == 0) near = 0;
  if (tid < BM_MAX_K) pick_b[tid] = -1;
  const int64_t own_stop = tid < min(a.stops, BM_MAX_K) ? a.stop[s * a.stop_stride + tid] : -1;
  for (int b = wave; b < a.W; b += WAVES) {
    const int r = s * a.W + b;
    const int64_t first = (int64_t)r * a.blocks;
    const float2* list = a.lists + (first + lane) * a.k;
    const float2 none = make_float2(-INFINITY, 0.f);
    // all loads at once; what a row that is not in use has there is not looked at
    const float score = a.scores[r];
    const bool in = fabsf(score) < INFINITY, over = bm_done(a, r), mine = lane < a.blocks;
    const float2 own = mine ? a.sums[first + lane] : make_float2(-INFINITY, 0.f);
    float2 head[BM_AHEAD];
#pragma unroll
    for (int j = 0; j < BM_AHEAD; ++j) head[j] = mine && j < a.k ? list[j] : none;
    if (lane == 0) ended[b] = over;
    if (!in || over) {
      if (lane == 0) {
        value[b][0] = (double)score;
        cand[b][0] = make_float2(0.f, 0.f);
        count[b] = in ? 1 : 0;
      }
      continue;
    }
    const float M = wave_top(own.x);
    BmRow row = {M, wave_total(M > -INFINITY ? (double)own.y * bm_shift(own.x) * bm_weight(own.x, M) : 0.0)};
    const int got = bm_merge(a, list, head, cand[b], M);
    const double log_z = log(row.z);
    for (int i = lane; i < got; i += 64) value[b][i] = bm_value(score, cand[b][i].x, row, log_z);
    if (lane == 0) {
      count[b] = got;
      rows[b] = row;
    }
  }
  if (tid < BM_MAX_K) stops[tid] = own_stop;
  __syncthreads();
  for (int turn = 0; turn < 2; ++turn) {
    const int all = a.W * a.k;
    if (all <= 64) {
      if (wave == 0) {
        const int b = (int)(((float)lane + 0.5f) * (1.f / (float)a.k)), i = lane - b * a.k;
        flat[lane] = lane < all && i < count[b] ? value[b][i] : -INFINITY;
        ranks[lane] = 0;
      }
      __syncthreads();
      // a value a lane; every wave counts some of the others
      const double v = flat[lane];
      int before = 0;
#pragma unroll
      for (int j = 0; j < 64 / WAVES; ++j) {
        const int o = wave * (64 / WAVES) + j;
        const double y = flat[o];
        before += y > v || (y == v && o < lane);    // of one row the lists are in order
      }
      if (before) atomicAdd(&ranks[lane], before);
      __syncthreads();
      if (wave == 0) {
        order[ranks[lane]] = lane;                         // a permutation: equal values by lane
        bm_wave_lds();
        const int up = order[lane], down = order[min(lane + 1, 63)];
        const double vu = flat[up], vd = flat[down], vk = flat[order[a.k - 1]];
        const int bu = (int)(((float)up + 0.5f) * (1.f / (float)a.k));
        if (lane < a.k && vu > -INFINITY) {
          pick_b[lane] = bu;
          pick_t[lane] = up - bu * a.k;
        }
        // next to one another, of two rows, and one of them may be among the k
        if (turn == 0 && vd > -INFINITY && vu - vd <= 2 * BM_ERR && vk - vd <= 2 * BM_ERR) {
          const int bd = (int)(((float)down + 0.5f) * (1.f / (float)a.k));
          if (bu != bd && !(ended[bu] && ended[bd])) atomicOr(&near, 1u << bu | 1u << bd);
        }
      }
    } else {
      // the k-th best of the rows' first few values, 3 k in all or more: what reaches that, or
      // stands close below, is in question
      const int q = min((3 * a.k + a.W - 1) / a.W, a.k), firsts_n = a.W * q;
      if (tid < firsts_n) {
        const int b = tid / q, i = tid - b * q;
        reach[tid] = i < count[b] ? value[b][i] : -INFINITY;
      }
      if (tid == 0) {
        asked = 0;
        least = -INFINITY;
      }
      __syncthreads();
      if (tid < firsts_n) {
        const double v = reach[tid];
        int above = 0;
#pragma unroll 8
        for (int j = 0; j < firsts_n; ++j) above += reach[j] > v || (reach[j] == v && j < tid);
        if (above == a.k - 1) least = v;
      }
      __syncthreads();
      const double from = least - 4 * BM_ERR;
      __syncthreads();
      for (int c = tid; c < all; c += 64 * WAVES) {
        const int b = c / a.k, i = c - b * a.k;
        const double v = i < count[b] ? value[b][i] : -INFINITY;
        if (v > -INFINITY && v >= from) {
          const int x = atomicAdd(&asked, 1);
          line[x] = (uint16_t)c;
          reach[x] = v;
        }
      }
      __syncthreads();
      const int n = asked;
      for (int x = tid; x < n; x += 64 * WAVES) {
        const int c = line[x];
        const double v = reach[x];
        int rank = 0;
#pragma unroll 8
        for (int y = 0; y < n; ++y) rank += reach[y] > v || (reach[y] == v && line[y] < c);
        place[rank] = (uint16_t)c;
      }
      __syncthreads();
      auto at = [&](int r) {
        const int c = place[r], b = c / a.k;
        return value[b][c - b * a.k];
      };
      const double vk = n ? at(min(a.k, n) - 1) : 0.0;
      for (int r = tid; r < n; r += 64 * WAVES) {
        const int bu = place[r] / a.k;
        if (r < a.k) {
          pick_b[r] = bu;
          pick_t[r] = place[r] - bu * a.k;
        }
        // next to one another, of two rows, and one of them may be among the k
        if (turn == 0 && r + 1 < n && at(r) - at(r + 1) <= 2 * BM_ERR && vk - at(r + 1) <= 2 * BM_ERR) {
          const int bd = place[r + 1] / a.k;
          if (bu != bd && !(ended[bu] && ended[bd])) atomicOr(&near, 1u << bu | 1u << bd);
        }
      }
    }
    __syncthreads();
    const uint32_t again = turn ? 0 : near;
    if (!again) break;
    for (int b = 0; b < a.W; ++b) {
      if (!(again >> b & 1) || ended[b]) continue;
      BmRow row = rows[b];
      row.z = bm_exact_sum<DT, WAVES>(a, s, b, row.m, lds);
      const double log_z = log(row.z);
      const float score = a.scores[s * a.W + b];
      for (int i = tid; i < count[b]; i += 64 * WAVES)
        value[b][i] = bm_value(score, cand[b][i].x, row, log_z);
    }
    __syncthreads();
  }
  for (int j = tid; j < a.k; j += 64 * WAVES) {
    int b = pick_b[j];
    int64_t t = -1;
    bool over = true;
    float v = -INFINITY;
    if (b >= 0) v = (float)value[b][pick_t[j]];
    if (v > -INFINITY) {
      over = ended[b];
      t = over ? a.pad : __builtin_bit_cast(int, cand[b][pick_t[j]].y);
    } else {
      b = -1;                                       // also a sum that is too low for 32 bits
    }
    for (int i = 0; i < min(a.stops, BM_MAX_K); ++i) over |= stops[i] == t;
    for (int i = BM_MAX_K; i < a.stops; ++i) over |= a.stop[s * a.stop_stride + i] == t;
    const int64_t o = (int64_t)s * a.k + j;
    a.out_scores[o] = v;
    a.parents[o] = b;
    a.tokens[o] = t;
    a.out_done[o] = over;
  }
}

// Tokens of a block, 256 times this: as many as leave a workgroup for every CU twice, or as few.  A call in
// a graph of ten (among others, with its outputs' allocation, 32 x 4 take 20.9) of 8 x 16 beams, k = 16, with
// 8192 tokens 34.3 us, with 4096 38.2 (more lists to merge); 32 x 4 19.2 and 21.8; 4 x 4 beams over 32003
// tokens with 2048 12.4, with 4096 12.9.
static int bm_ept(int64_t rows, int V) {
  for (int ept = 32; ept > 8; ept /= 2)
    if (rows * ceil_div(V, 256 * ept) >= 512 || V > 128 * ept * BM_MAX_BLOCKS) return ept;
  return 8;
}

static int64_t bm_work(int n, int W, int V, int k) {
  if (n < 0 || W < 1 || V < 1 || k < 1) return OMNI_EINVAL;
  if (n > 65535 || W > BM_MAX_BEAMS || k > BM_MAX_K || V > 8192 * BM_MAX_BLOCKS) return OMNI_EUNSUPPORTED;
  const int64_t rows = (int64_t)n * W;
  const int64_t blocks = ceil_div(V, 64 * BM_WAVES * bm_ept(rows, V));
  const int64_t work = rows * blocks * (k + 1);
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
  float2* sums = (float2*)workspace;
  const BeamArgs a = {logits, req_stride, row_stride, scores, (const uint8_t*)done, stop, stop_stride,
                      stops, n, beams, vocab, k, blocks, pad, sums + rows * blocks, sums,
                      out_scores, parents, tokens, (uint8_t*)out_done};
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid(blocks, beams, n), block(64 * BM_WAVES);
#define BM_SCAN(DT)                                                                          \
  if (ept == 8) hipLaunchKernelGGL((beam_scan_kernel<DT, 8>), grid, block, 0, st, a);        \
  else if (ept == 16) hipLaunchKernelGGL((beam_scan_kernel<DT, 16>), grid, block, 0, st, a); \
  else hipLaunchKernelGGL((beam_scan_kernel<DT, 32>), grid, block, 0, st, a);
  if (dtype == 0) {
    BM_SCAN(0)
  } else if (dtype == 1) {
    BM_SCAN(1)
  } else {
    BM_SCAN(2)
  }
#undef BM_SCAN
  OMNI_CHECK_LAUNCH();
#define BM_PICK(DT)                                                                                      \
  if (beams > 8) hipLaunchKernelGGL((beam_pick_kernel<DT, 16>), dim3(n), dim3(64 * 16), 0, st, a);       \
  else hipLaunchKernelGGL((beam_pick_kernel<DT, 8>), dim3(n), dim3(64 * 8), 0, st, a);
  if (dtype == 0) {
    BM_PICK(0)
  } else if (dtype == 1) {
    BM_PICK(1)
  } else {
    BM_PICK(2)
  }
#undef BM_PICK
  OMNI_CHECK_LAUNCH();
  return OMNI_OK;
}
