// Rows of logits as the kernels over a vocabulary read them: elements of three types, 64-bit
// weights, reductions over a wave.  Used by spec_verify.hip and beam.hip.
#pragma once

#include "common.h"

template <int DT>
__device__ __forceinline__ constexpr int sv_size() { return DT == 2 ? 4 : 2; }

template <int DT>   // 0 fp16, 1 bf16, 2 fp32; NaN as -inf
__device__ __forceinline__ float sv_logit(const void* row, int64_t v) {
  float x;
  if (DT == 2) x = ((const float*)row)[v];
  else x = ld16f<DT == 1>(((const unsigned short*)row)[v]);
  return x == x ? x : -INFINITY;
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
