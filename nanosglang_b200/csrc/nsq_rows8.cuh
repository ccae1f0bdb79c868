// Symmetric 8-bit quantisation of a row, shared by the int8 linear (tokens and
// weight rows) and the key/value cache:
//   s = max|x| / 127 (int8) or max|x| / 448 (e4m3), 1 where that is 0;
//   code = rint(x / s) or e4m3(x / s), both nearest-even of the fp32 quotient.
// A row with a NaN or an infinity gets that as its scale, so it reads back as NaN.
#pragma once

#include "nsq_common.cuh"

namespace nsq {

// fmax that keeps a NaN
__device__ __forceinline__ float nan_max(float m, float v) { return (v > m || v != v) ? v : m; }

template <bool FP8>
__device__ __forceinline__ float row_scale(float absmax) {
  const float s = __fdiv_rn(absmax, FP8 ? 448.0f : 127.0f);
  return s == 0.0f ? 1.0f : s;
}

// x / s, correctly rounded, for many x: the rounded reciprocal, one product
// and one residual step (P. Markstein, IBM J. Res. Dev. 34, 1990), exact where
// nothing under- or overflows, which s in [2^-96, 2^96] ensures for every
// quotient that matters (smaller ones round to code 0 either way). Other
// scales take the division.
struct RowDiv {
  float s, r;
  bool near;
  __device__ __forceinline__ explicit RowDiv(float scale) {
    s = scale;
    r = __frcp_rn(scale);
    near = scale >= 1.2621774e-29f && scale <= 7.9228163e28f;
  }
  __device__ __forceinline__ float operator()(float x) const {
    if (!near) return __fdiv_rn(x, s);
    const float q = x * r;
    return fmaf(fmaf(-q, s, x), r, q);
  }
};

// The quotient's code, saturated: |q| passes 127 or 448 only where s is
// subnormal. A NaN becomes 0 (int8) or the NaN code (e4m3).
template <bool FP8>
__device__ __forceinline__ uint8_t row_code(float q) {
  if constexpr (FP8) {
    return static_cast<uint8_t>(__nv_cvt_float_to_fp8(q, __NV_SATFINITE, __NV_E4M3));
  } else {
    return static_cast<uint8_t>(static_cast<int8_t>(max(-127, min(127, __float2int_rn(q)))));
  }
}

}  // namespace nsq
