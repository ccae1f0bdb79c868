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

// Four codes, x0's in the low byte. Within RowDiv's range nothing saturates and
// nothing is NaN: int8 then takes the low byte of q + 1.5 * 2^23, whose ulp is
// 1 (rint without the conversion pipe).
template <bool FP8>
__device__ __forceinline__ uint32_t row_codes4(const RowDiv& dv, float x0, float x1, float x2, float x3) {
  const float q0 = dv(x0), q1 = dv(x1), q2 = dv(x2), q3 = dv(x3);
  if constexpr (FP8) {
    return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(q0, q1), __NV_SATFINITE, __NV_E4M3) |
           ((uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(q2, q3), __NV_SATFINITE, __NV_E4M3) << 16);
  } else {
    if (!dv.near) {
      return (uint32_t)row_code<false>(q0) | ((uint32_t)row_code<false>(q1) << 8) |
             ((uint32_t)row_code<false>(q2) << 16) | ((uint32_t)row_code<false>(q3) << 24);
    }
    const uint32_t a = __float_as_uint(q0 + 12582912.f), b = __float_as_uint(q1 + 12582912.f);
    const uint32_t c = __float_as_uint(q2 + 12582912.f), d = __float_as_uint(q3 + 12582912.f);
    return prmt(prmt(a, b, 0x0040), prmt(c, d, 0x0040), 0x5410);
  }
}

// Eight 16-bit elements of x (two per word) as codes.
template <bool FP8, bool BF16>
__device__ __forceinline__ uint2 row_codes8(const RowDiv& dv, uint4 x) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  float f[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = elem_to_float<BF16>((uint16_t)(w[i / 2] >> (16 * (i & 1))));
  return make_uint2(row_codes4<FP8>(dv, f[0], f[1], f[2], f[3]), row_codes4<FP8>(dv, f[4], f[5], f[6], f[7]));
}

// The largest magnitude of 16-bit elements, two at a time as unsigned integers
// (the order of magnitudes; a NaN is above infinity, so it stays).
__device__ __forceinline__ uint32_t abs_max2(uint32_t m, uint4 x) {
  m = __vmaxu2(m, x.x & 0x7fff7fffu);
  m = __vmaxu2(m, x.y & 0x7fff7fffu);
  m = __vmaxu2(m, x.z & 0x7fff7fffu);
  return __vmaxu2(m, x.w & 0x7fff7fffu);
}
template <bool BF16>
__device__ __forceinline__ float abs_max_value(uint32_t m) {
  return elem_to_float<BF16>((uint16_t)max(m & 0xffffu, m >> 16));
}

}  // namespace nsq
