// 64-bit helpers of the token-level kernels: reductions by DPP, 2^t and log2 with few live registers.
// 64-bit vector operations run at the rate of 32-bit ones on this part, so what a result's exactness
// hangs on is simply computed in 64 bits.
#pragma once

#include <type_traits>

#include "fm_vocab.hip.h"

namespace fm {

constexpr double kLn2d = 0.69314718055994530942;
constexpr double kLog2ed = 1.4426950408889634074;

template <int CTRL>
__device__ __forceinline__ double dpp64(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, 0xf, 0xf, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, 0xf, 0xf, false);
  return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ double readlane64(double v, int l) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, l);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), l);
  return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}
struct Sum64 { __device__ static __forceinline__ double f(double a, double b) { return a + b; } };

// over aligned groups of G lanes (1, 2, 4, 8, 16 or 64), the result in every lane, fixed order
template <int G, typename Op>
__device__ __forceinline__ double group_reduce64(double v) {
  if constexpr (G >= 2) v = Op::f(v, dpp64<kDppXor1>(v));
  if constexpr (G >= 4) v = Op::f(v, dpp64<kDppXor2>(v));
  if constexpr (G >= 8) v = Op::f(v, dpp64<kDppHalfMirror>(v));
  if constexpr (G >= 16) v = Op::f(v, dpp64<kDppMirror>(v));
  if constexpr (G == 64)
    v = Op::f(Op::f(readlane64(v, 0), readlane64(v, 16)), Op::f(readlane64(v, 32), readlane64(v, 48)));
  return v;
}
__device__ __forceinline__ double wave_sum64(double v) { return group_reduce64<64, Sum64>(v); }

template <int CTRL>
__device__ __forceinline__ uint64_t dpp_u64(uint64_t v) {
  return __builtin_bit_cast(uint64_t, dpp64<CTRL>(__builtin_bit_cast(double, v)));
}
__device__ __forceinline__ uint64_t readlane_u64(uint64_t v, int l) {
  return __builtin_bit_cast(uint64_t, readlane64(__builtin_bit_cast(double, v), l));
}
__device__ __forceinline__ uint64_t wave_sum_u64(uint64_t v) {
  v += dpp_u64<kDppXor1>(v);
  v += dpp_u64<kDppXor2>(v);
  v += dpp_u64<kDppHalfMirror>(v);
  v += dpp_u64<kDppMirror>(v);
  return (readlane_u64(v, 0) + readlane_u64(v, 16)) + (readlane_u64(v, 32) + readlane_u64(v, 48));
}
// inclusive prefix sum over the wave in lane order: four shifts inside the rows of sixteen lanes, then
// the rows' totals
__device__ __forceinline__ uint64_t wave_incl_u64(uint64_t v) {
  const int lane = lane_id(), in_row = lane & 15;
  uint64_t t = dpp_u64<0x111>(v);            // row_shr:1
  v += in_row >= 1 ? t : 0ull;
  t = dpp_u64<0x112>(v);
  v += in_row >= 2 ? t : 0ull;
  t = dpp_u64<0x114>(v);
  v += in_row >= 4 ? t : 0ull;
  t = dpp_u64<0x118>(v);
  v += in_row >= 8 ? t : 0ull;
  const uint64_t a = readlane_u64(v, 15), b = readlane_u64(v, 31), c = readlane_u64(v, 47);
  v += lane >= 48 ? (a + b) + c : (lane >= 32 ? a + b : (lane >= 16 ? a : 0ull));
  return v;
}
// integer sum over the workgroup, the waves' by DPP
template <int NW>
__device__ __forceinline__ uint64_t block_sum_int64(uint64_t v, uint64_t* smem) {
  v = wave_sum_u64(v);
  if ((threadIdx.x & 63) == 0) smem[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0ull;
#pragma unroll
  for (int i = 0; i < NW; ++i) v += smem[i];
  __syncthreads();
  return v;
}

// across the NW waves of a workgroup; the waves' results are combined by lanes rather than by every
// thread reading all of them (32 registers beside a held row)
template <int NW, typename Op>
__device__ __forceinline__ double block_reduce64(double v, double* smem) {
  v = group_reduce64<64, Op>(v);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (lane == 0) smem[wave] = v;
  __syncthreads();
  v = group_reduce64<NW, Op>(smem[lane & (NW - 1)]);
  __syncthreads();
  return v;
}
// 2^t: degree-8 polynomial through the Chebyshev nodes of [-1/2, 1/2] (relative error 1.1e-12) and an
// exact scaling. Below 2^-1100 the result is zero; NaN stays.
__device__ __forceinline__ double exp2_64(double t) {
  t = t < -1100.0 ? -1100.0 : t;
  const double n = __builtin_rint(t);
  const double f = t - n;
  double r = 1.3255224878668817e-06;
  r = __builtin_fma(r, f, 1.5310079402249296e-05);
  r = __builtin_fma(r, f, 0.00015403455852453838);
  r = __builtin_fma(r, f, 0.0013333450568000645);
  r = __builtin_fma(r, f, 0.009618129159402558);
  r = __builtin_fma(r, f, 0.05550410941205933);
  r = __builtin_fma(r, f, 0.2402265069581299);
  r = __builtin_fma(r, f, 0.6931471805459335);
  r = __builtin_fma(r, f, 1.0);
  return __builtin_amdgcn_ldexp(r, (int)n);
}
// the fp32 logarithm of the mantissa, corrected by the first two terms of log(1 + r) for what is left
__device__ __forceinline__ double log2_64(double x) {
  const double m = __builtin_amdgcn_frexp_mant(x);
  const double y = (double)fast_log2((float)m);
  const double r = __builtin_fma(m, exp2_64(-y), -1.0);
  const double l = (double)__builtin_amdgcn_frexp_exp(x) + y + r * __builtin_fma(r, -0.5, 1.0) * kLog2ed;
  return x == 0.0 ? -__builtin_inf() : l;
}

}  // namespace fm
