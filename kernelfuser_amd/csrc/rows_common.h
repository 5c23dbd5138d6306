// The arithmetic of a prepared row (RMSNorm * gamma, rotate-half RoPE) and
// its lane exchanges, shared by the kernels that prepare rows.
#pragma once

#include "kfmi_device.h"
#include "kfmi_launch.h"

namespace kfmi {
namespace {

// Normalised element x*inv*gamma with the rounding points of a style.
template <int ST>
__device__ __forceinline__ float norm_elem(float x, float inv, float g) {
  if (ST == ST_HF) return round_bf16(round_bf16(x * inv) * g);  // rope:560-561
  if (ST == ST_LEGACY) return round_bf16(__fmul_rn(__fmul_rn(x, inv), g));  // rope:563
  return __fmul_rn(__fmul_rn(x, inv), g);  // FP32: rope:125, rope:298
}

// rotate-half output of one element: first half n*c - np*s, second half n*c + np*s.
template <int ST>
__device__ __forceinline__ float rope_elem(float n, float np, float c, float s, bool first) {
  if (ST == ST_FP32) {  // rope:129 / rope:164-167 (fp32=True): two products, one add
    // No contraction into an FMA: both products are rounded, then the sum
    // (HIP's __fmul_rn/__fadd_rn are plain * and + that the headers let the
    // compiler contract, so the operators are written here).
#pragma clang fp contract(off)
    const float p0 = n * c, p1 = np * s;
    return first ? p0 - p1 : p0 + p1;
  }
  float p0 = round_bf16(n * c), p1 = round_bf16(np * s);  // rope:578-579
  return first ? p0 - p1 : p0 + p1;  // rounded to BF16 at the store (rope:580-581)
}

template <int LPR>
__device__ __forceinline__ float row_sum(float x) {
  x = sum16(x);
  if constexpr (LPR == 32) x += __shfl_xor(x, 16);
  return x;
}

// 1 / sqrt(mean x^2 + eps) of a row of D values, 8 per lane.
template <int LPR, int D>
__device__ __forceinline__ float row_inv_rms(const float (&x)[8], float eps) {
  float ss = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) ss = __fmaf_rn(x[j], x[j], ss);
  ss = row_sum<LPR>(ss);
  return rsqrt_rn(ss * (1.0f / D) + eps);
}

// Normalised value held by the rotate-half partner lane (lane ^ LPR/2).
template <int LPR>
__device__ __forceinline__ float partner_f32(float x) {
  if constexpr (LPR == 16) return dpp_f32<DPP_ROW_ROR8>(x);
  else return __shfl_xor(x, LPR / 2);
}

}  // namespace
}  // namespace kfmi
