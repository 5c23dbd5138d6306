// Device code shared by the kernels of the paged cache and of the row
// preparation: the rounding chains of norm and rotation, e4m3 rows and
// their scales, device-resident indices.
#pragma once

#include "kfmi_device.h"
#include "kfmi_launch.h"

namespace kfmi {
namespace {

inline int log2_of(int64_t n) {
  int s = 0;
  while (((int64_t)1 << s) < n) ++s;
  return s;
}

__device__ __forceinline__ int64_t load_index(const void *p, bool wide, int64_t i) {
  return wide ? reinterpret_cast<const int64_t *>(p)[i] : (int64_t) reinterpret_cast<const int32_t *>(p)[i];
}

// The same in two words (low, high) through the constant address space: a wave-uniform
// index becomes scalar loads, which do not wait for the vector loads in
// flight.  For memory that nothing writes while the kernel runs.
typedef const __attribute__((address_space(4))) int32_t const_i32_t;
__device__ __forceinline__ int2 load_index_words(const void *p, bool wide, int64_t i) {
  const_i32_t *w = (const_i32_t *)(reinterpret_cast<uintptr_t>(p));
  const int lo = w[wide ? 2 * i : i], hi = w[wide ? 2 * i + 1 : i];
  return int2{lo, wide ? hi : lo >> 31};
}

// E8M0: 2^(byte - 127), 255 is NaN.  2^-127 (byte 0) is a subnormal float.
__device__ __forceinline__ float scale_value(uint32_t byte) {
  const uint32_t bits = byte << 23;
  return __uint_as_float(byte == 0 ? 0x00400000u : byte == 255 ? 0x7fc00000u : bits);
}

// Eight e4m3 values (exact in float).
__device__ __forceinline__ void unpack_e4m3(const u32x2_t &w, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const f32x2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], false);
    const f32x2_t hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], true);
    f[4 * i] = lo[0];
    f[4 * i + 1] = lo[1];
    f[4 * i + 2] = hi[0];
    f[4 * i + 3] = hi[1];
  }
}

// Maximum over the LPR lanes of a row (16 or 32).
template <int LPR>
__device__ __forceinline__ uint32_t row_max_u32(uint32_t x) {
  x = max(x, dpp_u32<DPP_QUAD_XOR1>(x));
  x = max(x, dpp_u32<DPP_QUAD_XOR2>(x));
  x = max(x, dpp_u32<DPP_ROW_HALF_MIRROR>(x));
  x = max(x, dpp_u32<DPP_ROW_MIRROR>(x));
  if constexpr (LPR == 32) x = max(x, (uint32_t)__shfl_xor((int)x, 16));
  return x;
}

}  // namespace
}  // namespace kfmi
