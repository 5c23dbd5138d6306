// Attention of the last few tokens of each sequence over its paged cache.
#include <cstdio>
#include <string>

#include "cache_common.h"
#include "kfmi_launch.h"

namespace kfmi {
namespace {

struct DecodeParams {
  const uint16_t *q;
  const char *k_cache, *v_cache;
  const uint8_t *k_scale, *v_scale;
  const void *pages, *lengths;
  uint16_t *out;
  int64_t qs[3], cs[3], es[2];
  int64_t pages_stride, lengths_stride, num_pages, capacity, window;
  int hq, hk, S;
  int page_shift, page_mask;
  bool pages64, len64;
  float scale, softcap, inv_softcap;
};

__device__ __forceinline__ float block_reduce(float x, bool max_, float *lds) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const float y = __shfl_xor(x, o);
    x = max_ ? fmaxf(x, y) : x + y;
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
  __syncthreads();
  return max_ ? fmaxf(fmaxf(lds[0], lds[1]), fmaxf(lds[2], lds[3])) : (lds[0] + lds[1]) + (lds[2] + lds[3]);
}

template <bool FP8>
__device__ __forceinline__ void load8(const char *p, float (&f)[8]) {
  if constexpr (FP8) unpack_e4m3(*reinterpret_cast<const u32x2_t *>(p), f);
  else unpack8(ld16(reinterpret_cast<const uint16_t *>(p)), f);
}

// One query of one head per workgroup; 256 keys at a time with the running
// maximum and sum of the softmax.  Only visible keys are read.
template <int D, bool FP8>
__global__ __launch_bounds__(256) void decode_kernel(DecodeParams p) {
  __shared__ float qf[D], pr[256], red[4], part[256];
  __shared__ int64_t rowoff[256];
  constexpr int ES = FP8 ? 1 : 2;
  const int tid = threadIdx.x;
  const int i = blockIdx.x % p.S, h = blockIdx.x / p.S;
  const int64_t b = blockIdx.y;
  const int hk = h / (p.hq / p.hk);
  const int64_t len = load_index(p.lengths, p.len64, b * p.lengths_stride);
  const bool bad_len = len < 0 || len > p.capacity;
  const int64_t t = bad_len ? -1 : len - p.S + i;
  const int64_t lo = p.window > 0 && t - p.window + 1 > 0 ? t - p.window + 1 : 0;
  for (int d = tid; d < D; d += 256)
    qf[d] = bf_lo((uint32_t)p.q[b * p.qs[0] + h * p.qs[1] + i * p.qs[2] + d]);
  __syncthreads();
  const int d = tid % D, part_of = tid / D;
  float m = -INFINITY, l = 0.f, acc = 0.f;
  bool bad = bad_len;
  for (int64_t j0 = lo; j0 <= t; j0 += 256) {
    const int n = t + 1 - j0 < 256 ? (int)(t + 1 - j0) : 256;
    float s = -INFINITY;
    bool bad_page = false;
    if (tid < n) {
      const int64_t j = j0 + tid;
      int64_t page = load_index(p.pages, p.pages64, b * p.pages_stride + (j >> p.page_shift));
      bad_page = page < 0 || page >= p.num_pages;
      if (bad_page) page = 0;
      const int64_t at = j & p.page_mask;
      const int64_t off = page * p.cs[0] + hk * p.cs[1] + at * p.cs[2];
      rowoff[tid] = off;
      float dot = 0.f;
      for (int c = 0; c < D; c += 8) {
        float f[8];
        load8<FP8>(p.k_cache + (off + c) * ES, f);
#pragma unroll
        for (int e = 0; e < 8; ++e) dot = fmaf(f[e], qf[c + e], dot);
      }
      if (FP8) dot *= scale_value(p.k_scale[page * p.es[0] + hk * p.es[1] + at]);
      s = dot * p.scale;
      if (p.softcap > 0.f) s = p.softcap * tanhf(s * p.inv_softcap);
    }
    bad |= __syncthreads_or(bad_page);
    const float mt = fmaxf(m, block_reduce(s, true, red));
    const float base = mt == -INFINITY ? 0.f : mt;
    float e = tid < n ? expf(s - base) : 0.f;
    const float alpha = expf(m - base);
    l = l * alpha + block_reduce(e, false, red);
    m = mt;
    if (FP8 && tid < n) {
      const int64_t j = j0 + tid;
      int64_t page = load_index(p.pages, p.pages64, b * p.pages_stride + (j >> p.page_shift));
      if (page < 0 || page >= p.num_pages) page = 0;
      e *= scale_value(p.v_scale[page * p.es[0] + hk * p.es[1] + (j & p.page_mask)]);
    }
    pr[tid] = e;
    __syncthreads();
    acc *= alpha;
    for (int k = part_of; k < n; k += 256 / D) {
      const char *row = p.v_cache + (rowoff[k] + d) * ES;
      const float v = FP8 ? __builtin_amdgcn_cvt_f32_fp8((int)*reinterpret_cast<const uint8_t *>(row), 0)
                          : bf_lo((uint32_t)*reinterpret_cast<const uint16_t *>(row));
      acc = fmaf(pr[k], v, acc);
    }
    __syncthreads();
  }
  part[tid] = acc;
  __syncthreads();
  if (tid < D) {
    float o = part[tid];
    if (D == 128) o += part[(tid + 128) & 255];
    o = bad ? __uint_as_float(0x7fc00000u) : t < lo ? 0.f : o / l;
    p.out[((b * p.hq + h) * p.S + i) * D + tid] = (uint16_t)(pack_bf16x2(o, 0.f) & 0xffffu);
  }
}

template <int D, bool FP8>
hipError_t launch_decode_t(const DecodeParams &p, int64_t B, hipStream_t stream) {
  const dim3 grid((unsigned)(p.hq * p.S), (unsigned)B);
  hipLaunchKernelGGL((decode_kernel<D, FP8>), grid, dim3(256), 0, stream, p);
  static const std::string name = [] {
    char b[96];
    snprintf(b, sizeof(b), "decode_kernel<%d, %s>", D, tf(FP8));
    return std::string(b);
  }();
  launch_log_add(reinterpret_cast<const void *>(&decode_kernel<D, FP8>), name.c_str(), (int64_t)grid.x * grid.y, 256);
  return hipGetLastError();
}

}  // namespace

int64_t decode_workspace_bytes(const kfmi_decode_args &) { return 0; }

hipError_t launch_decode(const kfmi_decode_args &a, hipStream_t stream) {
  DecodeParams p{};
  p.q = (const uint16_t *)a.q;
  p.k_cache = (const char *)a.k_cache; p.v_cache = (const char *)a.v_cache;
  p.k_scale = (const uint8_t *)a.k_scale; p.v_scale = (const uint8_t *)a.v_scale;
  p.pages = a.pages; p.lengths = a.lengths;
  p.out = (uint16_t *)a.out;
  for (int i = 0; i < 3; ++i) {
    p.qs[i] = a.q_stride[i];
    p.cs[i] = a.cache_stride[i];
  }
  for (int i = 0; i < 2; ++i) p.es[i] = a.scale_stride[i];
  p.pages_stride = a.pages_stride; p.lengths_stride = a.lengths_stride;
  p.num_pages = a.num_pages;
  p.capacity = a.max_pages * a.page_size;
  p.window = a.window;
  p.hq = (int)a.Hq; p.hk = (int)a.Hkv; p.S = (int)a.S;
  p.page_shift = log2_of(a.page_size);
  p.page_mask = (int)(a.page_size - 1);
  p.pages64 = a.index_flags & KFMI_I64_PAGES;
  p.len64 = a.index_flags & KFMI_I64_LENGTHS;
  p.scale = (float)a.scale;
  p.softcap = (float)a.softcap;
  p.inv_softcap = a.softcap > 0 ? (float)(1.0 / a.softcap) : 0.f;
  const bool fp8 = a.cache_type == KFMI_CACHE_E4M3;
  if (a.D == 128) return fp8 ? launch_decode_t<128, true>(p, a.B, stream) : launch_decode_t<128, false>(p, a.B, stream);
  return fp8 ? launch_decode_t<256, true>(p, a.B, stream) : launch_decode_t<256, false>(p, a.B, stream);
}

}  // namespace kfmi
