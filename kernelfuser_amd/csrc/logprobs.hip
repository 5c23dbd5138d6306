// Log probabilities of given tokens, entropy and top alternatives of rows of
// logits.
#include <hip/hip_fp16.h>

#include <cstdio>
#include <string>

#include "cache_common.h"
#include "kfmi_launch.h"

namespace kfmi {
namespace {

struct LogprobsParams {
  const void *logits, *ids;
  float *logprobs, *entropy, *top_logprobs;
  int64_t *top_ids;
  int64_t ls[2], is[2];
  int64_t N1, V;
  int top;
  bool ids64;
};

template <int TYPE>
__device__ __forceinline__ float load_logit(const void *p, int64_t i) {
  if constexpr (TYPE == KFMI_LOGITS_F32) return reinterpret_cast<const float *>(p)[i];
  else if constexpr (TYPE == KFMI_LOGITS_BF16) return bf_lo((uint32_t) reinterpret_cast<const uint16_t *>(p)[i]);
  else return __half2float(reinterpret_cast<const __half *>(p)[i]);
}

// (value, index) in the order of the alternatives as one whole number: larger
// values first, then lower indices.  -0 counts as 0.
__device__ __forceinline__ uint64_t rank_key(float x, uint32_t i) {
  uint32_t u = __float_as_uint(x + 0.0f);
  u = u & 0x80000000u ? ~u : u | 0x80000000u;
  return ((uint64_t)u << 32) | (uint32_t)~i;
}
__device__ __forceinline__ float key_value(uint64_t key) {
  const uint32_t u = (uint32_t)(key >> 32);
  return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}

// One row per workgroup: maximum, then sums, then one round per alternative.
template <int TYPE>
__global__ __launch_bounds__(256) void logprobs_kernel(LogprobsParams p) {
  __shared__ float red[2][4];
  __shared__ uint64_t best[4];
  const int tid = threadIdx.x, w = tid >> 6;
  const int64_t row = blockIdx.x;
  const int64_t n0 = row / p.N1, n1 = row - n0 * p.N1;
  const int64_t base = n0 * p.ls[0] + n1 * p.ls[1];
  float m = -INFINITY;
  for (int64_t i = tid; i < p.V; i += 256) m = fmaxf(m, load_logit<TYPE>(p.logits, base + i));
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
  if ((tid & 63) == 0) red[0][w] = m;
  __syncthreads();
  m = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
  __syncthreads();
  float z = 0.f, t = 0.f;
  for (int64_t i = tid; i < p.V; i += 256) {
    const float d = load_logit<TYPE>(p.logits, base + i) - m, e = expf(d);
    z += e;
    t += e * fmaxf(d, -1000.f);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    z += __shfl_xor(z, o);
    t += __shfl_xor(t, o);
  }
  if ((tid & 63) == 0) {
    red[0][w] = z;
    red[1][w] = t;
  }
  __syncthreads();
  z = (red[0][0] + red[0][1]) + (red[0][2] + red[0][3]);
  t = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
  const float nan = __uint_as_float(0x7fc00000u);
  const bool none = !(z >= 1.0f);  // NaN, +infinity or no finite logit
  const float lse = logf(z);
  if (tid == 0) {
    const int64_t id = load_index(p.ids, p.ids64, n0 * p.is[0] + n1 * p.is[1]);
    const bool in = id >= 0 && id < p.V;
    p.logprobs[row] = none || !in ? nan : load_logit<TYPE>(p.logits, base + (in ? id : 0)) - m - lse;
    p.entropy[row] = none ? nan : lse - t / z;
  }
  uint64_t last = ~0ull;
  for (int k = 0; k < p.top; ++k) {
    uint64_t mine = 0;
    if (!none) {
      for (int64_t i = tid; i < p.V; i += 256) {
        const uint64_t key = rank_key(load_logit<TYPE>(p.logits, base + i), (uint32_t)i);
        if (key < last && key > mine) mine = key;
      }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const uint64_t other = __shfl_xor((unsigned long long)mine, o);
      mine = other > mine ? other : mine;
    }
    __syncthreads();
    if ((tid & 63) == 0) best[w] = mine;
    __syncthreads();
    last = best[0];
    for (int i = 1; i < 4; ++i) last = best[i] > last ? best[i] : last;
    if (tid == 0) {
      p.top_ids[row * p.top + k] = none ? -1 : (int64_t)(uint32_t)~(uint32_t)last;
      p.top_logprobs[row * p.top + k] = none ? nan : key_value(last) - m - lse;
    }
  }
}

template <int TYPE>
hipError_t launch_logprobs_t(const LogprobsParams &p, int64_t rows, hipStream_t stream) {
  hipLaunchKernelGGL((logprobs_kernel<TYPE>), dim3((unsigned)rows), dim3(256), 0, stream, p);
  static const std::string name = [] {
    char b[96];
    snprintf(b, sizeof(b), "logprobs_kernel<%d>", TYPE);
    return std::string(b);
  }();
  launch_log_add(reinterpret_cast<const void *>(&logprobs_kernel<TYPE>), name.c_str(), rows, 256);
  return hipGetLastError();
}

}  // namespace

int64_t logprobs_workspace_bytes(const kfmi_logprobs_args &) { return 0; }

hipError_t launch_logprobs(const kfmi_logprobs_args &a, hipStream_t stream) {
  LogprobsParams p{};
  p.logits = a.logits; p.ids = a.ids;
  p.logprobs = a.logprobs; p.entropy = a.entropy; p.top_logprobs = a.top_logprobs; p.top_ids = a.top_ids;
  for (int i = 0; i < 2; ++i) {
    p.ls[i] = a.logits_stride[i];
    p.is[i] = a.ids_stride[i];
  }
  p.N1 = a.N1; p.V = a.V;
  p.top = a.top;
  p.ids64 = a.index_flags & KFMI_I64_IDS;
  switch (a.logits_type) {
    case KFMI_LOGITS_F32: return launch_logprobs_t<KFMI_LOGITS_F32>(p, a.N0 * a.N1, stream);
    case KFMI_LOGITS_BF16: return launch_logprobs_t<KFMI_LOGITS_BF16>(p, a.N0 * a.N1, stream);
    case KFMI_LOGITS_F16: return launch_logprobs_t<KFMI_LOGITS_F16>(p, a.N0 * a.N1, stream);
  }
  return hipErrorInvalidValue;
}

}  // namespace kfmi
