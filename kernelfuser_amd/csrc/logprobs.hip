// Log probabilities of given tokens, entropy and top alternatives of rows of
// logits (kfmi_token_logprobs).
//
// One pass over a row x: each lane keeps a running maximum m with
//   z = sum e^(x - m),  t = sum e^(x - m) (x - m)
// (rescaled when m grows: t' = a (t + (m - m') z), z' = a z, a = e^(m - m')),
// so that logp = x[id] - m - log z and the entropy is log z - t / z.  The
// alternatives are one sorted list per wave, entry i in lane i, of
// (value, index) as one whole number; a tile of logits is looked through only
// where its maximum exceeds the list's last entry, which a row of random logits
// does k log(V / k) times in all.  A list begins as the sorted maxima of the lanes'
// parts of the first tile.  -infinity never enters a list: what is missing at the end is
// filled with the lowest such indices.
//
// The bytes of the logits bound it; per bf16 logit there are also some eleven
// instruction slots (v_exp_f32 takes four), 12 bytes per cycle and CU, which
// is what the memory gives.
#include <cstdio>
#include <string>

#include "cache_common.h"
#include "kfmi_launch.h"

namespace kfmi {
namespace {

constexpr int LU = 4;          // 16-byte loads of a lane in flight
constexpr int MAX_SPLIT = 64;  // workgroups that share a row
constexpr int MAX_ROWS = KFMI_LOGPROBS_COUNTER_BYTES / 4;  // rows of a launch that splits them
constexpr int TOPM = KFMI_LOGPROBS_TOP_MAX;
constexpr float L2E = 1.44269504088896340736f;

// A workgroup's part of a split row.
struct Part {
  float m, z, t, unused;
  uint64_t keys[TOPM];
};

struct LogprobsParams {
  const void *logits, *ids;
  float *logprobs, *entropy, *top_logprobs;
  int64_t *top_ids;
  int *counters;
  Part *parts;
  int64_t ls[2], is[2];
  int64_t N1;
  int V, top, splits, vecs_per_split;  // 16-byte vectors of a row per workgroup
  bool ids64;
};

typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));

template <int TYPE>
constexpr int vec_of() { return TYPE == KFMI_LOGITS_F32 ? 4 : 8; }

template <int TYPE>
__device__ __forceinline__ float load_logit(const void *p, int64_t i) {
  if constexpr (TYPE == KFMI_LOGITS_F32) return reinterpret_cast<const float *>(p)[i];
  else if constexpr (TYPE == KFMI_LOGITS_BF16) return bf_lo((uint32_t) reinterpret_cast<const uint16_t *>(p)[i]);
  else return (float)reinterpret_cast<const _Float16 *>(p)[i];
}

template <int TYPE>
__device__ __forceinline__ void unpack(const u32x4_t &w, float *f) {
  if constexpr (TYPE == KFMI_LOGITS_F32) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(w[i]);
  } else if constexpr (TYPE == KFMI_LOGITS_BF16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = bf_lo(w[i]);
      f[2 * i + 1] = bf_hi(w[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f16x2_t h = __builtin_bit_cast(f16x2_t, (uint32_t)w[i]);
      f[2 * i] = (float)h[0];
      f[2 * i + 1] = (float)h[1];
    }
  }
}

// (value, index) in the order of the alternatives as one whole number: larger
// values first, then lower indices; 0 stands for none (-infinity, NaN).  -0 counts as 0.
__device__ __forceinline__ uint64_t rank_key(float x, uint32_t i) {
  uint32_t u = __float_as_uint(x + 0.0f);
  u = u & 0x80000000u ? ~u : u | 0x80000000u;
  return x > -INFINITY ? ((uint64_t)u << 32) | (uint32_t)~i : 0ull;
}
__device__ __forceinline__ float key_value(uint64_t key) {
  const uint32_t u = (uint32_t)(key >> 32);
  return key == 0 ? -INFINITY : __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ uint64_t lane_of(uint64_t x, int lane) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), lane) << 32 |
         (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)x, lane);
}

// A sorted list over the lanes of a wave, largest first; tau is entry top - 1.
struct TopList {
  uint64_t key, tau;

  // The lanes' keys in order.
  __device__ __forceinline__ void sort(uint64_t x, int lane, int top) {
    int r = 0;
#pragma unroll 8
    for (int i = 0; i < 64; ++i) {
      const uint64_t y = lane_of(x, i);
      r += y > x || (y == x && i < lane) ? 1 : 0;
    }
    const uint32_t lo = (uint32_t)__builtin_amdgcn_ds_permute(4 * r, (int)(uint32_t)x);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_ds_permute(4 * r, (int)(x >> 32));
    key = (uint64_t)hi << 32 | lo;
    tau = lane_of(key, top - 1);
  }

  // One candidate per lane (0: none); keys are unique.
  __device__ __forceinline__ void insert(uint64_t x, int lane, int top) {
    uint64_t todo = __ballot(x > tau);
    while (todo) {
      const int l = __builtin_ctzll(todo);
      const uint64_t c = lane_of(x, l);
      const int pos = __builtin_popcountll(__ballot(key > c));
      const uint32_t lo = (uint32_t)__shfl_up((int)(uint32_t)key, 1), hi = (uint32_t)__shfl_up((int)(key >> 32), 1);
      const uint64_t up = (uint64_t)hi << 32 | lo;
      key = lane < pos ? key : lane == pos ? c : up;
      tau = lane_of(key, top - 1);
      todo = __ballot(x > tau) & ~((2ull << l) - 1);
    }
  }
};

// Running maximum and sums of one lane, wave or workgroup.
struct Sums {
  float m, z, t;
  __device__ __forceinline__ void move(float to) {  // to >= m; to -infinity only from -infinity
    const float base = to == -INFINITY ? 0.f : to;
    const float dm = m == -INFINITY ? 0.f : fmaxf(m - base, -1e4f);  // finite, for the product with a = 0
    const float a = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(dm * L2E);
    t = a * fmaf(dm, z, t);
    z = a * z;
    m = to;
  }
  __device__ __forceinline__ void join(Sums o) {
    const float to = fmaxf(m, o.m);
    // a NaN in z or t (a row that is no distribution) goes through the sums
    Sums a = *this;
    a.move(to);
    o.move(to);
    m = to;
    z = a.z + o.z;
    t = a.t + o.t;
  }
};

template <int TYPE, bool TOP>
__global__ __launch_bounds__(256) void logprobs_kernel(LogprobsParams p) {
  constexpr int VEC = vec_of<TYPE>();
  constexpr int SIZE = 16 / VEC;
  constexpr int NE = LU * VEC;  // logits of a lane and tile
  __shared__ uint64_t keys[4 * TOPM];
  __shared__ float sums[4][3];
  __shared__ uint32_t arrived;
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int row = (int)(blockIdx.x / (uint32_t)p.splits), part = (int)(blockIdx.x % (uint32_t)p.splits);
  const int64_t n0 = row / p.N1, n1 = row - n0 * p.N1;
  const int64_t base = n0 * p.ls[0] + n1 * p.ls[1];
  const char *first = reinterpret_cast<const char *>(p.logits) + base * SIZE;
  // Vectors start at the 16-byte boundary at or before the row; logits outside the row are not read.
  const int head = (int)(reinterpret_cast<uintptr_t>(first) & 15u) / SIZE;
  const int vecs = (head + p.V + VEC - 1) / VEC;
  const int v0 = part * p.vecs_per_split;
  const int v1 = part == p.splits - 1 ? vecs : min(vecs, v0 + p.vecs_per_split);

  Sums s{-INFINITY, 0.f, 0.f};
  TopList list{0ull, 0ull};
  bool begun = false;
  for (int vt = v0 + w * (64 * LU); vt < v1; vt += 4 * 64 * LU) {
    float x[NE];
    u32x4_t raw[LU];
    const bool inner = vt * VEC >= head && (vt + 64 * LU) * VEC - head <= p.V && vt + 64 * LU <= v1;  // wave-uniform
    if (inner) {
#pragma unroll
      for (int u = 0; u < LU; ++u)
        raw[u] = __builtin_nontemporal_load(
            reinterpret_cast<const u32x4_t *>(first - head * SIZE + (int64_t)(vt + 64 * u + lane) * 16));
#pragma unroll
      for (int u = 0; u < LU; ++u) unpack<TYPE>(raw[u], x + u * VEC);
    } else {
#pragma unroll
      for (int u = 0; u < LU; ++u) {
        const int v = vt + 64 * u + lane, i0 = v * VEC - head;
        if (v < v1 && i0 >= 0 && i0 + VEC <= p.V) {
          unpack<TYPE>(*reinterpret_cast<const u32x4_t *>(first + (int64_t)i0 * SIZE), x + u * VEC);
        } else {
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const int i = i0 + e;
            x[u * VEC + e] = v < v1 && i >= 0 && i < p.V ? load_logit<TYPE>(first, i) : -INFINITY;
          }
        }
      }
    }
    float vm[LU], top = -INFINITY;
#pragma unroll
    for (int u = 0; u < LU; ++u) {
      vm[u] = x[u * VEC];
#pragma unroll
      for (int e = 1; e < VEC; ++e) vm[u] = fmaxf(vm[u], x[u * VEC + e]);
      top = fmaxf(top, vm[u]);
    }
    if (top > s.m) s.move(top);
    const float b = s.m == -INFINITY ? 0.f : s.m;
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      const float d = x[i] - b, e = __builtin_amdgcn_exp2f(d * L2E);
      s.z += e;
      s.t = fmaf(e, fmaxf(d, -1000.0f), s.t);  // e is 0 (or NaN) where this matters
    }
    if constexpr (TOP) {
      const uint32_t i0 = (uint32_t)((vt + lane) * VEC - head);  // index of x[0]
      if (!begun) {
        begun = true;
        // the lane's largest, the first of equals
        float best = x[0];
        int at = 0;
#pragma unroll
        for (int i = 1; i < NE; ++i) {
          const bool more = x[i] > best || !(best > -INFINITY);
          best = more ? x[i] : best;
          at = more ? i : at;
        }
        const uint32_t bi = i0 + (uint32_t)(at / VEC * 64 * VEC + at % VEC);
        list.sort(rank_key(best, bi), lane, p.top);
        const float tv = key_value(list.tau);
        if (__any(top >= tv && top > -INFINITY)) {
#pragma unroll
          for (int u = 0; u < LU; ++u) {
            if (!__any(vm[u] >= tv && vm[u] > -INFINITY)) continue;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
              const uint32_t i = i0 + (uint32_t)(u * 64 * VEC + e);
              const uint64_t key = i == bi ? 0ull : rank_key(x[u * VEC + e], i);
              list.insert(key, lane, p.top);
            }
          }
        }
      } else if (__any(top > key_value(list.tau))) {
#pragma unroll
        for (int u = 0; u < LU; ++u) {
          if (!__any(vm[u] > key_value(list.tau))) continue;
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const uint32_t i = i0 + (uint32_t)(u * 64 * VEC + e);
            if (__any(x[u * VEC + e] > key_value(list.tau))) list.insert(rank_key(x[u * VEC + e], i), lane, p.top);
          }
        }
      }
    }
  }

  auto join_waves = [&](Sums x) {  // x of the wave's lanes, then of the waves
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) x.join(Sums{__shfl_xor(x.m, o), __shfl_xor(x.z, o), __shfl_xor(x.t, o)});
    if (lane == 0) {
      sums[w][0] = x.m;
      sums[w][1] = x.z;
      sums[w][2] = x.t;
    }
    if (TOP && lane < p.top) keys[w * p.top + lane] = list.key;
    __syncthreads();
    x = Sums{sums[0][0], sums[0][1], sums[0][2]};
#pragma unroll
    for (int i = 1; i < 4; ++i) x.join(Sums{sums[i][0], sums[i][1], sums[i][2]});
    return x;
  };
  // This thread's key of the four lists and its place among them all.
  auto place = [&](uint64_t &key) {
    key = tid < 4 * p.top ? keys[tid] : 0ull;
    int r = 0;
    for (int i = 0; i < 4 * p.top; ++i) r += keys[i] > key ? 1 : 0;
    return r;
  };

  Sums all = join_waves(s);
  if (p.splits > 1) {
    // Parts are written and read with agent-coherent accesses and the last
    // workgroup of a row joins them, as in the decode kernel.
    Part *mine = p.parts + (int64_t)row * p.splits + part;
    if constexpr (TOP) {
      uint64_t key;
      const int r = place(key);
      if (key != 0 && r < p.top) __hip_atomic_store(&mine->keys[r], key, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      // places that no key takes: there are fewer keys than `top`
      const int have = __syncthreads_count(key != 0);
      if (tid >= have && tid < p.top) __hip_atomic_store(&mine->keys[tid], 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    if (tid == 0) {
      __hip_atomic_store(&mine->m, all.m, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      __hip_atomic_store(&mine->z, all.z, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      __hip_atomic_store(&mine->t, all.t, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (tid == 0)
      arrived = (uint32_t)__hip_atomic_fetch_add(p.counters + row, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (arrived != (uint32_t)p.splits - 1) return;
    const Part *parts = p.parts + (int64_t)row * p.splits;
    s = Sums{-INFINITY, 0.f, 0.f};
    if (w == 0 && lane < p.splits) {
      s.m = __hip_atomic_load(&parts[lane].m, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      s.z = __hip_atomic_load(&parts[lane].z, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      s.t = __hip_atomic_load(&parts[lane].t, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    if constexpr (TOP) {
      list = TopList{0ull, 0ull};
      const int n = p.splits * p.top;
      for (int i = w * 64; i < n; i += 256) {
        uint64_t key = 0;
        if (i + lane < n)
          key = __hip_atomic_load(&parts[(i + lane) / p.top].keys[(i + lane) % p.top], __ATOMIC_RELAXED,
                                  __HIP_MEMORY_SCOPE_AGENT);
        if (i == w * 64) list.sort(key, lane, p.top);
        else list.insert(key, lane, p.top);
      }
    }
    if (tid == 0) __hip_atomic_store(p.counters + row, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    all = join_waves(s);
  }

  const float nan = __uint_as_float(0x7fc00000u);
  const bool none = !(all.z > 0.f);  // NaN, +infinity or no logit above -infinity
  const float lse = logf(all.z);
  if (tid == 0) {
    const int64_t id = load_index(p.ids, p.ids64, n0 * p.is[0] + n1 * p.is[1]);
    const bool in = id >= 0 && id < p.V;
    p.logprobs[row] = none || !in ? nan : load_logit<TYPE>(first, in ? id : 0) - all.m - lse;
    p.entropy[row] = none ? nan : lse - all.t / all.z;
  }
  if constexpr (TOP) {
    uint64_t key;
    const int r = place(key);
    const int64_t out = (int64_t)row * p.top;
    const int have = __syncthreads_count(key != 0);
    if (none) {
      if (tid < p.top) {
        p.top_ids[out + tid] = -1;
        p.top_logprobs[out + tid] = nan;
      }
    } else {
      if (key != 0 && r < p.top) {
        p.top_ids[out + r] = (int64_t)(uint32_t)~(uint32_t)key;
        p.top_logprobs[out + r] = key_value(key) - all.m - lse;
      }
      if (w == 0) {  // the lowest indices of -infinity take the places left
        int at = have;
        for (int i = lane; at < p.top; i += 64) {
          const bool hit = i < p.V && load_logit<TYPE>(first, i < p.V ? i : 0) == -INFINITY;
          const uint64_t hits = __ballot(hit);
          const int to = at + __builtin_popcountll(hits & ((1ull << lane) - 1));
          if (hit && to < p.top) {
            p.top_ids[out + to] = i;
            p.top_logprobs[out + to] = -INFINITY;
          }
          at += __builtin_popcountll(hits);
          if (i - lane >= p.V) break;
        }
      }
    }
  }
}

// Workgroups per row: enough for four per CU, each with a tile per wave at least.
int splits_of(const kfmi_logprobs_args &a) {
  const int64_t rows = a.N0 * a.N1;
  if (rows > MAX_ROWS) return 1;
  const int64_t vec = a.logits_type == KFMI_LOGITS_F32 ? 4 : 8;
  const int64_t tiles = (a.V + vec * 64 * LU * 4 - 1) / (vec * 64 * LU * 4);
  int64_t n = (1024 + rows - 1) / rows;
  n = n < tiles ? n : tiles;
  return (int)(n < 1 ? 1 : n > MAX_SPLIT ? MAX_SPLIT : n);
}

template <int TYPE, bool TOP>
hipError_t launch_logprobs_t(const LogprobsParams &p, int64_t rows, hipStream_t stream) {
  const int64_t grid = rows * p.splits;
  hipLaunchKernelGGL((logprobs_kernel<TYPE, TOP>), dim3((unsigned)grid), dim3(256), 0, stream, p);
  static const std::string name = [] {
    char b[96];
    snprintf(b, sizeof(b), "logprobs_kernel<%d, %s>", TYPE, tf(TOP));
    return std::string(b);
  }();
  launch_log_add(reinterpret_cast<const void *>(&logprobs_kernel<TYPE, TOP>), name.c_str(), grid, 256);
  launch_log_plan("splits=%d", p.splits);
  return hipGetLastError();
}

template <int TYPE>
hipError_t dispatch_logprobs(const LogprobsParams &p, int64_t rows, hipStream_t stream) {
  return p.top > 0 ? launch_logprobs_t<TYPE, true>(p, rows, stream) : launch_logprobs_t<TYPE, false>(p, rows, stream);
}

}  // namespace

int64_t logprobs_workspace_bytes(const kfmi_logprobs_args &a) {
  const int n = splits_of(a);
  return n > 1 ? KFMI_LOGPROBS_COUNTER_BYTES + a.N0 * a.N1 * n * (int64_t)sizeof(Part) : 0;
}

hipError_t launch_logprobs(const kfmi_logprobs_args &a, hipStream_t stream) {
  LogprobsParams p{};
  p.logits = a.logits; p.ids = a.ids;
  p.logprobs = a.logprobs; p.entropy = a.entropy; p.top_logprobs = a.top_logprobs; p.top_ids = a.top_ids;
  for (int i = 0; i < 2; ++i) {
    p.ls[i] = a.logits_stride[i];
    p.is[i] = a.ids_stride[i];
  }
  p.N1 = a.N1;
  p.V = (int)a.V;
  p.top = a.top;
  p.ids64 = a.index_flags & KFMI_I64_IDS;
  p.splits = 1;
  const int64_t need = logprobs_workspace_bytes(a);
  if (need > 0 && a.work && a.work_bytes >= need) {
    p.splits = splits_of(a);
    p.counters = (int *)a.work;
    p.parts = (Part *)((char *)a.work + KFMI_LOGPROBS_COUNTER_BYTES);
  }
  // whole tiles of the four waves per workgroup (the last takes what the row's alignment adds)
  const int64_t vec = a.logits_type == KFMI_LOGITS_F32 ? 4 : 8, tile = 4 * 64 * LU;
  const int64_t vecs = (a.V + vec - 1) / vec;
  p.vecs_per_split = (int)(((vecs + p.splits - 1) / p.splits + tile - 1) / tile * tile);
  switch (a.logits_type) {
    case KFMI_LOGITS_F32: return dispatch_logprobs<KFMI_LOGITS_F32>(p, a.N0 * a.N1, stream);
    case KFMI_LOGITS_BF16: return dispatch_logprobs<KFMI_LOGITS_BF16>(p, a.N0 * a.N1, stream);
    case KFMI_LOGITS_F16: return dispatch_logprobs<KFMI_LOGITS_F16>(p, a.N0 * a.N1, stream);
  }
  return hipErrorInvalidValue;
}

}  // namespace kfmi
