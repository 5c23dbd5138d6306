// Log probabilities of given tokens, entropy and top alternatives of rows of
// logits (kfmi_token_logprobs).
//
// One pass over a row x: each lane keeps a running maximum m with
//   z = sum e^(x - m),  t = sum e^(x - m) (x - m)
// (rescaled when m grows: t' = a (t + (m - m') z), z' = a z, a = e^(m - m')),
// so that logp = x[id] - m - log z and the entropy is log z - t / z, the exponents in
// units of log 2, which is what v_exp_f32 takes.
//
// The alternatives are one sorted list per wave, entry i in lane i, of
// (value, index) as one whole number.  The top-th largest of the lanes' maxima is a bar below which nothing can
// belong; what a tile has above it is gathered in LDS and sorted into the list 64 at a time, which
// raises the bar: a row of random logits has k log(V / k) such values in all.  -infinity never
// enters a list: what is missing at the end is filled with the lowest such indices.
//
// The bytes of the logits bound it; per bf16 logit there are also some eleven
// instruction slots (v_exp_f32 takes four), 12 bytes per cycle and CU, which
// is what the memory gives: 4096 rows of 32000 in bf16 47 us (5.6 TB/s), with 20 alternatives 68.  64 rows of
// 131071 in 32 bits, mostly -infinity, with 20 alternatives: 15.7 us, of which the loads are 5, the launch and the
// join of a row's eight workgroups 6, the alternatives 4.
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
// Rows from which each is one wave's, a wave per SIMD: nothing is joined (4096 rows of 32000 in bf16 with one
// alternative 57 us, 71 with four waves a row).
constexpr int WAVE_ROWS = 1024;
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
  int V, top, rows, splits, vecs_per_split;  // 16-byte vectors of a row per workgroup
  int waves;                                 // of a row: 4, or 1 (never split)
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
__device__ __forceinline__ uint32_t value_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  return x > -INFINITY ? (u & 0x80000000u ? ~u : u | 0x80000000u) : 0u;
}
__device__ __forceinline__ uint64_t rank_key(float x, uint32_t i) {
  const uint32_t u = value_key(x);
  return u ? (uint64_t)u << 32 | (uint32_t)~i : 0ull;
}
__device__ __forceinline__ float key_value(uint32_t u) {
  return u == 0 ? -INFINITY : __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ float key_value(uint64_t key) { return key_value((uint32_t)(key >> 32)); }
__device__ __forceinline__ uint64_t lane_of(uint64_t x, int lane) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), lane) << 32 |
         (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)x, lane);
}

// The value of lane ^ M.
template <int M>
__device__ __forceinline__ uint32_t exchange32(uint32_t x, int lane) {
  if constexpr (M == 1) return dpp_u32<DPP_QUAD_XOR1>(x);
  else if constexpr (M == 2) return dpp_u32<DPP_QUAD_XOR2>(x);
  else if constexpr (M == 4) return dpp_u32<0x1B>(dpp_u32<DPP_ROW_HALF_MIRROR>(x));  // 7 - i, then 3 - i in each quad
  else if constexpr (M == 8) return dpp_u32<DPP_ROW_ROR8>(x);
  else if constexpr (M == 15) return dpp_u32<DPP_ROW_MIRROR>(x);
  else if constexpr (M == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    return lane & 16 ? r[0] : r[1];
  } else {
    const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return lane & 32 ? r[0] : r[1];
  }
}
template <int M>
__device__ __forceinline__ uint64_t exchange(uint64_t x, int lane) {
  return (uint64_t)exchange32<M>((uint32_t)(x >> 32), lane) << 32 | exchange32<M>((uint32_t)x, lane);
}

// One step of a bitonic network: lanes with `keep` take the larger of the two.
template <int M>
__device__ __forceinline__ uint64_t step(uint64_t x, int lane, bool keep) {
  const uint64_t y = exchange<M>(x, lane);
  return (x > y) == keep ? x : y;
}
template <int M>
__device__ __forceinline__ uint64_t steps(uint64_t x, int lane, bool up) {  // a bitonic run of 2 M lanes, sorted
  x = step<M>(x, lane, ((lane & M) == 0) != up);
  if constexpr (M > 1) x = steps<M / 2>(x, lane, up);
  return x;
}
// The 64 lanes' keys, smallest first.
__device__ __forceinline__ uint64_t sort_up(uint64_t x, int lane) {
  x = steps<1>(x, lane, (lane & 2) == 0);
  x = steps<2>(x, lane, (lane & 4) == 0);
  x = steps<4>(x, lane, (lane & 8) == 0);
  x = steps<8>(x, lane, (lane & 16) == 0);
  x = steps<16>(x, lane, (lane & 32) == 0);
  return steps<32>(x, lane, true);
}

// The top-th largest of the lanes' values (ordered as whole numbers).
template <int M>
__device__ __forceinline__ uint32_t steps32(uint32_t x, int lane, bool up) {
  const uint32_t y = exchange32<M>(x, lane);
  x = ((lane & M) == 0) != up ? max(x, y) : min(x, y);
  if constexpr (M > 1) x = steps32<M / 2>(x, lane, up);
  return x;
}
__device__ __forceinline__ uint32_t nth_largest(uint32_t x, int lane, int top) {
  x = steps32<1>(x, lane, (lane & 2) == 0);
  x = steps32<2>(x, lane, (lane & 4) == 0);
  x = steps32<4>(x, lane, (lane & 8) == 0);
  x = steps32<8>(x, lane, (lane & 16) == 0);
  x = steps32<16>(x, lane, (lane & 32) == 0);
  x = steps32<32>(x, lane, false);
  return (uint32_t)__builtin_amdgcn_readlane((int)x, top - 1);
}

// A sorted list over the lanes of a wave, largest first; tau is entry top - 1.
// Keys are unique, so the order in which they arrive does not matter.
struct TopList {
  uint64_t key, tau;

  // 64 more keys, smallest first.
  __device__ __forceinline__ void merge_up(uint64_t x, int lane, int top) {
    key = steps<32>(x > key ? x : key, lane, false);
    tau = lane_of(key, top - 1);
  }
  // Another list.
  __device__ __forceinline__ void merge(uint64_t x, int lane, int top) {
    if (lane_of(x, 0) <= tau) return;
    if (lane_of(key, 0) == 0) {
      key = x;
      tau = lane_of(x, top - 1);
      return;
    }
    merge_up(exchange<32>(exchange<16>(exchange<15>(x, lane), lane), lane), lane, top);
  }
  // One key per lane (0: none): a few are put in one by one, some 250 cycles each,
  // more by a sort, which takes as long as five of them.
  __device__ __forceinline__ void insert(uint64_t x, int lane, int top) {
    uint64_t todo = __ballot(x > tau);
    if (__builtin_popcountll(todo) > 5) {
      merge_up(sort_up(x, lane), lane, top);
      return;
    }
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

// max of three; a NaN among them is ignored (as by fmaxf, for which the compiler first
// makes each operand a quiet one: an instruction each).
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

// Over the lanes of a wave.
__device__ __forceinline__ float wave_max(float x, int lane) {
  auto with = [&](uint32_t y) { x = fmaxf(x, __uint_as_float(y)); };
  with(exchange32<1>(__float_as_uint(x), lane));
  with(exchange32<2>(__float_as_uint(x), lane));
  with(exchange32<4>(__float_as_uint(x), lane));
  with(exchange32<8>(__float_as_uint(x), lane));
  with(exchange32<16>(__float_as_uint(x), lane));
  with(exchange32<32>(__float_as_uint(x), lane));
  return x;
}
__device__ __forceinline__ float wave_sum(float x, int lane) {
  auto with = [&](uint32_t y) { x += __uint_as_float(y); };
  with(exchange32<1>(__float_as_uint(x), lane));
  with(exchange32<2>(__float_as_uint(x), lane));
  with(exchange32<4>(__float_as_uint(x), lane));
  with(exchange32<8>(__float_as_uint(x), lane));
  with(exchange32<16>(__float_as_uint(x), lane));
  with(exchange32<32>(__float_as_uint(x), lane));
  return x;
}

// A maximum that overflows in units of log 2 (a row of the type's lowest values, say).
__device__ __forceinline__ bool is_huge(float m) { return !(fabsf(m) <= 1e38f); }

// Running maximum m and sums of one lane, wave or workgroup:
// z = sum 2^d, t = sum 2^d d with d = fma(x, log2(e), -b), b = m log2(e) rounded,
// one instruction per logit; where b would overflow, d = (x - m) log2(e).
struct Sums {
  float m, z, t;
  __device__ __forceinline__ void move(float to) {  // to >= m; to -infinity only from -infinity
#pragma clang fp contract(off)  // both products are rounded, as b is
    // finite, for the product with a = 0; NaN (m and `to` are +infinity) meets a z that is NaN
    const float by = is_huge(to) ? (m - to) * L2E : m * L2E - to * L2E;
    const float dm = m == -INFINITY ? 0.f : fmaxf(by, -1e4f);
    const float a = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(dm);
    t = a * fmaf(dm, z, t);
    z = a * z;
    m = to;
  }
  __device__ __forceinline__ void over_lanes(int lane) {
    move(wave_max(m, lane));
    z = wave_sum(z, lane);
    t = wave_sum(t, lane);
  }
};

template <int TYPE, bool TOP>
__global__ __launch_bounds__(256) void logprobs_kernel(LogprobsParams p) {
  constexpr int VEC = vec_of<TYPE>();
  constexpr int SIZE = 16 / VEC;
  constexpr int NE = LU * VEC;  // logits of a lane and tile
  __shared__ uint64_t keys[4][TOPM], joined[TOPM];
  __shared__ uint64_t found[TOP ? 4 : 1][TOP ? 128 : 1];
  __shared__ float sums[4][3];
  __shared__ uint32_t arrived;
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const bool alone = p.waves == 1;  // a row is one wave's, and no wave meets another
  const int row = alone ? (int)blockIdx.x * 4 + w : (int)(blockIdx.x / (uint32_t)p.splits);
  const int part = alone ? 0 : (int)(blockIdx.x % (uint32_t)p.splits);
  if (alone && row >= p.rows) return;
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
  bool ruled_out = false;  // wave-uniform
  // Whether a tile lies within the row (wave-uniform), and its loads, which run while the
  // tile before it is summed.
  auto inner = [&](int vt) { return vt * VEC >= head && (vt + 64 * LU) * VEC - head <= p.V && vt + 64 * LU <= v1; };
  u32x4_t raw[LU];
  auto request = [&](int vt) {
#pragma unroll
    for (int u = 0; u < LU; ++u)
      raw[u] = __builtin_nontemporal_load(
          reinterpret_cast<const u32x4_t *>(first - head * SIZE + (int64_t)(vt + 64 * u + lane) * 16));
  };
  // What may belong to the list: values above the bar, gathered in LDS until there are more than 64.
  float bar = -INFINITY, seen = -INFINITY;
  int have = 0, tiles = 0, rank_at = 1;
  auto flush = [&] {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    for (int o = 0; o < have; o += 64) list.insert(o + lane < have ? found[w][o + lane] : 0ull, lane, p.top);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    have = 0;
    bar = fmaxf(bar, key_value(list.tau));
  };
  const int vt0 = v0 + (alone ? 0 : w) * (64 * LU), stride = p.waves * 64 * LU;
  bool requested = vt0 < v1 && inner(vt0);
  if (requested) request(vt0);
  for (int vt = vt0; vt < v1; vt += stride) {
    float x[NE];
    if (requested) {
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
    requested = vt + stride < v1 && inner(vt + stride);
    if (requested) request(vt + stride);
    float vm[LU], top = -INFINITY;
#pragma unroll
    for (int u = 0; u < LU; ++u) {
      vm[u] = max3(x[u * VEC], x[u * VEC + 1], x[u * VEC + 2]);
      if constexpr (VEC == 8) vm[u] = max3(max3(vm[u], x[u * VEC + 3], x[u * VEC + 4]), x[u * VEC + 5], x[u * VEC + 6]);
    }
#pragma unroll
    for (int u = 0; u < LU; ++u) {
      vm[u] = fmaxf(vm[u], x[u * VEC + VEC - 1]);
      top = fmaxf(top, vm[u]);
    }
    if (top > s.m) s.move(top);
    float b = s.m == -INFINITY ? 0.f : s.m * L2E;
    // 0 * -infinity is NaN: a wave that meets -infinity does the tile again and goes on with the exponents
    // held above -1000, which costs an instruction per logit.
    const bool huge = __any(is_huge(s.m) && s.m != -INFINITY);
    if (!ruled_out && !huge) {
      const Sums kept = s;
#pragma unroll
      for (int i = 0; i < NE; ++i) {
        const float d = fmaf(x[i], L2E, -b), e = __builtin_amdgcn_exp2f(d);
        s.z += e;
        s.t = fmaf(e, d, s.t);
      }
      ruled_out = __any(s.t != s.t);
      if (ruled_out) s = kept;
      else goto summed;
      // computed again, not kept: 64 registers
      asm volatile("" : "+v"(b));
    }
    if (!huge) {
#pragma unroll
      for (int i = 0; i < NE; ++i) {
        const float d = fmaf(x[i], L2E, -b), e = __builtin_amdgcn_exp2f(d);
        s.z += e;
        s.t = fmaf(e, fmaxf(d, -1000.0f), s.t);
      }
    } else {
#pragma unroll
      for (int i = 0; i < NE; ++i) {
        const float d = is_huge(s.m) && s.m != -INFINITY ? (x[i] - s.m) * L2E : fmaf(x[i], L2E, -b);
        const float e = __builtin_amdgcn_exp2f(d);
        s.z += e;
        s.t = fmaf(e, fmaxf(d, -1000.0f), s.t);
      }
    }
  summed:
    if constexpr (TOP) {
      const uint32_t i0 = (uint32_t)((vt + lane) * VEC - head);  // index of x[0]
      ++tiles;
      seen = fmaxf(seen, top);
      if (__any(top > bar)) {
        // The lanes' maxima of all tiles so far bound the top-th largest from below; they are
        // ranked again whenever the number of tiles has doubled.  What exceeds the bar is gathered in LDS and enters
        // the list 64 at a time.  A value equal to a bar that was there before this tile has `top`
        // others of lower indices before it; one equal to a bar that this tile raises may not.
        float above = bar;
        if (tiles >= rank_at) {
          const uint32_t to = nth_largest(value_key(seen), lane, p.top);
          rank_at = 2 * tiles;
          if (key_value(to) > bar) {
            bar = key_value(to);
            above = key_value(to - (to == 0x80000000u ? 2 : 1));  // the next lower number
          }
        }
        uint32_t mine = 0;  // this lane's
#pragma unroll
        for (int e = NE - 1; e >= 0; --e) mine = mine << 1 | (x[e] > above ? 1u : 0u);
        for (;;) {  // one of each lane
          const uint64_t who = __ballot(mine != 0);
          if (!who) break;
          if (have > 64) flush();
          const int e = mine ? __builtin_ctz(mine) : 0;
          uint32_t y[NE];  // x[e], bit by bit of e
#pragma unroll
          for (int k = 0; k < NE; ++k) y[k] = __float_as_uint(x[k]);
#pragma unroll
          for (int o = 1; o < NE; o *= 2) {
            const uint32_t m = e & o ? ~0u : 0u;
#pragma unroll
            for (int k = 0; k < NE; k += 2 * o) y[k] = (y[k + o] & m) | (y[k] & ~m);
          }
          if (mine)
            found[w][have + __builtin_popcountll(who & ((1ull << lane) - 1))] =
                rank_key(__uint_as_float(y[0]), i0 + (uint32_t)(e / VEC * (64 * VEC) + e % VEC));
          have += __builtin_popcountll(who);
          mine &= mine - 1;
        }
      }
    }
  }
  if constexpr (TOP) {
    if (have > 0) flush();
  }

  // The lanes' sums and lists of all waves, in the first wave (lists: each wave's in LDS).
  auto join_waves = [&](Sums x) {
    x.over_lanes(lane);
    if (alone) return x;
    if (lane == 0) {
      sums[w][0] = x.m;
      sums[w][1] = x.z;
      sums[w][2] = x.t;
    }
    if (TOP && lane < p.top) keys[w][lane] = list.key;
    if (TOP && tid < TOPM) joined[tid] = 0ull;
    __syncthreads();
    if (w == 0) {
      const float top = fmaxf(fmaxf(sums[0][0], sums[1][0]), fmaxf(sums[2][0], sums[3][0]));
      float z = 0.f, t = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        Sums y{sums[i][0], sums[i][1], sums[i][2]};
        y.move(top);
        z += y.z;
        t += y.t;
      }
      x = Sums{top, z, t};
    }
    return x;
  };
  // The waves' lists as one, in the first wave: a key's place is the number of larger ones in
  // all four sorted lists, found by halving.
  auto join_lists = [&] {
    if (!TOP || alone) return;
    const uint32_t top = (uint32_t)p.top;
    uint32_t larger[3] = {0, 0, 0};
    for (uint32_t o = 1u << (31 - __builtin_clz(top)); o > 0; o /= 2) {
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        const uint32_t at = larger[i] + o;
        larger[i] = (keys[(w + i + 1) & 3][min(at, top) - 1] > list.key) & (at <= top) ? at : larger[i];
      }
    }
    const uint32_t place = (uint32_t)lane + larger[0] + larger[1] + larger[2];
    if (list.key != 0 && place < top) joined[place] = list.key;
    __syncthreads();
    if (w == 0) list.key = lane < p.top ? joined[lane] : 0ull;
  };

  Sums all = join_waves(s);
  if (p.splits > 1) {
    // Parts are written and read with agent-coherent accesses and the last
    // workgroup of a row joins them, as in the decode kernel.
    Part *mine = p.parts + (int64_t)row * p.splits + part;
    join_lists();
    if (TOP && tid < p.top) __hip_atomic_store(&mine->keys[tid], list.key, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
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
      for (int i = w; i < p.splits; i += 16) {  // four lists on their way at once
        uint64_t part_keys[4];
#pragma unroll
        for (int q = 0; q < 4; ++q)
          part_keys[q] = lane < p.top && i + 4 * q < p.splits
                             ? __hip_atomic_load(&parts[i + 4 * q].keys[lane], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)
                             : 0ull;
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (i + 4 * q < p.splits) list.merge(part_keys[q], lane, p.top);
      }
    }
    if (tid == 0) __hip_atomic_store(p.counters + row, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    all = join_waves(s);
  }

  join_lists();
  if (w != 0 && !alone) return;
  constexpr float LN2 = 0.693147180559945309417f;
  const float nan = __uint_as_float(0x7fc00000u);
  const bool none = !(all.z > 0.f);  // NaN, +infinity or no logit above -infinity
  const float lz = log2f(all.z);
  // log2 of the sum relative to m itself: b's rounding goes back in
  const float lm = is_huge(all.m) ? lz : lz - fmaf(all.m, L2E, -(all.m * L2E));
  auto logp = [&](float x) { return x - all.m - lm * LN2; };
  if (lane == 0) {
    const int64_t id = load_index(p.ids, p.ids64, n0 * p.is[0] + n1 * p.is[1]);
    const bool in = id >= 0 && id < p.V;
    p.logprobs[row] = none || !in ? nan : logp(load_logit<TYPE>(first, in ? id : 0));
    p.entropy[row] = none ? nan : (lz - all.t / all.z) * LN2;
  }
  if constexpr (TOP) {
    const int64_t out = (int64_t)row * p.top;
    if (none) {
      if (lane < p.top) {
        p.top_ids[out + lane] = -1;
        p.top_logprobs[out + lane] = nan;
      }
      return;
    }
    if (lane < p.top && list.key != 0) {
      p.top_ids[out + lane] = (int64_t)(uint32_t)~(uint32_t)list.key;
      p.top_logprobs[out + lane] = logp(key_value(list.key));
    }
    // the lowest indices of -infinity take the places left
    int at = __builtin_popcountll(__ballot(list.key != 0));
    for (int i0 = 0; at < p.top && i0 < p.V; i0 += 64) {
      const int i = i0 + lane;
      const bool hit = i < p.V && load_logit<TYPE>(first, i < p.V ? i : 0) == -INFINITY;
      const uint64_t hits = __ballot(hit);
      const int to = at + __builtin_popcountll(hits & ((1ull << lane) - 1));
      if (hit && to < p.top) {
        p.top_ids[out + to] = i;
        p.top_logprobs[out + to] = -INFINITY;
      }
      at += __builtin_popcountll(hits);
    }
  }
}

// Workgroups per row: two per CU, each with a tile per wave at least (64 rows of 131071 in 32 bits:
// 11.7 us; with four per CU 13.8, with one 14.5).
int splits_of(const kfmi_logprobs_args &a) {
  const int64_t rows = a.N0 * a.N1;
  if (rows > MAX_ROWS) return 1;
  const int64_t vec = a.logits_type == KFMI_LOGITS_F32 ? 4 : 8;
  const int64_t tiles = (a.V + vec * 64 * LU * 4 - 1) / (vec * 64 * LU * 4);
  int64_t n = (512 + rows - 1) / rows;
  n = n < tiles ? n : tiles;
  return (int)(n < 1 ? 1 : n > MAX_SPLIT ? MAX_SPLIT : n);
}

template <int TYPE, bool TOP>
hipError_t launch_logprobs_t(const LogprobsParams &p, int64_t rows, hipStream_t stream) {
  const int64_t grid = p.waves == 1 ? (rows + 3) / 4 : rows * p.splits;
  hipLaunchKernelGGL((logprobs_kernel<TYPE, TOP>), dim3((unsigned)grid), dim3(256), 0, stream, p);
  static const std::string name = [] {
    char b[96];
    snprintf(b, sizeof(b), "logprobs_kernel<%d, %s>", TYPE, tf(TOP));
    return std::string(b);
  }();
  launch_log_add(reinterpret_cast<const void *>(&logprobs_kernel<TYPE, TOP>), name.c_str(), grid, 256);
  launch_log_plan("splits=%d waves=%d", p.splits, p.waves);
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
  p.rows = (int)(a.N0 * a.N1);
  p.splits = 1;
  p.waves = p.rows >= WAVE_ROWS ? 1 : 4;
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
