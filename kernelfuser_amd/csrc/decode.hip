// Attention of the last few tokens of each sequence over its paged cache
// (kfmi_attention_decode_bf16).
//
// out_i = sum_j softmax_j(cap(q_i . k_j * scale)) v_j over the keys that
// query i sees.  Every key and value is read once per KV head, so the cache's bytes
// bound the call: 4 * D * 2 bytes (bf16) per key and head against 4 * D * R flops for the R = group * S query rows
// that share them, at most 64 rows a pass.  The design:
//
//  * the R rows of a KV head are the columns of 16x16x32 matrix
//    instructions: S^T = K Q^T with 16 keys, O^T = V^T P^T with 16 values of d.
//    K rows go from memory to registers as they lie (a lane's 16 bytes are its eight k's).  A
//    lane of S^T holds the weights of keys 4c..4c+3 (c = lane / 16) of two
//    16-key groups for one row, which is its part of the second product's operand if the 32
//    keys of a step are numbered so; V is then loaded so that a lane has 8
//    consecutive d of those eight keys (coalesced rows) and turned by 32 v_perm per
//    32 keys.  Nothing goes through LDS in the loop, no wave waits for another;
//  * a weight is the sum of two bf16 numbers, two products each: its rounding to one
//    would be as large as the result's own (2^-9), and the matrix
//    units have time for it;
//  * the work of a launch (units of 32 keys per wave, all heads and sequences)
//    is dealt evenly to one round of workgroups, whatever the lengths: each
//    finds its share by a scan of the lengths.  A head's sequence that
//    crosses a border is joined, in order, by the workgroup that arrives last.
#include <cstdio>
#include <string>

#include "cache_common.h"
#include "kfmi_launch.h"

namespace kfmi {
namespace {

constexpr int WV = 4;            // waves per workgroup
constexpr int NTHR = 64 * WV;
constexpr int UNIT = 32 * WV;    // keys per unit of work
constexpr int SC1 = 16;          // cache policy of agent-coherent accesses
constexpr float LOG2E = 1.44269504088896340736f;

struct DecodeParams {
  const uint16_t *q;
  const char *k_cache, *v_cache;
  const uint8_t *k_scale, *v_scale;
  const void *pages, *lengths;
  uint16_t *out;
  int *counters;    // NULL: no workspace, no sequence is split
  float *partials;  // 2 slots per workgroup
  int64_t qs[3], cs[3], es[2];
  int64_t pages_stride, lengths_stride, num_pages;
  int B, hq, hk, S, group, rows, rblocks;  // rows = group * S, in blocks of 16 * NT
  int capacity, window, min_units;
  int page_shift, page_mask;
  bool pages64, len64;
  float scale, softcap;  // softcap 0: none
};

// What a launch reads of one sequence.
struct Sequence {
  int len;    // 0 where the given one is wrong
  int start;  // first key of the first unit: below every key that a query sees, a multiple of 32
  int units;
  bool bad;
};

__device__ __forceinline__ Sequence sequence(const DecodeParams &p, int b) {
  Sequence s;
  const int64_t len = load_index(p.lengths, p.len64, (int64_t)b * p.lengths_stride);
  s.bad = len < 0 || len > p.capacity;
  s.len = s.bad ? 0 : (int)len;
  const int lo = p.window > 0 ? max(0, s.len - p.S - p.window + 1) : 0;
  s.start = lo & ~31;
  s.units = max(1, (s.len - s.start + UNIT - 1) / UNIT);
  return s;
}

__device__ __forceinline__ float max_rows4(float x) {  // over lanes l, l^16, l^32, l^48
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  return max_halves(x);
}
__device__ __forceinline__ float sum_rows4(float x) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  return sum_halves(x);
}

__device__ __forceinline__ f32x4_t mfma(const u32x4_t &a, const u32x4_t &b, const f32x4_t &c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0,
                                                 0, 0);
}

__device__ __forceinline__ uint32_t bf16_of_e4m3(uint32_t w, bool high) {
  return __builtin_bit_cast(uint32_t, high ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w, 1.0f, true)
                                           : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w, 1.0f, false));
}

// The d that element (m, t) of O^T is: lane group m of V's loads, product t.
template <int D, bool FP8>
__device__ __forceinline__ int d_of(int m, int x) {  // of t = 8 * x
  return FP8 && D == 256 ? 16 * m + 8 * x : 128 * x + 8 * m;
}

// V of 32 keys: v[j] is 8 (or 16) values of d of one key; the operand of product
// t takes d t of all eight keys.
template <int D, bool FP8>
struct VTile {
  static constexpr int W = FP8 ? D / 64 : D / 32;  // dwords per key and lane
  uint32_t w[8][W];
  __device__ __forceinline__ u32x4_t operand(int t) const {
    u32x4_t r;
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      if constexpr (FP8) {
        const uint32_t a = w[2 * y][t / 4], b = w[2 * y + 1][t / 4];
        const uint32_t pair = __builtin_amdgcn_perm(b, a, t & 2 ? 0x07030602u : 0x05010400u);
        r[y] = bf16_of_e4m3(pair, t & 1);
      } else {
        r[y] = __builtin_amdgcn_perm(w[2 * y + 1][t / 2], w[2 * y][t / 2], t & 1 ? 0x07060302u : 0x05040100u);
      }
    }
    return r;
  }
  // Whether a value of key j is an infinity or NaN.
  __device__ __forceinline__ bool odd(int j) const {
    bool any = false;
#pragma unroll
    for (int x = 0; x < W; ++x) {
      const uint32_t u = w[j][x];
      if constexpr (FP8) {
#pragma unroll
        for (int e = 0; e < 4; ++e) any |= ((u >> (8 * e)) & 0x7fu) == 0x7fu;
      } else {
        any |= (u & 0x7f80u) == 0x7f80u || (u & 0x7f800000u) == 0x7f800000u;
      }
    }
    return any;
  }
};

// MULTI: S > 1.
template <int D, bool FP8, int NT, bool MULTI>
__global__ __launch_bounds__(NTHR, NT * D <= 256 ? 2 : 1) void decode_kernel(DecodeParams p) {
  constexpr int NK = D / 32;    // matrix steps of q . k
  constexpr int ND = D / 16;    // products of P V
  constexpr int NX = ND / 8;
  constexpr int ES = FP8 ? 1 : 2;
  constexpr int ROWS = 16 * NT;
  constexpr int SLOT = ROWS * (D + 2);  // floats: O row by row, then (m, l) of each row
  constexpr int LDX = 36;               // floats per row of the exchange (32 and padding)
  constexpr int MG = NTHR / (D / 8);    // groups of the join
  constexpr int EX = WV * ROWS * LDX > MG * 4 * D ? WV * ROWS * LDX : MG * 4 * D;
  __shared__ __attribute__((aligned(16))) float ex[EX];
  __shared__ float ml[(WV * ROWS > MG * 4 ? WV * ROWS : MG * 4) * 2];
  __shared__ uint32_t plan[WV + 3];
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, c = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const bool split = p.counters != nullptr;
  const uint32_t ipb = (uint32_t)(p.hk * p.rblocks);  // items (head, block of rows) per sequence

  // This workgroup's share [g0, g1) of all units: sequences in the order
  // 0, NTHR, 2 NTHR, .., 1, NTHR + 1, .. (thread by thread).
  uint32_t mine = 0;
  for (int b = tid; b < p.B; b += NTHR) mine += (split ? (uint32_t)sequence(p, b).units : 1u) * ipb;
  uint32_t incl = mine;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t y = (uint32_t)__shfl_up((int)incl, o);
    if (lane >= o) incl += y;
  }
  if (lane == 63) plan[w] = incl;
  __syncthreads();
  uint32_t total = 0, before = 0;
#pragma unroll
  for (int i = 0; i < WV; ++i) {
    if (i < w) before += plan[i];
    total += plan[i];
  }
  incl += before;
  const uint32_t per = max((total + gridDim.x - 1) / gridDim.x, (uint32_t)p.min_units);
  const uint32_t g0 = blockIdx.x * per, g1 = min(g0 + per, total);
  if (g0 >= total) return;  // workgroup-uniform
  if (incl - mine <= g0 && g0 < incl) {
    uint32_t rem = g0 - (incl - mine);
    int b = tid;
    for (;;) {
      const uint32_t u = (split ? (uint32_t)sequence(p, b).units : 1u) * ipb;
      if (rem < u) break;
      rem -= u;
      b += NTHR;
    }
    plan[WV] = (uint32_t)b;
    plan[WV + 1] = rem;
  }
  __syncthreads();
  int b = __builtin_amdgcn_readfirstlane((int)plan[WV]);
  uint32_t rem = (uint32_t)__builtin_amdgcn_readfirstlane((int)plan[WV + 1]);

  for (uint32_t g = g0; g < g1;) {
    const Sequence s = sequence(p, b);
    const uint32_t units = split ? (uint32_t)s.units : 1u;
    const uint32_t item = rem / units, k0 = rem - item * units;
    const uint32_t k1 = min(units, k0 + (g1 - g));
    const int h = (int)(item / (uint32_t)p.rblocks), rb = (int)(item % (uint32_t)p.rblocks);
    const int key0 = s.start + (int)k0 * UNIT;
    const int key1 = split ? min(s.len, s.start + (int)k1 * UNIT) : s.len;
    const int seq_lo = p.window > 0 ? max(0, s.len - p.S - p.window + 1) : 0;
    // keys that every query sees: [all_lo, all_hi)
    const int all_hi = s.len - p.S + 1, all_lo = p.window > 0 ? max(0, s.len - p.window) : 0;

    int hi[NT], lo[NT], token[NT];
    u32x4_t qf[NT][NK];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int r = rb * ROWS + 16 * t + n;
      const bool live = r < p.rows;
      const int rr = live ? r : 0;
      const int gi = rr / p.S;
      token[t] = rr - gi * p.S;
      hi[t] = live ? s.len - p.S + token[t] + 1 : 0;
      lo[t] = p.window > 0 ? max(0, hi[t] - p.window) : 0;
      const uint16_t *src = p.q + b * p.qs[0] + (int64_t)(h * p.group + gi) * p.qs[1] + token[t] * p.qs[2];
#pragma unroll
      for (int k = 0; k < NK; ++k) {
        const int d = FP8 ? 64 * (k / 2) + 16 * c + 8 * (k & 1) : 32 * k + 8 * c;
        qf[t][k] = ld16(src + d);
      }
    }
    f32x4_t acc[NT][ND];
    float m[NT], l[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      m[t] = -INFINITY;
      l[t] = 0.f;
#pragma unroll
      for (int d = 0; d < ND; ++d) acc[t][d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
    bool bad = s.bad;

    for (int j0 = key0 + 32 * w; j0 < key1; j0 += UNIT) {
      // pages of the two groups of 16 keys; a group that no query sees is not looked up
      const char *kb[2], *vb[2];
      const uint8_t *ksb[2], *vsb[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int j = j0 + 16 * t;
        const bool seen = j < s.len && j + 16 > seq_lo;
        int64_t page = 0;
        if (seen) page = load_index(p.pages, p.pages64, (int64_t)b * p.pages_stride + (j >> p.page_shift));
        if (page < 0 || page >= p.num_pages) {
          bad = true;
          page = 0;
        }
        const int64_t at = j & p.page_mask;
        const int64_t off = (page * p.cs[0] + h * p.cs[1] + at * p.cs[2]) * ES;
        kb[t] = p.k_cache + off;
        vb[t] = p.v_cache + off;
        if constexpr (FP8) {
          const int64_t so = page * p.es[0] + h * p.es[1] + at;
          ksb[t] = p.k_scale + so;
          vsb[t] = p.v_scale + so;
        }
      }
      const uint32_t row = (uint32_t)p.cs[2] * ES;  // bytes from token to token
      u32x4_t kw[2][FP8 ? NK / 2 : NK];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int k = 0; k < (FP8 ? NK / 2 : NK); ++k)
          kw[t][k] = *reinterpret_cast<const u32x4_t *>(kb[t] + (n * row + 16 * c + 64 * k));
      uint32_t ksw[2], vsw[2];
      if constexpr (FP8) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          ksw[t] = *reinterpret_cast<const uint32_t *>(ksb[t] + 4 * c);
          vsw[t] = *reinterpret_cast<const uint32_t *>(vsb[t] + 4 * c);
        }
      }
      VTile<D, FP8> v;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const char *src = vb[j / 4] + (4 * c + (j & 3)) * row;
        if constexpr (FP8 && D == 128) {
          const u32x2_t x = *reinterpret_cast<const u32x2_t *>(src + 8 * n);
          v.w[j][0] = x[0];
          v.w[j][1] = x[1];
        } else {
#pragma unroll
          for (int x = 0; x < VTile<D, FP8>::W / 4; ++x) {
            const u32x4_t y = *reinterpret_cast<const u32x4_t *>(src + 16 * n + 256 * x);
#pragma unroll
            for (int e = 0; e < 4; ++e) v.w[j][4 * x + e] = y[e];
          }
        }
      }

      const bool edge = j0 < all_lo || j0 + 32 > all_hi;  // wave-uniform
      u32x4_t ph[NT], pl[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float sc[8];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          f32x4_t z = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int k = 0; k < NK; ++k) {
            u32x4_t a;
            if constexpr (FP8) {
              const uint32_t x0 = kw[u][k / 2][2 * (k & 1)], x1 = kw[u][k / 2][2 * (k & 1) + 1];
              a = u32x4_t{bf16_of_e4m3(x0, false), bf16_of_e4m3(x0, true), bf16_of_e4m3(x1, false), bf16_of_e4m3(x1, true)};
            } else {
              a = kw[u][k];
            }
            z = mfma(a, qf[t][k], z);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float x = z[i] * p.scale;
            if constexpr (FP8) x *= scale_value((ksw[u] >> (8 * i)) & 255u);
            sc[4 * u + i] = x;
          }
        }
        if (p.softcap > 0.f) {
          // cap * tanh(x / cap), tanh y = 1 - 2 / (e^2y + 1)
          const float a = 2.0f * LOG2E / p.softcap, cap = p.softcap;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float e = __builtin_amdgcn_exp2f(sc[i] * a);
            sc[i] = fmaf(-2.0f * cap, __builtin_amdgcn_rcpf(e + 1.0f), cap);
          }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) sc[i] *= LOG2E;
        if (edge) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int j = j0 + 16 * (i / 4) + 4 * c + (i & 3);
            if (j < lo[t] || j >= hi[t]) sc[i] = -INFINITY;
          }
        }
        float mx = sc[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) mx = fmaxf(mx, sc[i]);
        mx = fmaxf(max_rows4(mx), m[t]);
        const float base = mx == -INFINITY ? 0.f : mx;  // no key so far: the weights below are 0
        if (__any(mx > m[t])) {
          const float alpha = __builtin_amdgcn_exp2f(m[t] - base);
          l[t] *= alpha;
#pragma unroll
          for (int d = 0; d < ND; ++d) acc[t][d] *= alpha;
          m[t] = mx;
        }
        float sum = 0.f;
        float pr[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          pr[i] = __builtin_amdgcn_exp2f(sc[i] - base);
          sum += pr[i];
        }
        l[t] += sum;
        if constexpr (FP8) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float x = pr[i] * scale_value((vsw[i / 4] >> (8 * (i & 3))) & 255u);
            const int j = j0 + 16 * (i / 4) + 4 * c + (i & 3);
            pr[i] = edge && (j < lo[t] || j >= hi[t]) ? 0.f : x;  // a scale that is not seen may be NaN
          }
        }
        // p = hi + lo, both bf16 and both positive where p is: lo keeps 2^-7
        // to 2^-6 of p, so that an infinite v, which meets both, stays an infinity.
        float lo_[8];
        uint32_t hb[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          hb[i] = __float_as_uint(pr[i] * 0.9921875f);
          lo_[i] = pr[i] - __uint_as_float(hb[i] & 0xffff0000u);
        }
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          ph[t][y] = __builtin_amdgcn_perm(hb[2 * y + 1], hb[2 * y], 0x07060302u);
          pl[t][y] = pack_bf16x2(lo_[2 * y], lo_[2 * y + 1]);
        }
      }

      if (edge) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int key = j0 + 16 * (j / 4) + 4 * c + (j & 3);
          bool drop = key < seq_lo || key >= s.len;
          if constexpr (MULTI) {
            // A value that is not finite, of a key that only some of the queries
            // see, would reach the others as 0 * NaN: the key is taken out, and the
            // rows that see it are NaN.
            const uint64_t odd = __ballot(!drop && (key < all_lo || key >= all_hi) && v.odd(j));
            if (odd >> (16 * c) & 0xffffu) {
              drop = true;
#pragma unroll
              for (int t = 0; t < NT; ++t)
                if (key >= lo[t] && key < hi[t]) l[t] = __uint_as_float(0x7fc00000u);
            }
          }
          if (drop) {
#pragma unroll
            for (int x = 0; x < VTile<D, FP8>::W; ++x) v.w[j][x] = 0u;
          }
        }
      }
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        const u32x4_t a = v.operand(d);
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[t][d] = mfma(a, pl[t], mfma(a, ph[t], acc[t][d]));
      }
    }

    // Join the waves: maxima and sums first, then O in pieces of 32 columns.
    const bool any_bad = __syncthreads_or(bad);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const float sum = sum_rows4(l[t]);
      if (c == 0) {
        ml[(w * ROWS + 16 * t + n) * 2] = m[t];
        ml[(w * ROWS + 16 * t + n) * 2 + 1] = sum;
      }
    }
    const uint32_t istart = g - k0;
    const uint32_t w0 = istart / per, w1 = split ? (istart + units - 1) / per : w0;
    const bool whole = w0 == w1;
    const int rows_here = min(ROWS, p.rows - rb * ROWS);
    const int64_t out0 = ((int64_t)(b * p.hq + h * p.group) * p.S + rb * ROWS) * D;
    float *slot = nullptr;
    __amdgpu_buffer_rsrc_t rs;
    if (!whole) {
      slot = p.partials + (int64_t)(2 * blockIdx.x + (w0 == blockIdx.x ? 1 : 0)) * SLOT;
      rs = __builtin_amdgcn_make_buffer_rsrc(slot, 0, SLOT * 4, 0x00020000);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int x = 0; x < NX; ++x) {
        __syncthreads();
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          float *dst = ex + (w * ROWS + 16 * t + n) * LDX + 8 * c;
#pragma unroll
          for (int e = 0; e < 8; ++e) dst[e] = acc[t][8 * x + e][i];
        }
        __syncthreads();
        for (int piece = tid; piece < 4 * rows_here; piece += NTHR) {
          const int r = piece >> 2, cc = piece & 3;
          float mm = -INFINITY;
#pragma unroll
          for (int y = 0; y < WV; ++y) mm = fmaxf(mm, ml[(y * ROWS + r) * 2]);
          const float base = mm == -INFINITY ? 0.f : mm;
          float o[8] = {}, sum = 0.f;
#pragma unroll
          for (int y = 0; y < WV; ++y) {
            const float a = __builtin_amdgcn_exp2f(ml[(y * ROWS + r) * 2] - base);
            sum = fmaf(a, ml[(y * ROWS + r) * 2 + 1], sum);
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = fmaf(a, ex[(y * ROWS + r) * LDX + 8 * cc + e], o[e]);
          }
          const int d = d_of<D, FP8>(4 * cc + i, x);
          if (whole) {
            const int tk = (rb * ROWS + r) % p.S;
            const bool none = s.len - p.S + tk < 0;  // no key at all
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e)
              y[e] = any_bad ? __uint_as_float(0x7fc00000u) : none ? 0.f : o[e] / sum;
            st16(p.out + out0 + (int64_t)r * D + d, pack8(y));
          } else {
            __builtin_amdgcn_raw_buffer_store_b128(
                __builtin_bit_cast(u32x4_t, f32x4_t{o[0], o[1], o[2], o[3]}), rs, (r * D + d) * 4, 0, SC1);
            __builtin_amdgcn_raw_buffer_store_b128(
                __builtin_bit_cast(u32x4_t, f32x4_t{o[4], o[5], o[6], o[7]}), rs, (r * D + d + 4) * 4, 0, SC1);
            if (i == 0 && x == 0 && cc == 0) {
              // a wrong page is handed on as a sum that is NaN
              const float su = any_bad ? __uint_as_float(0x7fc00000u) : sum;
              __builtin_amdgcn_raw_buffer_store_b64(u32x2_t{__float_as_uint(mm), __float_as_uint(su)}, rs,
                                                    (ROWS * D + 2 * r) * 4, 0, SC1);
            }
          }
        }
      }
    }
    if (!whole) {
      // Every store of this thread has completed, then one arrival per
      // workgroup (release before, acquire after, at agent scope).
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      if (tid == 0) {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "agent");
        plan[WV + 2] = (uint32_t)atomicAdd(p.counters + w0, 1);
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
      }
      __syncthreads();
      if (plan[WV + 2] == w1 - w0) {  // the last: join the parts w0 .. w1 in order
        const int piece = tid % (D / 8), grp = tid / (D / 8);
        const uint32_t parts = w1 - w0 + 1;
        const auto all = __builtin_amdgcn_make_buffer_rsrc(p.partials, 0, 2 * gridDim.x * (SLOT * 4), 0x00020000);
#pragma unroll 1
        for (int r0 = 0; r0 < rows_here; r0 += 4) {
          float o[4][8] = {}, mm[4], sum[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            mm[r] = -INFINITY;
            sum[r] = 0.f;
          }
#pragma unroll 1
          for (uint32_t k = grp; k < parts; k += MG) {
            const uint32_t from = w0 + k;
            const uint32_t at = (2 * from + (from == w0 ? 1 : 0)) * (SLOT * 4);
            u32x4_t po[4][2];
            u32x2_t pm[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const int rr = min(r0 + r, rows_here - 1);
              pm[r] = __builtin_amdgcn_raw_buffer_load_b64(all, at + (ROWS * D + 2 * rr) * 4, 0, SC1);
              po[r][0] = __builtin_amdgcn_raw_buffer_load_b128(all, at + (rr * D + 8 * piece) * 4, 0, SC1);
              po[r][1] = __builtin_amdgcn_raw_buffer_load_b128(all, at + (rr * D + 8 * piece + 4) * 4, 0, SC1);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const float pmax = __uint_as_float(pm[r][0]);
              const float top = fmaxf(mm[r], pmax), base = top == -INFINITY ? 0.f : top;
              const float a = __builtin_amdgcn_exp2f(mm[r] - base), a1 = __builtin_amdgcn_exp2f(pmax - base);
              mm[r] = top;
              sum[r] = fmaf(__uint_as_float(pm[r][1]), a1, sum[r] * a);
#pragma unroll
              for (int e = 0; e < 8; ++e) o[r][e] = fmaf(__uint_as_float(po[r][e / 4][e % 4]), a1, o[r][e] * a);
            }
          }
          __syncthreads();
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            if (piece == 0) {
              ml[(grp * 4 + r) * 2] = mm[r];
              ml[(grp * 4 + r) * 2 + 1] = sum[r];
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) ex[(grp * 4 + r) * D + 8 * piece + e] = o[r][e];
          }
          __syncthreads();
          for (int k = tid; k < 4 * (D / 8); k += NTHR) {
            const int r = k / (D / 8), pc = k % (D / 8);
            if (r0 + r >= rows_here) continue;
            float top = -INFINITY;
#pragma unroll
            for (int y = 0; y < MG; ++y) top = fmaxf(top, ml[(y * 4 + r) * 2]);
            const float base = top == -INFINITY ? 0.f : top;
            float y8[8] = {}, su = 0.f;
#pragma unroll
            for (int y = 0; y < MG; ++y) {
              const float a = __builtin_amdgcn_exp2f(ml[(y * 4 + r) * 2] - base);
              su = fmaf(a, ml[(y * 4 + r) * 2 + 1], su);
#pragma unroll
              for (int e = 0; e < 8; ++e) y8[e] = fmaf(a, ex[(y * 4 + r) * D + 8 * pc + e], y8[e]);
            }
            const int tk = (rb * ROWS + r0 + r) % p.S;
            const bool none = s.len - p.S + tk < 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) y8[e] = none && su == su ? 0.f : y8[e] / su;
            st16(p.out + out0 + (int64_t)(r0 + r) * D + 8 * pc, pack8(y8));
          }
        }
        if (tid == 0) atomicExch(p.counters + w0, 0);
      }
    }
    __syncthreads();  // the exchange's memory is free again
    g += k1 - k0;
    rem += k1 - k0;
    if (rem == units * ipb) {
      rem = 0;
      b += NTHR;
      if (b >= p.B) b = b % NTHR + 1;
    }
  }
}

// Rows of a pass and workgroups of a launch.
struct Plan {
  int nt, rblocks;
  int64_t grid, slot_floats;
};

Plan plan_of(const kfmi_decode_args &a) {
  Plan r{};
  const int64_t rows = a.Hq / a.Hkv * a.S;
  const int most = a.D == 128 ? 4 : 2;
  r.nt = rows <= 16 ? 1 : rows <= 32 || most == 2 ? 2 : 4;
  r.rblocks = (int)((rows + 16 * r.nt - 1) / (16 * r.nt));
  const int64_t units = a.B * a.Hkv * r.rblocks * ((a.max_pages * a.page_size + UNIT - 1) / UNIT);
  const int64_t round = r.nt * a.D <= 256 ? 512 : 256;  // workgroups that run at once: two or one per CU
  r.grid = units < round ? units : round;
  r.slot_floats = 16 * r.nt * (a.D + 2);
  return r;
}

template <int D, bool FP8, int NT, bool MULTI>
hipError_t launch_decode_t(const DecodeParams &p, int64_t grid, hipStream_t stream) {
  hipLaunchKernelGGL((decode_kernel<D, FP8, NT, MULTI>), dim3((unsigned)grid), dim3(NTHR), 0, stream, p);
  static const std::string name = [] {
    char b[96];
    snprintf(b, sizeof(b), "decode_kernel<%d, %s, %d, %s>", D, tf(FP8), NT, tf(MULTI));
    return std::string(b);
  }();
  launch_log_add(reinterpret_cast<const void *>(&decode_kernel<D, FP8, NT, MULTI>), name.c_str(), grid, NTHR);
  launch_log_plan("split=%d rblocks=%d", p.counters != nullptr, p.rblocks);
  return hipGetLastError();
}

template <int D, bool FP8, int NT>
hipError_t launch_decode_s(const DecodeParams &p, int64_t grid, hipStream_t stream) {
  return p.S > 1 ? launch_decode_t<D, FP8, NT, true>(p, grid, stream) : launch_decode_t<D, FP8, NT, false>(p, grid, stream);
}

template <int D, bool FP8>
hipError_t dispatch_decode(const DecodeParams &p, int nt, int64_t grid, hipStream_t stream) {
  if (nt == 1) return launch_decode_s<D, FP8, 1>(p, grid, stream);
  if (nt == 2) return launch_decode_s<D, FP8, 2>(p, grid, stream);
  if constexpr (D == 128) return launch_decode_s<D, FP8, 4>(p, grid, stream);
  return hipErrorInvalidValue;
}

}  // namespace

int64_t decode_workspace_bytes(const kfmi_decode_args &a) {
  const Plan r = plan_of(a);
  return r.grid > 1 ? KFMI_DECODE_COUNTER_BYTES + 2 * r.grid * r.slot_floats * 4 : 0;
}

hipError_t launch_decode(const kfmi_decode_args &a, hipStream_t stream) {
  const Plan plan = plan_of(a);
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
  p.capacity = (int)(a.max_pages * a.page_size);
  p.window = (int)(a.window < p.capacity ? a.window : 0);  // a window of all keys is none
  p.min_units = 1;
  p.B = (int)a.B; p.hq = (int)a.Hq; p.hk = (int)a.Hkv; p.S = (int)a.S;
  p.group = p.hq / p.hk;
  p.rows = p.group * p.S;
  p.rblocks = plan.rblocks;
  p.page_shift = log2_of(a.page_size);
  p.page_mask = (int)(a.page_size - 1);
  p.pages64 = a.index_flags & KFMI_I64_PAGES;
  p.len64 = a.index_flags & KFMI_I64_LENGTHS;
  p.scale = (float)a.scale;
  p.softcap = (float)a.softcap;
  const int64_t need = decode_workspace_bytes(a);
  if (need > 0 && a.work && a.work_bytes >= need) {
    p.counters = (int *)a.work;
    p.partials = (float *)((char *)a.work + KFMI_DECODE_COUNTER_BYTES);
  }
  const int64_t grid = p.counters || need == 0 ? plan.grid
                                               : (plan.grid < a.B * a.Hkv * plan.rblocks ? plan.grid : a.B * a.Hkv * plan.rblocks);
  const bool fp8 = a.cache_type == KFMI_CACHE_E4M3;
  if (a.D == 128)
    return fp8 ? dispatch_decode<128, true>(p, plan.nt, grid, stream) : dispatch_decode<128, false>(p, plan.nt, grid, stream);
  return fp8 ? dispatch_decode<256, true>(p, plan.nt, grid, stream) : dispatch_decode<256, false>(p, plan.nt, grid, stream);
}

}  // namespace kfmi
