// Attention of the last few tokens of each sequence over its paged cache
// (kfmi_attention_decode_bf16).
//
// out_i = sum_j softmax_j(cap(q_i . k_j * scale)) v_j over the keys that
// query i sees.  Every key and value is read once per KV head, so the cache's bytes
// bound the call: 4 * D bytes (bf16) per key and head against 4 * D * R flops for the R = group * S query rows
// that share them, at most 64 rows a pass.  64 sequences of 4096 keys, 8 heads of D = 128, take
// 169 us (1.07 GB, 6.4 TB/s; a bare read of such pages reaches 6.8), one of 32768 28.4 us, one of 333 8.2; at 32
// rows in e4m3 the softmax and the conversions bound it instead: 16 sequences of 4096 keys 41 us (137 MB).  The design:
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
//    units have time for it.  An e4m3 row becomes bf16, times its scale, in the conversion, exactly;
//  * the work of a launch (units of 32 keys per wave, all heads and sequences)
//    is dealt evenly to one round of workgroups, whatever the lengths: each
//    finds its share by a scan of the lengths.  A head's sequence that
//    crosses a border is joined, in order, by the workgroup that arrives last.
#include <cstdio>
#include <string>
#include <type_traits>

#include "cache_common.h"
#include "kfmi_launch.h"

namespace kfmi {
namespace {

constexpr int WV = 4;            // waves per workgroup
constexpr int NTHR = 64 * WV;
constexpr int UNIT = 32 * WV;    // keys per unit of work
constexpr int SC1 = 16;          // cache policy of agent-coherent accesses
constexpr float LARGE_CAP = 128.0f * 1.44269504f;  // caps from here keep small scores' digits, see the kernel

struct DecodeParams {
  const uint16_t *q;
  const char *k_cache, *v_cache;
  const uint8_t *k_scale, *v_scale;
  const void *pages, *lengths;
  uint16_t *out;
  int *counters;    // NULL: no workspace, no sequence is split
  float *partials;  // 2 slots per workgroup
  int64_t qs[3], cs[3], es[2];
  int64_t pages_stride, lengths_stride;
  int num_pages, B, hq, hk, S, group, rows, rblocks;  // rows = group * S, in blocks of 16 * NT
  int capacity, window;
  int page_shift, page_mask;
  bool pages64, len64;
  float score_scale;  // of q . k: to the argument 2 a log2(e) of c tanh a
  float cap;          // softcap * log2(e); 0: none
  float slope, offset;  // of the scores (exponents of 2), see the kernel
};

// What a launch reads of one sequence.
struct Sequence {
  int len;    // 0 where the given one is wrong
  int lo;     // first key that a query sees
  int start;  // first key of the first unit: lo or below, a multiple of 32
  int units;
  bool bad;
};

__device__ __forceinline__ Sequence sequence(const DecodeParams &p, int b) {
  Sequence s;
  const int2 len = load_index_words(p.lengths, p.len64, (int64_t)b * p.lengths_stride);
  s.bad = len.y != 0 || (uint32_t)len.x > (uint32_t)p.capacity;
  s.len = s.bad ? 0 : len.x;
  s.lo = p.window > 0 ? max(0, s.len - p.S - p.window + 1) : 0;
  s.start = s.lo & ~31;
  s.units = p.counters ? max(1, (s.len - s.start + UNIT - 1) / UNIT) : 1;  // never split: one unit of all keys
  return s;
}

// Units of work per workgroup: an even share, but
//  * where two workgroups per CU would have up to four units each (eight at D = 256), one
//    has them all (e4m3, 32 sequences of 1024 keys at D = 128: 17.4 instead of 20.6 us, 32 of 2048 at
//    D = 256 49 instead of 54; with more two are faster, 64 of 1024 at D = 128 28.3 instead of 31.2,
//    64 of up to 8192 at D = 256 180 instead of 189).  bf16 has two only where one would have at least
//    two whole sequences (256 of 100 keys 31.5 instead of 41.5 us, 64 of 300 18 instead of 20; one of
//    32768 keys, in pieces, 38 instead of 30);
//  * a sequence (`most` units, the longest) of up to three units is not split: the join
//    takes as long as two (one of 333 keys: 9.3 instead of 9.5 us), and a longer
//    one not into more parts than its join, some 0.8 us for 64 rows of
//    parts, leaves worth it: units / parts * 1.2 us + rows * parts / 64 * 0.8 us is least at
//    parts = sqrt(96 * units / rows) (one head of 16 rows, 32768 keys at D = 256: 49 us, 94 in as many parts as
//    there are units, 59 in half of these parts).
__device__ __forceinline__ uint32_t units_per_workgroup(uint32_t total, uint32_t most, uint32_t grid, uint32_t rows,
                                                        uint32_t few) {
  uint32_t even = (total + grid - 1) / grid;
  const uint32_t alone = (total + 255) / 256;
  if (grid > 256 && (few ? even <= few : alone < 2 * most)) even = alone;
  const uint32_t least = most <= 3 ? most : min(most, (uint32_t)__builtin_sqrtf((float)(most * rows) * (1.0f / 96.0f)));
  return max(even, max(least, 1u));
}

// A workgroup's part of one sequence, head and block of rows: units k0 .. k1 - 1.
struct Item {
  Sequence s;
  int b, h, rb;
  uint32_t k0, k1;
  int key0, key1;
};

__device__ __forceinline__ Item item_at(const DecodeParams &p, int b, uint32_t rem, uint32_t left) {
  Item it;
  it.s = sequence(p, b);
  it.b = b;
  const uint32_t units = (uint32_t)it.s.units, item = rem / units;
  it.k0 = rem - item * units;
  it.k1 = min(units, it.k0 + left);
  it.h = (int)(item / (uint32_t)p.rblocks);
  it.rb = (int)(item % (uint32_t)p.rblocks);
  it.key0 = it.s.start + (int)it.k0 * UNIT;
  it.key1 = p.counters ? min(it.s.len, it.s.start + (int)it.k1 * UNIT) : it.s.len;
  return it;
}

// x, of which the compiler knows nothing: what is computed from it stays where it
// is used, instead of in registers across the whole of the kernel's loop.
__device__ __forceinline__ int opaque(int x) {
  asm volatile("" : "+v"(x));
  return x;
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

// Two e4m3 values of w times a scale, whose byte is the exponent of `scale`, as bf16: exact
// for what a cache holds, NaN where the byte is 255.
__device__ __forceinline__ uint32_t bf16_of_e4m3(uint32_t w, uint32_t scale, bool high) {
  const float f = __uint_as_float(scale);
  return __builtin_bit_cast(uint32_t, high ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w, f, true)
                                           : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w, f, false));
}
__device__ __forceinline__ uint32_t scale_byte(uint32_t w, int i) { return ((w >> (8 * i)) & 255u) << 23; }

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
  uint32_t scale[FP8 ? 8 : 1];
  // Values 2 x and 2 x + 1 of key j in bf16.
  __device__ __forceinline__ uint32_t pair(int j, int x) const {
    if constexpr (FP8) return bf16_of_e4m3(w[j][x / 2], scale[j], x & 1);
    else return w[j][x];
  }
  // The operands of products 2 x and 2 x + 1.
  __device__ __forceinline__ void operands(int x, u32x4_t (&a)[2]) const {
    uint32_t c[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) c[j] = pair(j, x);
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      a[0][y] = __builtin_amdgcn_perm(c[2 * y + 1], c[2 * y], 0x05040100u);
      a[1][y] = __builtin_amdgcn_perm(c[2 * y + 1], c[2 * y], 0x07060302u);
    }
  }
  // Whether a value of key j is an infinity or NaN.
  __device__ __forceinline__ bool odd(int j) const {
    bool any = false;
    if constexpr (FP8) any = scale[j] == 255u << 23;
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

// Waves per SIMD that the registers leave room for.  A wave alone reads bf16 as fast as two do, and half
// the workgroups make half the parts of a split sequence; many short sequences and e4m3, which takes twice the
// arithmetic per byte, are faster with two (e4m3, 64 sequences of 4096 keys at D = 128: 92
// instead of 104 us).
constexpr int waves_per_simd(int d, bool fp8, int nt) { return fp8 ? (d * nt <= 256 ? 2 : 1) : d * nt <= 128 ? 2 : 1; }

// GENERAL: several queries or a cap.  Without it (one token per sequence, no cap) neither is in the code: one sequence
// of 333 keys 8.2 instead of 8.7 us, 64 of up to 8192 in bf16 175 instead of 176.5.
template <int D, bool FP8, int NT, bool GENERAL>
__global__ __launch_bounds__(NTHR, waves_per_simd(D, FP8, NT)) void decode_kernel(DecodeParams p) {
  constexpr int NK = D / 32;    // matrix steps of q . k
  constexpr int ND = D / 16;    // products of P V
  constexpr int NX = ND / 8;
  constexpr int JU = D == 128 && !FP8 && NT <= 2 ? 2 : 1;  // parts in flight in the join
  constexpr int ES = FP8 ? 1 : 2;
  constexpr int ROWS = 16 * NT;
  constexpr int SLOT = ROWS * (D + 2);  // floats: O row by row, then (m, l) of each row
  constexpr int LDX = D + 4;            // floats per row of the exchange
  constexpr int MG = NTHR / (D / 8);    // groups of the join
  constexpr int EX = WV * ROWS * LDX > MG * 4 * D ? WV * ROWS * LDX : MG * 4 * D;
  __shared__ __attribute__((aligned(16))) float ex[EX];
  __shared__ float ml[(WV * ROWS > MG * 4 ? WV * ROWS : MG * 4) * 2];
  __shared__ uint32_t arrived;
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, c = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const float offset = GENERAL ? p.offset : 0.f;
  const uint32_t ipb = (uint32_t)(p.hk * p.rblocks);  // items (head, block of rows) per sequence

  // This workgroup's share [g0, g1) of all units, the sequences in the order
  // 0, 64, 128, .., 1, 65, .. (lane by lane); every wave finds it by itself.
  uint32_t mine = 0, incl, most = 0;  // units of this lane's sequences, of all up to it; the longest's
  if (p.B == 1) {
    most = (uint32_t)sequence(p, 0).units;
    mine = lane == 0 ? most * ipb : 0u;
    incl = most * ipb;
  } else {
    for (int b = lane; b < p.B; b += 64) {
      const uint32_t u = (uint32_t)sequence(p, b).units;
      mine += u * ipb;
      most = max(most, u);
    }
    incl = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t y = (uint32_t)__shfl_up((int)incl, o);
      if (lane >= o) incl += y;
      most = max(most, (uint32_t)__shfl_xor((int)most, o));
    }
  }
  most = (uint32_t)__builtin_amdgcn_readfirstlane((int)most);
  const uint32_t total = (uint32_t)__builtin_amdgcn_readlane((int)incl, 63);
  const uint32_t per = units_per_workgroup(total, most, gridDim.x, (uint32_t)min(ROWS, p.rows), FP8 ? D / 32 : 0);
  const uint32_t g0 = blockIdx.x * per, g1 = min(g0 + per, total);
  if (g0 >= total) return;  // workgroup-uniform
  int b = __builtin_ctzll(__ballot(incl > g0));
  uint32_t rem = g0 - (uint32_t)__builtin_amdgcn_readlane((int)(incl - mine), b);
  for (;;) {
    const uint32_t u = (uint32_t)sequence(p, b).units * ipb;
    if (rem < u) break;
    rem -= u;
    b += 64;
  }

  // The pages of the two groups of 16 keys from j on.  A group that no query
  // sees takes the nearest page that one does: its own entry may be anything.
  int2 pg[2];
  auto request_pages = [&](const Item &it, int j0) {
    const int64_t row0 = (int64_t)it.b * p.pages_stride;
    const int lo = it.s.lo >> p.page_shift, hi = max(it.s.len - 1, 0) >> p.page_shift;
#pragma unroll
    for (int t = 0; t < 2; ++t)
      pg[t] = load_index_words(p.pages, p.pages64, row0 + min(max((j0 + 16 * t) >> p.page_shift, lo), hi));
  };
  const uint32_t row = (uint32_t)p.cs[2] * ES;  // bytes from token to token
  const char *kb[2], *vb[2];
  const uint8_t *ksb[2], *vsb[2];
  auto look_up = [&](const Item &it, int j0, bool &bad) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const bool wrong = pg[t].y != 0 || (uint32_t)pg[t].x >= (uint32_t)p.num_pages;
      bad |= wrong;
      const int64_t page = wrong ? 0 : pg[t].x;
      const int64_t at = (j0 + 16 * t) & p.page_mask;
      const int64_t off = (page * p.cs[0] + it.h * p.cs[1] + at * p.cs[2]) * ES;
      kb[t] = p.k_cache + off;
      vb[t] = p.v_cache + off;
      if constexpr (FP8) {
        const int64_t so = page * p.es[0] + it.h * p.es[1] + at;
        ksb[t] = p.k_scale + so;
        vsb[t] = p.v_scale + so;
      }
    }
  };
  u32x4_t qf[NT][NK];
  auto load_q = [&](const Item &it) {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int r = it.rb * ROWS + 16 * t + opaque(n), rr = r < p.rows ? r : 0, gi = rr / p.S;
      const uint16_t *src = p.q + it.b * p.qs[0] + (int64_t)(it.h * p.group + gi) * p.qs[1] + (rr - gi * p.S) * p.qs[2];
#pragma unroll
      for (int k = 0; k < NK; ++k)
        qf[t][k] = ld16(src + (FP8 ? 64 * (k / 2) + 16 * c + 8 * (k & 1) : 32 * k + 8 * c));
    }
  };
  u32x4_t kw[2][FP8 ? NK / 2 : NK];
  uint32_t ksw[2], vsw[2];
  VTile<D, FP8> v;
  auto load_k = [&]() {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int k = 0; k < (FP8 ? NK / 2 : NK); ++k)
        kw[t][k] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t *>(kb[t] + (n * row + 16 * c + 64 * k)));
      if constexpr (FP8) ksw[t] = ksb[t][n];
    }
  };
  auto load_v = [&]() {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const char *src = vb[j / 4] + (4 * c + (j & 3)) * row;
      if constexpr (FP8 && D == 128) {
        const u32x2_t x = __builtin_nontemporal_load(reinterpret_cast<const u32x2_t *>(src + 8 * n));
        v.w[j][0] = x[0];
        v.w[j][1] = x[1];
      } else {
#pragma unroll
        for (int x = 0; x < VTile<D, FP8>::W / 4; ++x) {
          const u32x4_t y = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t *>(src + 16 * n + 256 * x));
#pragma unroll
          for (int e = 0; e < 4; ++e) v.w[j][4 * x + e] = y[e];
        }
      }
    }
    if constexpr (FP8) {
#pragma unroll
      for (int t = 0; t < 2; ++t) vsw[t] = *reinterpret_cast<const uint32_t *>(vsb[t] + 4 * c);
    }
  };

  // The item's first step of this wave: whether there is one, and its loads.
  auto begin = [&](const Item &it, bool &bad) {
    load_q(it);
    const int j0 = it.key0 + 32 * w;
    if (j0 >= it.key1) return false;
    request_pages(it, j0);
    look_up(it, j0, bad);
    load_k();
    load_v();
    request_pages(it, j0 + UNIT);
    return true;
  };

  uint32_t g = g0;
  Item it = item_at(p, b, rem, g1 - g);
  bool bad = it.s.bad, some = begin(it, bad);
  for (;;) {
    const Sequence s = it.s;
    // keys that every query sees: [all_lo, all_hi)
    const int all_hi = s.len - p.S + 1, all_lo = p.window > 0 ? max(0, s.len - p.window) : 0;
    int hi[NT], lo[NT];
    f32x4_t acc[NT][ND];
    float m[NT], l[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int r = it.rb * ROWS + 16 * t + opaque(n);
      hi[t] = r < p.rows ? s.len - p.S + r % p.S + 1 : 0;
      lo[t] = p.window > 0 ? max(0, hi[t] - p.window) : 0;
      m[t] = -INFINITY;
      l[t] = 0.f;
#pragma unroll
      for (int d = 0; d < ND; ++d) acc[t][d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
    if (some) {
      // Q is waited for here, once: in the loop the wait would be one for the
      // youngest loads, K and V of the next step.
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int k = 0; k < NK; ++k) asm volatile("" ::"v"(qf[t][k]));
      // K of the next step is requested as soon as this step's K has been used,
      // V likewise; the last step has none to request.
      int j0 = it.key0 + 32 * w;
      auto step = [&](auto more) {
      if constexpr (more.value) {
        look_up(it, j0 + UNIT, bad);
        request_pages(it, j0 + 2 * UNIT);
      }
      const bool edge = j0 < all_lo || j0 + 32 > all_hi;  // wave-uniform
      f32x4_t z[NT][2];
#pragma unroll
      for (int t = 0; t < NT; ++t) z[t][0] = z[t][1] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int k = 0; k < NK; ++k) {
          u32x4_t a;
          if constexpr (FP8) {
            const uint32_t x0 = kw[u][k / 2][2 * (k & 1)], x1 = kw[u][k / 2][2 * (k & 1) + 1], ks = ksw[u] << 23;
            a = u32x4_t{bf16_of_e4m3(x0, ks, false), bf16_of_e4m3(x0, ks, true), bf16_of_e4m3(x1, ks, false),
                        bf16_of_e4m3(x1, ks, true)};
          } else {
            a = kw[u][k];
          }
#pragma unroll
          for (int t = 0; t < NT; ++t) z[t][u] = mfma(a, qf[t][k], z[t][u]);
        }
      }
      __builtin_amdgcn_sched_barrier(0);  // the loads take the registers of what they follow
      if constexpr (more.value) load_k();
      __builtin_amdgcn_sched_barrier(0);
      u32x4_t ph[NT], pl[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        // Scores are p.slope * y + p.offset: y is q . k, or under a cap c with
        // c tanh a = c - 2 c / (e^2a + 1) that last quotient's -1 / (e^2a + 1).  The sum is good to 2^-22 of the
        // cap: 2^-15 in a score capped at 128.  Under a larger cap y is the score, where a
        // is small by the series a (1 - a^2 / 3 + 2 a^4 / 15), below 1/16 good
        // to 2^-26 of itself (for every cap it would make 16 sequences of 4096 keys, 32 rows a head,
        // 48 us; without it they take 45).
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = z[t][i / 4][i & 3];
        if (GENERAL && p.cap > 0.f) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            y[i] = -__builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(y[i] * p.score_scale) + 1.0f);
          if (p.cap > LARGE_CAP) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float w = z[t][i / 4][i & 3] * p.score_scale, a = w * 0.34657359027997264f, a2 = a * a;
              const float near = p.cap * a * fmaf(a2, fmaf(a2, 0.13333333333f, -0.33333333333f), 1.0f);
              y[i] = fabsf(w) < 0.18033688f ? near : fmaf(2.0f * p.cap, y[i], p.cap);
            }
          }
        }
        if (edge) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int j = j0 + 16 * (i / 4) + 4 * c + (i & 3);
            if (j < lo[t] || j >= hi[t]) y[i] = -INFINITY;
          }
        }
        float mx = y[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) mx = fmaxf(mx, y[i]);
        mx = fmaxf(fmaf(p.slope, max_rows4(mx), offset), m[t]);
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
          pr[i] = __builtin_amdgcn_exp2f(fmaf(p.slope, y[i], offset - base));
          sum += pr[i];
        }
        l[t] += sum;
        // p = hi + lo, both bf16.  For a bf16 cache both are positive where p is: lo keeps 2^-7
        // to 2^-6 of p, so that an infinite v, which meets both, stays an infinity.
        float lo_[8];
        uint32_t hb[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          hb[i] = __float_as_uint(FP8 ? pr[i] : pr[i] * 0.9921875f);
          lo_[i] = pr[i] - __uint_as_float(hb[i] & 0xffff0000u);
        }
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          ph[t][y] = __builtin_amdgcn_perm(hb[2 * y + 1], hb[2 * y], 0x07060302u);
          pl[t][y] = pack_bf16x2(lo_[2 * y], lo_[2 * y + 1]);
        }
      }

      if constexpr (FP8) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v.scale[j] = scale_byte(vsw[j / 4], j & 3);
      }
      if (edge) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int key = j0 + 16 * (j / 4) + 4 * c + (j & 3);
          bool drop = key < s.lo || key >= s.len;
          if constexpr (GENERAL) {
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
            if constexpr (FP8) v.scale[j] = 0u;
          }
        }
      }
#pragma unroll
      for (int d = 0; d < ND; d += 2) {
        u32x4_t a[2];
        v.operands(d / 2, a);
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int t = 0; t < NT; ++t) acc[t][d + x] = mfma(a[x], pl[t], mfma(a[x], ph[t], acc[t][d + x]));
      }
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (more.value) load_v();
      __builtin_amdgcn_sched_barrier(0);
      };
      for (; j0 + UNIT < it.key1; j0 += UNIT) step(std::true_type{});
      step(std::false_type{});
    }

    // The next item's first loads run while this one is written.
    const uint32_t istart = g - it.k0;
    const uint32_t w0 = istart / per, w1 = (istart + (uint32_t)s.units - 1) / per;  // the workgroups that share the item
    g += it.k1 - it.k0;
    rem += it.k1 - it.k0;
    if (rem == (uint32_t)s.units * ipb) {
      rem = 0;
      b += 64;
      if (b >= p.B) b = b % 64 + 1;
    }
    const bool again = g < g1;
    Item next = it;
    bool next_bad = false, next_some = false;
    if (again) {
      next = item_at(p, b, rem, g1 - g);
      next_bad = next.s.bad;
      next_some = begin(next, next_bad);
    }

    // Join the waves: maxima, sums and O of the rows in use through LDS.
    const bool whole = w0 == w1;
    const int rows_here = min(ROWS, p.rows - it.rb * ROWS);
    const int xtid = opaque(tid), xn = xtid & 15, xc = (xtid & 63) >> 4;
    const int64_t out0 = ((int64_t)(it.b * p.hq + it.h * p.group) * p.S + it.rb * ROWS) * D;
    float *slot = p.partials + (int64_t)(2 * blockIdx.x + (w0 == blockIdx.x ? 1 : 0)) * SLOT;
    const auto rs = __builtin_amdgcn_make_buffer_rsrc(whole ? p.partials : slot, 0, whole ? 0 : SLOT * 4, 0x00020000);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const float sum = sum_rows4(l[t]);
      if (16 * t + xn < rows_here) {
        float *dst = ex + (w * ROWS + 16 * t + xn) * LDX;
        if (xc == 0) {
          ml[(w * ROWS + 16 * t + xn) * 2] = m[t];
          ml[(w * ROWS + 16 * t + xn) * 2 + 1] = sum;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int x = 0; x < NX; ++x) {
            float *o = dst + d_of<D, FP8>(4 * xc + i, x);
#pragma unroll
            for (int e = 0; e < 8; e += 4)
              *reinterpret_cast<f32x4_t *>(o + e) =
                  f32x4_t{acc[t][8 * x + e][i], acc[t][8 * x + e + 1][i], acc[t][8 * x + e + 2][i], acc[t][8 * x + e + 3][i]};
          }
      }
    }
    const bool any_bad = __syncthreads_or(bad);
    const float nan = __uint_as_float(0x7fc00000u);
    for (int piece = xtid; piece < rows_here * (D / 4); piece += NTHR) {
      const int r = piece / (D / 4), d = piece % (D / 4) * 4;
      float mm[WV], ll[WV], top = -INFINITY;
      f32x4_t o[WV];
#pragma unroll
      for (int y = 0; y < WV; ++y) {
        mm[y] = ml[(y * ROWS + r) * 2];
        ll[y] = ml[(y * ROWS + r) * 2 + 1];
        o[y] = *reinterpret_cast<const f32x4_t *>(ex + (y * ROWS + r) * LDX + d);
      }
#pragma unroll
      for (int y = 0; y < WV; ++y) top = fmaxf(top, mm[y]);
      const float base = top == -INFINITY ? 0.f : top;
      f32x4_t sum4 = {0.f, 0.f, 0.f, 0.f};
      float sum = 0.f;
#pragma unroll
      for (int y = 0; y < WV; ++y) {
        const float a = __builtin_amdgcn_exp2f(mm[y] - base);
        sum = fmaf(a, ll[y], sum);
#pragma unroll
        for (int e = 0; e < 4; ++e) sum4[e] = fmaf(a, o[y][e], sum4[e]);
      }
      if (whole) {
        const bool none = s.len - p.S + (it.rb * ROWS + r) % p.S < 0;  // no key at all
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = any_bad ? nan : none ? 0.f : sum4[e] / sum;
        *reinterpret_cast<u32x2_t *>(p.out + out0 + (int64_t)r * D + d) =
            u32x2_t{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
      } else {
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, sum4), rs, (r * D + d) * 4, 0, SC1);
        if (d == 0)  // a wrong page is handed on as a sum that is NaN
          __builtin_amdgcn_raw_buffer_store_b64(u32x2_t{__float_as_uint(top), __float_as_uint(any_bad ? nan : sum)}, rs,
                                                (ROWS * D + 2 * r) * 4, 0, SC1);
      }
    }
    if (!whole) {
      // The parts are written and read with agent-coherent accesses (SC1), which
      // pass the caches of an XCD by: a store that has completed (vmcnt) is what
      // any later SC1 load gets.  So the arrival needs no L2 writeback or
      // invalidation (release and acquire fences cost 18 us a launch here).
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      if (tid == 0)
        arrived = (uint32_t)__hip_atomic_fetch_add(p.counters + w0, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      __syncthreads();
      if (arrived == w1 - w0) {  // the last: join the parts w0 .. w1 in order
        // A thread sums 8 columns of 4 rows over every pgs-th part; the groups of threads
        // that the parts leave over take other rows.
        const int tid_ = opaque(tid);
        const uint32_t parts = w1 - w0 + 1;
        const int piece = tid_ % (D / 8), grp = tid_ / (D / 8);
        int pgs = 1;
        while (pgs < MG && (uint32_t)pgs < parts) pgs *= 2;
        const int pgi = grp % pgs, step = 4 * (MG / pgs);
        const auto all = __builtin_amdgcn_make_buffer_rsrc(p.partials, 0, 2 * gridDim.x * (SLOT * 4), 0x00020000);
#pragma unroll 1
        for (int rb0 = 0; rb0 < rows_here; rb0 += step) {
          const int r0 = rb0 + grp / pgs * 4;
          float o[4][8] = {}, mm[4], sum[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            mm[r] = -INFINITY;
            sum[r] = 0.f;
          }
#pragma unroll 1
          for (uint32_t k = pgi; k < parts; k += JU * pgs) {
            u32x4_t po[JU][4][2];
            u32x2_t pm[JU][4];
#pragma unroll
            for (int q = 0; q < JU; ++q) {
              const uint32_t from = w0 + min(k + q * pgs, parts - 1);
              const uint32_t at = (2 * from + (from == w0 ? 1 : 0)) * (SLOT * 4);
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                const int rr = min(r0 + r, rows_here - 1);
                pm[q][r] = __builtin_amdgcn_raw_buffer_load_b64(all, at + (ROWS * D + 2 * rr) * 4, 0, SC1);
                po[q][r][0] = __builtin_amdgcn_raw_buffer_load_b128(all, at + (rr * D + 8 * piece) * 4, 0, SC1);
                po[q][r][1] = __builtin_amdgcn_raw_buffer_load_b128(all, at + (rr * D + 8 * piece + 4) * 4, 0, SC1);
              }
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int q = 0; q < JU; ++q) {
              if (k + q * pgs >= parts) break;
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                const float pmax = __uint_as_float(pm[q][r][0]);
                const float top = fmaxf(mm[r], pmax), base = top == -INFINITY ? 0.f : top;
                const float a = __builtin_amdgcn_exp2f(mm[r] - base), a1 = __builtin_amdgcn_exp2f(pmax - base);
                mm[r] = top;
                sum[r] = fmaf(__uint_as_float(pm[q][r][1]), a1, sum[r] * a);
#pragma unroll
                for (int e = 0; e < 8; ++e) o[r][e] = fmaf(__uint_as_float(po[q][r][e / 4][e % 4]), a1, o[r][e] * a);
              }
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
            for (int e = 0; e < 8; e += 4)
              *reinterpret_cast<f32x4_t *>(ex + (grp * 4 + r) * D + 8 * piece + e) =
                  f32x4_t{o[r][e], o[r][e + 1], o[r][e + 2], o[r][e + 3]};
          }
          __syncthreads();
          for (int k = tid_; k < step * (D / 4); k += NTHR) {
            const int rr = k / (D / 4), d = k % (D / 4) * 4;
            const int r = rb0 + rr, g4 = rr / 4 * pgs, r4 = rr % 4;
            if (r >= rows_here) continue;
            float top = -INFINITY;
#pragma unroll 4
            for (int y = 0; y < pgs; ++y) top = fmaxf(top, ml[((g4 + y) * 4 + r4) * 2]);
            const float base = top == -INFINITY ? 0.f : top;
            f32x4_t y4 = {0.f, 0.f, 0.f, 0.f};
            float su = 0.f;
#pragma unroll 4
            for (int y = 0; y < pgs; ++y) {
              const int at = (g4 + y) * 4 + r4;
              const float a = __builtin_amdgcn_exp2f(ml[at * 2] - base);
              const f32x4_t v4 = *reinterpret_cast<const f32x4_t *>(ex + at * D + d);
              su = fmaf(a, ml[at * 2 + 1], su);
#pragma unroll
              for (int e = 0; e < 4; ++e) y4[e] = fmaf(a, v4[e], y4[e]);
            }
            *reinterpret_cast<u32x2_t *>(p.out + out0 + (int64_t)r * D + d) =
                u32x2_t{pack_bf16x2(y4[0] / su, y4[1] / su), pack_bf16x2(y4[2] / su, y4[3] / su)};
          }
          __syncthreads();
        }
        if (tid == 0) __hip_atomic_store(p.counters + w0, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
    }
    if (!again) break;
    __syncthreads();  // the exchange's memory is free again
    it = next;
    bad = next_bad;
    some = next_some;
  }
}

// Blocks of 16 query rows of a pass: all of a head's rows, up to 64; at D = 256 up to 32 in e4m3 and 16 in bf16,
// whose 32 need more registers than there are (16 sequences of 4096 keys, 32 rows: 171 us in two passes, 176 in one).
int widest(const kfmi_decode_args &a, bool fp8) {
  const int64_t rows = a.Hq / a.Hkv * a.S;
  if (rows <= 16 || (a.D == 256 && !fp8)) return 1;
  return rows <= 32 || a.D == 256 ? 2 : 4;
}

// Workgroups and partial results of a launch.
struct Plan {
  int nt, rblocks;
  int64_t grid;
};

// Few sequences leave most of the chip idle, and the exchange and the join of 64 rows take 25 us: their
// rows are dealt to more workgroups in smaller blocks, which read the same keys again, mostly from the caches.  A
// pass takes half the rows where what is read (of the pages' capacity) is then at most 64 MB, or 256 MB by few
// heads and blocks (64 rows, one sequence of 2048 keys: 17.6 instead of 44.5 us, one of 16384 40 instead
// of 76, eight of 2048 35 instead of 49; but eight of 16384 173 instead of 122).
Plan plan_of(const kfmi_decode_args &a) {
  Plan r{};
  const bool fp8 = a.cache_type == KFMI_CACHE_E4M3;
  const int64_t rows = a.Hq / a.Hkv * a.S, capacity = a.max_pages * a.page_size;
  const int64_t keys = a.window > 0 && a.window < capacity - a.S ? a.window + a.S : capacity;
  auto blocks = [&](int nt) { return (rows + 16 * nt - 1) / (16 * nt); };
  r.nt = widest(a, fp8);
  while (r.nt > 1) {
    const int half = r.nt / 2;
    const int64_t items = a.B * a.Hkv * blocks(half);
    const double mb = (double)(items * keys) * (double)(a.D * (fp8 ? 2 : 4)) / (1 << 20);
    if (!(mb <= 64.0 || (mb <= 256.0 && items <= 64 * half))) break;
    r.nt = half;
  }
  r.rblocks = (int)blocks(r.nt);
  const int64_t items = a.B * a.Hkv * r.rblocks, units = items * ((capacity + UNIT - 1) / UNIT);
  // bf16 has two workgroups per CU only where there are as many heads (units_per_workgroup)
  const int64_t round = fp8 || items >= 512 ? 256 * waves_per_simd((int)a.D, fp8, r.nt) : 256;
  r.grid = units < round ? units : round;
  return r;
}

template <int D, bool FP8, int NT, bool GENERAL>
hipError_t launch_decode_t(const DecodeParams &p, int64_t grid, hipStream_t stream) {
  hipLaunchKernelGGL((decode_kernel<D, FP8, NT, GENERAL>), dim3((unsigned)grid), dim3(NTHR), 0, stream, p);
  static const std::string name = [] {
    char b[96];
    snprintf(b, sizeof(b), "decode_kernel<%d, %s, %d, %s>", D, tf(FP8), NT, tf(GENERAL));
    return std::string(b);
  }();
  launch_log_add(reinterpret_cast<const void *>(&decode_kernel<D, FP8, NT, GENERAL>), name.c_str(), grid, NTHR);
  launch_log_plan("split=%d rblocks=%d", p.counters != nullptr, p.rblocks);
  return hipGetLastError();
}

template <int D, bool FP8, int NT>
hipError_t launch_decode_s(const DecodeParams &p, int64_t grid, hipStream_t stream) {
  return p.S > 1 || p.cap > 0.f ? launch_decode_t<D, FP8, NT, true>(p, grid, stream) : launch_decode_t<D, FP8, NT, false>(p, grid, stream);
}

template <int D, bool FP8>
hipError_t dispatch_decode(const DecodeParams &p, int nt, int64_t grid, hipStream_t stream) {
  if (nt == 1) return launch_decode_s<D, FP8, 1>(p, grid, stream);
  if constexpr (D == 128 || FP8)
    if (nt == 2) return launch_decode_s<D, FP8, 2>(p, grid, stream);
  if constexpr (D == 128)
    if (nt == 4) return launch_decode_s<D, FP8, 4>(p, grid, stream);
  return hipErrorInvalidValue;
}

}  // namespace

// For any plan of these sizes: two slots of its widest pass for each of at most 512 workgroups.
int64_t decode_workspace_bytes(const kfmi_decode_args &a) {
  const int64_t rows = a.Hq / a.Hkv * a.S;
  const int64_t units = a.B * a.Hkv * ((rows + 15) / 16) * ((a.max_pages * a.page_size + UNIT - 1) / UNIT);
  const int64_t slots = units < 512 ? units : 512;
  return slots > 1 ? KFMI_DECODE_COUNTER_BYTES + 2 * slots * 16 * widest(a, true) * (a.D + 2) * 4 : 0;
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
  p.num_pages = (int)a.num_pages;
  p.capacity = (int)(a.max_pages * a.page_size);
  p.window = (int)(a.window < p.capacity ? a.window : 0);  // a window of all keys is none
  p.B = (int)a.B; p.hq = (int)a.Hq; p.hk = (int)a.Hkv; p.S = (int)a.S;
  p.group = p.hq / p.hk;
  p.rows = p.group * p.S;
  p.rblocks = plan.rblocks;
  p.page_shift = log2_of(a.page_size);
  p.page_mask = (int)(a.page_size - 1);
  p.pages64 = a.index_flags & KFMI_I64_PAGES;
  p.len64 = a.index_flags & KFMI_I64_LENGTHS;
  constexpr double log2e = 1.4426950408889634;
  p.cap = (float)(a.softcap * log2e);
  // (a ratio of scale and cap beyond a float's range caps any score but 0)
  p.score_scale = a.softcap > 0 ? (float)fmin(2.0 * log2e * a.scale / a.softcap, 3.0e38) : 0.0f;
  p.slope = a.softcap == 0 ? (float)(a.scale * log2e) : p.cap > LARGE_CAP ? 1.0f : 2.0f * p.cap;
  p.offset = a.softcap == 0 || p.cap > LARGE_CAP ? 0.0f : p.cap;
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
