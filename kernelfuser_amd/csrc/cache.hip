// The paged key-value cache: rows prepared and written into it, and its pages
// read back as dense tensors (the layout is described in kfmi.h).
//
// Both are memory-bound: a row of D values is D/8 lanes of 8 values each (one
// 16-lane DPP row at D = 128), 16 bytes of bf16 or 8 bytes of e4m3 per lane.
//
// Writing: norm y = bf16 chain of x / sqrt(mean x^2 + eps) * gamma, rotation y cos + partner sin at the
// token's own table row (rows_common.h), then, for e4m3, y / 2^e rounded.  8192 tokens of 32 + 2 x 8 heads of
// D = 128 take 35 us (205 MB, 5.9 TB/s), 4000 e4m3 tokens of 16 + 2 x 8 of D = 256 26 us (116 MB), where the
// row arithmetic and the conversion fill 70% of the vector slots; one token 2.6 us, a launch.
// Reading: 8 sequences of 4096 e4m3 keys, 8 heads of D = 256, 60 us (344 MB, 5.7 TB/s).
#include <cstdio>
#include <string>

#include "cache_common.h"
#include "kfmi_launch.h"
#include "rows_common.h"

namespace kfmi {
namespace {

struct WriteParams {
  const uint16_t *q, *k, *v, *gq, *gk, *cos, *sin;
  const void *positions, *slots;
  uint16_t *qn, *kn;
  char *k_cache, *v_cache;
  uint8_t *k_scale, *v_scale;
  int64_t qs[3], ks[3], vs[3];  // strides of B, H, S in elements
  int64_t ps[2], ss[2];
  int64_t cs[3], es[2];
  uint32_t S, T, hq, hk;  // T = B * S tokens; heads of q (0: none) and of k
  int64_t table_rows, slot_end;
  int page_shift, page_mask;
  bool pos64, slot64;
  float eps;
};

// Rows from which a lane takes four heads of its token instead of one (32 + 2 x 8 heads of D = 128:
// 24576 rows 4.9 us with one, 5.6 with four; 98304 rows 14.9 and 10.9).
constexpr int64_t WIDE_ROWS = 1 << 15;

// Bytes (read and written) from which reading the cache back leaves the caches alone: what
// is larger than them comes from memory in any case, and then faster (268 MB of bf16 45.8 instead
// of 51.1 us); what is smaller may be in them (201 MB of e4m3 25.3 instead of 35.0 us).
constexpr int64_t STREAM_BYTES = 1 << 28;

// A row of 8 values per lane in e4m3 with its scale 2^e: e is the smallest
// exponent (at least -124: e4m3's smallest step, 2^-9, times 2^-124 is bf16's) with max|row| <= 448 * 2^e over the finite values, so that the
// division by the scale is exact and the conversion (round to nearest even)
// cannot overflow.  448 = 0.875 * 2^9: with max = m * 2^x, 0.5 <= m < 1, e is
// x - 9, one more where m > 0.875.  Only at e = 120 could a rounding up (to
// 256 * 2^120 = 2^128) leave bf16's range: 240 is the most there.  Returns the
// payload; byte = e + 127.
template <int LPR>
__device__ __forceinline__ u32x2_t quantise_row(const float (&y)[8], uint32_t &byte) {
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(y[j]) & 0x7fffffffu);
  top = row_max_u32<LPR>(top);
  const bool large = __any(top >= 0x7f000000u);  // 2^127 and more, infinities, NaN: rarely
  if (large) {
    top = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t a = __float_as_uint(y[j]) & 0x7fffffffu;
      top = max(top, a < 0x7f800000u ? a : 0u);
    }
    top = row_max_u32<LPR>(top);
  }
  const int ex = (int)(top >> 23) - 126 - 9 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
  const int e = top == 0 ? 0 : max(ex, -124);
  byte = (uint32_t)(e + 127);
  const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
  float z[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) z[j] = y[j] * inv;
  if (large) {
    const float most = e == 120 ? 240.0f : 448.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      z[j] = __builtin_amdgcn_fmed3f(z[j], -most, most);
      if ((__float_as_uint(y[j]) & 0x7f800000u) == 0x7f800000u) z[j] = __uint_as_float(0x7fc00000u);
    }
  }
  u32x2_t w;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    int x = __builtin_amdgcn_cvt_pk_fp8_f32(z[4 * i], z[4 * i + 1], 0, false);
    x = __builtin_amdgcn_cvt_pk_fp8_f32(z[4 * i + 2], z[4 * i + 3], x, true);
    w[i] = (uint32_t)x;
  }
  return w;
}

// A workgroup takes 256 / LPR consecutive tokens (blockIdx.x) of a unit of U
// heads of q, of k or of v (blockIdx.y), one 16-byte chunk per lane and row.  A lane's U
// rows share the token's table rows, gamma, position and slot.  Every load is
// issued before the first is waited for, and every row is finished before one is stored
// (stores and loads share a counter).
template <int D, int ST, bool ROPE, bool FP8, int U>
__global__ __launch_bounds__(256) void cache_write_kernel(WriteParams p) {
  constexpr int LPR = D / 8;
  constexpr int HALF = LPR / 2;
  const uint32_t t_ = blockIdx.x * (256 / LPR) + threadIdx.x / LPR, lc = threadIdx.x % LPR;
  const bool live = t_ < p.T;
  const uint32_t t = live ? t_ : p.T - 1;  // loads stay in bounds; nothing is stored for this lane
  const uint32_t b = t / p.S, s = t - b * p.S;
  const uint32_t uq = (p.hq + U - 1) / U, uk = (p.hk + U - 1) / U;
  const uint32_t unit = blockIdx.y;  // everything from here to the row is workgroup-uniform
  const bool is_q = unit < uq, is_v = unit >= uq + uk;
  const uint32_t nh = is_q ? p.hq : p.hk;
  const uint32_t h0 = (is_q ? unit : is_v ? unit - uq - uk : unit - uq) * U;
  const uint16_t *src = is_q ? p.q : is_v ? p.v : p.k;
  const int64_t s0 = is_q ? p.qs[0] : is_v ? p.vs[0] : p.ks[0];
  const int64_t s1 = is_q ? p.qs[1] : is_v ? p.vs[1] : p.ks[1];
  const int64_t s2 = is_q ? p.qs[2] : is_v ? p.vs[2] : p.ks[2];
  const uint16_t *row = src + b * s0 + s * s2 + lc * 8;
  u32x4_t held[U];  // the row as it is, then prepared
#pragma unroll
  for (int i = 0; i < U; ++i) held[i] = ld16_nt(row + min(h0 + i, nh - 1) * s1);
  const int64_t slot = load_index(p.slots, p.slot64, b * p.ss[0] + s * p.ss[1]);
  const bool bad_slot = slot >= p.slot_end;
  const uint32_t nan2 = 0x7fc07fc0u;
  if (!is_v) {
    const u32x4_t gw = ld16((is_q ? p.gq : p.gk) + lc * 8);
    bool bad_pos = false;
    u32x4_t cw, sw;
    if constexpr (ROPE) {
      int64_t pos = load_index(p.positions, p.pos64, b * p.ps[0] + s * p.ps[1]);
      bad_pos = pos < 0 || pos >= p.table_rows;
      pos = bad_pos ? 0 : pos;
      cw = ld16(p.cos + pos * D + lc * 8);
      sw = ld16(p.sin + pos * D + lc * 8);
    }
    asm volatile("" ::: "memory");
    float g[8], c[8], sn[8];
    unpack8(gw, g);
    if constexpr (ROPE) {
      const uint32_t flip = lc < HALF ? 0x80008000u : 0u;  // first half: n*c - np*s
      sw ^= u32x4_t{flip, flip, flip, flip};
      unpack8(cw, c);
      unpack8(sw, sn);
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      float x[8], y[8];
      unpack8(held[i], x);
      const float inv = row_inv_rms<LPR, D>(x, p.eps);
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = norm_elem<ST>(x[j], inv, g[j]);
      if constexpr (ROPE) {
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = rope_elem<ST>(y[j], partner_f32<LPR>(y[j]), c[j], sn[j], false);
      }
      held[i] = pack8(y);
      if (bad_pos) held[i] = u32x4_t{nan2, nan2, nan2, nan2};
      asm volatile("" ::"v"(held[i]));  // finished here, with every lane active, not in the stores' branches
    }
  }
  u32x2_t payload[U];
  uint32_t byte[U];
  if constexpr (FP8) {
    if (!is_q) {
#pragma unroll
      for (int i = 0; i < U; ++i) {
        float f[8];
        unpack8(held[i], f);
        payload[i] = quantise_row<LPR>(f, byte[i]);
        asm volatile("" ::"v"(payload[i]), "v"(byte[i]));
      }
    }
  }
  if (!live) return;
  if (is_q || (p.kn && !is_v)) {
    uint16_t *dst = (is_q ? p.qn : p.kn) + ((int64_t)(b * nh + h0) * p.S + s) * D + lc * 8;
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (h0 + i < nh)
        st16_nt(dst + (int64_t)i * p.S * D, bad_slot ? u32x4_t{nan2, nan2, nan2, nan2} : held[i]);
  }
  if (is_q || slot < 0 || bad_slot) return;
  const int64_t page = slot >> p.page_shift, at = slot & p.page_mask;
  const int64_t off = page * p.cs[0] + h0 * p.cs[1] + at * p.cs[2] + lc * 8;
  char *cache = (is_v ? p.v_cache : p.k_cache) + off * (FP8 ? 1 : 2);
#pragma unroll
  for (int i = 0; i < U; ++i) {
    if (h0 + i >= nh) break;
    if constexpr (FP8) {
      __builtin_nontemporal_store(payload[i], reinterpret_cast<u32x2_t *>(cache + i * p.cs[1]));
      if (lc == 0) (is_v ? p.v_scale : p.k_scale)[page * p.es[0] + (h0 + i) * p.es[1] + at] = (uint8_t)byte[i];
    } else {
      st16_nt(reinterpret_cast<uint16_t *>(cache) + i * p.cs[1], held[i]);
    }
  }
}

template <int D, int ST, bool ROPE, bool FP8, int U>
hipError_t launch_write_t(const WriteParams &p, hipStream_t stream) {
  constexpr uint32_t tokens = 256 / (D / 8);
  const dim3 grid((p.T + tokens - 1) / tokens, (p.hq + U - 1) / U + 2 * ((p.hk + U - 1) / U));
  hipLaunchKernelGGL((cache_write_kernel<D, ST, ROPE, FP8, U>), grid, dim3(256), 0, stream, p);
  static const std::string name = [] {
    char b[96];
    snprintf(b, sizeof(b), "cache_write_kernel<%d, %d, %s, %s, %d>", D, ST, tf(ROPE), tf(FP8), U);
    return std::string(b);
  }();
  launch_log_add(reinterpret_cast<const void *>(&cache_write_kernel<D, ST, ROPE, FP8, U>), name.c_str(),
                 (int64_t)grid.x * grid.y, 256);
  return hipGetLastError();
}

template <int D, int ST, bool ROPE, bool FP8>
hipError_t launch_write_u(const WriteParams &p, hipStream_t stream) {
  const int64_t rows = (int64_t)p.T * (p.hq + 2 * p.hk);
  return rows >= WIDE_ROWS ? launch_write_t<D, ST, ROPE, FP8, 4>(p, stream) : launch_write_t<D, ST, ROPE, FP8, 1>(p, stream);
}

template <int D, int ST>
hipError_t dispatch_write(const WriteParams &p, bool rope, bool fp8, hipStream_t s) {
  if (rope) return fp8 ? launch_write_u<D, ST, true, true>(p, s) : launch_write_u<D, ST, true, false>(p, s);
  return fp8 ? launch_write_u<D, ST, false, true>(p, s) : launch_write_u<D, ST, false, false>(p, s);
}

struct ReadParams {
  const char *k_cache, *v_cache;
  const uint8_t *k_scale, *v_scale;
  const void *pages, *lengths;
  uint16_t *k, *v;
  int64_t cs[3], es[2];
  int64_t pages_stride, lengths_stride, num_pages, capacity;
  uint32_t L, hk;
  int page_shift, page_mask;
  bool pages64, len64;
};

// 256 / LPR rows of K and V of head blockIdx.y of sequence blockIdx.z per
// workgroup.  NT: loads that leave the caches alone (see STREAM_BYTES).
template <int D, bool FP8, bool NT>
__global__ __launch_bounds__(256) void cache_read_kernel(ReadParams p) {
  constexpr int LPR = D / 8;
  const int64_t b = blockIdx.z, h = blockIdx.y;
  const uint32_t lc = threadIdx.x % LPR, j = blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
  if (j >= p.L) return;
  const int64_t len = load_index(p.lengths, p.len64, b * p.lengths_stride);
  const uint32_t nan2 = 0x7fc07fc0u;
  u32x4_t out[2] = {{0u, 0u, 0u, 0u}, {0u, 0u, 0u, 0u}};
  bool bad = len < 0 || len > p.capacity;
  if (!bad && j < len) {
    const int64_t page = load_index(p.pages, p.pages64, b * p.pages_stride + (j >> p.page_shift));
    bad = page < 0 || page >= p.num_pages;
    if (!bad) {
      const int64_t at = j & p.page_mask;
      const int64_t off = page * p.cs[0] + h * p.cs[1] + at * p.cs[2] + lc * 8;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const char *c = x ? p.v_cache : p.k_cache;
        if constexpr (FP8) {
          const u32x2_t *src = reinterpret_cast<const u32x2_t *>(c + off);
          const u32x2_t w = NT ? __builtin_nontemporal_load(src) : *src;
          const float sc = scale_value((x ? p.v_scale : p.k_scale)[page * p.es[0] + h * p.es[1] + at]);
          float f[8];
          unpack_e4m3(w, f);
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] *= sc;
          out[x] = pack8(f);
        } else {
          const uint16_t *src = reinterpret_cast<const uint16_t *>(c) + off;
          out[x] = NT ? ld16_nt(src) : ld16(src);
        }
      }
    }
  }
  if (bad) out[0] = out[1] = u32x4_t{nan2, nan2, nan2, nan2};
  const int64_t o = ((b * p.hk + h) * p.L + j) * D + lc * 8;
  st16_nt(p.k + o, out[0]);
  st16_nt(p.v + o, out[1]);
}

template <int D, bool FP8, bool NT>
hipError_t launch_read_t(const ReadParams &p, int64_t B, hipStream_t stream) {
  constexpr uint32_t rows = 256 / (D / 8);
  const dim3 grid((p.L + rows - 1) / rows, p.hk, (unsigned)B);
  hipLaunchKernelGGL((cache_read_kernel<D, FP8, NT>), grid, dim3(256), 0, stream, p);
  static const std::string name = [] {
    char b[96];
    snprintf(b, sizeof(b), "cache_read_kernel<%d, %s, %s>", D, tf(FP8), tf(NT));
    return std::string(b);
  }();
  launch_log_add(reinterpret_cast<const void *>(&cache_read_kernel<D, FP8, NT>), name.c_str(),
                 (int64_t)grid.x * grid.y * grid.z, 256);
  return hipGetLastError();
}

template <int D, bool FP8>
hipError_t launch_read_n(const ReadParams &p, int64_t B, hipStream_t stream) {
  const int64_t bytes = 2 * B * p.hk * p.L * D * (FP8 ? 3 : 4);
  return bytes >= STREAM_BYTES ? launch_read_t<D, FP8, true>(p, B, stream) : launch_read_t<D, FP8, false>(p, B, stream);
}

}  // namespace

hipError_t launch_cache_write(const kfmi_cache_write_args &a, int style, hipStream_t stream) {
  WriteParams p{};
  p.q = (const uint16_t *)a.q; p.k = (const uint16_t *)a.k; p.v = (const uint16_t *)a.v;
  p.gq = (const uint16_t *)a.gq; p.gk = (const uint16_t *)a.gk;
  p.cos = (const uint16_t *)a.cos; p.sin = (const uint16_t *)a.sin;
  p.positions = a.positions; p.slots = a.slots;
  p.qn = (uint16_t *)a.qn; p.kn = (uint16_t *)a.kn;
  p.k_cache = (char *)a.k_cache; p.v_cache = (char *)a.v_cache;
  p.k_scale = (uint8_t *)a.k_scale; p.v_scale = (uint8_t *)a.v_scale;
  for (int i = 0; i < 3; ++i) {
    p.qs[i] = a.q_stride[i]; p.ks[i] = a.k_stride[i]; p.vs[i] = a.v_stride[i]; p.cs[i] = a.cache_stride[i];
  }
  for (int i = 0; i < 2; ++i) {
    p.ps[i] = a.position_stride[i]; p.ss[i] = a.slot_stride[i]; p.es[i] = a.scale_stride[i];
  }
  p.S = (uint32_t)a.S;
  p.T = (uint32_t)(a.B * a.S);
  p.hq = a.q ? (uint32_t)a.Hq : 0u;
  p.hk = (uint32_t)a.Hkv;
  p.table_rows = a.table_rows;
  p.slot_end = a.num_pages * a.page_size;
  p.page_shift = log2_of(a.page_size);
  p.page_mask = (int)(a.page_size - 1);
  p.pos64 = a.index_flags & KFMI_I64_POSITIONS;
  p.slot64 = a.index_flags & KFMI_I64_SLOTS;
  p.eps = (float)a.eps;
  const bool rope = a.cos != nullptr, fp8 = a.cache_type == KFMI_CACHE_E4M3;
#define KFMI_STYLES(D)                                                 \
  switch (style) {                                                     \
    case ST_HF: return dispatch_write<D, ST_HF>(p, rope, fp8, stream); \
    case ST_LEGACY: return dispatch_write<D, ST_LEGACY>(p, rope, fp8, stream); \
    case ST_FP32: return dispatch_write<D, ST_FP32>(p, rope, fp8, stream); \
  }
  if (a.D == 128) {
    KFMI_STYLES(128)
  } else {
    KFMI_STYLES(256)
  }
#undef KFMI_STYLES
  return hipErrorInvalidValue;
}

hipError_t launch_cache_read(const kfmi_cache_read_args &a, hipStream_t stream) {
  ReadParams p{};
  p.k_cache = (const char *)a.k_cache; p.v_cache = (const char *)a.v_cache;
  p.k_scale = (const uint8_t *)a.k_scale; p.v_scale = (const uint8_t *)a.v_scale;
  p.pages = a.pages; p.lengths = a.lengths;
  p.k = (uint16_t *)a.k; p.v = (uint16_t *)a.v;
  for (int i = 0; i < 3; ++i) p.cs[i] = a.cache_stride[i];
  for (int i = 0; i < 2; ++i) p.es[i] = a.scale_stride[i];
  p.pages_stride = a.pages_stride; p.lengths_stride = a.lengths_stride;
  p.num_pages = a.num_pages;
  p.capacity = a.max_pages * a.page_size;
  p.L = (uint32_t)a.L;
  p.hk = (uint32_t)a.Hkv;
  p.page_shift = log2_of(a.page_size);
  p.page_mask = (int)(a.page_size - 1);
  p.pages64 = a.index_flags & KFMI_I64_PAGES;
  p.len64 = a.index_flags & KFMI_I64_LENGTHS;
  const bool fp8 = a.cache_type == KFMI_CACHE_E4M3;
  if (a.D == 128) return fp8 ? launch_read_n<128, true>(p, a.B, stream) : launch_read_n<128, false>(p, a.B, stream);
  return fp8 ? launch_read_n<256, true>(p, a.B, stream) : launch_read_n<256, false>(p, a.B, stream);
}

}  // namespace kfmi
