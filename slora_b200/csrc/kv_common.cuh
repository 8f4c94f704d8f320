// 8-bit paged KV cache: argument blocks, page lookup, 8-bit conversions and the exact rounding of quotients that the
// append, read, attention and eviction kernels share.
//
// A page holds `page` tokens of every KV head: values [page id][head][token][d] of one byte, one FP32 scale per (page,
// head) for k and one for v.  One (page, head) is a contiguous run of page * d bytes, so a head's tokens stream in
// runs of 1 to 32 KB wherever the pages lie, and the scale costs 4 bytes per run.
#pragma once

#include "lora_common.cuh"

namespace slora {

constexpr int kStatusNonfinite = SLORA_STATUS_NONFINITE;

struct KvCache {
  uint8_t* k;
  uint8_t* v;
  float* ks;
  float* vs;
  float* w;
  int64_t n_pages;
  int shift;  // log2 of the tokens of a page
  int hkv;
  int d;
};

struct KvBatch {
  const int64_t* table;
  int64_t table_stride;
  const int32_t* kv_len;
  const int32_t* q_start;
  const int32_t* q_len;
  int32_t* status;
  int n_seq;
  int max_q;
  int64_t max_tokens;  // max_pages * page: no sequence may be longer
  int64_t T;           // rows of q, k, v
};

// One sequence, checked: a bad one has no new tokens and no keys.
struct KvSeq {
  int kv, q, row;  // tokens in the cache, new ones among them, first row of the new ones
  bool bad;
};
__device__ __forceinline__ KvSeq kv_seq(const KvBatch& b, int i) {
  KvSeq s;
  s.kv = b.kv_len[i];
  s.q = b.q_len[i];
  s.row = b.q_start[i];
  s.bad = s.kv < 0 || s.kv > b.max_tokens || s.q < 0 || s.q > b.max_q || s.row < 0 ||
          (s.q > 0 && static_cast<int64_t>(s.row) + s.q > b.T);
  if (s.bad) s.kv = s.q = s.row = 0;
  return s;
}

// Page of position `pos` of sequence i, -1 when the table's entry is no page.
__device__ __forceinline__ int64_t kv_page(const KvCache& c, const KvBatch& b, int i, int pos) {
  const int64_t p = b.table[i * b.table_stride + (pos >> c.shift)];
  return p >= 0 && p < c.n_pages ? p : -1;
}

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
  return __byte_perm(a, b, sel);
}

// ---- 8-bit values ---------------------------------------------------------------------------------------------------
// Pairs of stored bytes become pairs of f16.  int8, without a conversion instruction: the byte with its sign bit flipped
// under the exponent byte 0x64 is 1024 + 128 + q, exact, and one packed subtraction (on the FMA pipe) leaves q.  e4m3: the
// conversion instruction for pairs; moving the fields by shifts and masks took three more on the ALU pipe and 17 % more
// time over the decode of 32 sequences.
template <int KIND>
struct Kv8;
template <>
struct Kv8<SLORA_KV_INT8> {
  static constexpr float kTop = 127.f;
  static constexpr float kScale = 1.f;  // what a converted pair still has to be multiplied by
  static constexpr bool kInt = true;
  // bytes -> bytes that pair() takes
  __device__ static __forceinline__ uint32_t prepare(uint32_t w) { return w ^ 0x80808080u; }
  __device__ static __forceinline__ uint32_t finish(uint32_t v) {  // v = (0x64, b1, 0x64, b0)
    uint32_t r;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(v), "r"(0x64806480u));
    return r;
  }
  // f16x2 of bytes 0, 1 / 2, 3 of a prepared word
  __device__ static __forceinline__ uint32_t lo(uint32_t w) { return finish(prmt(w, 0x64646464u, 0x4140)); }
  __device__ static __forceinline__ uint32_t hi(uint32_t w) { return finish(prmt(w, 0x64646464u, 0x4342)); }
  // the four values of a word
  __device__ static __forceinline__ void values(uint32_t w, float (&v)[4]) {
    const uint32_t x = w ^ 0x80808080u;  // under the exponent of 2^23: 2^23 + 128 + q, exact
    v[0] = __uint_as_float(prmt(x, 0x4b000000u, 0x7440)) - 8388736.f;
    v[1] = __uint_as_float(prmt(x, 0x4b000000u, 0x7441)) - 8388736.f;
    v[2] = __uint_as_float(prmt(x, 0x4b000000u, 0x7442)) - 8388736.f;
    v[3] = __uint_as_float(prmt(x, 0x4b000000u, 0x7443)) - 8388736.f;
  }
};
template <>
struct Kv8<SLORA_KV_E4M3> {
  static constexpr float kTop = 448.f;
  static constexpr float kScale = 1.f;
  static constexpr bool kInt = false;
  __device__ static __forceinline__ uint32_t prepare(uint32_t w) { return w; }
  __device__ static __forceinline__ uint32_t pair(uint32_t v) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<unsigned short>(v)));
    return r;
  }
  __device__ static __forceinline__ uint32_t lo(uint32_t w) { return pair(w); }
  __device__ static __forceinline__ uint32_t hi(uint32_t w) { return pair(w >> 16); }
  __device__ static __forceinline__ void values(uint32_t w, float (&v)[4]) {
    const uint32_t a = lo(w), b = hi(w);
    const float2 x = __half22float2(reinterpret_cast<const __half2&>(a)), y = __half22float2(reinterpret_cast<const __half2&>(b));
    v[0] = x.x, v[1] = x.y, v[2] = y.x, v[3] = y.y;
  }
};

// round((x + lo) / s) in the 8-bit type, to nearest, ties to even, of the exact quotient (s > 0; x + lo exact in two FP32
// words, |lo| <= ulp(x) / 2): the stored byte.  The FP32 quotient is within an ulp or so of the exact one, so it decides
// everywhere but next to a border between two 8-bit values; there the sign of x + lo - border * s does (fma: one
// rounding, and the difference is small).  Pages that are scaled anew sit on such borders often: their ratios are small
// fractions.
template <int KIND>
__device__ __noinline__ uint32_t kv_round(float x, float lo, float s) {
  const float y = __fdiv_rn(x, s);
  float m = fabsf(y);
  float step = 1.f, inv = 1.f;
  if (!Kv8<KIND>::kInt) {  // spacing of the type at m: three bits behind the leading one, 2^-9 below 2^-6
    const uint32_t e = max(__float_as_uint(m) >> 23, 121u);
    step = __uint_as_float((e - 3u) << 23);
    inv = __uint_as_float((257u - e) << 23);  // 2^(3 - (e - 127)), e <= 254 - 3 for every value below the clamp
    if (m > 1024.f) return (__float_as_uint(y) >> 31 << 7) | 0x7eu;
  } else {
    m = fminf(m, 1024.f);
  }
  const float k = m * inv;  // in steps, exact
  const float f = floorf(k);
  const float off = k - f;
  float r = off > 0.5f || (off == 0.5f && (static_cast<int>(f) & 1)) ? f + 1.f : f;
  if (fabsf(off - 0.5f) < 2e-4f) {
    const float border = copysignf((f + 0.5f) * step, y);
    const float diff = copysignf(1.f, y) * (__fmaf_rn(-border, s, x) + lo);
    r = diff > 0.f ? f + 1.f : diff < 0.f ? f : f + static_cast<float>(static_cast<int>(f) & 1);
  }
  const uint32_t sign = __float_as_uint(y) >> 31;
  if (Kv8<KIND>::kInt) {
    const int q = static_cast<int>(fminf(r, 127.f));
    return static_cast<uint32_t>(sign ? -q : q) & 0xffu;
  }
  const float v = fminf(r * step, 448.f);  // a value of the type
  const uint32_t h = __half_as_ushort(__float2half_rn(v * (1.f / 256.f)));  // sign-less f16 fields, exact
  return (sign << 7) | (h >> 7);
}

// The same for four values x[e] = from[e] * by (by: what the values were scaled with; 1 for new ones) at once, packed into
// a word.  y[e] = from[e] * mul with mul = by / s is, up to roundings, within 2^-22 of the exact quotient; only where that
// is next to a border kv_round decides (for e4m3 also below 2^-6, where the steps no longer follow the exponent).
template <int KIND>
__device__ __forceinline__ uint32_t kv_round4(const float (&from)[4], float by, float mul, float s) {
  uint32_t w;
  bool near = !(mul < 1e37f);  // a scale next to FP32's smallest numbers has no inverse
  if (Kv8<KIND>::kInt) {
    float t[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float y = fminf(fmaxf(from[e] * mul, -127.f), 127.f);
      t[e] = y + 12582912.f;  // 1.5 * 2^23: the sum's last bits are y rounded to a whole number
      near = near || fabsf(y - (t[e] - 12582912.f)) > 0.4999f;
    }
    w = prmt(prmt(__float_as_uint(t[0]), __float_as_uint(t[1]), 0x0040), prmt(__float_as_uint(t[2]), __float_as_uint(t[3]), 0x0040), 0x5410);
  } else {
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      y[e] = from[e] * mul;
      const uint32_t b = __float_as_uint(y[e]) & 0x7fffffffu;
      near = near || (b & 0xfffffu) - 0x7ffe0u < 0x40u || b - 1u < 0x3c800000u - 1u;
    }
    unsigned short lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(y[1]), "f"(y[0]));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(y[3]), "f"(y[2]));
    w = lo | static_cast<uint32_t>(hi) << 16;
  }
  if (near) {
    w = 0;
#pragma unroll 1
    for (int e = 0; e < 4; ++e) {
      const float f = e == 0 ? from[0] : e == 1 ? from[1] : e == 2 ? from[2] : from[3];
      const float x = f * by;
      w |= kv_round<KIND>(x, __fmaf_rn(f, by, -x), s) << (8 * e);
    }
  }
  return w;
}
}  // namespace slora
