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

// The larger magnitudes of two pairs of f16.
__device__ __forceinline__ uint32_t max_abs_f16(uint32_t a, uint32_t b) {
  uint32_t r, t;
  asm("abs.f16x2 %0, %1;" : "=r"(t) : "r"(b));
  asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(t));
  return r;
}
// The largest stored magnitude of 16 bytes.
template <int KIND>
__device__ __forceinline__ float kv_top(const uint4& v) {
  using V8 = Kv8<KIND>;
  uint32_t m = 0;
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t x = V8::prepare(w[i]);
    m = max_abs_f16(max_abs_f16(m, V8::lo(x)), V8::hi(x));
  }
  const float2 f = __half22float2(reinterpret_cast<const __half2&>(m));
  return fmaxf(f.x, f.y) * V8::kScale;
}

// Scales below FP32's smallest normal number count as 0 (their inverse need not exist).
constexpr float kLeastScale = 1.17549435e-38f;
__device__ __forceinline__ float kv_scale(float s) { return s < kLeastScale ? 0.f : s; }

// round(from[e] * by / s) in the 8-bit type for four values (by: what they were scaled with; 1 for new ones), to nearest,
// ties to even, of the exact quotient, packed into a word.  s >= kLeastScale, mul = by / s.
//
// from * mul is, up to two or three roundings, within 2^-21.4 of the quotient, so it decides everywhere but next to a border
// between two 8-bit values (for e4m3 also below 2^-6, where the steps no longer follow the exponent); there the sign of
// from * by - border * s does, exactly: from * by in two words, an fma with one rounding, and the difference is small.
// Pages that are scaled anew sit on such borders often: their ratios are small fractions.
// int8: from * mul + 384 lies in [256, 512), whose FP32 numbers are 2^-15 apart: one fma leaves 128 + the quotient in fixed
// point, twice that plus a half its rounding in byte 2 and what was rounded in the lower half.
// far: some value may lie beyond the type's range (an infinity): all take the exact way, which clamps.
template <int KIND>
__device__ __forceinline__ uint32_t kv_round4(const float (&from)[4], float by, float mul, float s, bool far = false) {
  uint32_t r[4];
  float y[4];
  bool near = far;
  if (Kv8<KIND>::kInt) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      r[e] = __float_as_uint(__fmaf_rn(from[e], mul, 384.f)) * 2u + 0x8000u;
      near = near || r[e] * 0x10000u + 0x40000u <= 0x80000u;  // within two steps of a half
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      y[e] = from[e] * mul;
      near = near || __float_as_uint(y[e]) * 0x1000u - 0x7ffe0000u < 0x40000u || (fabsf(y[e]) < 0.015625f && from[e] != 0.f);
    }
  }
  if (near) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float top = Kv8<KIND>::kTop;
      const float q = fminf(fmaxf(from[e] * mul, -top), top);
      // steps of the type at q: 1, or three bits behind the leading one and 2^-9 below 2^-6
      float step = 1.f, inv = 1.f;
      if (!Kv8<KIND>::kInt) {
        const uint32_t x = max(__float_as_uint(fabsf(q)) >> 23, 121u);
        step = __uint_as_float((x - 3u) << 23);
        inv = __uint_as_float((257u - x) << 23);
      }
      const float low = floorf(q * inv);  // the value is low or low + 1 steps
      const float x = from[e] * by;
      const float over = __fmaf_rn(-(low + 0.5f) * step, s, x) + __fmaf_rn(from[e], by, -x);
      const float odd = static_cast<float>(static_cast<int>(low) & 1);
      const float k = over > 0.f ? low + 1.f : over < 0.f ? low : low + odd;
      y[e] = k * step;
      r[e] = static_cast<uint32_t>(static_cast<int>(fminf(fmaxf(k, -top), top)) + 128) << 16;
    }
  }
  if (Kv8<KIND>::kInt) return prmt(prmt(r[0], r[1], 0x0062), prmt(r[2], r[3], 0x0062), 0x5410) ^ 0x80808080u;
  unsigned short lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(y[1]), "f"(y[0]));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(y[3]), "f"(y[2]));
  return lo | static_cast<uint32_t>(hi) << 16;
}

}  // namespace slora
