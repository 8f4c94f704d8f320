// Rotary embedding of q and k, the append of new tokens to the 8-bit cache, and reading it back.
//
// Rotary: element pairs (x0, x1) of a head turn by position * frequency.  The angle is reduced in 64 bits (position *
// turns, minus the nearest whole number: a position of 10^6 keeps 2^-30 of a turn, where FP32 would keep 2^-4) and only
// the remainder goes to sincospif.  Cosines and sines of a block of tokens are worked out once, in shared memory, and
// serve all heads.  A row of a head is 8 elements a lane (16-byte loads and stores); in the half layout the partner of a
// value sits rot / 16 lanes away (one shuffle per element), in the interleaved layout in the same lane.
// What bounds it: q, k read and written once (16-bit), at the copy rate; one token: launch and one chain of loads.
//
// Append: the new tokens of one page belong to one CTA (the scale of a (page, head) is a maximum over them) and a warp takes
// a (head, k or v): a first walk over the tokens for the maximum, a second that quantises (its loads come from L1).
// When the scale grows, the page's older values are rounded to the new one in place.
#pragma once

#include "kv_common.cuh"

namespace slora {

constexpr int kRowThreads = 256;
constexpr int kRowWarps = kRowThreads / 32;

struct RotaryArgs {
  const int64_t* positions;
  const double* turns;
  float factor;
  int rot;     // elements of a head that turn
  int layout;  // 0 half, 1 interleaved
  int inverse;
};

struct RowArgs {  // rotary alone
  RotaryArgs r;
  const void* src[2];  // q, k
  void* dst[2];
  int64_t src_stride[2], dst_stride[2];
  int heads[2];
  int64_t T;
  int tokens_per_cta;
  int head_splits;
};

struct AppendArgs {
  KvCache c;
  KvBatch b;
  RotaryArgs r;
  const void* q;
  void* q_out;
  const void* k;
  const void* v;
  int64_t q_stride, q_out_stride, k_stride, v_stride;
  int hq;
  int head_splits;
  int max_units;  // pages a sequence's new tokens touch, at most
};

// (cos, sin) of `n` tokens from `t0` on into cs[n][rot / 2].
__device__ __forceinline__ void rotary_table(const RotaryArgs& r, int64_t t0, int n, float2* cs) {
  const int half = r.rot >> 1;
  for (int i = threadIdx.x; i < n * half; i += blockDim.x) {
    const int t = i / half, p = i - t * half;
    const double a = static_cast<double>(r.positions[t0 + t]) * r.turns[p];
    float s, c;
    sincospif(2.f * static_cast<float>(a - rint(a)), &s, &c);
    cs[i] = make_float2(c * r.factor, (r.inverse ? -s : s) * r.factor);
  }
}

// Turns the eight elements `x` that this lane holds of a head row (elements 8 sub .. 8 sub + 7; all lanes of the warp take
// part) by the row's cosines and sines.
__device__ __forceinline__ void rotary_turn(float (&x)[8], const float2* cs, int sub, int rot, int layout) {
  if (layout == 0) {
    const int far = rot >> 4;  // lanes between the partners
    const bool low = sub < far, in = sub < 2 * far;
    const int lane = threadIdx.x & 31;
    const int other = low ? lane + far : in ? lane - far : lane;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float y = __shfl_sync(0xffffffffu, x[e], other);
      if (in) {
        const float2 w = cs[8 * (low ? sub : sub - far) + e];
        x[e] = low ? x[e] * w.x - y * w.y : y * w.y + x[e] * w.x;
      }
    }
  } else if (8 * sub < rot) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 w = cs[4 * sub + e];
      const float a = x[2 * e], b = x[2 * e + 1];
      x[2 * e] = a * w.x - b * w.y;
      x[2 * e + 1] = a * w.y + b * w.x;
    }
  }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  union {
    uint4 u;
    T e[8];
  } v;
#pragma unroll
  for (int e = 0; e < 8; ++e) v.e[e] = from_f32<T>(x[e]);
  *reinterpret_cast<uint4*>(p) = v.u;
}

// Heads [h0, h1) of tokens [t0, t0 + n): turned rows src -> dst.  Rows of a warp's step: 256 / D.
template <int D, typename T>
__device__ __forceinline__ void rotary_rows(const RotaryArgs& r, const T* src, T* dst, int64_t src_stride, int64_t dst_stride,
                                            int64_t t0, int n, int h0, int h1, const float2* cs) {
  constexpr int kLanes = D / 8, kRows = 32 / kLanes;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane % kLanes;
  const int heads = h1 - h0, rows = n * heads, half = r.rot >> 1;
  for (int base = warp * kRows; base < rows; base += kRowWarps * kRows) {
    const int row = base + lane / kLanes;
    const bool real = row < rows;
    const int t = real ? row / heads : 0, h = h0 + (real ? row - t * heads : 0);
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (real) cvt8<T>(*reinterpret_cast<const uint4*>(src + (t0 + t) * src_stride + h * D + 8 * sub), x);
    rotary_turn(x, cs + t * half, sub, r.rot, r.layout);
    if (real) store8<T>(dst + (t0 + t) * dst_stride + h * D + 8 * sub, x);
  }
}

template <int D, typename T>
__global__ void __launch_bounds__(kRowThreads) rotary_kernel(const RowArgs a) {
  extern __shared__ float2 cs[];
  pdl_launch_dependents();
  pdl_wait();
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * a.tokens_per_cta;
  const int n = static_cast<int>(a.T - t0 < a.tokens_per_cta ? a.T - t0 : a.tokens_per_cta);
  rotary_table(a.r, t0, n, cs);
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const int h0 = static_cast<int>(static_cast<int64_t>(a.heads[w]) * blockIdx.y / a.head_splits);
    const int h1 = static_cast<int>(static_cast<int64_t>(a.heads[w]) * (blockIdx.y + 1) / a.head_splits);
    if (h1 > h0)
      rotary_rows<D, T>(a.r, static_cast<const T*>(a.src[w]), static_cast<T*>(a.dst[w]), a.src_stride[w], a.dst_stride[w], t0,
                        n, h0, h1, cs);
  }
}

// The (sequence, page) of a CTA: units are the pages that a sequence's new tokens touch, over all sequences.
struct AppendUnit {
  int seq, block;
};
__device__ __forceinline__ int append_units(const AppendArgs& a, const KvSeq& s) {
  return s.q == 0 ? 0 : ((s.kv - 1) >> a.c.shift) - (max(s.kv - s.q, 0) >> a.c.shift) + 1;
}
// Unit u, and whether there is one.  Every thread adds up a run of sequences.
__device__ __forceinline__ bool append_find(const AppendArgs& a, int u, AppendUnit* out) {
  __shared__ int sums[kRowWarps];
  __shared__ AppendUnit found;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (a.b.n_seq + kRowThreads - 1) / kRowThreads;
  const int i0 = min(tid * per, a.b.n_seq), i1 = min(i0 + per, a.b.n_seq);
  int mine = 0;
  for (int i = i0; i < i1; ++i) {
    const KvSeq s = kv_seq(a.b, i);
    if ((s.bad || s.q > s.kv) && u == 0 && blockIdx.y == 0) set_status(a.b.status, SLORA_STATUS_BAD_TABLE);
    mine += append_units(a, s);
  }
  int incl = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int n = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += n;
  }
  if (lane == 31) sums[warp] = incl;
  if (tid == 0) found.seq = -1;
  __syncthreads();
  int before = incl - mine;
#pragma unroll
  for (int w = 0; w < kRowWarps; ++w)
    if (w < warp) before += sums[w];
  if (u >= before && u < before + mine) {
    for (int i = i0; i < i1; ++i) {
      const KvSeq s = kv_seq(a.b, i);
      const int n = append_units(a, s);
      if (u < before + n) {
        found.seq = i;
        found.block = (max(s.kv - s.q, 0) >> a.c.shift) + u - before;
        break;
      }
      before += n;
    }
  }
  __syncthreads();
  *out = found;
  return found.seq >= 0;
}

// NaN -> 0, infinities -> the largest FP32; tells whether x was one of them.
__device__ __forceinline__ bool kv_finite(float& x) {
  if (fabsf(x) <= 3.4028234663852886e38f) return true;
  x = x == x ? copysignf(3.4028234663852886e38f, x) : 0.f;
  return false;
}

// One (page, head) of k or v: new tokens in slots [n0, n1) whose rows start at `src`, older ones in slots [0, n0).
template <int D, int KIND, typename T>
__device__ __forceinline__ void append_page(const AppendArgs& a, const T* src, int64_t stride, int n0, int n1, uint8_t* page,
                                            float* scale, const float2* cs, bool turn) {
  constexpr int kLanes = D / 8, kRows = 32 / kLanes;
  using V8 = Kv8<KIND>;
  const int lane = threadIdx.x & 31, sub = lane % kLanes, rr = lane / kLanes, half = a.r.rot >> 1;
  const float s_old = n0 > 0 ? *scale : 0.f;
  float x[8];
  auto load = [&](int base) {
    const int i = base + rr;
    const bool real = i < n1;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = 0.f;
    if (real) cvt8<T>(*reinterpret_cast<const uint4*>(src + static_cast<int64_t>(i - n0) * stride + 8 * sub), x);
    if (turn) rotary_turn(x, cs + (real ? i - n0 : 0) * half, sub, a.r.rot, a.r.layout);
    return real;
  };
  float top = 0.f;
  bool fine = true;
  for (int base = n0; base < n1; base += kRows) {
    load(base);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const bool ok = kv_finite(x[e]);
      fine = fine && ok;
      top = fmaxf(top, ok ? fabsf(x[e]) : 0.f);
    }
  }
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  if (!fine) set_status(a.b.status, kStatusNonfinite);
  const float s_new = fmaxf(s_old, __fdiv_rn(top, V8::kTop));
  if (s_new != s_old && n0 > 0) {
    // older values at the new scale: 16 bytes a lane
    const float mul = __fdiv_rn(s_old, s_new);
#pragma unroll 2
    for (int i = lane; i < n0 * D / 16; i += 32) {
      const uint4 w = reinterpret_cast<const uint4*>(page)[i];
      float q[4];
      uint4 y;
      V8::values(w.x, q);
      y.x = kv_round4<KIND>(q, s_old, mul, s_new);
      V8::values(w.y, q);
      y.y = kv_round4<KIND>(q, s_old, mul, s_new);
      V8::values(w.z, q);
      y.z = kv_round4<KIND>(q, s_old, mul, s_new);
      V8::values(w.w, q);
      y.w = kv_round4<KIND>(q, s_old, mul, s_new);
      reinterpret_cast<uint4*>(page)[i] = y;
    }
  }
  const float mul = s_new > 0.f ? __fdiv_rn(1.f, s_new) : 0.f;
#pragma unroll 2
  for (int base = n0; base < n1; base += kRows) {
    const bool real = load(base);
    uint2 w = make_uint2(0, 0);
    if (s_new > 0.f) {
#pragma unroll
      for (int e = 0; e < 8; ++e) kv_finite(x[e]);
      const float lo[4] = {x[0], x[1], x[2], x[3]}, hi[4] = {x[4], x[5], x[6], x[7]};
      w.x = kv_round4<KIND>(lo, 1.f, mul, s_new);
      w.y = kv_round4<KIND>(hi, 1.f, mul, s_new);
    }
    if (real) *reinterpret_cast<uint2*>(page + (base + rr) * D + 8 * sub) = w;
  }
  __syncwarp();
  if (lane == 0) *scale = s_new;
}

// The new tokens of one page: their q rows, and k and v of this CTA's share of the heads.
template <int D, int KIND, typename T>
__device__ __forceinline__ void append_unit(const AppendArgs& a, const AppendUnit& u, float2* cs) {
  const KvSeq s = kv_seq(a.b, u.seq);
  const int page = 1 << a.c.shift, old = max(s.kv - s.q, 0), begin = u.block << a.c.shift;
  const int n0 = max(old - begin, 0), n1 = min(s.kv - begin, page);  // slots of this page's new tokens
  // rows of q, k, v; with q_len > kv_len (already reported) the first rows have no place and are left out
  const int64_t row = static_cast<int64_t>(s.row) + (s.q - s.kv) + begin + n0;
  const bool turn = a.r.turns != nullptr;
  if (turn) rotary_table(a.r, row, n1 - n0, cs);
  __syncthreads();
  const int split = blockIdx.y;
  if (turn && a.q != nullptr) {
    const int h0 = static_cast<int>(static_cast<int64_t>(a.hq) * split / a.head_splits);
    const int h1 = static_cast<int>(static_cast<int64_t>(a.hq) * (split + 1) / a.head_splits);
    rotary_rows<D, T>(a.r, static_cast<const T*>(a.q), static_cast<T*>(a.q_out), a.q_stride, a.q_out_stride, row, n1 - n0, h0, h1, cs);
  }
  const int64_t p = kv_page(a.c, a.b, u.seq, begin);
  if (p < 0) {
    if (threadIdx.x == 0) set_status(a.b.status, SLORA_STATUS_BAD_TABLE);
    return;
  }
  // (head, k or v) of this CTA's share, one warp each
  const int g0 = static_cast<int>(2ll * a.c.hkv * split / a.head_splits), g1 = static_cast<int>(2ll * a.c.hkv * (split + 1) / a.head_splits);
  for (int i = g0 + (threadIdx.x >> 5); i < g1; i += kRowWarps) {
    const int h = i >> 1;
    const int64_t ph = p * a.c.hkv + h;
    uint8_t* bytes = ((i & 1) ? a.c.v : a.c.k) + (ph << a.c.shift) * D;
    const int64_t stride = (i & 1) ? a.v_stride : a.k_stride;
    const T* src = static_cast<const T*>((i & 1) ? a.v : a.k) + row * stride + h * D;
    append_page<D, KIND, T>(a, src, stride, n0, n1, bytes, ((i & 1) ? a.c.vs : a.c.ks) + ph, cs, turn && !(i & 1));
    if (a.c.w != nullptr && !(i & 1))
      for (int x = n0 + (threadIdx.x & 31); x < n1; x += 32) a.c.w[(ph << a.c.shift) + x] = 0.f;
  }
}

template <int D, int KIND, typename T>
__global__ void __launch_bounds__(kRowThreads) kv_append_kernel(const AppendArgs a) {
  extern __shared__ float2 cs[];
  pdl_launch_dependents();
  pdl_wait();
  // the grid holds every unit unless sequences share rows
  AppendUnit u;
  for (int at = blockIdx.x; append_find(a, at, &u); at += gridDim.x) append_unit<D, KIND, T>(a, u, cs);
}

struct ReadArgs {
  KvCache c;
  KvBatch b;
  const int32_t* first;
  int64_t count;
  void* out[2];
};

// Cached values back to 16 bits: a warp takes rows (token, head) of one sequence, k and v; eight elements a lane.
template <int D, int KIND, typename T>
__global__ void __launch_bounds__(kRowThreads) kv_read_kernel(const ReadArgs a) {
  constexpr int kLanes = D / 8, kRows = 32 / kLanes;
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, sub = lane % kLanes;
  const int64_t rows = a.b.n_seq * a.count * a.c.hkv;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kRowWarps * kRows;
  for (int64_t i = (static_cast<int64_t>(blockIdx.x) * kRowWarps + (threadIdx.x >> 5)) * kRows + lane / kLanes; i < rows; i += step) {
    const int64_t token = i / a.c.hkv;
    const int h = static_cast<int>(i - token * a.c.hkv);
    const int seq = static_cast<int>(token / a.count);
    const int64_t pos = token - seq * a.count + (a.first ? a.first[seq] : 0);
    int kv = a.b.kv_len[seq];
    if (kv < 0 || kv > a.b.max_tokens) {
      if (sub == 0) set_status(a.b.status, SLORA_STATUS_BAD_TABLE);
      kv = 0;
    }
    int64_t p = -1;
    if (pos >= 0 && pos < kv) {
      p = kv_page(a.c, a.b, seq, static_cast<int>(pos));
      if (p < 0 && sub == 0) set_status(a.b.status, SLORA_STATUS_BAD_TABLE);
    }
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (p >= 0) {
        const int64_t ph = p * a.c.hkv + h;
        const uint8_t* src = (w ? a.c.v : a.c.k) + ((ph << a.c.shift) + (pos & ((1 << a.c.shift) - 1))) * D + 8 * sub;
        const uint2 v = *reinterpret_cast<const uint2*>(src);
        const float s = (w ? a.c.vs : a.c.ks)[ph];
        float q[4];
        Kv8<KIND>::values(v.x, q);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = q[e] * s;
        Kv8<KIND>::values(v.y, q);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[4 + e] = q[e] * s;
      }
      store8<T>(static_cast<T*>(a.out[w]) + i * D + 8 * sub, x);
    }
  }
}

}  // namespace slora
