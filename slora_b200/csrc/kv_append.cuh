// Rotary embedding of q and k, the append of new tokens to the 8-bit cache, and reading it back.
//
// Rotary: element pairs (x0, x1) of a head turn by position * frequency.  The angle is reduced in 64 bits (position *
// turns, minus the nearest whole number: a position of 10^6 keeps 2^-30 of a turn, where FP32 would keep 2^-4) and only
// the remainder goes to sincospif.  Cosines and sines of a block of tokens are worked out once, in shared memory, and
// serve all heads.  A row of a head is 8 elements a lane (16-byte loads and stores); in the half layout the partner of a
// value sits rot / 16 lanes away (one shuffle per element), in the interleaved layout in the same lane.
// What bounds it: q, k read and written once (16-bit), at the copy rate: 8191 tokens of 64 + 8 heads of 128, half of each
// turned: 53 us, 0.86 of it.  One token: 10 us, all of them the call's and the launch's.
//
// Append: the new tokens of one page belong to one CTA (the scale of a (page, head) is a maximum over them): all warps take
// a (head, k or v) together when there are many tokens, one warp each when there are few (decode).  When the scale grows,
// the page's older values are rounded to the new one in place.  Batches with more than kAppendWarpTokens new tokens of a
// sequence (max_q_len) take two launches, q by tokens and k, v by heads: one kernel for both had too many registers and instructions (236 against 152 us
// then, 7983 tokens of 64 + 8 + 8 heads of 128; now 50 and 73 us).  What bounds it there is instructions (angles, exact
// rounding) and the barriers of the two walks over a page; at decode every CTA's scan over the lengths, with two barriers, and
// then a chain of loads: table, scale, values (77 sequences of 32 heads: 16 us).
#pragma once

#include "kv_common.cuh"
#include "lora_mma.cuh"

namespace slora {

constexpr int kRowThreads = 256;
constexpr int kRowWarps = kRowThreads / 32;
constexpr int kAppendWarpTokens = 4;  // new tokens of a sequence up to which a warp takes a (head, k or v) by itself

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
  int rows_at, rows_step;  // shared memory behind the cosines: rows of one (page, head), and of the next (0: one buffer)
};

__device__ __forceinline__ float2 rotary_pair(const RotaryArgs& r, int64_t token, int pair) {
  const double a = static_cast<double>(r.positions[token]) * r.turns[pair];
  float s, c;
  sincospif(2.f * static_cast<float>(a - rint(a)), &s, &c);
  return make_float2(c * r.factor, (r.inverse ? -s : s) * r.factor);
}
// (cos, sin) of `n` tokens from `t0` on into cs[n][rot / 2].
__device__ __forceinline__ void rotary_table(const RotaryArgs& r, int64_t t0, int n, float2* cs) {
  const int half = r.rot >> 1;
  for (int i = threadIdx.x; i < n * half; i += blockDim.x) {
    const int t = i / half;
    cs[i] = rotary_pair(r, t0 + t, i - t * half);
  }
}
// The same for CTAs of a cluster that work on the same tokens: each works out its share of the angles (150 instructions
// apiece, what the rows' own work comes to) and stores it into every CTA's shared memory.
__device__ __forceinline__ void rotary_table_cluster(const RotaryArgs& r, int64_t t0, int n, float2* cs, int size) {
  const int half = r.rot >> 1, rank = static_cast<int>(cluster_rank());
  cluster_sync_all();  // every CTA of the cluster runs, and is done with its last table
  for (int i = rank * blockDim.x + threadIdx.x; i < n * half; i += size * blockDim.x) {
    const int t = i / half;
    const float2 v = rotary_pair(r, t0 + t, i - t * half);
    const uint32_t at = smem_u32(cs + i);
    for (int k = 0; k < size; ++k)
      asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(peer_smem(at, k)), "f"(v.x), "f"(v.y) : "memory");
  }
  cluster_sync_all();
}

// The cosines and sines that a lane needs for the eight elements 8 sub .. 8 sub + 7 of a head row of one token; in the half
// layout the sines carry the sign of the lane's part, so that both parts are x cos + partner sin.
struct RotaryLane {
  float2 w[8];
  int other;  // half layout: lane with the partners
  bool in;    // these elements turn
  __device__ __forceinline__ void load(const float2* cs, int sub, int rot, int layout) {
    if (layout == 0)
      load_as<0>(cs, sub, rot);
    else
      load_as<1>(cs, sub, rot);
  }
  __device__ __forceinline__ void turn(float (&x)[8], int layout) const {  // all lanes of the warp take part
    if (layout == 0)
      turn_as<0>(x);
    else
      turn_as<1>(x);
  }
  template <int LAYOUT>
  __device__ __forceinline__ void load_as(const float2* cs, int sub, int rot) {
    const int lane = threadIdx.x & 31;
    other = lane;
    in = 8 * sub < rot;
    if (LAYOUT == 0) {
      const int far = rot >> 4;  // lanes between the partners
      const bool low = sub < far;
      if (in) other = low ? lane + far : lane - far;
      const float4* p = reinterpret_cast<const float4*>(cs + (in ? 8 * (low ? sub : sub - far) : 0));
      const float sign = low ? -1.f : 1.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float4 v = p[e];
        w[2 * e] = make_float2(v.x, v.y * sign);
        w[2 * e + 1] = make_float2(v.z, v.w * sign);
      }
    } else if (in) {
      const float4* p = reinterpret_cast<const float4*>(cs + 4 * sub);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float4 v = p[e];
        w[2 * e] = make_float2(v.x, v.y);
        w[2 * e + 1] = make_float2(v.z, v.w);
      }
    }
  }
  template <int LAYOUT>
  __device__ __forceinline__ void turn_as(float (&x)[8]) const {
    if (LAYOUT == 0) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float y = __shfl_sync(0xffffffffu, x[e], other);
        const float z = x[e] * w[e].x + y * w[e].y;
        x[e] = in ? z : x[e];
      }
    } else if (in) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float a = x[2 * e], b = x[2 * e + 1];
        x[2 * e] = a * w[e].x - b * w[e].y;
        x[2 * e + 1] = a * w[e].y + b * w[e].x;
      }
    }
  }
};

// The largest magnitude of eight values into top; `odd` stays 0 while all are finite (NaN and infinities make it NaN).
__device__ __forceinline__ void append_top(const float (&x)[8], float* top, float* odd) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    *top = fmaxf(*top, fabsf(x[e]));
    *odd = __fmaf_rn(x[e], 0.f, *odd);
  }
}
// The same without what is not finite.
__device__ __forceinline__ void append_top_finite(const float (&x)[8], float* top) {
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (fabsf(x[e]) <= 3.4028234663852886e38f) *top = fmaxf(*top, fabsf(x[e]));
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

// Heads [h0, h1) of tokens [t0, t0 + n): turned rows src -> dst.  A warp takes a token and a few heads at a time: the
// token's cosines stay in registers, and kRowUnroll loads of 512 bytes are in flight.
constexpr int kRowUnroll = 4;
template <int D, typename T, int LAYOUT>
__device__ __forceinline__ void rotary_rows_as(const RotaryArgs& r, const T* src, T* dst, int64_t src_stride, int64_t dst_stride,
                                            int64_t t0, int n, int h0, int h1, const float2* cs) {
  constexpr int kLanes = D / 8, kRows = 32 / kLanes, kHeads = kRows * kRowUnroll;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane % kLanes, rr = lane / kLanes;
  const int chunks = (h1 - h0 + kHeads - 1) / kHeads, half = r.rot >> 1;
  for (int item = warp; item < n * chunks; item += kRowWarps) {
    const int t = item / chunks, h = h0 + (item - t * chunks) * kHeads + rr;
    const T* from = src + (t0 + t) * src_stride + 8 * sub;
    T* to = dst + (t0 + t) * dst_stride + 8 * sub;
    uint4 raw[kRowUnroll];
#pragma unroll
    for (int u = 0; u < kRowUnroll; ++u) {
      raw[u] = make_uint4(0, 0, 0, 0);
      if (h + u * kRows < h1) raw[u] = *reinterpret_cast<const uint4*>(from + (h + u * kRows) * D);
    }
    RotaryLane w;
    w.load_as<LAYOUT>(cs + t * half, sub, r.rot);
#pragma unroll
    for (int u = 0; u < kRowUnroll; ++u) {
      float x[8];
      cvt8<T>(raw[u], x);
      w.turn_as<LAYOUT>(x);
      if (h + u * kRows < h1) store8<T>(to + (h + u * kRows) * D, x);
    }
  }
}

template <int D, typename T>
__device__ __forceinline__ void rotary_rows(const RotaryArgs& r, const T* src, T* dst, int64_t src_stride, int64_t dst_stride,
                                            int64_t t0, int n, int h0, int h1, const float2* cs) {
  if (r.layout == 0)
    rotary_rows_as<D, T, 0>(r, src, dst, src_stride, dst_stride, t0, n, h0, h1, cs);
  else
    rotary_rows_as<D, T, 1>(r, src, dst, src_stride, dst_stride, t0, n, h0, h1, cs);
}

template <int D, typename T>
__global__ void __launch_bounds__(kRowThreads) rotary_kernel(const RowArgs a) {
  extern __shared__ __align__(16) float2 cs[];
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

// NaN -> 0, infinities -> the largest FP32.
__device__ __forceinline__ void kv_finite(float& x) {
  if (!(fabsf(x) <= 3.4028234663852886e38f)) x = x == x ? copysignf(3.4028234663852886e38f, x) : 0.f;
}

// Older values of a (page, head), `bytes` of them, rounded to a grown scale: 16 bytes a lane.  s_old 0 (a scale that counts
// as 0): they become 0, and s_new may be 0 too.
template <int KIND>
__device__ __forceinline__ void append_rescale(uint8_t* page, int bytes, float s_old, float s_new, int id, int step) {
  using V8 = Kv8<KIND>;
  const float mul = __fdiv_rn(s_old, s_new);
#pragma unroll 1
  for (int i = id; i < bytes / 16; i += step) {
    if (!(s_old > 0.f)) {
      reinterpret_cast<uint4*>(page)[i] = make_uint4(0, 0, 0, 0);
      continue;
    }
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

// Eight values at scale s_new, packed; fine: all of them are finite.
template <int KIND>
__device__ __forceinline__ uint2 append_pack(float (&x)[8], float mul, float s_new, bool fine) {
  uint2 w = make_uint2(0, 0);
  if (s_new > 0.f) {
    if (!fine) {
#pragma unroll
      for (int e = 0; e < 8; ++e) kv_finite(x[e]);
    }
    const float lo[4] = {x[0], x[1], x[2], x[3]}, hi[4] = {x[4], x[5], x[6], x[7]};
    w.x = kv_round4<KIND>(lo, 1.f, mul, s_new, !fine);
    w.y = kv_round4<KIND>(hi, 1.f, mul, s_new, !fine);
  }
  return w;
}

// New rows of one (page, head) of k or v into shared memory, [token][d], asynchronously.
template <int D, typename T>
__device__ __forceinline__ void append_fetch(uint8_t* to, const T* src, int64_t stride, int n) {
  for (int x = threadIdx.x; x < n * (D / 8); x += kRowThreads) {
    const int i = x / (D / 8), c = x % (D / 8);
    cp_async16(smem_u32(to + x * 16), src + i * stride + 8 * c);
  }
  cp_async_commit();
}

// One (page, head) of k or v by the whole CTA, for pages with more than a few new tokens, from its rows in shared memory.
template <int D, int KIND, typename T>
__device__ __forceinline__ void append_page_cta(const AppendArgs& a, const uint8_t* rows, int n0, int n1, uint8_t* page,
                                                float* scale, const float2* cs, bool turn) {
  constexpr int kLanes = D / 8, kRows = 32 / kLanes, kPass = kRowWarps * kRows;
  using V8 = Kv8<KIND>;
  __shared__ float tops[kRowWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane % kLanes, half = a.r.rot >> 1;
  const int mine = warp * kRows + lane / kLanes, n = n1 - n0, passes = (n + kPass - 1) / kPass;
  const float was = n0 > 0 ? *scale : 0.f, s_old = kv_scale(was);
  auto row = [&](int p, float (&x)[8]) {
    const int i = min(mine + p * kPass, n - 1);  // lanes without a row repeat the last one
    cvt8<T>(*reinterpret_cast<const uint4*>(rows + (i * kLanes + sub) * 16), x);
    if (turn) {
      RotaryLane w;
      w.load(cs + i * half, sub, a.r.rot, a.r.layout);
      w.turn(x, a.r.layout);
    }
  };
  float top = 0.f, odd = 0.f;
#pragma unroll 1
  for (int p = 0; p < passes; ++p) {
    float x[8];
    row(p, x);
    append_top(x, &top, &odd);
  }
  const bool fine = !__any_sync(0xffffffffu, odd != 0.f);
  if (!fine) {
    top = 0.f;
#pragma unroll 1
    for (int p = 0; p < passes; ++p) {
      float x[8];
      row(p, x);
      append_top_finite(x, &top);
    }
    if (lane == 0) set_status(a.b.status, kStatusNonfinite);
  }
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  if (lane == 0) tops[warp] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kRowWarps; ++w) top = fmaxf(top, tops[w]);
  const float s_new = kv_scale(fmaxf(s_old, __fdiv_rn(top, V8::kTop)));
  if (s_new != was && n0 > 0) append_rescale<KIND>(page, n0 * D, s_old, s_new, threadIdx.x, kRowThreads);
  const float mul = s_new > 0.f ? __fdiv_rn(1.f, s_new) : 0.f;
#pragma unroll 1
  for (int p = 0; p < passes; ++p) {
    float x[8];
    row(p, x);
    const uint2 w = append_pack<KIND>(x, mul, s_new, fine);
    const int i = mine + p * kPass;
    if (i < n) *reinterpret_cast<uint2*>(page + (n0 + i) * D + 8 * sub) = w;
  }
  __syncthreads();  // every thread has read the rows, the old scale and tops
  if (threadIdx.x == 0) *scale = s_new;
}

// One (page, head) of k or v by a warp: new tokens in slots [n0, n1) whose rows start at `src`, older ones in slots [0, n0).
template <int D, int KIND, typename T>
__device__ __forceinline__ void append_page(const AppendArgs& a, const T* src, int64_t stride, int n0, int n1, uint8_t* page,
                                            float* scale, const float2* cs, bool turn) {
  constexpr int kLanes = D / 8, kRows = 32 / kLanes;
  using V8 = Kv8<KIND>;
  const int lane = threadIdx.x & 31, sub = lane % kLanes, rr = lane / kLanes, half = a.r.rot >> 1;
  const float was = n0 > 0 ? *scale : 0.f, s_old = kv_scale(was);
  float x[8];
  auto load = [&](int base) {
    const int i = base + rr;
    const bool real = i < n1;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = 0.f;
    if (real) cvt8<T>(*reinterpret_cast<const uint4*>(src + static_cast<int64_t>(i - n0) * stride + 8 * sub), x);
    if (turn) {
      RotaryLane w;
      w.load(cs + (real ? i - n0 : 0) * half, sub, a.r.rot, a.r.layout);
      w.turn(x, a.r.layout);
    }
    return real;
  };
  float top = 0.f, odd = 0.f;
  for (int base = n0; base < n1; base += kRows) {
    load(base);
    append_top(x, &top, &odd);
  }
  const bool fine = !__any_sync(0xffffffffu, odd != 0.f);
  if (!fine) {
    top = 0.f;
    for (int base = n0; base < n1; base += kRows) {
      load(base);
      append_top_finite(x, &top);
    }
    if (lane == 0) set_status(a.b.status, kStatusNonfinite);
  }
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  const float s_new = kv_scale(fmaxf(s_old, __fdiv_rn(top, V8::kTop)));
  if (s_new != was && n0 > 0) append_rescale<KIND>(page, n0 * D, s_old, s_new, lane, 32);
  const float mul = s_new > 0.f ? __fdiv_rn(1.f, s_new) : 0.f;
  for (int base = n0; base < n1; base += kRows) {
    const bool real = load(base);
    const uint2 w = append_pack<KIND>(x, mul, s_new, fine);
    if (real) *reinterpret_cast<uint2*>(page + (base + rr) * D + 8 * sub) = w;
  }
  __syncwarp();
  if (lane == 0) *scale = s_new;
}

// The new tokens of one page: their q rows, and k and v of this CTA's share of the heads.  Where pages have many new tokens
// (WIDE) the two are launches of their own: q's wants few registers and many CTAs.
enum AppendPart { APPEND_FEW = 0, APPEND_Q = 1, APPEND_KV = 2 };
template <int D, int KIND, typename T, int PART>
__device__ __forceinline__ void append_unit(const AppendArgs& a, const AppendUnit& u, float2* cs) {
  const KvSeq s = kv_seq(a.b, u.seq);
  const int page = 1 << a.c.shift, old = max(s.kv - s.q, 0), begin = u.block << a.c.shift;
  const int n0 = max(old - begin, 0), n1 = min(s.kv - begin, page);  // slots of this page's new tokens
  // rows of q, k, v; with q_len > kv_len (already reported) the first rows have no place and are left out
  const int64_t row = static_cast<int64_t>(s.row) + (s.q - s.kv) + begin + n0;
  const bool turn = a.r.turns != nullptr;
  if (PART == APPEND_Q) {
    // the CTAs of a page share its tokens, so each works out its own angles only
    const int t0 = (n1 - n0) * static_cast<int>(blockIdx.y) / a.head_splits, t1 = (n1 - n0) * static_cast<int>(blockIdx.y + 1) / a.head_splits;
    rotary_table(a.r, row + t0, t1 - t0, cs);
    __syncthreads();
    rotary_rows<D, T>(a.r, static_cast<const T*>(a.q), static_cast<T*>(a.q_out), a.q_stride, a.q_out_stride, row + t0, t1 - t0, 0, a.hq, cs);
    return;
  }
  if (turn) {
    if (a.head_splits > 1 && (n1 - n0) * a.r.rot > 2 * kRowThreads)
      rotary_table_cluster(a.r, row, n1 - n0, cs, a.head_splits);
    else
      rotary_table(a.r, row, n1 - n0, cs);
  }
  __syncthreads();
  const int split = blockIdx.y;  // the CTAs of a page are one cluster
  if (PART == APPEND_FEW && turn && a.q != nullptr) {
    const int h0 = static_cast<int>(static_cast<int64_t>(a.hq) * split / a.head_splits);
    const int h1 = static_cast<int>(static_cast<int64_t>(a.hq) * (split + 1) / a.head_splits);
    rotary_rows<D, T>(a.r, static_cast<const T*>(a.q), static_cast<T*>(a.q_out), a.q_stride, a.q_out_stride, row, n1 - n0, h0, h1, cs);
  }
  const int64_t p = kv_page(a.c, a.b, u.seq, begin);
  if (p < 0) {
    if (threadIdx.x == 0) set_status(a.b.status, SLORA_STATUS_BAD_TABLE);
    return;
  }
  // (head, k or v) of this CTA's share: all warps on one where the page has many new tokens, else one warp each
  const int g0 = static_cast<int>(2ll * a.c.hkv * split / a.head_splits), g1 = static_cast<int>(2ll * a.c.hkv * (split + 1) / a.head_splits);
  auto source = [&](int i, int64_t* stride) {
    *stride = (i & 1) ? a.v_stride : a.k_stride;
    return static_cast<const T*>((i & 1) ? a.v : a.k) + row * *stride + (i >> 1) * D;
  };
  auto place = [&](int i, float** scale) {
    const int64_t ph = p * a.c.hkv + (i >> 1);
    *scale = ((i & 1) ? a.c.vs : a.c.ks) + ph;
    return ((i & 1) ? a.c.v : a.c.k) + (ph << a.c.shift) * D;
  };
  const int n = n1 - n0;
  int64_t stride;
  float* scale;
  if (PART == APPEND_KV) {
    uint8_t* rows[2] = {reinterpret_cast<uint8_t*>(cs) + a.rows_at, reinterpret_cast<uint8_t*>(cs) + a.rows_at + a.rows_step};
    const bool two = a.rows_step > 0;  // two buffers: the next rows come in while these are rounded
    if (two && g0 < g1) {
      const T* src = source(g0, &stride);
      append_fetch<D, T>(rows[0], src, stride, n);
    }
    for (int i = g0; i < g1; ++i) {
      const int buf = two ? (i - g0) & 1 : 0;
      if (!two || i + 1 < g1) {
        const T* src = source(two ? i + 1 : i, &stride);
        append_fetch<D, T>(rows[two ? buf ^ 1 : 0], src, stride, n);
        if (two)
          cp_async_wait<1>();
        else
          cp_async_wait<0>();
      } else {
        cp_async_wait<0>();
      }
      __syncthreads();
      uint8_t* bytes = place(i, &scale);
      append_page_cta<D, KIND, T>(a, rows[buf], n0, n1, bytes, scale, cs, turn && !(i & 1));
    }
  } else {
    for (int i = g0 + static_cast<int>(threadIdx.x >> 5); i < g1; i += kRowWarps) {
      const T* src = source(i, &stride);
      uint8_t* bytes = place(i, &scale);
      append_page<D, KIND, T>(a, src, stride, n0, n1, bytes, scale, cs, turn && !(i & 1));
    }
  }
  // weights of new tokens start at 0; the CTA that has a head's k writes them
  if (a.c.w != nullptr)
    for (int x = threadIdx.x; x < ((g1 + 1) / 2 - (g0 + 1) / 2) * n; x += kRowThreads)
      a.c.w[((p * a.c.hkv + (g0 + 1) / 2 + x / n) << a.c.shift) + n0 + x % n] = 0.f;
}

template <int D, int KIND, typename T, int PART>
__global__ void __launch_bounds__(kRowThreads, PART == APPEND_Q ? 4 : 3) kv_append_kernel(const AppendArgs a) {
  extern __shared__ __align__(16) float2 cs[];
  pdl_launch_dependents();
  pdl_wait();
  // the grid holds every unit unless sequences share rows
  AppendUnit u;
  for (int at = blockIdx.x; append_find(a, at, &u); at += gridDim.x) append_unit<D, KIND, T, PART>(a, u, cs);
}

struct ReadArgs {
  KvCache c;
  KvBatch b;
  const int32_t* first;
  int64_t count;
  void* out[2];
};

// Cached values back to 16 bits: a warp takes kReadAhead rows a half warp (eight heads at d 128) of one token, with one look at
// its page, eight elements a lane, and has all their k and v on their way at once. 7983 tokens of 8 heads: 17 -> 14 us against
// a warp per token and head.
constexpr int kReadAhead = 4;
template <int D, int KIND, typename T>
__global__ void __launch_bounds__(kRowThreads) kv_read_kernel(const ReadArgs a) {
  constexpr int kLanes = D / 8, kRows = 32 / kLanes, kGroup = kReadAhead * kRows;
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, sub = lane % kLanes, rr = lane / kLanes;
  const int groups = (a.c.hkv + kGroup - 1) / kGroup;
  const int64_t units = a.b.n_seq * a.count * groups;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kRowWarps;
  for (int64_t unit = static_cast<int64_t>(blockIdx.x) * kRowWarps + (threadIdx.x >> 5); unit < units; unit += step) {
    int64_t token, seq64;
    int group;
    if (units <= 0xffffffffll) {
      token = static_cast<uint32_t>(unit) / static_cast<uint32_t>(groups);
      seq64 = static_cast<uint32_t>(token) / static_cast<uint32_t>(a.count);
    } else {
      token = unit / groups;
      seq64 = token / a.count;
    }
    group = static_cast<int>(unit - token * groups);
    const int seq = static_cast<int>(seq64);
    const int64_t pos = token - seq * a.count + (a.first ? a.first[seq] : 0);
    int kv = a.b.kv_len[seq];
    if (kv < 0 || kv > a.b.max_tokens) {
      if (lane == 0) set_status(a.b.status, SLORA_STATUS_BAD_TABLE);
      kv = 0;
    }
    int64_t p = -1;
    if (pos >= 0 && pos < kv) {
      p = kv_page(a.c, a.b, seq, static_cast<int>(pos));
      if (p < 0 && lane == 0) set_status(a.b.status, SLORA_STATUS_BAD_TABLE);
    }
    const int slot = static_cast<int>(pos & ((1 << a.c.shift) - 1));
    T* const out[2] = {static_cast<T*>(a.out[0]) + token * a.c.hkv * D + 8 * sub, static_cast<T*>(a.out[1]) + token * a.c.hkv * D + 8 * sub};
    const int h0 = group * kGroup + rr;
    uint2 v[kReadAhead][2];
    float s[kReadAhead][2];
#pragma unroll
    for (int u = 0; u < kReadAhead; ++u) {
      const int h = h0 + u * kRows;
      v[u][0] = v[u][1] = make_uint2(0, 0);
      s[u][0] = s[u][1] = 0.f;
      if (p >= 0 && h < a.c.hkv) {
        const int64_t ph = p * a.c.hkv + h, at = ((ph << a.c.shift) + slot) * D + 8 * sub;
        v[u][0] = *reinterpret_cast<const uint2*>(a.c.k + at);
        v[u][1] = *reinterpret_cast<const uint2*>(a.c.v + at);
        s[u][0] = a.c.ks[ph];
        s[u][1] = a.c.vs[ph];
      }
    }
#pragma unroll
    for (int u = 0; u < kReadAhead; ++u) {
      const int h = h0 + u * kRows;
      if (h >= a.c.hkv) break;
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        float x[8], q[4];
        Kv8<KIND>::values(v[u][w].x, q);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = q[e] * s[u][w];
        Kv8<KIND>::values(v[u][w].y, q);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[4 + e] = q[e] * s[u][w];
        store8<T>(out[w] + h * D, x);
      }
    }
  }
}

}  // namespace slora
