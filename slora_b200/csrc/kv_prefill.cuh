// Attention over the 8-bit cache for many query rows per sequence and KV head (chunks of prompts): tcgen05.
//
// 4 d multiply-adds per key and row against 2 d bytes per key: from some dozens of rows on the tensor pipe bounds it, and
// the exponentials next to it: 128 keys x 128 rows take 1024 cycles of the pipe (d 128) and as many of the SM's 16
// exponentials a cycle.  Hence two row tiles of 128 per CTA that take turns: while one is in its softmax, the tensor pipe
// works on the other.
//   rows of a tile = (new token, q head of the KV head) pairs in that order, one thread each in the softmax
//   S = Q K^T    128 x 128, Q and K in shared memory (f16, 128-byte swizzle, inner dimension d)
//   P            over S in tensor memory (f16 pairs), the A operand of the second product
//   O += P V     V in shared memory as it lies in the cache, keys outside: the outer-major form of the same layout
// Roles: seven warps convert 8-bit pages to f16 operands (values exact, as in kv_attend.cuh; with four of them the tensor
// pipe waited for operands), one lane issues the MMAs, four warps per row tile do the softmax.  Scales never touch the
// operands: a page's k scale multiplies its 16-column groups of S (the maximum of a group is taken before it), its v
// scale, relative to the row's reference, goes into the exponent of p, and comes out of the sum of p again per group.
// The reference is a power of two, a row's own; it follows the largest v scale that the row sees in a step of 128 keys,
// so pages that a row does not see (later tokens, what a window has left behind) cost it nothing, and a change rescales
// the row's O by a power of two, which rounds nothing.  p * vs is one f16 number (64 p vs / 2^ref; for f16 outputs too:
// its 2^-11 shows as 1.4 times the error of the output's own rounding, a second number would double the product): off by
// 2^-11 of itself or, where it is small, by 2^-31 of the reference, which is 2 to 2^9 times the step's largest scale.
// The running maximum is raised only when a score passes it by 2^8; then the row's O is rescaled in tensor memory.  P(j)
// replaces S(j) and S(j + 1) replaces P(j): the MMAs of a CTA run in order, so the commit behind S(j + 1) also says that
// O has P(j) V(j).
//
// Chunks of 4 prompts (3521 new tokens behind 2002 to 4352 cached ones, 64 q heads on 8, d 128, int8): 735 us, 536 TFLOP/s, 0.32
// of the measured rate of a large matrix product (d 64: 566 us); the simple form of the same loop took 3136 us.  What bounds
// it is the chain of one row tile (scores out of tensor memory, p back: 3700 cycles for four warps; then the product and
// the next scores), of which two run side by side.  Without the exponentials it takes as long; without the conversion 6 %
// less; with one reference for all rows of a CTA (which let pages that a row does not see round its p) 3 to 4 % less.
//
// Every wait is bounded; a CTA that gives up records SLORA_STATUS_TIMEOUT and frees its tensor memory.
#pragma once

#include "kv_attend.cuh"
#include "lora_mma.cuh"

namespace slora {

constexpr int kPreSoftWarps = 8, kPreCvtWarps = 7;  // and one that issues the MMAs
// Registers of a thread after the roles have parted: 2 x 152 + 2 x 104 for the four groups of four warps, which is what the
// launch gave them (4 x 128).
constexpr int kPreSoftRegs = 152, kPreOtherRegs = 104;
constexpr int kPreThreads = (kPreSoftWarps + kPreCvtWarps + 1) * 32;
constexpr int kPreKeys = 128;                // keys of a step
constexpr int kPreRows = 256;                // rows of a CTA
constexpr int kPreGroups = kPreKeys / 16;    // 16 keys share their scales whatever the page size
constexpr int kPreScaleSlots = 4;            // steps whose scales are kept: the softmax of a step reads them after its K is gone
constexpr float kPreRange = 6.f;             // log2: p * vs / reference * 2^6 <= 2^8 * 2^6: inside f16
constexpr float kPreLower = 8.f;             // octaves that a step's largest v scale may lie below the reference
constexpr float kPreFar = 40.f;              // octaves below the reference from which a scale's p * vs is 0 in f16 (p only counts)
constexpr float kPreRise = 64.f;             // octaves that the reference may sink from its highest: O stays inside FP32
constexpr float kNoScale = -1000.f;          // exponent of a scale that counts as 0, or of no page
constexpr float kNoRef = -200.f;             // no reference yet (the smallest is above -126)

template <int D>
struct PreSmem {
  uint8_t q[2][128 * D * 2];   // row tiles; [64 elements][row][128 bytes]
  uint8_t k[2][kPreKeys * D * 2];
  uint8_t v[2][kPreKeys * D * 2];
  uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], o_full;
  uint32_t tmem;
  int bad;
  // Per 16 keys, v scale = m 2^e with m in [0.5, 1), top the largest e of the step: k scale, log2 m (-inf: a bad page), e + 6
  // and 1 / m (part, for rows that see a part of the step), or 2^(top - e - 6) / m (whole).
  alignas(16) float4 whole[kPreScaleSlots][kPreGroups], part[kPreScaleSlots][kPreGroups];
  float top[kPreScaleSlots];
  KvFind find;
};

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, "
      "%18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
        "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
        "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};\n" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
      "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// D[tmem] (+)= A[tmem] * B[smem], one K = 16 step: A's 16 columns of f16 lie in eight columns of tensor memory.
__device__ __forceinline__ void umma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n"
      "}\n" ::"r"(tmem_d),
      "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate), "r"(0u)
      : "memory");
}
// Outer-major operand with the 128-byte swizzle: rows (keys) of 64 elements of the outer dimension (d), eight of them 1024
// bytes, the next eight keys 1024 bytes on, the next 64 elements `lbo` bytes on.
__device__ __forceinline__ uint64_t umma_smem_desc_sw128_mn(uint32_t addr, uint32_t lbo) {
  uint64_t d = static_cast<uint64_t>((addr & 0x3ffffu) >> 4);
  d |= static_cast<uint64_t>(lbo >> 4) << 16;
  d |= static_cast<uint64_t>(1024 >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(2) << 61;
  return d;
}

// The largest score (log2 units) of this thread's row of S: groups of 16 columns share their scale.  The next 32 columns are on
// their way from tensor memory while 32 are looked at.  MASKED: only columns [from, to) count.
template <int D, bool MASKED>
__device__ __forceinline__ float pre_max(const PreSmem<D>& sm, int slot, uint32_t t_s, float down, int from, int to) {
  float top = kNegInf;
  uint32_t raw[2][32];
  tmem_ld32(t_s, raw[0]);
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    tmem_ld_wait();
    if (c < 3) tmem_ld32(t_s + 32 * (c + 1), raw[(c + 1) & 1]);
    uint32_t(&x)[32] = raw[c & 1];
    if (MASKED) {
#pragma unroll
      for (int e = 0; e < 32; ++e)
        if (32 * c + e < from || 32 * c + e >= to) x[e] = 0xff800000u;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float g0 = __uint_as_float(x[16 * h]), g1 = __uint_as_float(x[16 * h + 1]);
#pragma unroll
      for (int e = 2; e < 16; e += 2) {
        g0 = fmaxf(g0, __uint_as_float(x[16 * h + e]));
        g1 = fmaxf(g1, __uint_as_float(x[16 * h + e + 1]));
      }
      g0 = fmaxf(g0, g1);
      const float4 w = sm.whole[slot][2 * c + h];
      if (g0 > kNegInf && w.y > kNegInf) top = fmaxf(top, g0 * (down * w.x));
    }
  }
  return top;
}

// 2^e for a whole number e from -126 to 127: e + 127 in the low bits of 1.5 * 2^23 + e + 127, moved to the exponent's place.
__device__ __forceinline__ float pre_pow2(float e) { return __uint_as_float(__float_as_uint(e + 12583039.f) << 23); }

// The largest exponent of a v scale in the step among the keys [from, to).
template <int D>
__device__ __forceinline__ float pre_largest(const PreSmem<D>& sm, int slot, int from, int to) {
  float e = kNoScale;
#pragma unroll
  for (int g = 0; g < kPreGroups; ++g)
    if (16 * g < to && 16 * g + 16 > from) e = fmaxf(e, sm.part[slot][g].z - kPreRange);
  return e;
}

// p of this thread's row, relative to m0, times v scale / 2^ref, as f16 pairs, and the sum of p; tells whether one passes
// 2^14 (a score far above m0).  MASKED: groups the row does not see may have any scale.
template <int D, bool MASKED>
__device__ __forceinline__ bool pre_exp(const PreSmem<D>& sm, int slot, uint32_t t_s, float down, float m0, float ref, float* sum, int from,
                                        int to, uint32_t (&y)[64]) {
  uint32_t x[32];  // (a second buffer, for the columns to come, cost the converters more registers than it saved time)
  float l = 0.f;
  uint32_t high = 0;
  const float most = sm.top[slot];
  if (!MASKED) ref = most > kNoScale ? fminf(ref, most + kPreFar) : kNoScale;
  const float base = m0 + ref;  // what a score's exponent is taken relative to
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const float4 w0 = MASKED ? sm.part[slot][2 * c] : sm.whole[slot][2 * c];
    const float4 w1 = MASKED ? sm.part[slot][2 * c + 1] : sm.whole[slot][2 * c + 1];
    tmem_ld32(t_s + 32 * c, x);
    tmem_ld_wait();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float4 w = h ? w1 : w0;
      const float e2 = MASKED ? fminf(fmaxf(w.z, ref - kPreFar + kPreRange), ref + 20.f) : w.z;
      const float f = down * w.x, add = w.y + (e2 - base), back = MASKED ? w.w * pre_pow2(ref - e2) : w.w;
      float s0 = 0.f, s1 = 0.f;
#pragma unroll
      for (int e = 0; e < 16; e += 2) {
        float x0 = ex2(__fmaf_rn(__uint_as_float(x[16 * h + e]), f, add));
        float x1 = ex2(__fmaf_rn(__uint_as_float(x[16 * h + e + 1]), f, add));
        if (MASKED) {
          const int at = 32 * c + 16 * h + e;
          if (at < from || at >= to) x0 = 0.f;
          if (at + 1 < from || at + 1 >= to) x1 = 0.f;
        }
        s0 += x0;
        s1 += x1;
        const uint32_t p = pack_f16(x0, x1);
        y[16 * c + 8 * h + e / 2] = p;
        asm("max.f16x2 %0, %1, %2;" : "=r"(high) : "r"(high), "r"(p));
      }
      l = __fmaf_rn(s0 + s1, back, l);
    }
  }
  *sum = MASKED ? l : l * pre_pow2(ref - most);
  const float2 top = __half22float2(reinterpret_cast<const __half2&>(high));
  return fmaxf(top.x, top.y) > 16384.f;
}

// (sequence, 256 rows, head) items; the last rows of a sequence see the most keys and come first.
__device__ __forceinline__ long long pre_items(const KvAttendArgs& a, const KvSeq& s) {
  if (s.q < a.min_q || s.q > a.lim_q || s.q == 0) return 0;
  return static_cast<long long>((s.q * a.group + kPreRows - 1) / kPreRows) * a.c.hkv;
}

template <int D, int KIND, typename T>
__global__ void __launch_bounds__(kPreThreads, 1) kv_prefill_kernel(const KvAttendArgs a) {
  using V8 = Kv8<KIND>;
  constexpr int kHalf = kPreKeys * 128;  // bytes of 64 elements of a 128-row operand
  extern __shared__ uint8_t smem_raw[];
  PreSmem<D>& sm = *reinterpret_cast<PreSmem<D>*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_launch_dependents();
  pdl_wait();
  const long long item = blockIdx.x;
  const long long total = kv_find<kPreThreads / 32, 1>(
      a.b.n_seq, &sm.find, [&](int i) { return pre_items(a, kv_seq(a.b, i)); }, [&](long long, int) { return item; });
  // the grid holds every item unless sequences share rows
  if (total > static_cast<long long>(gridDim.x) && item == 0 && tid == 0) set_status(a.b.status, SLORA_STATUS_BAD_TABLE);
  if (item >= total) return;
  const int seq = sm.find.seq[0];
  const KvSeq s = kv_seq(a.b, seq);
  const int rows = s.q * a.group, blocks = (rows + kPreRows - 1) / kPreRows;
  const int idx = static_cast<int>(item - sm.find.at[0]);
  const int head = idx % a.c.hkv, row0 = (blocks - 1 - idx / a.c.hkv) * kPreRows;
  // keys that the CTA's rows see: [key0, key_end), in steps of 128
  const int last_row = min(row0 + kPreRows, rows) - 1;
  const int base_to = s.kv - s.q + 1;  // keys that new token 0 sees end here
  const int key_end = max(base_to + last_row / a.group, 0);
  const int key0 = a.window > 0 ? max(max(base_to + row0 / a.group, 0) - a.window, 0) / kPreKeys * kPreKeys : 0;
  const int steps = key_end > key0 ? (key_end - key0 + kPreKeys - 1) / kPreKeys : 0;

  if (warp == kPreThreads / 32 - 1) {
    tmem_alloc(&sm.tmem, 512);
    tmem_relinquish();
  }
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sm.k_full[i], kPreCvtWarps * 32);
      mbar_init(&sm.v_full[i], kPreCvtWarps * 32);
      mbar_init(&sm.k_empty[i], 1);
      mbar_init(&sm.v_empty[i], 1);
      mbar_init(&sm.s_full[i], 1);
      mbar_init(&sm.p_full[i], 128);
    }
    mbar_init(&sm.o_full, 1);
    sm.bad = 0;
    fence_barrier_init();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem;
  bool ok = true;

  if (warp < kPreSoftWarps) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPreSoftRegs));
    // ---- softmax: one thread per row --------------------------------------------------------------------------------
    const int tile = warp >> 2, r = tid & 127;  // warp % 4 is the tensor-memory quarter that the warp may touch
    const int row = row0 + tile * 128 + r;
    const bool real = row < rows;
    const int j = real ? row / a.group : 0;
    float down = 0.f;
    {
      uint8_t* dst = sm.q[tile];
      const T* src = static_cast<const T*>(a.q) + (static_cast<int64_t>(s.row) + j) * a.q_stride + (head * a.group + row - j * a.group) * D;
      float top = 0.f;
#pragma unroll 4
      for (int c = 0; c < D / 8; ++c) {
        float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (real) cvt8<T>(*reinterpret_cast<const uint4*>(src + 8 * c), x);
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[e]));
      }
      const int e2 = top > 0.f ? min(max(141 - static_cast<int>(__float_as_uint(top) >> 23), -100), 100) : 0;
      float up = __uint_as_float(static_cast<uint32_t>(127 + e2) << 23);
      down = __uint_as_float(static_cast<uint32_t>(127 - e2) << 23) * fabsf(a.scale2) * V8::kScale;
      if (a.scale2 < 0.f) up = -up;
#pragma unroll 4
      for (int c = 0; c < D / 8; ++c) {
        float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (real) cvt8<T>(*reinterpret_cast<const uint4*>(src + 8 * c), x);
        uint4 w;
        w.x = pack_f16(x[0] * up, x[1] * up);
        w.y = pack_f16(x[2] * up, x[3] * up);
        w.z = pack_f16(x[4] * up, x[5] * up);
        w.w = pack_f16(x[6] * up, x[7] * up);
        *reinterpret_cast<uint4*>(dst + (c >> 3) * kHalf + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = w;
      }
      fence_proxy_async();
      mbar_arrive(&sm.p_full[tile]);  // phase 0: Q is there
    }
    const int to = real ? max(base_to + j, 0) : 0, from = a.window > 0 ? max(to - a.window, 0) : 0;
    int to_min = to, from_max = from;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      to_min = min(to_min, __shfl_xor_sync(0xffffffffu, to_min, d));
      from_max = max(from_max, __shfl_xor_sync(0xffffffffu, from_max, d));
    }
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + lane_off + tile * 128, t_o = tmem + lane_off + 256 + tile * D;
    float m = kNegInf, l = 0.f;
    float ref = kNoRef, highest = kNoRef;  // log2 of the row's reference, and its highest so far
    for (int i = 0; i < steps && ok; ++i) {
      // the step's scales were written before k_full, which the MMAs behind this barrier waited for
      ok = __all_sync(0xffffffffu, mbar_wait(&sm.s_full[tile], i & 1));
      if (!ok) break;
      tc_fence_after();
      const int key = key0 + i * kPreKeys, slot = i & (kPreScaleSlots - 1);
      const bool masked = key < from_max || key + kPreKeys > to_min;
      uint32_t p[64];
      float sum = 0.f;
      // the reference: above the largest scale that the row sees, and not far above
      const float was = ref;
      bool again = i == 0;
      {
        const float e = masked ? pre_largest<D>(sm, slot, from - key, to - key) : sm.top[slot];
        if (e > kNoScale && (e > ref || (e < ref - kPreLower && ref > highest - kPreRise))) {
          const float now = fmaxf(e + 1.f, highest - kPreRise);
          ref = now;
          highest = fmaxf(highest, now);
        }
      }
      // p relative to the maximum so far; only where a score lies far above it (and in the first step) is the maximum taken
      // anew, O and the sum so far rescaled, and p computed again (S is still there)
      if (!again)
        again = masked ? pre_exp<D, true>(sm, slot, t_s, down, m == kNegInf ? 0.f : m, ref, &sum, from - key, to - key, p)
                       : pre_exp<D, false>(sm, slot, t_s, down, m == kNegInf ? 0.f : m, ref, &sum, 0, 0, p);
      again = again || (m == kNegInf && to > key && from < key + kPreKeys);  // a row's first keys (a row without any waits for none)
      if (__any_sync(0xffffffffu, again || ref != was)) {
        float f = was > kNoRef ? pre_pow2(fmaxf(was - ref, -126.f)) : 1.f;
        const bool anew = __any_sync(0xffffffffu, again);
        if (anew) {
          const float top = masked ? pre_max<D, true>(sm, slot, t_s, down, from - key, to - key) : pre_max<D, false>(sm, slot, t_s, down, 0, 0);
          const float now = again ? fmaxf(m, top) : m;  // only rows that need it: a row's p do not depend on the others
          const float fall = now == kNegInf ? 1.f : ex2(m - now);
          m = now;
          l *= fall;
          f *= fall;
        }
        if (i > 0) {
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            uint32_t w[32];
            tmem_ld32(t_o + 32 * c, w);
            tmem_ld_wait();
            uint32_t y[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) y[e] = __float_as_uint(__uint_as_float(w[e]) * f);
            tmem_st16(t_o + 32 * c, y);
#pragma unroll
            for (int e = 0; e < 16; ++e) y[e] = __float_as_uint(__uint_as_float(w[16 + e]) * f);
            tmem_st16(t_o + 32 * c + 16, y);
          }
        }
        if (anew)
          pre_exp<D, true>(sm, slot, t_s, down, m == kNegInf ? 0.f : m, ref, &sum, masked ? from - key : 0, masked ? to - key : kPreKeys, p);
      }
      l += sum;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t y[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) y[e] = p[16 * c + e];
        tmem_st16(t_s + 16 * c, y);
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&sm.p_full[tile]);
    }
    // ---- epilogue ---------------------------------------------------------------------------------------------------
    if (ok && steps > 0) ok = __all_sync(0xffffffffu, mbar_wait(&sm.o_full, 0));
    if (ok) {
      tc_fence_after();
      const float inv = l > 0.f ? ldexpf(V8::kScale, static_cast<int>(fmaxf(ref, -140.f) - kPreRange)) / l : (l == 0.f ? 0.f : l);
      T* dst = static_cast<T*>(a.out) + (static_cast<int64_t>(s.row) + j) * a.out_stride + (head * a.group + row - j * a.group) * D;
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t w[32];
        if (steps > 0) {
          tmem_ld32(t_o + 32 * c, w);
          tmem_ld_wait();
        }
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          union {
            uint4 u;
            T e[8];
          } p;
#pragma unroll
          for (int e = 0; e < 8; ++e) p.e[e] = from_f32<T>(l == 0.f ? 0.f : __uint_as_float(w[8 * h + e]) * inv);
          if (real) *reinterpret_cast<uint4*>(dst + 32 * c + 8 * h) = p.u;
        }
      }
      if (real && a.lse) {
        a.lse[(static_cast<int64_t>(s.row) + j) * a.hq + head * a.group + row - j * a.group] =
            l == 0.f ? kNegInf : (m + log2f(l)) * 0.69314718055994531f;
      }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPreOtherRegs));
  }
  if (warp >= kPreSoftWarps && warp < kPreSoftWarps + kPreCvtWarps) {
    // ---- 8-bit pages -> f16 operands ----------------------------------------------------------------------------------
    // Unit x of an operand: 16 bytes of a key.  Eight lanes of a store take chunks that fall on all banks: for d 128 units
    // 0 - 3 the first half of key 2 y, 4 - 7 that of key 2 y + 1, 8 - 15 their second halves.
    constexpr int kUnits = kPreKeys * (D / 16), kCvtThreads = kPreCvtWarps * 32;
    constexpr int kPer = (kUnits + kCvtThreads - 1) / kCvtThreads;  // units of a thread and operand
    const int ct = tid - kPreSoftWarps * 32;
    const int l2 = ct & 31, cw = ct >> 5;
    auto unit_key = [&](int x) { return D == 128 ? 2 * (x >> 4) + (x >> 2 & 1) : x >> 2; };
    auto unit_sub = [&](int x) { return D == 128 ? (x & 3) + (x >> 3 & 1) * 4 : x & 3; };
    const int in_page = (1 << a.c.shift) - 1;
    uint4 kr[kPer], vr[kPer];
    int page_l = -1;  // lane g: page * hkv + head of 16-key group g of the step that is loaded next, its scales
    float ks_l = 0.f, vs_l = 0.f;
    int64_t entry_l = -1;  // the page table's entry for that group of the step after it: loaded a step ahead
    auto look_up = [&](int i) {
      const int pos = key0 + i * kPreKeys + 16 * (l2 & (kPreGroups - 1));
      entry_l = -1;
      if (i < steps && pos < s.kv) {
        entry_l = a.b.table[seq * a.b.table_stride + (pos >> a.c.shift)];
        if (entry_l < 0) entry_l = a.c.n_pages;  // told apart from "no keys" below
      }
    };
    auto take_up = [&]() {  // entry_l -> page_l and its scales
      page_l = -1;
      if (entry_l >= a.c.n_pages) set_status(a.b.status, SLORA_STATUS_BAD_TABLE);
      if (entry_l >= 0 && entry_l < a.c.n_pages) {
        page_l = static_cast<int>(entry_l * a.c.hkv + head);
        ks_l = a.c.ks[page_l];
        vs_l = a.c.vs[page_l];
      }
    };
    auto fetch = [&](int i, const uint8_t* base, uint4 (&regs)[kPer]) {
#pragma unroll
      for (int p = 0; p < kPer; ++p) {
        const int x = p * kCvtThreads + ct, key = min(unit_key(x), kPreKeys - 1);
        const int ph = __shfl_sync(0xffffffffu, page_l, key >> 4);
        regs[p] = make_uint4(0, 0, 0, 0);
        // keys behind the sequence's end may hold anything, NaN bytes among it
        if (ph >= 0 && x < kUnits && key0 + i * kPreKeys + key < s.kv)
          regs[p] = ld_stream16(base + static_cast<int64_t>((ph << a.c.shift) + ((key0 + i * kPreKeys + key) & in_page)) * D + 16 * unit_sub(x));
      }
    };
    auto put = [&](const uint4 (&regs)[kPer], uint8_t* dst) {
#pragma unroll
      for (int p = 0; p < kPer; ++p) {
        const int u = p * kCvtThreads + ct, key = unit_key(u);
        if (u >= kUnits) continue;
        const uint32_t x = V8::prepare(regs[p].x), y = V8::prepare(regs[p].y), z = V8::prepare(regs[p].z), w = V8::prepare(regs[p].w);
        const int c = 2 * unit_sub(u);
        uint8_t* row = dst + (c >> 3) * kHalf + key * 128;
        *reinterpret_cast<uint4*>(row + (((c & 7) ^ (key & 7)) << 4)) = make_uint4(V8::lo(x), V8::hi(x), V8::lo(y), V8::hi(y));
        *reinterpret_cast<uint4*>(row + ((((c + 1) & 7) ^ (key & 7)) << 4)) = make_uint4(V8::lo(z), V8::hi(z), V8::lo(w), V8::hi(w));
      }
    };
    look_up(0);
    take_up();
    look_up(1);
    int page_now = page_l;
    fetch(0, a.c.k, kr);
    fetch(0, a.c.v, vr);
    for (int i = 0; i < steps && ok; ++i) {
      const int st = i & 1, slot = i & (kPreScaleSlots - 1);
      page_now = page_l;
      const float ks_now = ks_l, vs_now = vs_l;
      take_up();
      look_up(i + 2);
      if (i >= 2) ok = mbar_wait(&sm.k_empty[st], ((i >> 1) - 1) & 1);
      if (!(ok = __all_sync(0xffffffffu, ok))) break;
      // lane g of each warp: scales of 16-key group g (lanes 8 and up repeat them)
      const bool counts = vs_now >= kLeastScale;  // a smaller scale: the values count as zero, p only in the sum
      if (cw == 0) {
        const uint32_t bits = __float_as_uint(vs_now);
        const bool there = page_now >= 0;
        const float e = there && counts ? static_cast<float>(static_cast<int>(bits >> 23) - 126) : kNoScale;
        float top = e;
#pragma unroll
        for (int d = 1; d < kPreGroups; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        const float m = counts ? __uint_as_float((bits & 0x7fffffu) | 0x3f000000u) : 1.f;
        const float e2 = fmaxf(e, top - kPreFar) + kPreRange, log2m = there ? __log2f(m) : kNegInf, ks = there ? ks_now : 0.f;
        const float inv = __fdividef(1.f, m);  // within 2^-22, as log2m: next to nothing beside p's rounding
        if (l2 < kPreGroups) {
          sm.whole[slot][l2] = make_float4(ks, log2m, e2, pre_pow2(top - e2) * inv);
          sm.part[slot][l2] = make_float4(ks, log2m, e + kPreRange, inv);
          if (l2 == 0) sm.top[slot] = top;
        }
      }
      put(kr, sm.k[st]);
      fence_proxy_async();
      mbar_arrive(&sm.k_full[st]);
      if (i + 1 < steps) fetch(i + 1, a.c.k, kr);
      if (i >= 2) ok = mbar_wait(&sm.v_empty[st], ((i >> 1) - 1) & 1);
      if (!(ok = __all_sync(0xffffffffu, ok))) break;
      // values of pages whose scale does not count
#pragma unroll
      for (int p = 0; p < kPer; ++p) {
        const int group = min(unit_key(p * kCvtThreads + ct), kPreKeys - 1) >> 4;
        if (!__shfl_sync(0xffffffffu, counts, group)) vr[p] = make_uint4(0, 0, 0, 0);
      }
      put(vr, sm.v[st]);
      fence_proxy_async();
      mbar_arrive(&sm.v_full[st]);
      if (i + 1 < steps) fetch(i + 1, a.c.v, vr);
    }
  } else if (warp == kPreSoftWarps + kPreCvtWarps && lane == 0 && steps > 0) {
    // ---- MMAs -----------------------------------------------------------------------------------------------------
    const uint32_t idesc_s = umma_idesc<__half>(kPreKeys), idesc_o = umma_idesc<__half>(D) | (1u << 16);  // V: outer-major
    auto score = [&](int tile, int st) {
      const uint32_t qa = smem_u32(sm.q[tile]), kb = smem_u32(sm.k[st]);
#pragma unroll
      for (int x = 0; x < D / 16; ++x) {
        const uint32_t off = (x >> 2) * kHalf + (x & 3) * 32;
        umma_f16(tmem + tile * 128, umma_smem_desc_sw128(qa + off), umma_smem_desc_sw128(kb + off), idesc_s, x > 0);
      }
      umma_commit(&sm.s_full[tile]);
    };
    auto value = [&](int tile, int st, bool more) {
      const uint32_t vb = smem_u32(sm.v[st]);
#pragma unroll
      for (int x = 0; x < kPreKeys / 16; ++x)
        umma_f16_ts(tmem + 256 + tile * D, tmem + tile * 128 + 8 * x, umma_smem_desc_sw128_mn(vb + x * 2048, kHalf), idesc_o,
                    more || x > 0);
    };
    ok = mbar_wait(&sm.p_full[0], 0) && mbar_wait(&sm.p_full[1], 0) && mbar_wait(&sm.k_full[0], 0);
    if (ok) {
      tc_fence_after();
      score(0, 0);
      score(1, 0);
      umma_commit(&sm.k_empty[0]);
    }
    for (int i = 0; i < steps && ok; ++i) {
      const int st = i & 1, nx = (i + 1) & 1;
      const bool next = i + 1 < steps;
      ok = mbar_wait(&sm.v_full[st], (i >> 1) & 1) && mbar_wait(&sm.p_full[0], (i + 1) & 1);
      if (!ok) break;
      tc_fence_after();
      value(0, st, i > 0);
      if (next) {
        if (!(ok = mbar_wait(&sm.k_full[nx], ((i + 1) >> 1) & 1))) break;
        tc_fence_after();
        score(0, nx);
      }
      if (!(ok = mbar_wait(&sm.p_full[1], (i + 1) & 1))) break;
      tc_fence_after();
      value(1, st, i > 0);
      umma_commit(&sm.v_empty[st]);
      if (next) {
        score(1, nx);
        umma_commit(&sm.k_empty[nx]);
      } else {
        umma_commit(&sm.o_full);
      }
    }
  }
  if (!ok) sm.bad = 1;
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (sm.bad && tid == 0) set_status(a.b.status, SLORA_STATUS_TIMEOUT);
  if (warp == kPreThreads / 32 - 1) tmem_dealloc(tmem, 512);
}

}  // namespace slora
