// Attention over the 8-bit cache for few query rows per sequence and KV head (decode, a handful of drafted tokens).
//
//   s[key][row] = scale * ks[page] * (k8[key] . q[row])          p = exp(s - lse[row])
//   o[row]      = sum_key p[key][row] * vs[page] * v8[key]       w[key] += sum_row p[key][row]
//
// What bounds it: the cache is read once, 2 d bytes per key and KV head against 4 d multiply-adds per row, so up to some
// dozens of rows the copy rate does.  Hence: no shared memory on the way of k and v.  A tile is 16 keys of one page; a warp
// loads it with 16-byte loads straight into the registers that mma.sync.m16n8k16 takes as its A operand.
//   S^T [16 keys x 8 rows] = K [16 x d] Q^T     thread (g, t) holds keys g, g + 8 and, of every 64 elements, the 16 from
//                                               16 t on: any order of the inner dimension will do as long as q's is the
//                                               same, so it is the order the bytes lie in.
//   O^T [d x 8 rows] += V^T [d x 16 keys] P^T   thread (g, t) holds keys 2t, 2t + 1, 2t + 8, 2t + 9 and 16 elements from
//                                               16 g on; the pairs (key, key + 1) that the operand wants come out of two
//                                               words by byte permutes, which the conversion to f16 needs anyway.
// P^T is the transpose of S^T's accumulator layout: one movmatrix per 8 x 8.  q is scaled by a power of two per row into
// f16's upper range, the 8-bit values are exact in f16 and so are their products in FP32: the only rounding before the
// sums is p's to f16 (2^-12 relative in the mean).  p is multiplied by vs (relative to a running power of two, so its f16
// range holds for any scales) and the maximum is only raised when some score passes it by 2^8: no shuffles in most steps.
//
// Work is split over the whole batch at once: units of 64 keys of every (sequence, row block, KV head) in one row, cut
// into equal runs, one per CTA; four warps take the 16-key tiles of a unit.  Every CTA adds up the lengths itself (one
// round trip for a few hundred sequences), so there is no plan to build or to keep.  A run that ends inside a (sequence,
// rows, head) leaves its part in the workspace and kv_join_kernel adds the parts in order: results do not depend on timing.
#pragma once

#include "kv_common.cuh"

namespace slora {

constexpr int kAttendWarps = 4;
constexpr int kAttendThreads = kAttendWarps * 32;
constexpr int kAttendUnit = 64;        // keys: one 16-key tile per warp
constexpr int kAttendMinUnits = 2;     // per CTA: shorter runs cost more in the join than they save
constexpr float kLazyMax = 8.f;        // log2 of how far a score may pass the running maximum before it is raised
constexpr float kPRange = 32.f;        // p * vs / ref * 32 <= 2^8 * 2 * 2^5: inside f16
constexpr float kNegInf = -INFINITY;

struct KvAttendArgs {
  KvCache c;
  KvBatch b;
  const void* q;
  void* out;
  float* lse;
  int64_t q_stride, out_stride;
  int hq, group;
  int rows_per_block;  // 8 * NT
  float scale2;        // scale * log2(e)
  int window;
  int min_q, lim_q;    // sequences with min_q <= q_len <= lim_q are this launch's
  float* part;         // [2 * grid][rows_per_block * (d + 2)]
  int* rec;            // [grid][4]: the (sequence, row block, head) that CTA is the first of and does not finish, its parts
};

// ---- the run of units of a CTA -----------------------------------------------------------------------------------------
struct KvRange {
  int lo, hi;  // units [lo, hi) of a sequence's keys that some row of the step sees
};
__device__ __forceinline__ KvRange kv_units(const KvSeq& s, int window) {
  KvRange r;
  r.hi = s.q > 0 ? (s.kv + kAttendUnit - 1) / kAttendUnit : 0;
  r.lo = 0;
  if (window > 0 && s.q > 0) r.lo = max(0, s.kv - s.q + 1 - window) / kAttendUnit;
  if (r.hi <= r.lo && s.q > 0) r.hi = r.lo + 1;  // no key at all: one empty unit, so that the rows are written
  return r;
}
__device__ __forceinline__ int64_t kv_seq_units(const KvAttendArgs& a, const KvSeq& s) {
  if (s.q < a.min_q || s.q > a.lim_q || s.q == 0) return 0;
  const KvRange r = kv_units(s, a.window);
  const int blocks = (s.q * a.group + a.rows_per_block - 1) / a.rows_per_block;
  return static_cast<int64_t>(r.hi - r.lo) * blocks * a.c.hkv;
}

// Sum over all sequences and the sequence that holds unit `want(total)`.  Every thread adds up a run of sequences.
struct KvFind {
  long long sums[16];
  long long at;  // units before the sequence
  int seq;
};
template <int WARPS, typename Units, typename Want>
__device__ __forceinline__ long long kv_find(int n_seq, KvFind* sh, const Units& units, const Want& want) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (n_seq + 32 * WARPS - 1) / (32 * WARPS);
  const int i0 = min(tid * per, n_seq), i1 = min(i0 + per, n_seq);
  long long mine = 0;
  for (int i = i0; i < i1; ++i) mine += units(i);
  long long incl = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long n = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += n;
  }
  if (lane == 31) sh->sums[warp] = incl;
  __syncthreads();
  long long before = incl - mine, total = 0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    if (w < warp) before += sh->sums[w];
    total += sh->sums[w];
  }
  const long long u = want(total);
  if (u >= before && u < before + mine) {
    for (int i = i0; i < i1; ++i) {
      const long long n = units(i);
      if (u < before + n) {
        sh->seq = i;
        sh->at = before;
        break;
      }
      before += n;
    }
  }
  __syncthreads();
  return total;
}
__device__ __forceinline__ long long kv_run(long long total, int grid) {
  const long long r = (total + grid - 1) / grid;
  return r < kAttendMinUnits ? kAttendMinUnits : r;
}

// ---- registers and mma -------------------------------------------------------------------------------------------------
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// What sums taken relative to maximum m weigh relative to `now`; sums that no finite score entered have m = -inf and
// l = 0, or l = NaN (a row of q with a NaN), which has to come through.
__device__ __forceinline__ float part_factor(float m, float l, float now) { return m == kNegInf ? l : ex2(m - now); }
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return reinterpret_cast<const uint32_t&>(h);
}
__device__ __forceinline__ uint4 ld_stream16(const uint8_t* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ uint2 ld_stream8(const uint8_t* p) {
  uint2 v;
  asm volatile("ld.global.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}

// The words of a 16-key tile that this thread feeds to the tensor pipe.
template <int D>
struct KTile {
  static constexpr int C = D / 64;
  uint32_t w[2][C][4];  // [key g, g + 8][64 elements][words of 16 bytes]
  __device__ __forceinline__ void load(const uint8_t* tile, int g, int t) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const uint4 v = ld_stream16(tile + (g + 8 * h) * D + 64 * c + 16 * t);
        w[h][c][0] = v.x, w[h][c][1] = v.y, w[h][c][2] = v.z, w[h][c][3] = v.w;
      }
  }
};
template <int D>
struct VTile {
  static constexpr int N = D / 32;       // words per key: D / 8 bytes in runs of 16 (8 for d 64)
  uint32_t w[4][N];                      // keys 2t, 2t + 1, 2t + 8, 2t + 9
  // element of word i, byte j: VTile::elem(g, i) + j
  __device__ static __forceinline__ int elem(int g, int i) {
    return D == 64 ? 8 * g + 4 * i : 128 * (i >> 2) + 16 * g + 4 * (i & 3);
  }
  __device__ __forceinline__ void load(const uint8_t* tile, int g, int t) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint8_t* row = tile + (2 * t + (j & 1) + 8 * (j >> 1)) * D;
      if (D == 64) {
        const uint2 v = ld_stream8(row + 8 * g);
        w[j][0] = v.x, w[j][1] = v.y;
      } else {
#pragma unroll
        for (int r = 0; r < D / 128; ++r) {
          const uint4 v = ld_stream16(row + 128 * r + 16 * g);
          w[j][4 * r] = v.x, w[j][4 * r + 1] = v.y, w[j][(4 * r + 2) % N] = v.z, w[j][(4 * r + 3) % N] = v.w;
        }
      }
    }
  }
};

// q of one row block as mma B operands: thread (g, t) holds row g of each n-tile, 16 elements of every 64.
template <int D, int NT, typename T>
struct QTile {
  static constexpr int C = D / 64;
  uint32_t w[NT][4 * C][2];
  float mul[NT][2];  // what the products of rows 2t, 2t + 1 still have to be multiplied by
  __device__ __forceinline__ void load(const KvAttendArgs& a, const KvSeq& s, int rb, int head, int g, int t, float kscale) {
    const T* q = static_cast<const T*>(a.q);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = rb * a.rows_per_block + nt * 8 + g;
      float f[C][16];
      float top = 0.f;
      const bool real = r < s.q * a.group;
      const int j = r / a.group;
      const T* row = q + (static_cast<int64_t>(s.row) + j) * a.q_stride + (head * a.group + r - j * a.group) * D;
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
          if (real) cvt8<T>(*reinterpret_cast<const uint4*>(row + 64 * c + 16 * t + 8 * h), x);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            f[c][8 * h + e] = x[e];
            top = fmaxf(top, fabsf(x[e]));
          }
        }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // 2^e with top * 2^e in [2^14, 2^15); the exponent is kept where both it and its inverse are normal numbers
      const int e = top > 0.f ? min(max(141 - static_cast<int>(__float_as_uint(top) >> 23), -100), 100) : 0;
      const float up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
      const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23) * kscale;
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          w[nt][4 * c + i][0] = pack_f16(f[c][4 * i] * up, f[c][4 * i + 1] * up);
          w[nt][4 * c + i][1] = pack_f16(f[c][4 * i + 2] * up, f[c][4 * i + 3] * up);
        }
      mul[nt][0] = __shfl_sync(0xffffffffu, down, 8 * t);
      mul[nt][1] = __shfl_sync(0xffffffffu, down, 8 * t + 4);
    }
  }
};

template <int D, int NT, int KIND>
__device__ __forceinline__ void kv_scores(float (&c)[NT][4], const KTile<D>& k, const uint32_t (&q)[NT][D / 16][2]) {
  using V8 = Kv8<KIND>;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) c[nt][0] = c[nt][1] = c[nt][2] = c[nt][3] = 0.f;
#pragma unroll
  for (int s = 0; s < D / 16; ++s) {
    const uint32_t x = V8::prepare(k.w[0][s >> 2][s & 3]), y = V8::prepare(k.w[1][s >> 2][s & 3]);
    const uint32_t a0 = V8::lo(x), a2 = V8::hi(x), a1 = V8::lo(y), a3 = V8::hi(y);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) mma_f16(c[nt], a0, a1, a2, a3, q[nt][s][0], q[nt][s][1]);
  }
}

// What a warp carries through its tiles of one (sequence, row block, head).
template <int D, int NT>
struct AttendState {
  float o[NT][D / 16][4];  // O^T: element elem(g, i) + 2 (mt & 1) (+ 1: entries 2, 3), rows 2t, 2t + 1; mt = 2 i + ...
  float m[NT][2], l[NT][2];
  float ref;               // power of two the value scales are taken relative to; 0: none yet
};

template <int D, int NT, int KIND, typename T>
struct AttendTypes {
  static constexpr int kRows = 8 * NT;
  static constexpr int kRegs = NT * D / 4;           // accumulator words of a thread
  static constexpr int kPartWords = kRows * (D + 2);
  struct Smem {
    KvFind find;
    float o[kAttendWarps][kRegs][32];
    float m[kAttendWarps][kRows], l[kAttendWarps][kRows], ref[kAttendWarps];
  };
};

// Rows 8 nt + 2 t + c of the row block: where their output goes.
template <int D, int KIND, typename T>
__device__ __forceinline__ void store_row4(const KvAttendArgs& a, const KvSeq& s, int head, int r, int elem, const float (&v)[4]) {
  const int j = r / a.group;
  T* row = static_cast<T*>(a.out) + (static_cast<int64_t>(s.row) + j) * a.out_stride + (head * a.group + r - j * a.group) * D + elem;
  union {
    uint2 u;
    T e[4];
  } p;
#pragma unroll
  for (int i = 0; i < 4; ++i) p.e[i] = from_f32<T>(v[i]);
  *reinterpret_cast<uint2*>(row) = p.u;
}

template <int D, int NT, int KIND, typename T>
__global__ void __launch_bounds__(kAttendThreads, NT == 1 && D <= 128 ? 4 : 2) kv_attend_kernel(const KvAttendArgs a) {
  using V8 = Kv8<KIND>;
  using Ty = AttendTypes<D, NT, KIND, T>;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  typename Ty::Smem& sm = *reinterpret_cast<typename Ty::Smem*>(smem_raw);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  pdl_launch_dependents();
  pdl_wait();
  const long long me = blockIdx.x, grid = gridDim.x;
  if (tid == 0) *reinterpret_cast<int4*>(a.rec + 4 * me) = make_int4(-1, 0, 0, 0);
  const long long total = kv_find<kAttendWarps>(
      a.b.n_seq, &sm.find,
      [&](int i) {
        const KvSeq x = kv_seq(a.b, i);
        if (x.bad && me == 0) set_status(a.b.status, SLORA_STATUS_BAD_TABLE);
        return static_cast<long long>(kv_seq_units(a, x));
      },
      [&](long long n) { return me * kv_run(n, static_cast<int>(grid)); });
  const long long run = kv_run(total, static_cast<int>(grid));
  long long u = me * run;
  const long long u_end = min(u + run, total);
  if (u >= u_end) return;
  int seq = sm.find.seq;
  long long seq_at = sm.find.at;  // units before the sequence
  KvSeq s = kv_seq(a.b, seq);

  while (u < u_end) {
    // the piece of the run inside one (sequence, row block, head)
    long long n = kv_seq_units(a, s);
    while (u >= seq_at + n) {
      seq_at += n;
      s = kv_seq(a.b, ++seq);
      n = kv_seq_units(a, s);
    }
    const KvRange range = kv_units(s, a.window);
    const int per = range.hi - range.lo;
    const int idx = static_cast<int>((u - seq_at) / per);   // row block * hkv + head
    const int first = static_cast<int>((u - seq_at) - static_cast<long long>(idx) * per);
    const int count = static_cast<int>(min(static_cast<long long>(per - first), u_end - u));
    const int rb = idx / a.c.hkv, head = idx - rb * a.c.hkv;

    QTile<D, NT, T> q;
    q.load(a, s, rb, head, g, t, a.scale2 * V8::kScale);
    // keys that rows 2t, 2t + 1 of each n-tile see: [from, to)
    int to[NT][2], from[NT][2], to_min = s.kv, from_max = 0;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int r = rb * a.rows_per_block + nt * 8 + 2 * t + c;
        const int j = min(r / a.group, s.q - 1);
        to[nt][c] = max(s.kv - s.q + j + 1, 0);
        from[nt][c] = a.window > 0 ? max(to[nt][c] - a.window, 0) : 0;
        to_min = min(to_min, to[nt][c]);
        from_max = max(from_max, from[nt][c]);
      }
#pragma unroll
    for (int d = 1; d < 4; d <<= 1) {
      to_min = min(to_min, __shfl_xor_sync(0xffffffffu, to_min, d));
      from_max = max(from_max, __shfl_xor_sync(0xffffffffu, from_max, d));
    }

    AttendState<D, NT> st;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < D / 16; ++i) st.o[nt][i][0] = st.o[nt][i][1] = st.o[nt][i][2] = st.o[nt][i][3] = 0.f;
      st.m[nt][0] = st.m[nt][1] = kNegInf;
      st.l[nt][0] = st.l[nt][1] = 0.f;
    }
    st.ref = 0.f;

    // this warp's tiles: 16 keys from key0 + 64 i on; lane l knows page and scales of tile base + l
    const int key0 = (range.lo + first) * kAttendUnit + 16 * warp;
    const int tiles = key0 < s.kv ? min(count, (s.kv - key0 + kAttendUnit - 1) / kAttendUnit) : 0;
    const int in_page = (1 << a.c.shift) - 1;
    int64_t off_l = -1;
    float ks_l = 0.f, vs_l = 0.f;
    auto fetch = [&](int base) {
      off_l = -1;
      if (base + lane < tiles) {
        const int key = key0 + (base + lane) * kAttendUnit;
        const int64_t p = kv_page(a.c, a.b, seq, key);
        if (p >= 0) {
          const int64_t ph = p * a.c.hkv + head;
          off_l = ((ph << a.c.shift) + (key & in_page)) * D;
          ks_l = a.c.ks[ph];
          vs_l = a.c.vs[ph];
        } else {
          set_status(a.b.status, SLORA_STATUS_BAD_TABLE);
        }
      }
    };
    fetch(0);
    int64_t off = __shfl_sync(0xffffffffu, off_l, 0);
    KTile<D> k;
    VTile<D> v;
    if (off >= 0) {
      k.load(a.c.k + off, g, t);
      v.load(a.c.v + off, g, t);
    }
    for (int i = 0; i < tiles; ++i) {
      const float ks = __shfl_sync(0xffffffffu, ks_l, i & 31);
      const float vs = __shfl_sync(0xffffffffu, vs_l, i & 31);
      if (((i + 1) & 31) == 0) fetch(i + 1);
      const int64_t next = i + 1 < tiles ? __shfl_sync(0xffffffffu, off_l, (i + 1) & 31) : -1;
      const bool here = off >= 0;  // the same in all lanes
      off = next;
      if (!here) {
        if (next >= 0) {
          k.load(a.c.k + next, g, t);
          v.load(a.c.v + next, g, t);
        }
        continue;
      }
      float c[NT][4];
      kv_scores<D, NT, KIND>(c, k, q.w);
      if (next >= 0) k.load(a.c.k + next, g, t);
      const int key = key0 + i * kAttendUnit;
      bool raise = vs > st.ref;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float f0 = q.mul[nt][0] * ks, f1 = q.mul[nt][1] * ks;
        c[nt][0] *= f0;
        c[nt][1] *= f1;
        c[nt][2] *= f0;
        c[nt][3] *= f1;
      }
      if (key < from_max || key + 16 > to_min) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int pos = key + g + 8 * (e >> 1);
            if (pos < from[nt][e & 1] || pos >= to[nt][e & 1]) c[nt][e] = kNegInf;
          }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
        raise = raise || fmaxf(c[nt][0], c[nt][2]) > st.m[nt][0] + kLazyMax || fmaxf(c[nt][1], c[nt][3]) > st.m[nt][1] + kLazyMax;
      if (__any_sync(0xffffffffu, raise)) {
        float up = 1.f;
        if (vs > st.ref) {
          const float now = __uint_as_float(min(max((__float_as_uint(vs) >> 23) + 1u, 27u), 254u) << 23);  // above vs
          up = st.ref > 0.f ? st.ref / now : 0.f;
          st.ref = now;
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            float top = fmaxf(c[nt][x], c[nt][x + 2]);
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
            const float m = fmaxf(st.m[nt][x], top);
            const float f = m == kNegInf ? 1.f : ex2(st.m[nt][x] - m);
            st.m[nt][x] = m;
            st.l[nt][x] *= f;
#pragma unroll
            for (int mt = 0; mt < D / 16; ++mt) {
              st.o[nt][mt][x] *= f * up;
              st.o[nt][mt][x + 2] *= f * up;
            }
          }
      }
      const float w = st.ref > 0.f ? vs * (kPRange / st.ref) : 0.f;
      uint32_t p[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float m0 = st.m[nt][0] == kNegInf ? 0.f : st.m[nt][0], m1 = st.m[nt][1] == kNegInf ? 0.f : st.m[nt][1];
        const float e0 = ex2(c[nt][0] - m0), e1 = ex2(c[nt][1] - m1), e2 = ex2(c[nt][2] - m0), e3 = ex2(c[nt][3] - m1);
        st.l[nt][0] += e0 + e2;
        st.l[nt][1] += e1 + e3;
        p[nt][0] = transpose8x8(pack_f16(e0 * w, e1 * w));
        p[nt][1] = transpose8x8(pack_f16(e2 * w, e3 * w));
      }
#pragma unroll
      for (int x = 0; x < VTile<D>::N; ++x) {
        const uint32_t w0 = V8::prepare(v.w[0][x]), w1 = V8::prepare(v.w[1][x]);
        const uint32_t w2 = V8::prepare(v.w[2][x]), w3 = V8::prepare(v.w[3][x]);
        const uint32_t l01 = prmt(w0, w1, 0x5140), h01 = prmt(w0, w1, 0x7362);
        const uint32_t l23 = prmt(w2, w3, 0x5140), h23 = prmt(w2, w3, 0x7362);
        const uint32_t a0 = V8::lo(l01), a1 = V8::hi(l01), a2 = V8::lo(l23), a3 = V8::hi(l23);
        const uint32_t b0 = V8::lo(h01), b1 = V8::hi(h01), b2 = V8::lo(h23), b3 = V8::hi(h23);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          mma_f16(st.o[nt][2 * x], a0, a1, a2, a3, p[nt][0], p[nt][1]);
          mma_f16(st.o[nt][2 * x + 1], b0, b1, b2, b3, p[nt][0], p[nt][1]);
        }
      }
      if (next >= 0) v.load(a.c.v + next, g, t);
    }

    // join the warps: every warp leaves its sums, then each thread adds a quarter of the words over the warps
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) st.l[nt][x] += __shfl_xor_sync(0xffffffffu, st.l[nt][x], d);
        if (g == 0) {
          sm.m[warp][8 * nt + 2 * t + x] = st.m[nt][x];
          sm.l[warp][8 * nt + 2 * t + x] = st.l[nt][x];
        }
      }
    if (lane == 0) sm.ref[warp] = st.ref * (V8::kScale / kPRange);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int mt = 0; mt < D / 16; ++mt)
#pragma unroll
        for (int e = 0; e < 4; ++e) sm.o[warp][(nt * (D / 16) + mt) * 4 + e][lane] = st.o[nt][mt][e];
    __syncthreads();
    const bool whole = count == per;
    const int slot = whole ? -1 : static_cast<int>(2 * me) + (u == me * run ? 0 : 1);
    float* part = whole ? nullptr : a.part + static_cast<int64_t>(slot) * Ty::kPartWords;
#pragma unroll
    for (int x = warp; x < Ty::kRegs / 8; x += kAttendWarps) {
      // words [8 x, 8 x + 8) are m-tiles 2i, 2i + 1 of n-tile nt: elements elem(g, i) + 0 .. 3 of rows 2t, 2t + 1
      const int nt = x / (D / 32), i = x - nt * (D / 32);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int r = 8 * nt + 2 * t + c;
        float m = kNegInf;
#pragma unroll
        for (int w = 0; w < kAttendWarps; ++w) m = fmaxf(m, sm.m[w][r]);
        float l = 0.f, v4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kAttendWarps; ++w) {
          const float f = part_factor(sm.m[w][r], sm.l[w][r], m);
          l += f * sm.l[w][r];
          const float fo = f * sm.ref[w];
          if (fo != 0.f) {
            v4[0] += fo * sm.o[w][8 * x + c][lane];
            v4[1] += fo * sm.o[w][8 * x + 2 + c][lane];
            v4[2] += fo * sm.o[w][8 * x + 4 + c][lane];
            v4[3] += fo * sm.o[w][8 * x + 6 + c][lane];
          }
        }
        const int row = rb * a.rows_per_block + r;
        if (row >= s.q * a.group) continue;
        const int elem = VTile<D>::elem(g, i);
        if (whole) {
          const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
#pragma unroll
          for (int e = 0; e < 4; ++e) v4[e] *= inv;
          store_row4<D, KIND, T>(a, s, head, row, elem, v4);
          if (a.lse && i == 0 && g == 0) {
            const int j = row / a.group;
            a.lse[(static_cast<int64_t>(s.row) + j) * a.hq + head * a.group + row - j * a.group] =
                l == 0.f ? kNegInf : (m + log2f(l)) * 0.69314718055994531f;
          }
        } else {
          *reinterpret_cast<float4*>(part + r * D + elem) = make_float4(v4[0], v4[1], v4[2], v4[3]);
          if (i == 0 && g == 0) {
            part[Ty::kRows * D + 2 * r] = m;
            part[Ty::kRows * D + 2 * r + 1] = l;
          }
        }
      }
    }
    if (!whole && first == 0 && tid == 0) {
      // the first CTA of a cut piece names it for the join: the CTAs after it hold their parts in slot 0
      const long long end = seq_at + static_cast<long long>(idx + 1) * per;
      *reinterpret_cast<int4*>(a.rec + 4 * me) =
          make_int4(seq, idx, slot, static_cast<int>((end - 1) / run - me) + 1);
    }
    u += count;
    __syncthreads();
  }
}

// Adds the parts of the (sequence, row block, head) that CTA blockIdx.x of the attention left unfinished, in the order of
// its keys.  Threads own (row, four elements); kJoinGroups of them share the parts.
constexpr int kJoinThreads = 512;
template <int D, typename T>
__global__ void __launch_bounds__(kJoinThreads) kv_join_kernel(const KvAttendArgs a) {
  __shared__ float4 sh_o[kJoinThreads];
  __shared__ float2 sh_ml[kJoinThreads];
  pdl_launch_dependents();
  pdl_wait();
  const int4 rec = *reinterpret_cast<const int4*>(a.rec + 4 * static_cast<int64_t>(blockIdx.x));
  if (rec.x < 0) return;
  const KvSeq s = kv_seq(a.b, rec.x);
  const int rb = rec.y / a.c.hkv, head = rec.y - rb * a.c.hkv;
  const int rows = min(a.rows_per_block, s.q * a.group - rb * a.rows_per_block);
  const int64_t words = static_cast<int64_t>(a.rows_per_block) * (D + 2);
  const int per_row = D / 4, at_once = kJoinThreads / per_row;
  const int groups = rows >= at_once ? 1 : at_once / rows;    // threads that share an output's parts
  for (int r0 = 0; r0 < rows; r0 += at_once) {
    const int e = threadIdx.x % per_row, x = threadIdx.x / per_row;
    const int r = groups == 1 ? r0 + x : x % rows, grp = groups == 1 ? 0 : x / rows;
    float m = kNegInf, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    if (r < rows && grp < groups) {
      for (int p = grp; p < rec.w; p += groups) {
        const int slot = p == 0 ? rec.z : 2 * (static_cast<int>(blockIdx.x) + p);
        const float* part = a.part + slot * words;
        const float2 ml = *reinterpret_cast<const float2*>(part + static_cast<int64_t>(a.rows_per_block) * D + 2 * r);
        const float4 v = *reinterpret_cast<const float4*>(part + r * D + 4 * e);
        const float now = fmaxf(m, ml.x);
        const float f0 = part_factor(m, l, now), f1 = part_factor(ml.x, ml.y, now);
        l = l * f0 + ml.y * f1;
        o.x = o.x * f0 + v.x * f1;
        o.y = o.y * f0 + v.y * f1;
        o.z = o.z * f0 + v.z * f1;
        o.w = o.w * f0 + v.w * f1;
        m = now;
      }
    }
    sh_o[threadIdx.x] = o;
    sh_ml[threadIdx.x] = make_float2(m, l);
    __syncthreads();
    if (r < rows && grp == 0) {
      for (int k = 1; k < groups; ++k) {
        const int y = threadIdx.x + k * rows * per_row;
        const float2 ml = sh_ml[y];
        const float4 v = sh_o[y];
        const float now = fmaxf(m, ml.x);
        const float f0 = part_factor(m, l, now), f1 = part_factor(ml.x, ml.y, now);
        l = l * f0 + ml.y * f1;
        o.x = o.x * f0 + v.x * f1;
        o.y = o.y * f0 + v.y * f1;
        o.z = o.z * f0 + v.z * f1;
        o.w = o.w * f0 + v.w * f1;
        m = now;
      }
      const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
      const float v4[4] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv};
      const int row = rb * a.rows_per_block + r;
      store_row4<D, 0, T>(a, s, head, row, 4 * e, v4);
      if (a.lse && e == 0) {
        const int j = row / a.group;
        a.lse[(static_cast<int64_t>(s.row) + j) * a.hq + head * a.group + row - j * a.group] =
            l == 0.f ? kNegInf : (m + log2f(l)) * 0.69314718055994531f;
      }
    }
    __syncthreads();
  }
}

// Accumulated attention weights: with lse known, the keys' scores once more and their exponentials summed over the rows.
// Tiles are independent; a warp keeps the keys of a tile in registers and walks through the sequence's rows.
template <int D, int KIND, typename T>
__global__ void __launch_bounds__(kAttendThreads, D <= 128 ? 4 : 2) kv_weights_kernel(const KvAttendArgs a) {
  using V8 = Kv8<KIND>;
  __shared__ KvFind find;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  pdl_launch_dependents();
  pdl_wait();
  const long long me = blockIdx.x, grid = gridDim.x;
  auto units = [&](int i) {
    const KvSeq s = kv_seq(a.b, i);
    if (s.q == 0) return 0ll;
    const KvRange r = kv_units(s, a.window);
    return static_cast<long long>(r.hi - r.lo) * a.c.hkv;
  };
  const long long total = kv_find<kAttendWarps>(a.b.n_seq, &find, units, [&](long long n) { return me * ((n + grid - 1) / grid); });
  const long long run = (total + grid - 1) / grid;
  long long u = me * run;
  const long long u_end = min(u + run, total);
  if (u >= u_end) return;
  int seq = find.seq;
  long long seq_at = find.at;
  long long n = units(seq);
  KvSeq s = kv_seq(a.b, seq);
  QTile<D, 1, T> q;
  int have_seq = -1, have_head = -1;
  for (; u < u_end; ++u) {
    while (u >= seq_at + n) {
      seq_at += n;
      n = units(++seq);
      s = kv_seq(a.b, seq);
    }
    const KvRange range = kv_units(s, a.window);
    const int per = range.hi - range.lo;
    const int head = static_cast<int>((u - seq_at) / per);
    const int key = (range.lo + static_cast<int>((u - seq_at) - static_cast<long long>(head) * per)) * kAttendUnit + 16 * warp;
    if (key >= s.kv) continue;
    const int64_t p = kv_page(a.c, a.b, seq, key);
    if (p < 0) continue;
    const int64_t ph = p * a.c.hkv + head;
    const int in_page = key & ((1 << a.c.shift) - 1);
    const float ks = a.c.ks[ph];
    KTile<D> k;
    k.load(a.c.k + ((ph << a.c.shift) + in_page) * D, g, t);
    float sum0 = 0.f, sum1 = 0.f;
    const int rows = s.q * a.group;
    for (int rb = 0; 8 * rb < rows; ++rb) {
      if (rows > 8 || have_seq != seq || have_head != head) {
        q.load(a, s, rb, head, g, t, a.scale2 * V8::kScale);
        have_seq = seq;
        have_head = head;
      }
      float c[1][4];
      kv_scores<D, 1, KIND>(c, k, q.w);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int r = 8 * rb + 2 * t + x;
        if (r >= rows) continue;
        const int j = r / a.group;
        const int to = s.kv - s.q + j + 1, from = a.window > 0 ? to - a.window : 0;
        const float lse = a.lse[(static_cast<int64_t>(s.row) + j) * a.hq + head * a.group + r - j * a.group];
        const float lse2 = lse * 1.4426950408889634f;
        const float f = q.mul[0][x] * ks;
        if (lse == kNegInf) continue;
        if (key + g >= from && key + g < to) sum0 += ex2(c[0][x] * f - lse2);
        if (key + g + 8 >= from && key + g + 8 < to) sum1 += ex2(c[0][x + 2] * f - lse2);
      }
    }
#pragma unroll
    for (int d = 1; d < 4; d <<= 1) {
      sum0 += __shfl_xor_sync(0xffffffffu, sum0, d);
      sum1 += __shfl_xor_sync(0xffffffffu, sum1, d);
    }
    if (t < 2) {
      // an atomic add only because two sequences may share a page; a page of one sequence gets one add per token
      const int pos = in_page + g + 8 * t;
      const float add = t == 0 ? sum0 : sum1;
      if (key + g + 8 * t < s.kv && add != 0.f) atomicAdd(a.c.w + (ph << a.c.shift) + pos, add);
    }
  }
}

}  // namespace slora
