// Attention over the 8-bit cache for few query rows per sequence and KV head (decode, a handful of drafted tokens).
//
//   s[key][row] = scale * ks[page] * (k8[key] . q[row])          p = exp(s - lse[row])
//   o[row]      = sum_key p[key][row] * vs[page] * v8[key]       w[key] += sum_row p[key][row]
//
// What bounds it: the cache is read once, 2 d bytes per key and KV head against 4 d multiply-adds per row, so up to some
// dozens of rows the copy rate does.  Hence: no shared memory on the way of k and v.  A tile is 16 keys of one page; a warp
// loads it with 16-byte loads straight into the registers that mma.sync.m16n8k16 takes as its A operand, each operand of
// the next tile as soon as the present one has been multiplied.  (Rings in shared memory, filled by cp.async or by the
// copy engine, measured 20 % slower over long sequences: the copies' issue, 900 cycles a tile and warp, is more than
// the registers they free are worth.)
//   S^T [16 keys x 8 rows] = K [16 x d] Q^T     thread (g, t) holds keys g, g + 8 and, of every 64 elements, the 16 from
//                                               16 t on: any order of the inner dimension will do as long as q's is the
//                                               same, so it is the order the bytes lie in.
//   O^T [d x 8 rows] += V^T [d x 16 keys] P^T   thread (g, t) holds keys 2t, 2t + 1, 2t + 8, 2t + 9 and 16 elements from
//                                               16 g on; the pairs (key, key + 1) that the operand wants come out of two
//                                               words by byte permutes, which the conversion to f16 needs anyway.
// P^T is the transpose of S^T's accumulator layout: one movmatrix per 8 x 8.  q is scaled by a power of two per row into
// f16's upper range, the 8-bit values are exact in f16 and so are their products in FP32: the only rounding before the
// sums is that of p * vs to f16 (2^-12 relative in the mean; for f16 outputs it goes in as two f16 numbers).  It is taken
// times a power of two, a row's own, that follows the scales of the tiles the row sees: down to p of 2^-10 it keeps f16's
// full precision whatever the scales, and pages that only other rows see cost a row nothing.  The maximum is only raised
// when some score passes it by 2^8, the power of two only changed when a scale leaves its band: no shuffles in most steps.
// (One power of two for all rows of a warp, which only rose, let a page that some row sees round the p of the others; 0 to
// 2 % less time at the sizes below, 7 % less with 32 rows at d 64.)
//
// Work is split over the whole batch at once: the tiles of every (sequence, row block, KV head) in one row, cut into runs
// of equal cost, one per CTA (a piece costs kAttendPiece tiles before its first key: its q, its page table, its output).
// The four warps of a CTA take its tiles in turn, so that 8 KB of k and of v that lie together are read together (runs per
// warp, without any join inside the CTA, measured 15 % slower over long sequences).  While a piece ends the next one's
// first tiles are on their way.  Every CTA adds up the lengths itself (one round trip for a few hundred sequences), so
// there is no plan to build or to keep.  A run that ends inside a (sequence, rows, head) leaves its part in the workspace
// and kv_join_kernel adds the parts in order: results do not depend on timing.
//
// Measured (d 128): 16 sequences of 8271 to 46873 tokens, 64 q heads on 8, 681 MB of cache: 134 us with the join, 0.77 of the
// copy rate; 64 sequences of 65 to 3955 tokens, 32 heads on 32, f16, 491 MB: 115 us, 0.65 (2048 pieces: their starts, and
// the instructions of 16 warps per SM); one short sequence: 15.2 us, two launches and some 7 us from the first load to the
// first product; one token of 64 heads on one KV head over 32768 keys: 39 us.
//
// Attention weights (add_weights) need the softmax's sum first: the scores go to the workspace (4 bytes per key and row,
// against the 2 d that the key cost) and kv_weights_kernel adds up their exponentials (32 sequences of 1000 to 8192 tokens,
// 32 heads on 8, e4m3: 68 us in all); where that would take too much memory kv_reweigh_kernel computes the scores again.
#pragma once

#include <type_traits>

#include "kv_common.cuh"

namespace slora {

constexpr int kAttendWarps = 4;
constexpr int kAttendThreads = kAttendWarps * 32;
constexpr int kAttendTile = 16;        // keys
constexpr int kAttendPiece = 12;       // tiles that starting and ending a piece is worth
constexpr int kAttendMinRun = kAttendPiece + 8;  // per CTA: shorter runs cost more in the join than they save
constexpr float kLazyMax = 8.f;        // log2 of how far a score may pass the running maximum before it is raised
// p * vs * w, w a row's power of two: w is taken so that vs * w lies in [2^4, 2^5) and kept while it lies in [2^-4, 2^6), so
// p * vs * w <= 2^8 * 2^6 is inside f16; it never rises by more than kWRise in all, so that the sums stay inside FP32
constexpr uint32_t kWTaken = 4, kWLow = 4, kWHigh = 6;
constexpr float kWRise = 18446744073709551616.f;  // 2^64
constexpr float kNegInf = -INFINITY;
constexpr float kNoMax = -1e30f;       // maximum of no score: finite, so that differences of maxima are numbers

// CTAs of the attention per SM, by what their registers allow (4 x 128 or 2 x 255; three of 168 spilled: 71 -> 112 us).
__host__ __device__ constexpr int attend_ctas(int nt, int d) { return nt * d <= 128 ? 4 : 2; }

struct KvAttendArgs {
  KvCache c;
  KvBatch b;
  const void* q;
  void* out;
  float* lse;
  int64_t q_stride, out_stride;
  int hq, group;
  int rows_per_block;  // 8 * NT
  int part_rows;       // rows of a block that any sequence has
  int blocks;          // row blocks that a sequence may have
  float scale2;        // scale * log2(e)
  int window;
  int min_q, lim_q;    // sequences with min_q <= q_len <= lim_q are this launch's
  int runs;            // CTAs that share the work
  float* part;         // [2 * runs][part_rows * (d + 4)]: sums, maximum and sum of p per row (a multiple of 16 bytes)
  int* rec;            // [runs][4]: the (sequence, row block, head) that a run is the first of and does not finish, its parts
  float* scores;       // [cost units][part_rows][16] or null: scores of every tile, log2 units
};

// ---- the run of tiles of a CTA ------------------------------------------------------------------------------------------
struct KvRange {
  int lo, hi;  // tiles [lo, hi) of a sequence's keys that some row of the step sees
};
__device__ __forceinline__ KvRange kv_tiles(const KvSeq& s, int window) {
  KvRange r;
  r.hi = s.q > 0 ? (s.kv + kAttendTile - 1) / kAttendTile : 0;
  r.lo = 0;
  if (window > 0 && s.q > 0) r.lo = max(0, max(s.kv - s.q + 1, 0) - window) / kAttendTile;
  if (r.hi <= r.lo && s.q > 0) r.hi = r.lo + 1;  // no key at all: one empty tile, so that the rows are written
  return r;
}
__device__ __forceinline__ long long kv_seq_cost(const KvAttendArgs& a, const KvSeq& s) {
  if (s.q < a.min_q || s.q > a.lim_q || s.q == 0) return 0;
  const KvRange r = kv_tiles(s, a.window);
  const int blocks = (s.q * a.group + a.rows_per_block - 1) / a.rows_per_block;
  return static_cast<long long>(r.hi - r.lo + kAttendPiece) * blocks * a.c.hkv;
}

// Sum over all sequences and, for each of N targets, the sequence that holds unit want(total, k).  Every thread adds up a
// run of sequences.
constexpr int kFindTargets = 4;
struct KvFind {
  long long sums[16];
  long long at[kFindTargets];  // units before the sequence
  int seq[kFindTargets];
};
template <int WARPS, int N, typename Units, typename Want>
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
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const long long u = want(total, k);
    if (u >= before && u < before + mine) {
      long long b = before;
      for (int i = i0; i < i1; ++i) {
        const long long n = per == 1 ? mine : units(i);
        if (u < b + n) {
          sh->seq[k] = i;
          sh->at[k] = b;
          break;
        }
        b += n;
      }
    }
  }
  __syncthreads();
  return total;
}
// Units of a run.  (Totals beyond 2^32 are no real batch: the division is 32-bit wherever it can be.)
__device__ __forceinline__ long long kv_run(long long total, int runs) {
  const long long n = total + runs - 1;
  const long long r = n <= 0xffffffffll ? static_cast<long long>(static_cast<uint32_t>(n) / static_cast<uint32_t>(runs)) : n / runs;
  return r < kAttendMinRun ? kAttendMinRun : r;
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
  static constexpr int N = D / 32;       // words per key: 16 bytes of every 128 (8 of 64)
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

// q of one row block as mma B operands: thread (g, t) holds row g of each n-tile, the chunks of KTile.
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
  // two chains of sums per n-tile: an mma waits for the one before it in its chain
  float d[NT][4];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 4; ++e) c[nt][e] = d[nt][e] = 0.f;
#pragma unroll
  for (int s = 0; s < D / 16; ++s) {
    const uint32_t x = V8::prepare(k.w[0][s >> 2][s & 3]), y = V8::prepare(k.w[1][s >> 2][s & 3]);
    const uint32_t a0 = V8::lo(x), a2 = V8::hi(x), a1 = V8::lo(y), a3 = V8::hi(y);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) mma_f16(s & 1 ? d[nt] : c[nt], a0, a1, a2, a3, q[nt][s][0], q[nt][s][1]);
  }
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 4; ++e) c[nt][e] += d[nt][e];
}

// What a warp carries through its tiles of one (sequence, row block, head).
template <int D, int NT>
struct AttendState {
  float o[NT][D / 16][4];  // O^T: element elem(g, i) + 2 (mt & 1) (+ 1: entries 2, 3), rows 2t, 2t + 1; mt = 2 i + ...
  float m[NT][2], l[NT][2];
  float w[NT][2];          // the row's power of two; 0: none yet
};

// One piece of a run: tiles [first, first + count) of the `per` of one (sequence, row block, head).
struct KvPiece {
  KvSeq s;
  int seq, idx;  // idx: row block * hkv + head
  int lo, first, count, per;
  int tiles;       // of the count, those that hold keys (a sequence without keys has one empty tile)
  long long unit;  // cost unit of tile 0
};

// What a CTA needs between pieces only: in shared memory, so that the registers go to the tiles.
struct KvRun {
  KvPiece piece[4];        // piece p in slot p & 3; count 0: there is none
  long long u, u_end;      // what is left of the run
  long long at, cost;      // units before the sequence that was reached, units of it
  int2 see[2][32];         // keys [x, y) that each row of an even / odd piece sees
};

// The next piece of the run into *out; `from`: the one before it.  (Called by one warp, once per piece: not inlined.)
__device__ __noinline__ void kv_next_piece(const KvAttendArgs& a, KvRun* run, const KvPiece* from, KvPiece* out, int lane) {
  KvPiece p = *from;
  long long u = run->u, at = run->at, cost = run->cost;
  const long long u_end = run->u_end;
  p.count = 0;
  while (u < u_end && p.count <= 0) {
    while (u >= at + cost) {
      at += cost;
      p.s = kv_seq(a.b, ++p.seq);
      cost = kv_seq_cost(a, p.s);
    }
    const KvRange range = kv_tiles(p.s, a.window);
    // a cut inside a piece's first kAttendPiece units belongs to the run behind it
    p.lo = range.lo;
    p.per = range.hi - range.lo;
    const int each = p.per + kAttendPiece;
    const long long in = u - at;
    p.idx = in <= 0xffffffffll ? static_cast<int>(static_cast<uint32_t>(in) / static_cast<uint32_t>(each)) : static_cast<int>(in / each);
    const int begin = static_cast<int>(in - static_cast<long long>(p.idx) * each);
    const int until = static_cast<int>(min(static_cast<long long>(each), begin + (u_end - u)));
    p.first = max(begin - kAttendPiece, 0);
    p.count = max(until - kAttendPiece, 0) - p.first;
    p.unit = u - begin + kAttendPiece;
    p.tiles = max(min(p.count, (p.s.kv + kAttendTile - 1) / kAttendTile - p.lo - p.first), 0);
    u += until - begin;
  }
  if (p.count < 0) p.count = 0;
  if (p.count == 0) p.tiles = 0;
  __syncwarp();
  if (lane == 0) {
    *out = p;
    run->u = u;
    run->at = at;
    run->cost = cost;
  }
  __syncwarp();
}

// Place in the cache (-1: a bad page) of this warp's tile base + lane of a piece.
__device__ __noinline__ int kv_places(const KvAttendArgs& a, const KvPiece* piece, int base, int warp, int lane) {
  const int tile = warp + (base + lane) * kAttendWarps;
  if (tile >= piece->tiles) return -1;
  const int key = (piece->lo + piece->first + tile) * kAttendTile, head = piece->idx % a.c.hkv;
  const int64_t p = kv_page(a.c, a.b, piece->seq, key);
  if (p < 0) {
    set_status(a.b.status, SLORA_STATUS_BAD_TABLE);
    return -1;
  }
  return static_cast<int>(((p * a.c.hkv + head) << (a.c.shift - 4)) + ((key & ((1 << a.c.shift) - 1)) >> 4));
}

template <int D, int NT>
struct AttendSmem {
  struct {
    float o[kAttendWarps][NT * D / 4][32];
    float2 ml[kAttendWarps][8 * NT];
    float unit[kAttendWarps][8 * NT];
  } join[2];
  float low[kAttendWarps][8 * NT];  // the smallest w of a row while it saw tiles; infinity: it has seen none
  KvRun run;
  KvFind find;
};

template <int D, int NT, int KIND, typename T>
__global__ void __launch_bounds__(kAttendThreads, attend_ctas(NT, D)) kv_attend_kernel(const __grid_constant__ KvAttendArgs a) {
  using V8 = Kv8<KIND>;
  // f16 outputs show p's rounding to f16 (1.4 to 1.6 times the error of their own): there p goes in as two f16 numbers.
  // bf16 outputs, eight times coarser, do not.
  constexpr bool kTwoParts = std::is_same<T, __half>::value;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  AttendSmem<D, NT>& sm = *reinterpret_cast<AttendSmem<D, NT>*>(smem_raw);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  KvRun* const run_state = &sm.run;
  pdl_launch_dependents();
  pdl_wait();
  const int me = blockIdx.x;
  const long long total = kv_find<kAttendWarps, 1>(
      a.b.n_seq, &sm.find,
      [&](int i) {
        const KvSeq x = kv_seq(a.b, i);
        if (x.bad && me == 0) set_status(a.b.status, SLORA_STATUS_BAD_TABLE);
        return kv_seq_cost(a, x);
      },
      [&](long long n, int) { return static_cast<long long>(me) * kv_run(n, a.runs); });
  const long long run = kv_run(total, a.runs);
  if (tid == 0) *reinterpret_cast<int4*>(a.rec + 4 * static_cast<int64_t>(me)) = make_int4(-1, 0, 0, 0);
  if (me * run >= total) return;
  if (warp == 0) {
    if (lane == 0) {
      run_state->u = me * run;
      run_state->u_end = min(run_state->u + run, total);
      run_state->at = sm.find.at[0];
      KvPiece& p = run_state->piece[3];
      p.seq = sm.find.seq[0];
      p.s = kv_seq(a.b, p.seq);
      run_state->cost = kv_seq_cost(a, p.s);
    }
    __syncwarp();
    kv_next_piece(a, run_state, &run_state->piece[3], &run_state->piece[0], lane);
  }
  __syncthreads();

  KTile<D> k;
  VTile<D> v;
  float ks = 0.f, vs = 0.f;          // scales of the tile in k and v; vs < 0: a bad page, nothing is loaded
  int place = -1;                    // lane l: of this warp's tile base + l of the piece that is loaded from, and its scales
  float ks_l = 0.f, vs_l = -1.f;
  auto scales = [&]() {
    vs_l = -1.f;
    if (place >= 0) {
      ks_l = a.c.ks[place >> (a.c.shift - 4)];
      vs_l = a.c.vs[place >> (a.c.shift - 4)];
    }
  };
  int issued = 0, tiles = 0;         // of that piece, this warp's
  bool there = false;                // the first tile of the present piece is loaded
  for (int number = 0;; ++number) {
    const KvPiece* const cur = &run_state->piece[number & 3];
    const KvPiece* const pro = &run_state->piece[(number + 1) & 3];
    if (cur->count == 0) return;
    if (!there) {
      tiles = max((cur->tiles - warp + kAttendWarps - 1) / kAttendWarps, 0);
      issued = 0;
      if (tiles > 0) {
        place = kv_places(a, cur, 0, warp, lane);
        const int tile = __shfl_sync(0xffffffffu, place, 0);
        issued = 1;
        if (tile >= 0) {
          k.load(a.c.k + static_cast<int64_t>(tile) * (kAttendTile * D), g, t);
          v.load(a.c.v + static_cast<int64_t>(tile) * (kAttendTile * D), g, t);
        }
        scales();
      }
    }
    bool ahead = false;  // loads have gone over to `pro`
    QTile<D, NT, T> q;
    int2* const see = run_state->see[number & 1];
    int inside_lo, inside_hi, key, left;  // keys that every row sees; the tile's first key; this warp's tiles left
    float* scores = nullptr;
    {
      const KvSeq s = cur->s;
      const int rb = cur->idx / a.c.hkv, head = cur->idx - rb * a.c.hkv;
      q.load(a, s, rb, head, g, t, a.scale2 * V8::kScale);
      const int j = min((rb * a.rows_per_block + min(lane, 8 * NT - 1)) / a.group, s.q - 1);
      const int to = max(s.kv - s.q + j + 1, 0), from = a.window > 0 ? max(to - a.window, 0) : 0;
      see[lane] = make_int2(from, to);  // every warp writes the same
      inside_hi = to, inside_lo = from;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        inside_hi = min(inside_hi, __shfl_xor_sync(0xffffffffu, inside_hi, d));
        inside_lo = max(inside_lo, __shfl_xor_sync(0xffffffffu, inside_lo, d));
      }
      key = (cur->lo + cur->first + warp) * kAttendTile;
      left = tiles;
      if (a.scores != nullptr) scores = a.scores + (cur->unit + cur->first + warp) * (a.part_rows * kAttendTile);
      if (!there) {
        ks = __shfl_sync(0xffffffffu, ks_l, 0);
        vs = __shfl_sync(0xffffffffu, vs_l, 0);
      }
    }
    // the pieces to come, while the loads are on their way: number + 2 goes where number - 2 was, which nobody reads any more
    if (number == 0) {
      if (warp == 0) {
        kv_next_piece(a, run_state, &run_state->piece[0], &run_state->piece[1], lane);
        kv_next_piece(a, run_state, &run_state->piece[1], &run_state->piece[2], lane);
      }
      __syncthreads();
    } else if (warp == (number & 3)) {
      kv_next_piece(a, run_state, pro, &run_state->piece[(number + 2) & 3], lane);
    }
    __syncwarp();

    AttendState<D, NT> st;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < D / 16; ++i) st.o[nt][i][0] = st.o[nt][i][1] = st.o[nt][i][2] = st.o[nt][i][3] = 0.f;
      st.m[nt][0] = st.m[nt][1] = kNoMax;
      st.l[nt][0] = st.l[nt][1] = 0.f;
      st.w[nt][0] = st.w[nt][1] = 0.f;
    }
    bool mixed = false;  // the thread's rows have different w
    if (lane < 8 * NT) sm.low[warp][lane] = INFINITY;
    __syncwarp();

    for (; left > 0; --left, key += kAttendTile * kAttendWarps) {
      if (issued == tiles && !ahead) {
        ahead = true;
        tiles = max((pro->tiles - warp + kAttendWarps - 1) / kAttendWarps, 0);
        issued = 0;
        if (tiles > 0) {
          place = kv_places(a, pro, 0, warp, lane);
          scales();
        }
      }
      int next = -1;
      float ks_n = 0.f, vs_n = -1.f;
      if (issued < tiles) {
        if (issued > 0 && (issued & 31) == 0) {
          place = kv_places(a, ahead ? pro : cur, issued, warp, lane);
          scales();
        }
        next = __shfl_sync(0xffffffffu, place, issued & 31);
        ks_n = __shfl_sync(0xffffffffu, ks_l, issued & 31);
        vs_n = __shfl_sync(0xffffffffu, vs_l, issued & 31);
        ++issued;
      }
      const int64_t off = static_cast<int64_t>(next) * (kAttendTile * D);
      if (vs < 0.f) {  // a bad page: no key of it counts
        if (next >= 0) {
          k.load(a.c.k + off, g, t);
          v.load(a.c.v + off, g, t);
        }
        ks = ks_n;
        vs = vs_n;
        if (scores != nullptr) {
          for (int x = lane; x < a.part_rows * kAttendTile; x += 32) scores[x] = kNegInf;
          scores += kAttendWarps * a.part_rows * kAttendTile;
        }
        continue;
      }
      float c[NT][4];
      kv_scores<D, NT, KIND>(c, k, q.w);
      if (next >= 0) k.load(a.c.k + off, g, t);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float f0 = q.mul[nt][0] * ks, f1 = q.mul[nt][1] * ks;
        c[nt][0] *= f0;
        c[nt][1] *= f1;
        c[nt][2] *= f0;
        c[nt][3] *= f1;
      }
      if (key < inside_lo || key + kAttendTile > inside_hi) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int pos = key + g + 8 * (e >> 1);
            const int2 sees = see[nt * 8 + 2 * t + (e & 1)];
            if (pos < sees.x || pos >= sees.y) c[nt][e] = kNegInf;
          }
        // what lies behind the sequence's end may be anything, NaN bytes among it: no p of 0 makes that 0
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (key + 2 * t + (j & 1) + 8 * (j >> 1) < cur->s.kv) continue;
#pragma unroll
          for (int x = 0; x < VTile<D>::N; ++x) v.w[j][x] = 0;
        }
      }
      if (scores != nullptr) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int r = nt * 8 + 2 * t + (e & 1);
            if (r < a.part_rows) scores[r * kAttendTile + g + 8 * (e >> 1)] = c[nt][e];
          }
        scores += kAttendWarps * a.part_rows * kAttendTile;
      }
      // a scale that counts as 0 fits any w
      auto outside = [&](float w) {
        return __float_as_uint(vs * w) - ((127u - kWLow) << 23) >= (kWLow + kWHigh) << 23 && vs >= kLeastScale;
      };
      bool raise = outside(st.w[0][0]);
      if (mixed) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) raise = raise || outside(st.w[nt][0]) || outside(st.w[nt][1]);
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        raise = raise || fmaxf(c[nt][0], c[nt][2]) > st.m[nt][0] + kLazyMax || fmaxf(c[nt][1], c[nt][3]) > st.m[nt][1] + kLazyMax;
      }
      if (__any_sync(0xffffffffu, raise)) {
        float lowest[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float2 low = *reinterpret_cast<const float2*>(&sm.low[warp][8 * nt + 2 * t]);
          lowest[nt][0] = low.x;
          lowest[nt][1] = low.y;
        }
        __syncwarp();
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            float top = fmaxf(c[nt][x], c[nt][x + 2]);
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
            // only rows that need it: what a row computes does not depend on the others
            const float m = top > st.m[nt][x] + kLazyMax ? top : st.m[nt][x];
            float f = ex2(st.m[nt][x] - m);
            st.l[nt][x] *= f;
            // w: of rows that see the tile, or have seen none (their sums are 0)
            if (outside(st.w[nt][x]) && (top > kNegInf || st.m[nt][x] == kNoMax)) {
              const uint32_t e = 254u + kWTaken - max(__float_as_uint(vs) >> 23, kWTaken);
              const float w = fminf(__uint_as_float(e << 23), lowest[nt][x] * kWRise);
              if (lowest[nt][x] < INFINITY) f *= w * __uint_as_float((254u << 23) - __float_as_uint(st.w[nt][x]));  // both powers of two
              st.w[nt][x] = w;
            }
            if (top > kNegInf && st.w[nt][x] > 0.f && g == 0) sm.low[warp][8 * nt + 2 * t + x] = fminf(lowest[nt][x], st.w[nt][x]);
            st.m[nt][x] = m;
#pragma unroll
            for (int mt = 0; mt < D / 16; ++mt) {
              st.o[nt][mt][x] *= f;
              st.o[nt][mt][x + 2] *= f;
            }
          }
        mixed = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mixed = mixed || st.w[nt][0] != st.w[0][0] || st.w[nt][1] != st.w[0][0];
        __syncwarp();
      }
      uint32_t p[NT][2], p_lo[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float e0 = ex2(c[nt][0] - st.m[nt][0]), e1 = ex2(c[nt][1] - st.m[nt][1]);
        const float e2 = ex2(c[nt][2] - st.m[nt][0]), e3 = ex2(c[nt][3] - st.m[nt][1]);
        st.l[nt][0] += e0 + e2;
        st.l[nt][1] += e1 + e3;
        const float pv0 = vs * st.w[nt][0], pv1 = vs * st.w[nt][1];
        const uint32_t h0 = pack_f16(e0 * pv0, e1 * pv1), h1 = pack_f16(e2 * pv0, e3 * pv1);
        p[nt][0] = transpose8x8(h0);
        p[nt][1] = transpose8x8(h1);
        if (kTwoParts) {
          const float2 f0 = __half22float2(reinterpret_cast<const __half2&>(h0)), f1 = __half22float2(reinterpret_cast<const __half2&>(h1));
          p_lo[nt][0] = transpose8x8(pack_f16(__fmaf_rn(e0, pv0, -f0.x), __fmaf_rn(e1, pv1, -f0.y)));
          p_lo[nt][1] = transpose8x8(pack_f16(__fmaf_rn(e2, pv0, -f1.x), __fmaf_rn(e3, pv1, -f1.y)));
        }
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
          if (kTwoParts) {
            mma_f16(st.o[nt][2 * x], a0, a1, a2, a3, p_lo[nt][0], p_lo[nt][1]);
            mma_f16(st.o[nt][2 * x + 1], b0, b1, b2, b3, p_lo[nt][0], p_lo[nt][1]);
          }
        }
      }
      if (next >= 0) v.load(a.c.v + off, g, t);
      ks = ks_n;
      vs = vs_n;
    }

    // The piece's sums: every warp leaves its own, then each thread adds eight words (four elements of two rows) at a time
    // over the warps; to the output when the piece is whole, else to the workspace.  Two buffers take turns: one barrier.
    auto& home = sm.join[number & 1];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        float l = st.l[nt][x];
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
        if (g == 0) {
          home.ml[warp][8 * nt + 2 * t + x] = make_float2(st.m[nt][x], l);
          home.unit[warp][8 * nt + 2 * t + x] = st.w[nt][x] > 0.f ? V8::kScale / st.w[nt][x] : 0.f;
        }
      }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int mt = 0; mt < D / 16; ++mt)
#pragma unroll
        for (int e = 0; e < 4; ++e) home.o[warp][(nt * (D / 16) + mt) * 4 + e][lane] = st.o[nt][mt][e];
    __syncthreads();
    {
      const KvSeq s = cur->s;
      const int rb = cur->idx / a.c.hkv, head = cur->idx - rb * a.c.hkv;
      const bool whole = cur->count == cur->per;
      const int slot = 2 * me + (cur->first > 0 ? 0 : 1);
      float* part = a.part + static_cast<int64_t>(slot) * a.part_rows * (D + 4);
      for (int x = warp; x < NT * D / 32; x += kAttendWarps) {
        // words [8 x, 8 x + 8) are m-tiles 2i, 2i + 1 of n-tile nt: elements elem(g, i) + 0 .. 3 of rows 2t, 2t + 1
        const int nt = x / (D / 32), i = x - nt * (D / 32);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int r = 8 * nt + 2 * t + c, row = rb * a.rows_per_block + r;
          if (row >= s.q * a.group) continue;
          float m = kNoMax;
#pragma unroll
          for (int w = 0; w < kAttendWarps; ++w) m = fmaxf(m, home.ml[w][r].x);
          float l = 0.f, v4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int w = 0; w < kAttendWarps; ++w) {
            const float2 ml = home.ml[w][r];
            const float f = ex2(ml.x - m);
            l += f * ml.y;
            const float fo = f * home.unit[w][r];
            v4[0] += fo * home.o[w][8 * x + c][lane];
            v4[1] += fo * home.o[w][8 * x + 2 + c][lane];
            v4[2] += fo * home.o[w][8 * x + 4 + c][lane];
            v4[3] += fo * home.o[w][8 * x + 6 + c][lane];
          }
          const int elem = VTile<D>::elem(g, i);
          if (whole) {
            const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
            const int j = row / a.group, h = head * a.group + row - j * a.group;
            const int64_t token = static_cast<int64_t>(s.row) + j;
            union {
              uint2 u;
              T e[4];
            } y;
#pragma unroll
            for (int e = 0; e < 4; ++e) y.e[e] = from_f32<T>(v4[e] * inv);
            *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + token * a.out_stride + h * D + elem) = y.u;
            if (a.lse && i == 0 && g == 0) a.lse[token * a.hq + h] = l == 0.f ? kNegInf : (m + log2f(l)) * 0.69314718055994531f;
          } else {
            *reinterpret_cast<float4*>(part + r * D + elem) = make_float4(v4[0], v4[1], v4[2], v4[3]);
            if (i == 0 && g == 0) *reinterpret_cast<float2*>(part + a.part_rows * D + 2 * r) = make_float2(m, l);
          }
        }
      }
      if (!whole && cur->first == 0 && tid == 0) {
        // the first run of a cut piece names it for the join: the runs after it hold their parts in slot 0
        const long long end = cur->unit + cur->per;
        const long long behind = end - 1 - static_cast<long long>(me) * run;
        const int parts = (behind <= 0xffffffffll ? static_cast<int>(static_cast<uint32_t>(behind) / static_cast<uint32_t>(run)) : static_cast<int>(behind / run)) + 1;
        *reinterpret_cast<int4*>(a.rec + 4 * static_cast<int64_t>(me)) = make_int4(cur->seq, cur->idx, slot, parts);
      }
    }
    there = ahead && tiles > 0;
  }
}

// Adds the parts of the (sequence, row block, head) that a run of the attention left unfinished, in the order of its
// keys: what each part weighs first (all of them at once), then the sums, whose loads do not wait for one another.
// 32 lanes share a row, the warps rows and parts.
constexpr int kJoinThreads = 512;
constexpr int kJoinParts = 128;  // parts whose weights are held at a time
template <int D, typename T>
__global__ void __launch_bounds__(kJoinThreads) kv_join_kernel(const KvAttendArgs a) {
  constexpr int kLanes = D / 4 > 32 ? 32 : D / 4, kVec = D / 4 / kLanes;  // float4 of a lane
  constexpr int kTeams = kJoinThreads / kLanes;
  __shared__ float4 sh_o[kJoinThreads * kVec];
  __shared__ float sh_f[32][kJoinParts];
  __shared__ float sh_m[32], sh_l[32], sh_keep[32];
  const int tid = threadIdx.x;
  pdl_launch_dependents();
  pdl_wait();
  const int me = blockIdx.x;
  const int4 rec = *reinterpret_cast<const int4*>(a.rec + 4 * static_cast<int64_t>(me));
  if (rec.x < 0) return;
  const KvSeq s = kv_seq(a.b, rec.x);
  const int rb = rec.y / a.c.hkv, head = rec.y - rb * a.c.hkv;
  const int rows = min(a.rows_per_block, s.q * a.group - rb * a.rows_per_block);
  const int64_t words = static_cast<int64_t>(a.part_rows) * (D + 4);
  auto part_of = [&](int p) { return a.part + (p == 0 ? rec.z : 2 * (me + p)) * words; };
  const int e = tid % kLanes, team = tid / kLanes;
  static_assert(8 * (256 / D) <= kTeams, "a team has one row of the block at most (attend_tiles)");
  const int groups = kTeams / rows;  // teams that share a row's parts
  const int r = team % rows, grp = team / rows;
  const bool on = grp < groups;
  float4 o[kVec];
#pragma unroll
  for (int v = 0; v < kVec; ++v) o[v] = make_float4(0.f, 0.f, 0.f, 0.f);
  if (tid < 32) {
    sh_m[tid] = kNoMax;
    sh_l[tid] = 0.f;
  }
  for (int p0 = 0; p0 < rec.w; p0 += kJoinParts) {
    const int np = min(kJoinParts, rec.w - p0);
    __syncthreads();
    // one warp per row: the weights of this stretch of parts relative to the maximum so far
    for (int rr = tid >> 5; rr < rows; rr += kJoinThreads / 32) {
      float m = kNoMax;
      float2 ml[kJoinParts / 32];
#pragma unroll
      for (int k = 0; k < kJoinParts / 32; ++k) {
        const int p = k * 32 + (tid & 31);
        ml[k] = make_float2(kNoMax, 0.f);
        if (p < np) ml[k] = *reinterpret_cast<const float2*>(part_of(p0 + p) + static_cast<int64_t>(a.part_rows) * D + 2 * rr);
        m = fmaxf(m, ml[k].x);
      }
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
      const float was = sh_m[rr], now = fmaxf(was, m);
      float l = 0.f;
#pragma unroll
      for (int k = 0; k < kJoinParts / 32; ++k) {
        const float f = ex2(ml[k].x - now);
        sh_f[rr][k * 32 + (tid & 31)] = f;
        l += f * ml[k].y;
      }
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
      if ((tid & 31) == 0) {
        const float keep = ex2(was - now);
        sh_keep[rr] = keep;
        sh_l[rr] = sh_l[rr] * keep + l;
        sh_m[rr] = now;
      }
      __syncwarp();
    }
    __syncthreads();
    if (on) {
      const float keep = sh_keep[r];
#pragma unroll
      for (int v = 0; v < kVec; ++v) o[v].x *= keep, o[v].y *= keep, o[v].z *= keep, o[v].w *= keep;
#pragma unroll 8
      for (int p = grp; p < np; p += groups) {
        const float f = sh_f[r][p];
        const float* part = part_of(p0 + p) + r * D;
#pragma unroll
        for (int v = 0; v < kVec; ++v) {
          const float4 y = *reinterpret_cast<const float4*>(part + 4 * (v * kLanes + e));
          if (f != 0.f) {
            o[v].x += y.x * f;
            o[v].y += y.y * f;
            o[v].z += y.z * f;
            o[v].w += y.w * f;
          }
        }
      }
    }
  }
#pragma unroll
  for (int v = 0; v < kVec; ++v) sh_o[v * kJoinThreads + tid] = o[v];
  __syncthreads();
  if (on && grp == 0) {
    const float l = sh_l[r];
    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
    const int row = rb * a.rows_per_block + r, j = row / a.group, h = head * a.group + row - j * a.group;
    const int64_t token = static_cast<int64_t>(s.row) + j;
#pragma unroll
    for (int v = 0; v < kVec; ++v) {
      for (int k = 1; k < groups; ++k) {
        const float4 y = sh_o[v * kJoinThreads + tid + k * rows * kLanes];
        o[v].x += y.x, o[v].y += y.y, o[v].z += y.z, o[v].w += y.w;
      }
      union {
        uint2 u;
        T e[4];
      } p;
      p.e[0] = from_f32<T>(o[v].x * inv);
      p.e[1] = from_f32<T>(o[v].y * inv);
      p.e[2] = from_f32<T>(o[v].z * inv);
      p.e[3] = from_f32<T>(o[v].w * inv);
      *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + token * a.out_stride + h * D + 4 * (v * kLanes + e)) = p.u;
    }
    if (a.lse && e == 0) a.lse[token * a.hq + h] = l == 0.f ? kNegInf : (sh_m[r] + log2f(l)) * 0.69314718055994531f;
  }
}

// Accumulated attention weights from the stored scores: w[key] += sum over the rows of 2^(score - lse).  Runs of tiles, as in
// the attention but over (sequence, KV head) only.  A lane takes a key of a tile and half of a block's rows.  A warp has a run
// of its own and goes through a tile's row blocks in their order; with many of them (SPLIT) a CTA has the run, and teams of 2
// to 16 warps share a tile's row blocks and add up their sums in a fixed order.  Either way one addition per token to the
// cache, so that weights do not depend on timing.
template <int D, bool SPLIT>
__global__ void __launch_bounds__(SPLIT ? 512 : kAttendThreads) kv_weights_kernel(const KvAttendArgs a) {
  constexpr int kWarps = SPLIT ? 16 : kAttendWarps, kRuns = SPLIT ? 1 : kWarps;  // runs of a CTA
  __shared__ KvFind find;
  __shared__ float part[SPLIT ? 2 : 1][SPLIT ? kWarps : 1][4 * kAttendTile];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_launch_dependents();
  pdl_wait();
  const int me = blockIdx.x * kRuns + (SPLIT ? 0 : warp);
  const int runs = gridDim.x * kRuns;
  // units: what a sequence costs in the attention, a row block's worth of it
  auto units = [&](const KvSeq& s) {
    if (s.q < a.min_q || s.q > a.lim_q || s.q == 0) return 0ll;
    const KvRange r = kv_tiles(s, a.window);
    return static_cast<long long>(r.hi - r.lo + kAttendPiece) * a.c.hkv;
  };
  auto run_of = [&](long long n) { return SPLIT ? (n + runs - 1) / runs : kv_run(n, runs); };
  const long long total = kv_find<kWarps, kRuns>(
      a.b.n_seq, &find, [&](int i) { return units(kv_seq(a.b, i)); },
      [&](long long n, int k) { return static_cast<long long>(blockIdx.x * kRuns + k) * run_of(n); });
  const long long run = run_of(total);
  long long u = me * run;
  const long long u_end = min(u + run, total);
  if (u >= u_end) return;
  int seq = find.seq[SPLIT ? 0 : warp];
  long long seq_at = find.at[SPLIT ? 0 : warp];
  long long scores_at = seq_at;  // cost units of the attention before the sequence: where its scores start
  if (a.blocks > 1) {
    scores_at = 0;
    for (int i = lane; i < seq; i += 32) scores_at += kv_seq_cost(a, kv_seq(a.b, i));
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) scores_at += __shfl_xor_sync(0xffffffffu, scores_at, d);
  }
  KvSeq s = kv_seq(a.b, seq);
  long long n_units = units(s);
  const int key_in = lane & 15, half = lane >> 4;
  int buf = 0;
  while (u < u_end) {
    while (u >= seq_at + n_units) {
      seq_at += n_units;
      scores_at += kv_seq_cost(a, s);
      s = kv_seq(a.b, ++seq);
      n_units = units(s);
    }
    const KvRange range = kv_tiles(s, a.window);
    const int per = range.hi - range.lo, piece = per + kAttendPiece;
    const long long in = u - seq_at;
    const int head = in <= 0xffffffffll ? static_cast<int>(static_cast<uint32_t>(in) / static_cast<uint32_t>(piece)) : static_cast<int>(in / piece);
    const int at = static_cast<int>(in - static_cast<long long>(head) * piece);
    const int until = static_cast<int>(min(static_cast<long long>(piece), at + (u_end - u)));
    u += until - at;
    const int all_rows = s.q * a.group, blocks = (all_rows + a.rows_per_block - 1) / a.rows_per_block;
    const int team = SPLIT ? (blocks > 8 ? 16 : blocks > 4 ? 8 : blocks > 2 ? 4 : 2) : 1;  // warps that share a tile's blocks
    const int mate = SPLIT ? warp % team : 0, first = SPLIT ? 4 * (warp / team) : 0, step = SPLIT ? 4 * (kWarps / team) : 4;
    const float* const scores = a.scores + (scores_at + static_cast<long long>(head) * piece + kAttendPiece) * (a.part_rows * kAttendTile) + lane;
    const long long block_step = static_cast<long long>(a.c.hkv) * piece * (a.part_rows * kAttendTile);
    // lane r holds lse of row r of a block (32 rows at most)
    auto lse_of = [&](int rb) {
      const int row = rb * a.rows_per_block + lane, j = row / a.group;
      if (lane >= a.rows_per_block || row >= all_rows) return kNegInf;
      return a.lse[(static_cast<int64_t>(s.row) + j) * a.hq + head * a.group + row - j * a.group] * 1.4426950408889634f;
    };
    float lse_l = lse_of(0);
    // 32 tiles at a time: lane l looks up where tile l's weights are
    const int end = min(until - kAttendPiece, (s.kv + kAttendTile - 1) / kAttendTile - range.lo);
    for (int i0 = max(at - kAttendPiece, 0); i0 < end; i0 += 32) {
      int place = -1;  // token row of the cache
      const int key_l = (range.lo + i0 + lane) * kAttendTile;
      if (i0 + lane < end) {
        const int64_t p = kv_page(a.c, a.b, seq, key_l);
        if (p >= 0) place = static_cast<int>(((p * a.c.hkv + head) << a.c.shift) + (key_l & ((1 << a.c.shift) - 1)));
      }
      const int n = min(32, end - i0);
      // an atomic add only because sequences may share a page (then in no fixed order); else one add per token
      auto add = [&](int tile, int key, int to, float sum) {
        if (to >= 0 && (range.lo + i0 + tile) * kAttendTile + key < s.kv && sum != 0.f) atomicAdd(a.c.w + to + key, sum);
      };
      for (int i = 0; i < n; i += step) {  // four tiles a warp: their loads overlap
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
        for (int rb = mate; rb < blocks; rb += team) {
          if (blocks > 1) lse_l = lse_of(rb);
          const int rows = min(a.rows_per_block, all_rows - rb * a.rows_per_block);
          const float* const src = scores + rb * block_step + static_cast<int64_t>(i0 + i + first) * (a.part_rows * kAttendTile);
#pragma unroll 4
          for (int r0 = 0; r0 < rows; r0 += 2) {
            const float lse = __shfl_sync(0xffffffffu, lse_l, r0 + half);
#pragma unroll
            for (int t = 0; t < 4; ++t) {
              const float x = r0 + half < rows && i + first + t < n ? src[(t * a.part_rows + r0) * kAttendTile] : kNegInf;
              sum[t] += lse > kNegInf ? ex2(x - lse) : 0.f;
            }
          }
        }
#pragma unroll
        for (int t = 0; t < 4; ++t) sum[t] += __shfl_down_sync(0xffffffffu, sum[t], 16);
        if (!SPLIT) {
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            if (i + t >= n) break;
            const int to = __shfl_sync(0xffffffffu, place, i + t);
            if (half == 0) add(i + t, key_in, to, sum[t]);
          }
        } else {
          if (half == 0) {
#pragma unroll
            for (int t = 0; t < 4; ++t) part[buf][warp][t * kAttendTile + key_in] = sum[t];
          }
          __syncthreads();
          // two warps per team: a thread adds up its team's sums of one key
          if (tid < 64 * (kWarps / team)) {
            const int of = tid >> 6, tile = i + 4 * of + (tid >> 4 & 3);
            const int to = __shfl_sync(0xffffffffu, place, tile & 31);
            float all = 0.f;
            for (int x = 0; x < team; ++x) all += part[buf][of * team + x][tid & 63];
            if (tile < n) add(tile, key_in, to, all);
          }
          buf ^= 1;
        }
      }
    }
  }
}

// The same with the scores computed again: where they would take too much memory, or for many rows.
// Tiles are independent; a warp keeps the keys of a tile in registers and walks through the sequence's rows.
template <int D, int KIND, typename T>
__global__ void __launch_bounds__(kAttendThreads, D <= 128 ? 4 : 2) kv_reweigh_kernel(const KvAttendArgs a) {
  using V8 = Kv8<KIND>;
  __shared__ KvFind find;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  pdl_launch_dependents();
  pdl_wait();
  const long long me = blockIdx.x, grid = gridDim.x;
  auto units = [&](int i) {
    const KvSeq s = kv_seq(a.b, i);
    if (s.q == 0) return 0ll;
    const KvRange r = kv_tiles(s, a.window);
    return static_cast<long long>((r.hi - r.lo + kAttendWarps - 1) / kAttendWarps) * a.c.hkv;
  };
  const long long total = kv_find<kAttendWarps, 1>(a.b.n_seq, &find, units, [&](long long n, int) { return me * ((n + grid - 1) / grid); });
  const long long run = (total + grid - 1) / grid;
  long long u = me * run;
  const long long u_end = min(u + run, total);
  if (u >= u_end) return;
  int seq = find.seq[0];
  long long seq_at = find.at[0];
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
    const KvRange range = kv_tiles(s, a.window);
    const int per = (range.hi - range.lo + kAttendWarps - 1) / kAttendWarps;
    const int head = static_cast<int>((u - seq_at) / per);
    const int key = (range.lo + static_cast<int>((u - seq_at) - static_cast<long long>(head) * per) * kAttendWarps + warp) * kAttendTile;
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
        const int to = max(s.kv - s.q + j + 1, 0), from = a.window > 0 ? to - a.window : 0;
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
      // an atomic add only because sequences may share a page (then in no fixed order); else one add per token
      const int pos = in_page + g + 8 * t;
      const float add = t == 0 ? sum0 : sum1;
      if (key + g + 8 * t < s.kv && add != 0.f) atomicAdd(a.c.w + (ph << a.c.shift) + pos, add);
    }
  }
}

}  // namespace slora
