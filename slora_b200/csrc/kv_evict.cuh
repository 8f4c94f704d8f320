// Eviction from the 8-bit cache by accumulated attention weight: which tokens a (sequence, KV head) keeps, and their move
// to the front pages.
//
// Select: the budget-th largest weight by radix selection, 8 bits at a time, on the weights mapped to ordered integers
// (in shared memory when they fit); then one sweep in position order that places every kept position.  Ties go to the
// lowest position because the sweep counts them in order.  What bounds it: reading the weights once, and a chain of four
// histogram passes per (sequence, head).
//
// Move: the scale of a page belongs to its tokens, so a page with new neighbours gets a new scale and its values new
// roundings: max over tokens of |q| * s in 64 bits (exact), then the exact rounding of q * s / s_new.  Kept positions
// never move up, so in place a CTA can work through a head's pages in order, reading a round of pages before it writes
// them; with other destination pages all rounds run at once.  Bound by bytes: kept tokens read and written once.
#pragma once

#include "kv_common.cuh"

namespace slora {

constexpr int kSelectThreads = 1024;
constexpr int kSelectCopies = 8;             // histogram copies: weights share few exponents, so bins are contended
constexpr int kMoveThreads = 256;
constexpr int kMoveWarps = kMoveThreads / 32;

struct EvictArgs {
  KvCache c;
  KvBatch b;
  int budget, recent, sink;
  int32_t* kept;  // [n_seq][hkv][budget]
  const int64_t* dest;
  int64_t dest_stride;
  int in_place;
  int cached;     // weights that fit the select kernel's shared memory
  int chunks;     // CTAs per (sequence, head) of the move
};

__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t b = __float_as_uint(w == 0.f ? 0.f : w);
  return b >> 31 ? ~b : b | 0x80000000u;
}

// 256 (sequence, head) pairs of 3030 to 15912 weights, 2048 of them kept: 36 us; 32 pairs of 1225 to 1681: 10 us.  One CTA of
// 1024 threads per SM; two of 512 took 42 us.
__global__ void __launch_bounds__(kSelectThreads) kv_select_kernel(const EvictArgs a) {
  extern __shared__ uint32_t keys[];
  __shared__ int hist[kSelectCopies][256];
  __shared__ uint32_t s_prefix;
  __shared__ int s_left;
  __shared__ int s_count[2][32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_launch_dependents();
  pdl_wait();
  const int seq = blockIdx.x / a.c.hkv, head = blockIdx.x - seq * a.c.hkv;
  int n = a.b.kv_len[seq];
  if (n < 0 || n > a.b.max_tokens) {
    if (tid == 0) set_status(a.b.status, SLORA_STATUS_BAD_TABLE);
    n = 0;
  }
  int32_t* kept = a.kept + static_cast<int64_t>(blockIdx.x) * a.budget;
  if (n <= a.budget) {
    for (int j = tid; j < a.budget; j += kSelectThreads) kept[j] = j < n ? j : -1;
    return;
  }
  const int c0 = a.sink, c1 = n - a.recent;  // candidates
  const int want = a.budget - a.sink - a.recent;
  auto weight_at = [&](int i) {
    const int64_t p = kv_page(a.c, a.b, seq, i);
    if (p < 0) {
      set_status(a.b.status, SLORA_STATUS_BAD_TABLE);
      return 0u;
    }
    return weight_key(a.c.w[((p * a.c.hkv + head) << a.c.shift) + (i & ((1 << a.c.shift) - 1))]);
  };
  // four positions a thread and turn: their pages first, then their weights, so that the loads overlap
  for (int i0 = c0 + tid; i0 < c1 && i0 - c0 < a.cached; i0 += 4 * kSelectThreads) {
    int place[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = i0 + e * kSelectThreads;
      place[e] = -1;
      if (i < c1) {
        const int64_t p = kv_page(a.c, a.b, seq, i);
        place[e] = p < 0 ? -2 : static_cast<int>(((p * a.c.hkv + head) << a.c.shift) + (i & ((1 << a.c.shift) - 1)));
      }
    }
    float w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = place[e] >= 0 ? a.c.w[place[e]] : 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = i0 + e * kSelectThreads;
      if (place[e] == -2) set_status(a.b.status, SLORA_STATUS_BAD_TABLE);
      if (place[e] != -1 && i - c0 < a.cached) keys[i - c0] = place[e] == -2 ? 0u : weight_key(w[e]);
    }
  }
  auto key_at = [&](int i) { return i - c0 < a.cached ? keys[i - c0] : weight_at(i); };
  if (tid == 0) {
    s_prefix = 0;
    s_left = want;
  }
  // the want-th largest key: after the pass at `shift` the top bits of the threshold are known and s_left of the keys
  // that share them still have to be taken
  for (int shift = 24; shift >= 0 && want > 0; shift -= 8) {
    for (int i = tid; i < kSelectCopies * 256; i += kSelectThreads) hist[0][i] = 0;
    __syncthreads();
    const uint32_t prefix = s_prefix, mask = shift == 24 ? 0u : ~0u << (shift + 8);
    for (int i = c0 + tid; i < c1; i += kSelectThreads) {
      const uint32_t k = key_at(i);
      if ((k & mask) == prefix) atomicAdd(&hist[warp % kSelectCopies][(k >> shift) & 255u], 1);
    }
    __syncthreads();
    if (warp == 0) {
      // lane l holds bins 255 - 8 l .. 248 - 8 l; counts from the top
      int v[8], sum = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[e] = 0;
#pragma unroll
        for (int x = 0; x < kSelectCopies; ++x) v[e] += hist[x][255 - 8 * lane - e];
        sum += v[e];
      }
      int incl = sum;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += y;
      }
      int before = incl - sum;
      const int left = s_left;
      __syncwarp();
      if (before < left && left <= incl) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (before < left && left <= before + v[e]) {
            s_prefix = prefix | static_cast<uint32_t>(255 - 8 * lane - e) << shift;
            s_left = left - before;
          }
          before += v[e];
        }
      }
    }
    __syncthreads();
  }
  __syncthreads();
  const uint32_t limit = want > 0 ? s_prefix : 0xffffffffu;
  const int equal = want > 0 ? s_left : 0;  // keys equal to the limit that are kept, the first ones
  int above = 0, ties = 0;                  // kept above the limit / equal to it, before this sweep's positions
  int buf = 0;
  for (int base = 0; base < n; base += 4 * kSelectThreads, buf ^= 1) {
    const int i = base + 4 * tid;  // four positions a thread
    unsigned gt = 0, eq = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (i + e < c0 || (i + e >= c1 && i + e < n)) {
        gt |= 1u << e;
      } else if (i + e < c1 && want > 0) {
        const uint32_t k = key_at(i + e);
        gt |= (k > limit ? 1u : 0u) << e;
        eq |= (k == limit ? 1u : 0u) << e;
      }
    }
    const int own = __popc(gt) | __popc(eq) << 16;  // at most 4096 of each in a sweep
    int incl = own;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, incl, d);
      if (lane >= d) incl += y;
    }
    if (lane == 31) s_count[buf][warp] = incl;
    __syncthreads();
    int v = s_count[buf][lane];
    const int mine = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, v, d);
      if (lane >= d) v += y;
    }
    const int total = __shfl_sync(0xffffffffu, v, 31);
    const int before = __shfl_sync(0xffffffffu, v - mine, warp) + incl - own;
    int g = above + (before & 0xffff), q = ties + (before >> 16);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bool is_gt = gt >> e & 1u, is_eq = eq >> e & 1u;
      if (is_gt || (is_eq && q < equal)) kept[g + min(q, equal)] = i + e;
      g += is_gt;
      q += is_eq;
    }
    above += total & 0xffff;
    ties += total >> 16;
  }
}

// One page's part of a warp: 16 tokens of k or of v, 16 bytes a lane.
template <int D>
struct MoveRows {
  static constexpr int kLanes = D / 16, kRows = 32 / kLanes, kSteps = 16 / kRows;
  uint4 w[kSteps];
  float s[kSteps];
};

// Rounds the rows to the page's scale (or leaves them) and stores those that `write` has a bit for.
template <int D, int KIND>
__device__ __forceinline__ void move_store(MoveRows<D>& m, uint8_t* dst, bool same, float now, unsigned write) {
  using V8 = Kv8<KIND>;
  const float inv = now > 0.f ? __fdiv_rn(1.f, now) : 0.f;
#pragma unroll
  for (int i = 0; i < MoveRows<D>::kSteps; ++i) {
    if (!same) {
      const float mul = m.s[i] * inv;
      uint32_t words[4] = {m.w[i].x, m.w[i].y, m.w[i].z, m.w[i].w};
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        float v[4];
        V8::values(words[x], v);
        words[x] = now > 0.f ? kv_round4<KIND>(v, m.s[i], mul, now) : 0u;
      }
      m.w[i] = make_uint4(words[0], words[1], words[2], words[3]);
    }
    if (write >> i & 1u) *reinterpret_cast<uint4*>(dst + i * MoveRows<D>::kRows * D) = m.w[i];
  }
}

// The same 256 heads to other pages: 108 us for 0.27 GB moved.  The exact rounding bounds it (17 instructions a value, issue
// slots 63 % busy), then a round's wait for its loads and for the join of its maxima, which three CTAs per SM cover.
template <int D, int KIND>
__global__ void __launch_bounds__(kMoveThreads, D <= 128 ? 3 : 1) kv_move_kernel(const EvictArgs a) {
  using V8 = Kv8<KIND>;
  constexpr int kLanes = D / 16, kRows = 32 / kLanes, kSteps = 16 / kRows;
  __shared__ double s_top[2][2][kMoveWarps];  // [round's parity][k, v]
  __shared__ int s_same[2][kMoveWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane % kLanes, rr = lane / kLanes;
  pdl_launch_dependents();
  pdl_wait();
  const int sh = static_cast<int>(blockIdx.x);
  const int seq = sh / a.c.hkv, head = sh - seq * a.c.hkv;
  int n = a.b.kv_len[seq];
  if (n < 0 || n > a.b.max_tokens) n = 0;
  const int m = min(n, a.budget);
  if (a.in_place && n <= a.budget) return;
  const int32_t* kept = a.kept + static_cast<int64_t>(sh) * a.budget;
  const int shift = a.c.shift, page = 1 << shift, in_page = page - 1;
  const int team = page / 16;              // warps of a page
  const int at_once = kMoveWarps / team;   // pages of a round
  const int pages = (m + page - 1) >> shift;
  const int rounds = (pages + at_once - 1) / at_once;
  const int mine = warp / team, part = warp - mine * team;
  int turn = 0;
  for (int round = blockIdx.y; round < rounds; round += a.chunks, turn ^= 1) {
    const int block = round * at_once + mine;
    const bool active = block < pages;
    // places (token rows of the cache, -1 none) of this warp's 16 tokens: lane l < 16 looks up token l
    const int j = block * page + part * 16 + (lane & 15);
    int place = -1;
    bool same = true;
    if (active && j < m) {
      const int from = kept[j];
      same = from == j;
      const int64_t p = kv_page(a.c, a.b, seq, from);
      if (p >= 0)
        place = static_cast<int>(((p * a.c.hkv + head) << shift) + (from & in_page));
      else
        set_status(a.b.status, SLORA_STATUS_BAD_TABLE);
    }
    same = __all_sync(0xffffffffu, same);
    MoveRows<D> k, v;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      const int at = __shfl_sync(0xffffffffu, place, i * kRows + rr);
      k.w[i] = v.w[i] = make_uint4(0, 0, 0, 0);
      k.s[i] = v.s[i] = 0.f;
      if (at >= 0) {
        k.w[i] = *reinterpret_cast<const uint4*>(a.c.k + static_cast<int64_t>(at) * D + 16 * sub);
        v.w[i] = *reinterpret_cast<const uint4*>(a.c.v + static_cast<int64_t>(at) * D + 16 * sub);
        k.s[i] = a.c.ks[at >> shift];
        v.s[i] = a.c.vs[at >> shift];
      }
    }
    const float weight = place >= 0 ? a.c.w[place] : 0.f;
    double top_k = 0.0, top_v = 0.0;
    if (!same || team > 1) {
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        top_k = fmax(top_k, static_cast<double>(kv_top<KIND>(k.w[i])) * static_cast<double>(k.s[i]));
        top_v = fmax(top_v, static_cast<double>(kv_top<KIND>(v.w[i])) * static_cast<double>(v.s[i]));
      }
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        top_k = fmax(top_k, __shfl_xor_sync(0xffffffffu, top_k, d));
        top_v = fmax(top_v, __shfl_xor_sync(0xffffffffu, top_v, d));
      }
    }
    if (lane == 0) {
      s_top[turn][0][warp] = top_k;
      s_top[turn][1][warp] = top_v;
      s_same[turn][warp] = same;
    }
    // in place every warp has to have read its pages before any is written; else only the warps of a page exchange
    if (a.in_place)
      __syncthreads();
    else if (team > 1)
      asm volatile("bar.sync %0, %1;" ::"r"(1 + mine), "r"(32 * team) : "memory");
    else
      __syncwarp();
    for (int x = 0; x < team; ++x) {
      top_k = fmax(top_k, s_top[turn][0][mine * team + x]);
      top_v = fmax(top_v, s_top[turn][1][mine * team + x]);
      same = same && s_same[turn][mine * team + x];
    }
    if (active) {
      const int64_t dp = a.dest[seq * a.dest_stride + block];
      if (dp < 0 || dp >= a.c.n_pages) {
        if (lane == 0) set_status(a.b.status, SLORA_STATUS_BAD_TABLE);
      } else if (!(a.in_place && same)) {
        const int64_t ph = dp * a.c.hkv + head;
        unsigned write = 0;
#pragma unroll
        for (int i = 0; i < kSteps; ++i) write |= (block * page + part * 16 + i * kRows + rr < m ? 1u : 0u) << i;
        const int64_t at = ((ph << shift) + part * 16 + rr) * D + 16 * sub;
        const float was_k = __shfl_sync(0xffffffffu, k.s[0], 0), was_v = __shfl_sync(0xffffffffu, v.s[0], 0);
        const float now_k = same ? was_k : kv_scale(static_cast<float>(top_k * (1.0 / V8::kTop)));
        const float now_v = same ? was_v : kv_scale(static_cast<float>(top_v * (1.0 / V8::kTop)));
        move_store<D, KIND>(k, a.c.k + at, same, now_k, write);
        move_store<D, KIND>(v, a.c.v + at, same, now_v, write);
        if (part == 0 && lane == 0) {
          a.c.ks[ph] = now_k;
          a.c.vs[ph] = now_v;
        }
        if (lane < 16 && j < m) a.c.w[(ph << shift) + part * 16 + lane] = weight;
      }
    }
    if (a.in_place) __syncthreads();  // the round's pages are written before the next reads
  }
}

}  // namespace slora
