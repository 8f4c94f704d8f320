// 8-bit KV cache and rotary positions: host-side checks, dispatch and the C ABI of kv_attend.cuh, kv_append.cuh and
// kv_evict.cuh.  Every launch uses programmatic dependent launch: the kernels touch nothing before their grid-dependency
// wait, so only the launch itself overlaps what runs before.
#include <cstring>

#include "host_common.h"
#include "kv_append.cuh"
#include "kv_attend.cuh"
#include "kv_common.cuh"
#include "kv_evict.cuh"
#include "kv_prefill.cuh"
#include "smem_limit.h"

using namespace slora;

namespace {

// `cluster`: CTAs along y that form a cluster (1: none).
template <auto kernel, typename... A>
int launch_cluster(int cluster, dim3 grid, int threads, size_t smem, cudaStream_t stream, const char* what, const A&... args) {
  static SmemLimit limit;
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess) dev = -1;
  cudaError_t refused = cudaSuccess;
  const auto most = [&] {
    int all = 0;
    cudaFuncAttributes f;
    refused = cudaFuncGetAttributes(&f, kernel);
    if (refused == cudaSuccess) refused = cudaDeviceGetAttribute(&all, cudaDevAttrMaxSharedMemoryPerBlockOptin, dev < 0 ? 0 : dev);
    return refused == cudaSuccess ? static_cast<size_t>(all) - f.sharedSizeBytes : smem;
  };
  const auto set = [&](size_t bytes) {
    if (refused == cudaSuccess) refused = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
    return refused == cudaSuccess;
  };
  if (!limit.allow(dev, smem, most, set)) {
    cudaGetLastError();
    return fail(SLORA_ERR_LAUNCH, "%s: %zu bytes of shared memory: %s", what, smem, cudaGetErrorString(refused));
  }
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = grid;
  cfg.blockDim = dim3(static_cast<unsigned>(threads), 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cluster > 1) {
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 1;
    attr[1].val.clusterDim.y = static_cast<unsigned>(cluster);
    attr[1].val.clusterDim.z = 1;
    cfg.numAttrs = 2;
  }
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(SLORA_ERR_LAUNCH, "%s: %s", what, cudaGetErrorString(e));
  }
  g_launches[3].fetch_add(1, std::memory_order_relaxed);
  return SLORA_OK;
}

template <auto kernel, typename... A>
int launch_pdl(dim3 grid, int threads, size_t smem, cudaStream_t stream, const char* what, const A&... args) {
  return launch_cluster<kernel>(1, grid, threads, smem, stream, what, args...);
}

int sm_count() {
  static std::atomic<int> known[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) dev = 0;
  int n = known[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
    known[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

// ---- checks ----------------------------------------------------------------------------------------------------------
int check_dtype(int dtype) {
  return dtype == SLORA_F16 || dtype == SLORA_BF16 ? SLORA_OK : fail(SLORA_ERR_DTYPE, "unsupported dtype %d", dtype);
}

int check_head_dim(int d) {
  return d == 64 || d == 128 || d == 256 ? SLORA_OK
                                         : fail(SLORA_ERR_SHAPE, "No suitable kernel. head_dim=%d (64, 128 or 256)", d);
}

int check_cache(const slora_kv8_cache* c, KvCache* out) {
  if (!c) return fail(SLORA_ERR_NULL, "cache is null");
  if (!c->k || !c->v || !c->k_scale || !c->v_scale) return fail(SLORA_ERR_NULL, "cache: null buffer");
  if (c->kind != SLORA_KV_INT8 && c->kind != SLORA_KV_E4M3) return fail(SLORA_ERR_DTYPE, "cache: unknown kind %d", c->kind);
  int shift = 4;
  while (shift < 7 && (1 << shift) != c->page_tokens) ++shift;
  if ((1 << shift) != c->page_tokens)
    return fail(SLORA_ERR_SHAPE, "cache: page_tokens=%d (16, 32, 64 or 128)", c->page_tokens);
  if (const int rc = check_head_dim(c->head_dim)) return rc;
  if (c->kv_heads < 1 || c->kv_heads > 65535) return fail(SLORA_ERR_SHAPE, "cache: kv_heads=%d", c->kv_heads);
  if (c->n_pages < 1 || c->n_pages > 0x7fffffffLL) return fail(SLORA_ERR_SHAPE, "cache: n_pages=%lld", (long long)c->n_pages);
  if (((c->n_pages * c->kv_heads) << shift) > 0x7fffffffLL)
    return fail(SLORA_ERR_SHAPE, "cache: more than 2^31 rows (tokens x heads) in a layer");
  if (!aligned16(c->k) || !aligned16(c->v) || !aligned16(c->k_scale) || !aligned16(c->v_scale) || !aligned16(c->weights))
    return fail(SLORA_ERR_ALIGN, "cache: a buffer is not 16-byte aligned");
  out->k = static_cast<uint8_t*>(c->k);
  out->v = static_cast<uint8_t*>(c->v);
  out->ks = c->k_scale;
  out->vs = c->v_scale;
  out->w = c->weights;
  out->n_pages = c->n_pages;
  out->shift = shift;
  out->hkv = c->kv_heads;
  out->d = c->head_dim;
  return SLORA_OK;
}

int check_batch(const slora_kv8_batch* b, int shift, int64_t T, KvBatch* out) {
  if (!b) return fail(SLORA_ERR_NULL, "batch is null");
  if (b->n_seq < 0 || b->max_pages < 0 || b->max_q_len < 0 || T < 0 || T > 0x7fffffff)
    return fail(SLORA_ERR_SHAPE, "batch: negative or too large size");
  if (b->n_seq > 0 && (!b->page_table || !b->kv_len || !b->q_start || !b->q_len))
    return fail(SLORA_ERR_NULL, "batch: null table");
  if (b->n_seq > (1 << 20)) return fail(SLORA_ERR_SHAPE, "batch: n_seq=%d (at most 2^20)", b->n_seq);
  if (b->table_stride < b->max_pages) return fail(SLORA_ERR_SHAPE, "batch: table rows overlap");
  // positions are 32-bit, with room for a tile behind the last
  const int64_t tokens = static_cast<int64_t>(b->max_pages) << shift;
  if (tokens > 0x7ffff000) return fail(SLORA_ERR_SHAPE, "batch: max_pages=%d holds more than 2^31 tokens", b->max_pages);
  out->table = b->page_table;
  out->table_stride = b->table_stride;
  out->kv_len = b->kv_len;
  out->q_start = b->q_start;
  out->q_len = b->q_len;
  out->status = b->status;
  out->n_seq = b->n_seq;
  out->max_q = b->max_q_len;
  out->max_tokens = tokens;
  out->T = T;
  return SLORA_OK;
}

int check_rows(const void* p, int64_t stride, int64_t width, int64_t T, const char* name) {
  if (!p) return fail(SLORA_ERR_NULL, "%s is null", name);
  if (!aligned16(p) || stride % 8 != 0) return fail(SLORA_ERR_ALIGN, "%s rows are not 16-byte aligned", name);
  if (T > 1 && stride < width) return fail(SLORA_ERR_SHAPE, "%s rows overlap", name);
  return SLORA_OK;
}

// Do two sets of T rows of `width` 16-bit elements share memory?  (Rows side by side in one wider buffer do not.)
bool rows_overlap(const void* a, int64_t a_stride, const void* b, int64_t b_stride, int64_t width, int64_t T) {
  const int64_t d = (static_cast<const char*>(b) - static_cast<const char*>(a)) / 2;  // rows start on 16 bytes
  if (d >= (T - 1) * a_stride + width || -d >= (T - 1) * b_stride + width) return false;
  if (T > 1 && a_stride == b_stride) {
    const int64_t r = (d % a_stride + a_stride) % a_stride;
    return r < width || a_stride - r < width;
  }
  return true;
}
// Rows that are written while others are still read: the same ones, or none of them.
int check_in_place(const void* from, int64_t from_stride, const void* to, int64_t to_stride, int64_t width, int64_t T, const char* name) {
  if (from == to && (T <= 1 || from_stride == to_stride)) return SLORA_OK;
  return rows_overlap(from, from_stride, to, to_stride, width, T) ? fail(SLORA_ERR_SHAPE, "%s_out overlaps %s and is not the same rows", name, name)
                                                                  : SLORA_OK;
}

int check_rotary(int head_dim, int rot, int layout, const void* positions, const void* turns, RotaryArgs* out, float factor,
                 int inverse) {
  if (rot < 16 || rot > head_dim || rot % 16 != 0)
    return fail(SLORA_ERR_SHAPE, "No suitable kernel. rot=%d (a multiple of 16 up to head_dim=%d)", rot, head_dim);
  if (layout != 0 && layout != 1) return fail(SLORA_ERR_SHAPE, "rotary layout %d is neither 0 (half) nor 1 (interleaved)", layout);
  if (!positions || !turns) return fail(SLORA_ERR_NULL, "rotary: null positions or turns");
  out->positions = static_cast<const int64_t*>(positions);
  out->turns = static_cast<const double*>(turns);
  out->factor = factor;
  out->rot = rot;
  out->layout = layout;
  out->inverse = inverse;
  return SLORA_OK;
}

// CTAs that share a block of tokens, so that a small call still fills the GPU: about eight per SM, at least one row a warp.
int head_splits(int64_t units, int rows) {
  const int64_t want = (8 * sm_count() + units - 1) / (units > 0 ? units : 1);
  const int most = (rows + kRowWarps - 1) / kRowWarps;
  return static_cast<int>(want < 1 ? 1 : want > most ? most : want);
}

template <int D>
int rotary_d(const RowArgs& a, dim3 grid, size_t smem, int dtype, cudaStream_t s) {
  return dtype == SLORA_F16 ? launch_pdl<rotary_kernel<D, __half>>(grid, kRowThreads, smem, s, "rotary", a)
                            : launch_pdl<rotary_kernel<D, __nv_bfloat16>>(grid, kRowThreads, smem, s, "rotary", a);
}

// One instantiation per (head_dim, kind, I/O type).
#define KV_DISPATCH(D_, KIND_, DTYPE_, CALL)                                              \
  [&]() -> int {                                                                          \
    auto by_type = [&](auto d, auto kind) -> int {                                        \
      constexpr int D = decltype(d)::value;                                               \
      constexpr int KIND = decltype(kind)::value;                                         \
      if (DTYPE_ == SLORA_F16) {                                                          \
        using T = __half;                                                                 \
        return CALL;                                                                      \
      }                                                                                   \
      using T = __nv_bfloat16;                                                            \
      return CALL;                                                                        \
    };                                                                                    \
    auto by_kind = [&](auto d) -> int {                                                   \
      return KIND_ == SLORA_KV_INT8 ? by_type(d, std::integral_constant<int, SLORA_KV_INT8>()) \
                                    : by_type(d, std::integral_constant<int, SLORA_KV_E4M3>()); \
    };                                                                                    \
    return D_ == 64    ? by_kind(std::integral_constant<int, 64>())                       \
           : D_ == 128 ? by_kind(std::integral_constant<int, 128>())                      \
                       : by_kind(std::integral_constant<int, 256>());                     \
  }()

// ---- attention -------------------------------------------------------------------------------------------------------
// Tiles of eight rows (new tokens x q heads of a KV head) that a CTA of the attention holds.  One block of rows reads the
// keys once; the most is what the accumulators' registers allow (32 rows at head_dim 64, 16 at 128, 8 at 256).
int attend_tiles(int max_q, int group, int d) {
  const int64_t rows = static_cast<int64_t>(max_q) * group;
  const int most = 256 / d;
  return rows <= 8 || most == 1 ? 1 : rows <= 16 || most == 2 ? 2 : 4;
}
int attend_grid(int nt, int d) { return sm_count() * attend_ctas(nt, d); }

// Which sequences go to the tensor-memory kernel (kv_prefill.cuh): those with at least kPrefillRows rows, or, where a batch
// has few (sequence, KV head) pairs, with kPrefillShare / pairs.  That kernel does not split keys: an item of 256 rows takes
// 3 to 4 us per 128 keys on an SM of its own, however many SMs are idle, while the row kernel spreads any work over all
// of them at 8.6 ns per 128 keys and 16 rows.  Measured (d 128, us, row kernel / tensor-memory kernel):
//   24 sequences x 8 heads, 4096 keys:  56 rows 209 / -, 64 rows 211 / 333, 128 rows 398 / 323, 256 rows 774 / 271
//   4 sequences x 8 heads, 8192 keys:   64 rows 82 / 292, 128 rows 141 / 253, 256 rows 254 / 230
//   1 sequence, one KV head, 32768 keys: 64 rows 39 / 945, 256 rows 51 / 767
// head_dim 256 has no tensor-memory kernel: its operands do not fit.
constexpr int kPrefillRows = 64;
constexpr int64_t kPrefillShare = 6144;

// The scores that add_weights keeps take 4 bytes per key and row.  With them the row kernel takes all rows (128 keys and 16
// rows: 8.6 ns and 1.5 for the weights; the tensor-memory kernel 1.3, but 15 for the scores again).  Beyond this many bytes,
// if every sequence were as long as the table allows, they are computed again (32 sequences of 4096 keys, 32 heads on 8,
// one token each: weights kept 88 us, computed again 123): it bounds the workspace.
constexpr int64_t kMaxScoreBytes = int64_t(1) << 29;

// When the weights are added up, the warps of a CTA share a tile's row blocks where there are more than kSplitBlocks, or more
// than one and fewer (sequence, KV head) pairs than SMs.  Weights alone, us, a warp all blocks / shared (d 128):
//   24 sequences x 8 heads, 3 blocks, 4000 keys: 90 / 115;  5 blocks, 2000 keys: 141 / 145
//   4 x 8 heads, 8 blocks, 2000 keys: 185 / 34;  1 x 1 head, 400 blocks, 1000 keys: 6900 / 86
constexpr int kSplitBlocks = 4;

struct AttendLayout {
  int nt, grid, part_rows;
  int blocks;          // row blocks of a sequence, at most
  int split;           // q_len from which sequences are the prefill kernel's; above max_q: none
  int64_t pre_grid;    // its items, at most
  bool keep_scores;
  bool split_weights;
  size_t part, rec, lse, scores, total;
};
AttendLayout attend_layout(const KvCache& c, const KvBatch& b, int hq, int add_weights) {
  AttendLayout l;
  const int group = hq / c.hkv;
  const int64_t seqs = b.n_seq < b.T ? b.n_seq : b.T;
  double bytes = 0;  // of the scores
  // the row kernel's part, for sequences of up to most_q new tokens
  const auto rows_up_to = [&](int most_q) {
    l.nt = attend_tiles(most_q, group, c.d);
    const int64_t rows = static_cast<int64_t>(most_q) * group;
    l.part_rows = static_cast<int>(rows < 1 ? 1 : rows < 8 * l.nt ? rows : 8 * l.nt);
    l.blocks = static_cast<int>((rows + 8 * l.nt - 1) / (8 * l.nt));
    // cost units of all pieces (see kv_attend.cuh), if every sequence were as long as the page table allows
    const double units =
        static_cast<double>(b.n_seq) * (static_cast<double>(b.max_tokens / kAttendTile) + 1 + kAttendPiece) * c.hkv * l.blocks;
    bytes = units * l.part_rows * kAttendTile * sizeof(float);
  };
  l.split = 0x7fffffff;
  rows_up_to(b.max_q);
  l.keep_scores = add_weights && bytes <= static_cast<double>(kMaxScoreBytes);
  const int64_t pairs = seqs * c.hkv > 0 ? seqs * c.hkv : 1;
  l.split_weights = l.blocks > kSplitBlocks || (l.blocks > 1 && pairs < sm_count());
  if (!l.keep_scores && c.d <= 128) {
    const int64_t rows = kPrefillShare / pairs > kPrefillRows ? kPrefillShare / pairs : kPrefillRows;
    l.split = static_cast<int>((rows + group - 1) / group);
  }
  const bool pre = b.max_q >= l.split;
  if (pre) rows_up_to(l.split - 1);
  l.pre_grid = pre ? (b.T * group / kPreRows + seqs) * c.hkv : 0;
  l.grid = attend_grid(l.nt, c.d);
  const auto up = [](size_t x) { return (x + 15) & ~static_cast<size_t>(15); };
  const size_t runs = static_cast<size_t>(l.grid);
  l.part = 0;
  l.rec = up(2u * runs * l.part_rows * (c.d + 4) * sizeof(float));
  l.lse = l.rec + up(runs * 16);
  l.scores = l.lse + (add_weights ? up(static_cast<size_t>(b.T) * hq * sizeof(float)) : 0);
  l.total = l.scores + (l.keep_scores ? up(static_cast<size_t>(bytes)) : 0);
  return l;
}

template <int D, int NT, int KIND, typename T>
int attend_nt(const KvAttendArgs& a, int grid, cudaStream_t s) {
  return launch_pdl<kv_attend_kernel<D, NT, KIND, T>>(dim3(grid), kAttendThreads, sizeof(AttendSmem<D, NT>), s, "kv8_attend", a);
}
template <int D, int KIND, typename T>
int attend_launch(KvAttendArgs a, const AttendLayout& l, int add_weights, cudaStream_t s) {
  int rc = SLORA_OK;
  if (l.nt == 1) rc = attend_nt<D, 1, KIND, T>(a, l.grid, s);
  if constexpr (D <= 128) {
    if (l.nt == 2) rc = attend_nt<D, 2, KIND, T>(a, l.grid, s);
  }
  if constexpr (D == 64) {
    if (l.nt == 4) rc = attend_nt<D, 4, KIND, T>(a, l.grid, s);
  }
  if (rc) return rc;
  if constexpr (D <= 128) {
    if (l.pre_grid > 0) {
      KvAttendArgs p = a;
      p.min_q = l.split;
      p.lim_q = a.b.max_q;
      rc = launch_pdl<kv_prefill_kernel<D, KIND, T>>(dim3(static_cast<unsigned>(l.pre_grid)), kPreThreads, sizeof(PreSmem<D>) + 1024, s, "kv8_attend prefill", p);
      if (rc) return rc;
    }
  }
  rc = launch_pdl<kv_join_kernel<D, T>>(dim3(l.grid), kJoinThreads, 0, s, "kv8_attend join", a);
  if (rc || !add_weights) return rc;
  if (l.keep_scores)
    return l.split_weights ? launch_pdl<kv_weights_kernel<D, true>>(dim3(2 * sm_count()), 512, 0, s, "kv8_attend weights", a)
                           : launch_pdl<kv_weights_kernel<D, false>>(dim3(8 * sm_count()), kAttendThreads, 0, s, "kv8_attend weights", a);
  a.rows_per_block = 8;
  return launch_pdl<kv_reweigh_kernel<D, KIND, T>>(dim3(attend_grid(1, D)), kAttendThreads, 0, s, "kv8_attend weights", a);
}

int check_attend(const slora_kv8_cache* cache, const slora_kv8_batch* batch, int64_t T, int q_heads, int add_weights,
                 KvCache* c, KvBatch* b) {
  if (const int rc = check_cache(cache, c)) return rc;
  if (const int rc = check_batch(batch, c->shift, T, b)) return rc;
  if (q_heads < 1 || q_heads % c->hkv != 0 || q_heads > (1 << 20))
    return fail(SLORA_ERR_SHAPE, "q_heads=%d is not a multiple of kv_heads=%d", q_heads, c->hkv);
  if (static_cast<int64_t>(b->max_q) * (q_heads / c->hkv) > 0x3fffffff || T * q_heads > 0x3fffffffffLL)
    return fail(SLORA_ERR_SHAPE, "attend: too many rows");
  if (add_weights && !c->w) return fail(SLORA_ERR_NULL, "add_weights: the cache has no weights");
  return SLORA_OK;
}

// CTAs of a page's units (a cluster: 1, 2, 4 or 8) for `rows` head rows per token.
int append_splits(int64_t units, int rows) {
  const int splits = head_splits(units, rows);
  return splits >= 8 ? 8 : splits >= 4 ? 4 : splits >= 2 ? 2 : 1;
}
template <int D, int KIND, typename T>
int append_launch(AppendArgs a, int64_t units, int tokens, cudaStream_t s) {
  const size_t angles = a.r.turns ? static_cast<size_t>(tokens) * (a.r.rot / 2) * sizeof(float2) : 0;
  if (a.b.max_q <= kAppendWarpTokens) {
    a.head_splits = append_splits(units, a.hq + 2 * a.c.hkv);
    return launch_cluster<kv_append_kernel<D, KIND, T, APPEND_FEW>>(a.head_splits, dim3(static_cast<unsigned>(units), a.head_splits),
                                                                    kRowThreads, angles, s, "kv8_append", a);
  }
  if (a.q) {
    a.head_splits = (tokens + 7) / 8;  // about eight tokens a CTA
    if (const int rc = launch_pdl<kv_append_kernel<D, 0, T, APPEND_Q>>(dim3(static_cast<unsigned>(units), a.head_splits), kRowThreads,
                                                                       static_cast<size_t>(8) * (a.r.rot / 2) * sizeof(float2), s, "kv8_append q", a))
      return rc;
  }
  a.head_splits = append_splits(units, kRowWarps * 2 * a.c.hkv);
  const size_t rows = static_cast<size_t>(tokens) * D * 2;
  a.rows_at = static_cast<int>(angles);
  a.rows_step = angles + 2 * rows <= 200 * 1024 ? static_cast<int>(rows) : 0;
  return launch_cluster<kv_append_kernel<D, KIND, T, APPEND_KV>>(a.head_splits, dim3(static_cast<unsigned>(units), a.head_splits), kRowThreads,
                                                                 angles + (a.rows_step > 0 ? 2 : 1) * rows, s, "kv8_append k, v", a);
}
template <int D, int KIND, typename T>
int read_launch(const ReadArgs& a, int grid, cudaStream_t s) {
  return launch_pdl<kv_read_kernel<D, KIND, T>>(dim3(grid), kRowThreads, 0, s, "kv8_read", a);
}
template <int D, int KIND, typename T>
int move_launch(const EvictArgs& a, dim3 grid, cudaStream_t s) {
  return launch_pdl<kv_move_kernel<D, KIND>>(grid, kMoveThreads, 0, s, "kv8_evict move", a);
}

}  // namespace

extern "C" {

int slora_rotary(void* q_out, void* k_out, const void* q, const void* k, int64_t T, int q_heads, int k_heads,
                 int head_dim, int rot, int64_t q_out_stride, int64_t k_out_stride, int64_t q_stride, int64_t k_stride,
                 const int64_t* positions, const double* turns, float factor, int layout, int inverse, int dtype,
                 void* stream) {
  if (int rc = check_dtype(dtype)) return rc;
  if (int rc = check_head_dim(head_dim)) return rc;
  if (T < 0 || T > 0x7fffffff || q_heads < 0 || k_heads < 0 || q_heads > 65535 || k_heads > 65535)
    return fail(SLORA_ERR_SHAPE, "rotary: T=%lld, heads %d and %d", (long long)T, q_heads, k_heads);
  RowArgs a;
  memset(&a, 0, sizeof(a));
  if (T == 0 || q_heads + k_heads == 0) return SLORA_OK;
  if (int rc = check_rotary(head_dim, rot, layout, positions, turns, &a.r, factor, inverse)) return rc;
  const void* src[2] = {q, k};
  void* dst[2] = {q_out, k_out};
  const int heads[2] = {q_heads, k_heads};
  const int64_t ss[2] = {q_stride, k_stride}, ds[2] = {q_out_stride, k_out_stride};
  const char* names[2][2] = {{"q", "q_out"}, {"k", "k_out"}};
  for (int i = 0; i < 2; ++i) {
    if (heads[i] == 0) continue;
    if (int rc = check_rows(src[i], ss[i], static_cast<int64_t>(heads[i]) * head_dim, T, names[i][0])) return rc;
    if (int rc = check_rows(dst[i], ds[i], static_cast<int64_t>(heads[i]) * head_dim, T, names[i][1])) return rc;
    if (int rc = check_in_place(src[i], ss[i], dst[i], ds[i], static_cast<int64_t>(heads[i]) * head_dim, T, names[i][0])) return rc;
    a.src[i] = src[i];
    a.dst[i] = dst[i];
    a.src_stride[i] = ss[i];
    a.dst_stride[i] = ds[i];
    a.heads[i] = heads[i];
  }
  a.T = T;
  const int64_t per = (T + 8 * sm_count() - 1) / (8 * sm_count());
  a.tokens_per_cta = static_cast<int>(per < 1 ? 1 : per > 8 ? 8 : per);
  const int64_t blocks = (T + a.tokens_per_cta - 1) / a.tokens_per_cta;
  a.head_splits = head_splits(blocks, q_heads + k_heads);
  const size_t smem = static_cast<size_t>(a.tokens_per_cta) * (rot / 2) * sizeof(float2);
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(a.head_splits));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return head_dim == 64    ? rotary_d<64>(a, grid, smem, dtype, s)
         : head_dim == 128 ? rotary_d<128>(a, grid, smem, dtype, s)
                           : rotary_d<256>(a, grid, smem, dtype, s);
}

int slora_kv8_append(const slora_kv8_cache* cache, const slora_kv8_batch* batch, const void* k, const void* v,
                     int64_t k_stride, int64_t v_stride, int64_t T, const void* q, void* q_out, int q_heads,
                     int64_t q_stride, int64_t q_out_stride, const int64_t* positions, const double* turns, int rot,
                     float factor, int layout, int dtype, void* stream) {
  if (int rc = check_dtype(dtype)) return rc;
  AppendArgs a;
  memset(&a, 0, sizeof(a));
  if (int rc = check_cache(cache, &a.c)) return rc;
  if (int rc = check_batch(batch, a.c.shift, T, &a.b)) return rc;
  if (T == 0 || a.b.n_seq == 0 || a.b.max_q == 0) return SLORA_OK;
  const int64_t width = static_cast<int64_t>(a.c.hkv) * a.c.d;
  if (int rc = check_rows(k, k_stride, width, T, "k")) return rc;
  if (int rc = check_rows(v, v_stride, width, T, "v")) return rc;
  if (turns) {
    if (int rc = check_rotary(a.c.d, rot, layout, positions, turns, &a.r, factor, 0)) return rc;
  } else if (q) {
    return fail(SLORA_ERR_NULL, "append: q without a rotary table");
  }
  if (q) {
    if (q_heads < 1 || q_heads > 65535) return fail(SLORA_ERR_SHAPE, "append: q_heads=%d", q_heads);
    if (int rc = check_rows(q, q_stride, static_cast<int64_t>(q_heads) * a.c.d, T, "q")) return rc;
    if (int rc = check_rows(q_out, q_out_stride, static_cast<int64_t>(q_heads) * a.c.d, T, "q_out")) return rc;
    if (int rc = check_in_place(q, q_stride, q_out, q_out_stride, static_cast<int64_t>(q_heads) * a.c.d, T, "q")) return rc;
  }
  a.q = q;
  a.q_out = q_out;
  a.k = k;
  a.v = v;
  a.q_stride = q_stride;
  a.q_out_stride = q_out_stride;
  a.k_stride = k_stride;
  a.v_stride = v_stride;
  a.hq = q ? q_heads : 0;
  // pages that new tokens can touch: with T rows over the sequences, at most T / page + 2 each, and one per row
  const int64_t seqs = a.b.n_seq < T ? a.b.n_seq : T;
  int64_t units = (T >> a.c.shift) + 2 * seqs;
  if (units > T) units = T;
  if (a.b.max_q == 1 && units > seqs) units = seqs;
  const int page = 1 << a.c.shift;
  const int tokens = a.b.max_q < page ? a.b.max_q : page;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return KV_DISPATCH(a.c.d, cache->kind, dtype, (append_launch<D, KIND, T>(a, units, tokens, s)));
}

int slora_kv8_read(const slora_kv8_cache* cache, const slora_kv8_batch* batch, const int32_t* first, int64_t count,
                   void* k_out, void* v_out, int dtype, void* stream) {
  if (int rc = check_dtype(dtype)) return rc;
  ReadArgs a;
  memset(&a, 0, sizeof(a));
  if (int rc = check_cache(cache, &a.c)) return rc;
  if (int rc = check_batch(batch, a.c.shift, 0, &a.b)) return rc;
  if (count < 0 || count > 0x7fffffff) return fail(SLORA_ERR_SHAPE, "read: count=%lld", (long long)count);
  if (count == 0 || a.b.n_seq == 0) return SLORA_OK;
  if (!k_out || !v_out) return fail(SLORA_ERR_NULL, "read: null output");
  if (!aligned16(k_out) || !aligned16(v_out)) return fail(SLORA_ERR_ALIGN, "read: an output is not 16-byte aligned");
  a.first = first;
  a.count = count;
  a.out[0] = k_out;
  a.out[1] = v_out;
  const int64_t group = kReadAhead * (256 / a.c.d), units = count * a.b.n_seq * ((a.c.hkv + group - 1) / group);
  const int64_t blocks = (units + kRowWarps - 1) / kRowWarps, most = 8ll * sm_count();
  const int grid = static_cast<int>(blocks < most ? blocks : most);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return KV_DISPATCH(a.c.d, cache->kind, dtype, (read_launch<D, KIND, T>(a, grid, s)));
}

size_t slora_kv8_attend_workspace_bytes(const slora_kv8_cache* cache, const slora_kv8_batch* batch, int64_t T,
                                        int q_heads, int add_weights) {
  KvCache c;
  KvBatch b;
  if (check_attend(cache, batch, T, q_heads, add_weights, &c, &b)) return 0;
  return attend_layout(c, b, q_heads, add_weights).total;
}

int slora_kv8_attend(const slora_kv8_cache* cache, const slora_kv8_batch* batch, const void* q, int64_t q_stride,
                     int64_t T, int q_heads, void* out, int64_t out_stride, float* lse, float scale, int window,
                     int add_weights, void* workspace, size_t workspace_bytes, int dtype, void* stream) {
  if (int rc = check_dtype(dtype)) return rc;
  KvAttendArgs a;
  memset(&a, 0, sizeof(a));
  if (int rc = check_attend(cache, batch, T, q_heads, add_weights, &a.c, &a.b)) return rc;
  if (window < 0) return fail(SLORA_ERR_SHAPE, "attend: window=%d", window);
  if (T == 0 || a.b.n_seq == 0 || a.b.max_q == 0) return SLORA_OK;
  const int64_t width = static_cast<int64_t>(q_heads) * a.c.d;
  if (int rc = check_rows(q, q_stride, width, T, "q")) return rc;
  if (int rc = check_rows(out, out_stride, width, T, "out")) return rc;
  if (add_weights && rows_overlap(q, q_stride, out, out_stride, width, T))
    return fail(SLORA_ERR_SHAPE, "attend: out overlaps q, which add_weights reads again");
  const AttendLayout l = attend_layout(a.c, a.b, q_heads, add_weights);
  if (!workspace || workspace_bytes < l.total)
    return fail(SLORA_ERR_WORKSPACE, "attend: workspace of %zu bytes, %zu needed", workspace ? workspace_bytes : 0, l.total);
  if (!aligned16(workspace)) return fail(SLORA_ERR_ALIGN, "attend: the workspace is not 16-byte aligned");
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  a.q = q;
  a.out = out;
  a.lse = lse ? lse : add_weights ? reinterpret_cast<float*>(ws + l.lse) : nullptr;
  a.q_stride = q_stride;
  a.out_stride = out_stride;
  a.hq = q_heads;
  a.group = q_heads / a.c.hkv;
  a.rows_per_block = 8 * l.nt;
  a.scale2 = scale * 1.4426950408889634f;
  a.window = window;
  a.min_q = 0;
  a.lim_q = l.split - 1;
  a.part_rows = l.part_rows;
  a.blocks = l.blocks;
  a.runs = l.grid;
  a.scores = l.keep_scores ? reinterpret_cast<float*>(ws + l.scores) : nullptr;
  a.part = reinterpret_cast<float*>(ws + l.part);
  a.rec = reinterpret_cast<int*>(ws + l.rec);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return KV_DISPATCH(a.c.d, cache->kind, dtype, (attend_launch<D, KIND, T>(a, l, add_weights, s)));
}

int slora_kv8_evict(const slora_kv8_cache* cache, const slora_kv8_batch* batch, int budget, int recent, int sink,
                    int32_t* kept, const int64_t* dest_table, int64_t dest_stride, int dest_pages, void* stream) {
  EvictArgs a;
  memset(&a, 0, sizeof(a));
  if (int rc = check_cache(cache, &a.c)) return rc;
  if (int rc = check_batch(batch, a.c.shift, 0, &a.b)) return rc;
  if (!a.c.w) return fail(SLORA_ERR_NULL, "evict: the cache has no weights");
  if (budget < 1 || recent < 0 || sink < 0 || static_cast<int64_t>(recent) + sink > budget)
    return fail(SLORA_ERR_SHAPE, "evict: budget=%d must hold sink=%d and recent=%d tokens", budget, sink, recent);
  if (a.b.n_seq == 0) return SLORA_OK;
  if (!kept || !dest_table) return fail(SLORA_ERR_NULL, "evict: null kept or dest_table");
  const int64_t longest = budget < a.b.max_tokens ? budget : a.b.max_tokens;
  if (dest_pages < 0 || dest_stride < dest_pages || (static_cast<int64_t>(dest_pages) << a.c.shift) < longest)
    return fail(SLORA_ERR_SHAPE, "evict: %d destination pages cannot hold %lld tokens", dest_pages, (long long)longest);
  const int64_t heads = static_cast<int64_t>(a.b.n_seq) * a.c.hkv;
  if (heads > 0x7fffffff) return fail(SLORA_ERR_SHAPE, "evict: too many heads");
  a.budget = budget;
  a.recent = recent;
  a.sink = sink;
  a.kept = kept;
  a.dest = dest_table;
  a.dest_stride = dest_stride;
  a.in_place = dest_table == batch->page_table;
  // 40960 weights are what a CTA's shared memory takes (160 KB); a longer sequence's rest is read again in each pass
  a.cached = static_cast<int>(a.b.max_tokens < 40960 ? a.b.max_tokens : 40960);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (int rc = launch_pdl<kv_select_kernel>(dim3(static_cast<unsigned>(heads)), kSelectThreads,
                          static_cast<size_t>(a.cached) * sizeof(uint32_t), s, "kv8_evict select", a))
    return rc;
  const int64_t rounds = (((longest + (1 << a.c.shift) - 1) >> a.c.shift) * ((1 << a.c.shift) / 16) + kMoveWarps - 1) / kMoveWarps;
  int64_t chunks = a.in_place ? 1 : (16ll * sm_count() + heads - 1) / heads;
  if (chunks > rounds) chunks = rounds < 1 ? 1 : rounds;
  if (chunks > 65535) chunks = 65535;
  a.chunks = static_cast<int>(chunks);
  const dim3 grid(static_cast<unsigned>(heads), static_cast<unsigned>(chunks));
  return KV_DISPATCH(a.c.d, cache->kind, SLORA_F16, (move_launch<D, KIND, T>(a, grid, s)));
}

}  // extern "C"
