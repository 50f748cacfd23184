// cawq_layer.cu — the operators between the linears of a decoder layer: RMS
// norm with the residual, rotary embedding with the cache append, and
// attention over a paged cache. Kernels, their launchers and the extern "C"
// entry points (argument checks on the host; what only the device knows is
// bounded in the kernels, see cawq_paged.cuh).
#include <algorithm>
#include <cmath>

#include "cawq_common.cuh"

namespace cawq {

struct NormProblem {
  const void *x, *w, *res;
  void *y, *res_out;
  float* scales;  // non-null: y is e4m3
  size_t rows, d, ld_x, ld_res, ld_y, ld_res_out;
  float eps;
  int dtype, sm_count;
  cudaStream_t stream;
};

struct RopeProblem {
  const void *q, *k, *v;
  const float* rope;
  void* q_out;
  size_t rope_rows, tokens, n_q, d, ld_q, ld_k, ld_v, ld_q_out;
  int dtype;
  cudaStream_t stream;
};

struct AttentionProblem {
  const void* q;
  void* out;
  size_t tokens, n_q, d, ld_q, ld_out;
  float scale;
  int window, sinks;
  int dtype;
  void* workspace;
  int sm_count, device;
  cudaStream_t stream;
};

// Launch with programmatic dependent launch: every kernel of this file begins
// with griddepcontrol.wait.
template <typename K>
inline cudaError_t launch_pdl(K kern, dim3 grid, int threads, size_t smem, cudaStream_t stream,
                              void** args, uint32_t cluster = 1) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelExC(&cfg, reinterpret_cast<const void*>(kern), args);
}

// Dynamic shared memory past 48 KB has to be asked for once per device.
template <typename K>
inline cudaError_t allow_smem(K kern, int smem, int device, uint64_t* done) {
  if (device < 64 && (*done >> device & 1)) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(reinterpret_cast<const void*>(kern),
                                             cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e == cudaSuccess && device < 64) *done |= 1ull << device;
  return e;
}

cudaError_t read_layer_error(uint32_t* word, int reset) { return read_own_error_word(word, reset); }

}  // namespace cawq

#include "cawq_attention.cuh"
#include "cawq_attention_tile.cuh"
#include "cawq_norm.cuh"
#include "cawq_rope.cuh"

#define CAWQ_API extern "C" __attribute__((visibility("default")))

namespace cawq {

constexpr size_t kMaxInt = 0x7fffffff;

static bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

static cawq_status rms_norm(const void* x, const void* weight, const void* residual, void* y,
                            float* scales, void* residual_out, size_t rows, size_t d, size_t ld_x,
                            size_t ld_res, size_t ld_y, size_t ld_ro, float eps, cawq_dtype dtype,
                            void* stream) {
  if (dtype != CAWQ_F32 && dtype != CAWQ_F16 && dtype != CAWQ_BF16)
    return fail(CAWQ_ERR_DTYPE, "dtype must be CAWQ_F32, CAWQ_F16 or CAWQ_BF16");
  if (d == 0 || d > kMaxInt) return fail(CAWQ_ERR_INVALID_SHAPE, "d must be in 1 .. 2^31 - 1");
  if (rows > kMaxInt) return fail(CAWQ_ERR_INVALID_SHAPE, "rows must be below 2^31");
  size_t* lds[] = {&ld_x, &ld_res, &ld_y, &ld_ro};
  for (size_t* ld : lds) {
    if (*ld == 0) *ld = d;
    if (*ld < d) return fail(CAWQ_ERR_INVALID_SHAPE, "row strides must be >= d");
  }
  if (!(eps >= 0.f)) return fail(CAWQ_ERR_INVALID_ARGUMENT, "eps must be >= 0");
  if (residual_out && !residual)
    return fail(CAWQ_ERR_INVALID_ARGUMENT, "residual_out needs a residual");
  if (rows == 0) return CAWQ_OK;
  if (!x || !weight || !y) return fail(CAWQ_ERR_NULL_POINTER, "x, weight and y must be non-null");
  DeviceInfo dev;
  cawq_status st = require_sm100(&dev);
  if (st != CAWQ_OK) return st;
  const NormProblem p = {x, weight, residual, y, residual_out, scales, rows, d, ld_x, ld_res,
                         ld_y, ld_ro, eps, dtype, dev.sm_count, static_cast<cudaStream_t>(stream)};
  const cudaError_t e = launch_rms_norm(p);
  return e == cudaSuccess ? CAWQ_OK : cuda_fail(e, "RMS norm launch");
}

// The rules of a cache and its batch; `tokens` rows of new tokens.
static cawq_status check_paged(const cawq_paged_kv* kv, size_t tokens, size_t n_q) {
  if (!kv) return fail(CAWQ_ERR_NULL_POINTER, "kv must be non-null");
  if (kv->head_dim != 64 && kv->head_dim != 128)
    return fail(CAWQ_ERR_INVALID_SHAPE, fmt("head_dim = %zu must be 64 or 128", kv->head_dim));
  if (kv->page_size == 0 || kv->page_size % 8 != 0)
    return fail(CAWQ_ERR_INVALID_SHAPE,
                fmt("page_size = %zu must be a positive multiple of 8", kv->page_size));
  if (kv->n_kv == 0 || n_q == 0 || n_q % kv->n_kv != 0 || n_q / kv->n_kv > 128 || n_q > 65535)
    return fail(CAWQ_ERR_INVALID_SHAPE,
                fmt("n_q = %zu must be a multiple of n_kv = %zu, at most 128 times it and 65535",
                    n_q, kv->n_kv));
  if (kv->pages > kMaxInt || kv->batch > kMaxInt || tokens > kMaxInt ||
      kv->page_size > kMaxInt || kv->table_width > kMaxInt / kv->page_size)
    return fail(CAWQ_ERR_INVALID_SHAPE,
                "pages, batch, tokens and table_width * page_size must be below 2^31");
  if (tokens > kMaxInt / (n_q / kv->n_kv))
    return fail(CAWQ_ERR_INVALID_SHAPE, "tokens * n_q / n_kv must be below 2^31");
  if (kv->stride_page % 8 != 0 || kv->stride_head % 8 != 0 || kv->stride_token % 8 != 0)
    return fail(CAWQ_ERR_ALIGNMENT, "cache strides must be multiples of 8 elements");
  if (kv->ld_table < kv->table_width)
    return fail(CAWQ_ERR_INVALID_SHAPE, "ld_table must be >= table_width");
  if (!kv->q_start && tokens != kv->batch)
    return fail(CAWQ_ERR_INVALID_SHAPE, "without q_start there is one new token per sequence");
  if (tokens > 0 && kv->batch > 0) {
    if (!kv->seq_lens || (kv->table_width > 0 && !kv->block_table) ||
        (kv->pages > 0 && (!kv->k || !kv->v)))
      return fail(CAWQ_ERR_NULL_POINTER, "k, v, block_table and seq_lens must be non-null");
    if (!aligned16(kv->k) || !aligned16(kv->v))
      return fail(CAWQ_ERR_ALIGNMENT, "k and v must be 16-byte aligned");
  }
  return CAWQ_OK;
}

static PagedView paged_view(const cawq_paged_kv& kv, size_t elem, bool one_each) {
  PagedView v;
  v.k = static_cast<char*>(kv.k);
  v.v = static_cast<char*>(kv.v);
  v.sp = static_cast<int64_t>(kv.stride_page * elem);
  v.sh = static_cast<int64_t>(kv.stride_head * elem);
  v.st = static_cast<int64_t>(kv.stride_token * elem);
  v.table = kv.block_table;
  v.lens = kv.seq_lens;
  v.q_start = one_each ? nullptr : kv.q_start;
  v.ld_table = static_cast<int64_t>(kv.ld_table);
  v.pages = static_cast<uint32_t>(kv.pages);
  v.width = static_cast<uint32_t>(kv.table_width);
  v.batch = static_cast<uint32_t>(kv.batch);
  v.n_kv = static_cast<uint32_t>(kv.n_kv);
  v.page = FastDiv(static_cast<uint32_t>(kv.page_size));
  return v;
}

// A [tokens, heads, head_dim] operand: token stride (0 = dense) and alignment.
static cawq_status check_rows(const char* name, const void* p, size_t* ld, size_t width) {
  if (*ld == 0) *ld = width;
  if (*ld < width || *ld % 8 != 0)
    return fail(CAWQ_ERR_INVALID_SHAPE,
                fmt("%s: the token stride must be >= its heads * head_dim and a multiple of 8", name));
  if (!p) return fail(CAWQ_ERR_NULL_POINTER, fmt("%s must be non-null", name));
  if (!aligned16(p)) return fail(CAWQ_ERR_ALIGNMENT, fmt("%s must be 16-byte aligned", name));
  return CAWQ_OK;
}

static cawq_status attention(const void* q, void* out, const cawq_paged_kv* kv, size_t tokens,
                             size_t n_q, size_t ld_q, size_t ld_out, float scale, size_t window,
                             size_t sinks, cawq_dtype dtype, void* workspace,
                             size_t workspace_bytes, bool decode, void* stream) {
  if (dtype != CAWQ_F16 && dtype != CAWQ_BF16)
    return fail(CAWQ_ERR_DTYPE, "attention takes CAWQ_F16 or CAWQ_BF16");
  if (kv && !decode && !kv->q_start)
    return fail(CAWQ_ERR_NULL_POINTER, "q_start must be non-null");
  cawq_status st = check_paged(kv, tokens, n_q);
  if (st != CAWQ_OK) return st;
  if (tokens == 0 || kv->batch == 0) return CAWQ_OK;
  if ((st = check_rows("q", q, &ld_q, n_q * kv->head_dim)) != CAWQ_OK) return st;
  if ((st = check_rows("out", out, &ld_out, n_q * kv->head_dim)) != CAWQ_OK) return st;
  const size_t need = cawq_attention_workspace(kv, tokens, n_q);
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned16(workspace)))
    return fail(CAWQ_ERR_INVALID_ARGUMENT,
                fmt("the workspace must be 16-byte aligned and hold %zu bytes", need));
  DeviceInfo dev;
  if ((st = require_sm100(&dev)) != CAWQ_OK) return st;
  const AttentionProblem p = {q, out, tokens, n_q, kv->head_dim, ld_q, ld_out, scale,
                              static_cast<int>(std::min(window, kMaxInt)),
                              static_cast<int>(std::min(sinks, kMaxInt)), dtype, workspace,
                              dev.sm_count, dev.device, static_cast<cudaStream_t>(stream)};
  PagedView view = paged_view(*kv, 2, decode);
  // copies of no bytes, of keys that are masked, name the cache's first address:
  // of a cache without pages, which may have none, another valid one
  if (kv->pages == 0) view.k = view.v = static_cast<char*>(const_cast<void*>(q));
  // Sequences of few query rows go to the split kernel where splitting their
  // keys pays, the others to the tile kernel (AttLoad). The lengths are the
  // device's; the host goes by what it knows, the rows in all and the most keys
  // that the table or the window allow: one kernel for one sequence, for few
  // rows in all that pay at that length, for short tables and for batches of
  // prompts (1024 rows a sequence and more); else both, each on its own
  // sequences (an empty one costs 5 us).
  const size_t rows = tokens * (n_q / kv->n_kv);  // of a kv head, in all
  size_t keys = kv->table_width * kv->page_size;
  if (window > 0) keys = std::min(keys, std::min(window, kMaxInt) + std::min(sinks, kMaxInt) + tokens);
  bool split = decode || tile_heads_per_page(view) == 0, tile = !split;
  if (tile && keys > AttLoad::kLaunch && (kv->batch == 1 ? rows <= kAttFewRows : rows < 1024 * kv->batch)) {
    const size_t row_tiles = kv->batch == 1 ? (rows + 15) / 16 : rows / 16 + std::min(kv->batch, tokens);
    const uint32_t longest = static_cast<uint32_t>(std::min(keys, kMaxInt));
    tile = !(rows <= kAttFewRows && AttLoad{row_tiles * kv->n_kv * longest, longest}.splits());
    split = kv->batch > 1 || !tile;
  }
  cudaError_t e = cudaSuccess;
  if (tile) e = launch_attention_tile(p, view, split);
  if (split && e == cudaSuccess) e = launch_attention_split(p, view, tile);
  return e == cudaSuccess ? CAWQ_OK : cuda_fail(e, "attention launch");
}

}  // namespace cawq

using namespace cawq;

CAWQ_API cawq_status cawq_rms_norm(const void* x, const void* weight, const void* residual,
                                   void* y, void* residual_out, size_t rows, size_t d, size_t ld_x,
                                   size_t ld_residual, size_t ld_y, size_t ld_residual_out,
                                   float eps, cawq_dtype dtype, void* stream) {
  return rms_norm(x, weight, residual, y, nullptr, residual_out, rows, d, ld_x, ld_residual, ld_y,
                  ld_residual_out, eps, dtype, stream);
}

CAWQ_API cawq_status cawq_rms_norm_fp8(const void* x, const void* weight, const void* residual,
                                       void* y8, float* scales, void* residual_out, size_t rows,
                                       size_t d, size_t ld_x, size_t ld_residual, size_t ld_y8,
                                       size_t ld_residual_out, float eps, cawq_dtype dtype,
                                       void* stream) {
  if (rows > 0 && !scales) return fail(CAWQ_ERR_NULL_POINTER, "scales must be non-null");
  return rms_norm(x, weight, residual, y8, scales, residual_out, rows, d, ld_x, ld_residual, ld_y8,
                  ld_residual_out, eps, dtype, stream);
}

CAWQ_API cawq_status cawq_rope_append(const void* q, const void* k, const void* v,
                                      const float* rope, size_t rope_rows, void* q_out,
                                      const cawq_paged_kv* kv, size_t tokens, size_t n_q,
                                      size_t ld_q, size_t ld_k, size_t ld_v, size_t ld_q_out,
                                      cawq_dtype dtype, void* stream) {
  if (dtype != CAWQ_F16 && dtype != CAWQ_BF16)
    return fail(CAWQ_ERR_DTYPE, "the rotary append takes CAWQ_F16 or CAWQ_BF16");
  cawq_status st = check_paged(kv, tokens, n_q);
  if (st != CAWQ_OK) return st;
  if (rope_rows > kMaxInt) return fail(CAWQ_ERR_INVALID_SHAPE, "rope_rows must be below 2^31");
  if (tokens == 0 || kv->batch == 0) return CAWQ_OK;
  const size_t wq = n_q * kv->head_dim, wk = kv->n_kv * kv->head_dim;
  if ((st = check_rows("q", q, &ld_q, wq)) != CAWQ_OK) return st;
  if ((st = check_rows("k", k, &ld_k, wk)) != CAWQ_OK) return st;
  if ((st = check_rows("v", v, &ld_v, wk)) != CAWQ_OK) return st;
  if ((st = check_rows("q_out", q_out, &ld_q_out, wq)) != CAWQ_OK) return st;
  if (rope_rows > 0 && (!rope || !aligned16(rope)))
    return fail(CAWQ_ERR_ALIGNMENT, "rope must be non-null and 16-byte aligned");
  DeviceInfo dev;
  if ((st = require_sm100(&dev)) != CAWQ_OK) return st;
  const RopeProblem p = {q, k, v, rope, q_out, rope_rows, tokens, n_q, kv->head_dim, ld_q, ld_k,
                         ld_v, ld_q_out, dtype, static_cast<cudaStream_t>(stream)};
  const cudaError_t e = launch_rope_append(p, paged_view(*kv, 2, !kv->q_start));
  return e == cudaSuccess ? CAWQ_OK : cuda_fail(e, "rotary append launch");
}

CAWQ_API size_t cawq_attention_workspace(const cawq_paged_kv* kv, size_t tokens, size_t n_q) {
  if (!kv || kv->n_kv == 0 || tokens == 0) return 0;
  return attention_split_workspace(kv->batch, tokens, n_q / kv->n_kv, kv->n_kv,
                                   kv->table_width * kv->page_size, kv->head_dim,
                                   kv->q_start != nullptr);
}

CAWQ_API cawq_status cawq_attention_decode(const void* q, void* out, const cawq_paged_kv* kv,
                                           size_t n_q, size_t ld_q, size_t ld_out, float scale,
                                           size_t window, size_t sinks, cawq_dtype dtype,
                                           void* workspace, size_t workspace_bytes, void* stream) {
  return attention(q, out, kv, kv ? kv->batch : 0, n_q, ld_q, ld_out, scale, window, sinks, dtype,
                   workspace, workspace_bytes, true, stream);
}

CAWQ_API cawq_status cawq_attention_prefill(const void* q, void* out, const cawq_paged_kv* kv,
                                            size_t tokens, size_t n_q, size_t ld_q, size_t ld_out,
                                            float scale, size_t window, size_t sinks,
                                            cawq_dtype dtype, void* workspace,
                                            size_t workspace_bytes, void* stream) {
  return attention(q, out, kv, tokens, n_q, ld_q, ld_out, scale, window, sinks, dtype, workspace,
                   workspace_bytes, false, stream);
}
