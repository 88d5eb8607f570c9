// Host side of the attention operators: argument checks and launches.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdint>
#include <utility>

#include "../../include/svdmlp.h"
#include "attention_sm100.cuh"
#include "host.h"
#include "rope_pages.cuh"

namespace svdmlp {

static bool dtype_ok(int dtype) { return dtype == SVDMLP_BF16 || dtype == SVDMLP_F16; }

// Base and strides (elements of 2 bytes) on 16-byte boundaries.
static bool rows_aligned(const void* p, int64_t token, int64_t head) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && token % 8 == 0 && head % 8 == 0;
}

static bool elems_aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 1u) == 0; }

// A launch that may overlap the previous kernel on the stream: each of these
// kernels waits on the device (griddepcontrol.wait) before it reads or writes
// anything, and lets its own successor launch at once.
template <typename... Params, typename... Args>
static int launch_overlapped(void (*kernel)(Params...), dim3 grid, int threads, size_t smem, cudaStream_t s, Args&&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  SVD_CUDA(cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...));
  count_launch();
  return SVDMLP_OK;
}

// --------------------------------------------------------------------- rope
template <typename T, int E>
static int launch_rope(const RopeParams& p, bool interleaved, cudaStream_t s) {
  const int grid = (p.tokens + p.tile - 1) / p.tile;
  const size_t smem = static_cast<size_t>(p.tile) * p.half * sizeof(float2);
  return interleaved ? launch_overlapped(rope_kernel<T, E, true>, dim3(grid), kRopeThreads, smem, s, p)
                     : launch_overlapped(rope_kernel<T, E, false>, dim3(grid), kRopeThreads, smem, s, p);
}

static int rope_impl(const svdmlp_rope_args* a, cudaStream_t s) {
  if (!a || !a->q || !a->k || !a->positions || !a->inv_freq || !a->q_out) return SVDMLP_ERR_INVALID_VALUE;
  if (a->tokens <= 0 || a->q_heads <= 0 || a->kv_heads <= 0 || a->head_dim <= 0) return SVDMLP_ERR_INVALID_VALUE;
  if (!dtype_ok(a->dtype)) return SVDMLP_ERR_DTYPE;
  if (a->rotary_dim <= 0 || a->rotary_dim % 2 != 0 || a->rotary_dim > a->head_dim || a->head_dim > 512)
    return SVDMLP_ERR_SHAPE_MISMATCH;
  if (!std::isfinite(a->scale)) return SVDMLP_ERR_INVALID_VALUE;
  if ((a->k_cache == nullptr) != (a->v_cache == nullptr)) return SVDMLP_ERR_INVALID_VALUE;
  const bool cached = a->k_cache != nullptr;
  if (!cached && !a->k_out) return SVDMLP_ERR_INVALID_VALUE;
  if (cached && (!a->v || !a->slots || a->block_size <= 0 || a->num_blocks <= 0)) return SVDMLP_ERR_INVALID_VALUE;
  if (cached) {
    const int64_t inside = static_cast<int64_t>(a->kv_heads) * a->block_size * a->head_dim;
    if (a->k_block < inside || a->v_block < inside) return SVDMLP_ERR_SHAPE_MISMATCH;
  }
  RopeParams p{};
  p.tokens = a->tokens;
  p.q_heads = a->q_heads;
  p.kv_heads = a->kv_heads;
  p.head_dim = a->head_dim;
  p.half = a->rotary_dim / 2;
  p.block_size = a->block_size;
  p.scale = a->scale;
  p.q = a->q;
  p.k = a->k;
  p.v = a->v;
  p.q_token = a->q_token;
  p.q_head = a->q_head;
  p.k_token = a->k_token;
  p.k_head = a->k_head;
  p.v_token = a->v_token;
  p.v_head = a->v_head;
  p.positions = a->positions;
  p.slots = reinterpret_cast<const long long*>(a->slots);
  p.inv_freq = a->inv_freq;
  p.q_out = a->q_out;
  p.k_out = a->k_out;
  p.k_cache = a->k_cache;
  p.v_cache = a->v_cache;
  p.k_block = a->k_block;
  p.v_block = a->v_block;
  p.cache_slots = static_cast<long long>(a->block_size) * a->num_blocks;
  bool vec = p.half % 8 == 0 && p.head_dim % 8 == 0 && rows_aligned(p.q, p.q_token, p.q_head) &&
             rows_aligned(p.k, p.k_token, p.k_head) && rows_aligned(p.q_out, 0, 0) && rows_aligned(p.k_out, 0, 0);
  if (cached)
    vec = vec && rows_aligned(p.v, p.v_token, p.v_head) && rows_aligned(p.k_cache, p.k_block, 0) &&
          rows_aligned(p.v_cache, p.v_block, 0);
  if (!elems_aligned(p.q) || !elems_aligned(p.k) || !elems_aligned(p.v) || !elems_aligned(p.q_out) ||
      !elems_aligned(p.k_out) || !elems_aligned(p.k_cache) || !elems_aligned(p.v_cache))
    return SVDMLP_ERR_ALIGNMENT;
  const int e = vec ? 8 : 1;
  p.rot_units = p.half / e;
  p.head_units = p.rot_units + (p.head_dim - 2 * p.half) / e;
  p.v_units = p.head_dim / e;
  // fewer tokens per CTA where the tokens would not fill the SMs several times over
  p.tile = std::max(1, std::min(kRopeTile, a->tokens / (4 * planning_sms())));
  const bool inter = a->interleaved != 0;
  if (a->dtype == SVDMLP_BF16)
    return vec ? launch_rope<__nv_bfloat16, 8>(p, inter, s) : launch_rope<__nv_bfloat16, 1>(p, inter, s);
  return vec ? launch_rope<__half, 8>(p, inter, s) : launch_rope<__half, 1>(p, inter, s);
}

// -------------------------------------------------------------------- pages
static int pages_impl(const svdmlp_pages_args* a, cudaStream_t s) {
  if (!a || !a->table || !a->held || !a->added || !a->free_count || !a->cu || !a->lens || !a->count_out || !a->missing)
    return SVDMLP_ERR_INVALID_VALUE;
  if (a->batch <= 0 || a->tokens < 0 || a->block_size <= 0 || a->table_width <= 0 || a->free_capacity < 0)
    return SVDMLP_ERR_INVALID_VALUE;
  if (a->ld_table < a->table_width) return SVDMLP_ERR_SHAPE_MISMATCH;
  if ((a->tokens > 0 && (!a->slots || !a->positions)) || (a->free_capacity > 0 && !a->free_blocks))
    return SVDMLP_ERR_INVALID_VALUE;
  PagesParams p{};
  p.batch = a->batch;
  p.tokens = a->tokens;
  p.block_size = a->block_size;
  p.width = a->table_width;
  p.capacity = a->free_capacity;
  p.table = a->table;
  p.ld_table = a->ld_table;
  p.held = a->held;
  p.added = a->added;
  p.free_blocks = a->free_blocks;
  p.free_count = a->free_count;
  p.slots = reinterpret_cast<long long*>(a->slots);
  p.positions = a->positions;
  p.cu = a->cu;
  p.lens = a->lens;
  p.count_out = a->count_out;
  p.missing = a->missing;
  const int grid = std::max(1, std::min(planning_sms(), (a->tokens + kPagesThreads - 1) / kPagesThreads));
  return launch_overlapped(page_step_kernel, dim3(grid), kPagesThreads, 0, s, p);
}

// ---------------------------------------------------------------- attention
static int check_heads(int dtype, int q_heads, int kv_heads, int head_dim, float scale) {
  if (q_heads <= 0 || kv_heads <= 0) return SVDMLP_ERR_INVALID_VALUE;
  if (!dtype_ok(dtype)) return SVDMLP_ERR_DTYPE;
  if (q_heads % kv_heads != 0 || (head_dim != 64 && head_dim != 128)) return SVDMLP_ERR_SHAPE_MISMATCH;
  if (!std::isfinite(scale)) return SVDMLP_ERR_INVALID_VALUE;
  return SVDMLP_OK;
}

// ------------------------------------------------------------- tensor maps
static int attn_map(CUtensorMap* map, int dtype, const void* base, int rank, const int64_t* dims, const int64_t* strides,
                    const int* box) {
  auto fn = encode_fn();
  if (!fn) return cuda_fail(cudaErrorInitializationError);
  cuuint64_t d[5], st[5];
  cuuint32_t b[5], one[5] = {1, 1, 1, 1, 1};
  for (int i = 0; i < rank; ++i) {
    d[i] = static_cast<cuuint64_t>(dims[i]);
    b[i] = static_cast<cuuint32_t>(box[i]);
    if (i > 0) st[i - 1] = static_cast<cuuint64_t>(strides[i] * 2);
  }
  const CUresult r =
      fn(map, dtype == SVDMLP_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
         static_cast<cuuint32_t>(rank), const_cast<void*>(base), d, st, b, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? SVDMLP_OK : SVDMLP_ERR_ALIGNMENT;
}

// The query heads that share a key/value head lie in one tile, up to 64 of them.
static int pack_of(int group) { return group <= 64 ? group : 1; }

static int query_map(CUtensorMap* map, int dtype, const void* q, int tokens, int q_heads, int head_dim, int gp,
                     int64_t token, int64_t head) {
  const int64_t dims[4] = {head_dim, gp, q_heads / gp, tokens}, strides[4] = {1, head, head * gp, token};
  const int box[4] = {64, gp, 1, 128 / gp};
  return attn_map(map, dtype, q, 4, dims, strides, box);
}

// ------------------------------------------------------------------- launch
static constexpr int64_t kAttnCtlBytes = 256, kAttnCounterBytes = 1 << 20;  // as svdmlp_workspace_init lays them out
static constexpr int64_t kAttnSplitBytes = 2 * kAttnMaxGrid * sizeof(AttnSplit);

template <int D>
static int64_t attn_workspace() {
  return kAttnCtlBytes + kAttnCounterBytes + kAttnSplitBytes +
         static_cast<int64_t>(std::min(planning_sms(), kAttnMaxGrid)) * 2 * AttnCfg<D, true>::PART_FLOATS * 4;
}

template <typename T, int D, bool PAGED, bool PAIR>
static int launch_attention(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const AttnParams& p,
                            int grid, int join_rows, cudaStream_t s) {
  constexpr int SMEM = AttnCfg<D, PAIR>::SMEM_BYTES;
  static std::atomic<uint64_t> ready{0};  // devices whose shared-memory limit is set
  int dev = 0;
  SVD_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || !(ready.load() >> dev & 1)) {
    SVD_CUDA(cudaFuncSetAttribute(attention_kernel<T, D, PAGED, PAIR>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
    if (dev < 64) ready.fetch_or(1ull << dev);
  }
  SVD_CHECK(launch_overlapped(attention_kernel<T, D, PAGED, PAIR>, dim3(grid), kAttnThreads, SMEM, s, q, k, v, p));
  if (join_rows == 0) return SVDMLP_OK;
  constexpr int PER = PAIR ? 32 : kJoinThreads / 32 * (128 / D);
  return launch_overlapped(attention_join_kernel<T, D, PAIR>, dim3(grid * AttnCfg<D, PAIR>::WORKERS, (join_rows + PER - 1) / PER),
                           kJoinThreads, 0, s, p);
}

template <bool PAGED, bool PAIR>
static int dispatch_attention(int dtype, int head_dim, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v,
                              const AttnParams& p, int grid, int join_rows, cudaStream_t s) {
  if (dtype == SVDMLP_BF16)
    return head_dim == 128 ? launch_attention<__nv_bfloat16, 128, PAGED, PAIR>(q, k, v, p, grid, join_rows, s)
                           : launch_attention<__nv_bfloat16, 64, PAGED, PAIR>(q, k, v, p, grid, join_rows, s);
  return head_dim == 128 ? launch_attention<__half, 128, PAGED, PAIR>(q, k, v, p, grid, join_rows, s)
                         : launch_attention<__half, 64, PAGED, PAIR>(q, k, v, p, grid, join_rows, s);
}

// Units of up to so many keys are not divided: partials and the join cost more
// than the uneven end (measured, us).  Prompts, 512 / 1024 keys: 8 requests of
// 100 to 600 tokens 35.7 / 29.6, 16 of 400 47.9 / 38.  Trees, 512 / 256: 64
// requests of one token on some 800 keys 88 / 84, 8 on 2000 26 / 21.
static constexpr int kPromptSnap = 1024, kTreeSnap = 256;

// Keys per step.
static int attn_step(bool pair) { return pair ? AttnCfg<128, true>::STEP : AttnCfg<128, false>::STEP; }

// What both attentions set alike.
template <typename Args>
static void common_params(AttnParams* p, const Args* a, int q_tokens) {
  p->batch = a->batch;
  p->q_tokens = q_tokens;
  p->group = a->q_heads / a->kv_heads;
  p->gp = pack_of(p->group);
  p->head_groups = a->q_heads / p->gp;
  p->tt = 128 / p->gp;
  // a zero scale would turn masked scores (-inf) into NaN; the smallest one gives the same weights
  p->c = std::max(std::fabs(a->scale) * 1.4426950408889634f, 1e-30f);
  p->neg = a->scale < 0;
  p->cu_q = a->cu_q;
  p->q = a->q;
  p->q_token = a->q_token;
  p->q_head = a->q_head;
  p->out = a->out;
  p->out_token = a->out_token;
  p->out_head = a->out_head;
  uint8_t* ws = static_cast<uint8_t*>(a->workspace);
  p->err = reinterpret_cast<int*>(ws);
  p->splits = reinterpret_cast<AttnSplit*>(ws + kAttnCtlBytes + kAttnCounterBytes);
  p->partials = reinterpret_cast<float*>(ws + kAttnCtlBytes + kAttnCounterBytes + kAttnSplitBytes);
  p->timeout_ns = wait_limit_ns();
}

// One CTA per SM, or fewer where there cannot be work for all: at most `tokens`
// rows in `batch` requests, of at most `keys` keys each.  join_rows: rows of a
// unit that the join has to expect, 0 where no unit can be divided.
static int attn_grid(const AttnParams& p, bool pair, int64_t tokens, int64_t keys, int64_t unit_rows, int* grid,
                     int* join_rows) {
  SVD_CHECK(device_sms(grid));
  *grid = std::min(*grid, kAttnMaxGrid);
  const int64_t units = (tokens / (pair ? 2 * p.tt : p.tt) + p.batch) * p.head_groups;
  const int64_t steps = (keys + attn_step(pair) - 1) / attn_step(pair);
  const int64_t workers = units * (steps <= p.snap ? 1 : steps);
  *grid = static_cast<int>(std::min<int64_t>(*grid, pair ? workers : (workers + 1) / 2));
  *join_rows = steps <= p.snap ? 0 : static_cast<int>(std::min<int64_t>(unit_rows, pair ? 256 : 128));
  return SVDMLP_OK;
}

static int prompt_impl(const svdmlp_prompt_args* a, cudaStream_t s) {
  if (!a || !a->q || !a->k || !a->v || !a->cu_q || !a->cu_k || !a->out) return SVDMLP_ERR_INVALID_VALUE;
  if (a->batch <= 0 || a->q_tokens <= 0 || a->k_tokens <= 0) return SVDMLP_ERR_INVALID_VALUE;
  SVD_CHECK(check_heads(a->dtype, a->q_heads, a->kv_heads, a->head_dim, a->scale));
  if (!rows_aligned(a->q, a->q_token, a->q_head) || !rows_aligned(a->k, a->k_token, a->k_head) ||
      !rows_aligned(a->v, a->v_token, a->v_head) || !rows_aligned(a->out, a->out_token, a->out_head))
    return SVDMLP_ERR_ALIGNMENT;
  if (!a->workspace || (reinterpret_cast<uintptr_t>(a->workspace) & 255u) != 0) return SVDMLP_ERR_INVALID_VALUE;
  if (a->workspace_bytes < svdmlp_prompt_workspace_bytes()) return SVDMLP_ERR_WORKSPACE;
  AttnParams p{};
  common_params(&p, a, a->q_tokens);
  p.k_tokens = a->k_tokens;
  p.causal = a->causal != 0;
  // Two row tiles that share their keys pay once the key walks are long; shorter
  // requests gain more from two independent workers (measured, us, pair / solo:
  // 16 heads of 64, 16 sequences of 400 tokens 46.5 / 40.2, 8 of 1024 59.4 / 55.6,
  // 6 of 1300 79.8 / 71.7, 4 of 2000 89.5 / 92.0; 32 and 8 heads of 128, 16 of 400
  // 82.4 / 65.1, 8 of 512 58.0 / 52.0, 4 of 1300 107.8 / 104.7, 4 of 1500
  // 123.7 / 131.2, 2 of 2000 102.2 / 121.4).  At most 128 rows leave the second
  // tile empty.
  const bool pair =
      static_cast<int64_t>(a->q_tokens) * p.gp > 128ll * a->batch && a->k_tokens >= 1400ll * a->batch;
  p.cu_k = a->cu_k;
  p.k = a->k;
  p.v = a->v;
  p.k_token = a->k_token;
  p.k_head = a->k_head;
  p.v_token = a->v_token;
  p.v_head = a->v_head;
  const int step = attn_step(pair), box[3] = {64, 1, step};
  p.snap = kPromptSnap / step;
  int grid = 0, join_rows = 0;
  SVD_CHECK(attn_grid(p, pair, a->q_tokens, a->k_tokens, static_cast<int64_t>(a->q_tokens) * p.gp, &grid, &join_rows));
  CUtensorMap mq, mk, mv;
  SVD_CHECK(query_map(&mq, a->dtype, a->q, a->q_tokens, a->q_heads, a->head_dim, p.gp, a->q_token, a->q_head));
  const int64_t dims[3] = {a->head_dim, a->kv_heads, a->k_tokens};
  const int64_t ks[3] = {1, a->k_head, a->k_token}, vs[3] = {1, a->v_head, a->v_token};
  SVD_CHECK(attn_map(&mk, a->dtype, a->k, 3, dims, ks, box));
  SVD_CHECK(attn_map(&mv, a->dtype, a->v, 3, dims, vs, box));
  return pair ? dispatch_attention<false, true>(a->dtype, a->head_dim, mq, mk, mv, p, grid, join_rows, s)
              : dispatch_attention<false, false>(a->dtype, a->head_dim, mq, mk, mv, p, grid, join_rows, s);
}

static int tree_impl(const svdmlp_tree_args* a, cudaStream_t s) {
  if (!a || !a->q || !a->k_cache || !a->v_cache || !a->table || !a->lens || !a->cu_q || !a->out)
    return SVDMLP_ERR_INVALID_VALUE;
  if (a->batch <= 0 || a->tokens <= 0 || a->num_blocks <= 0 || a->table_width <= 0 || a->max_tree <= 0)
    return SVDMLP_ERR_INVALID_VALUE;
  SVD_CHECK(check_heads(a->dtype, a->q_heads, a->kv_heads, a->head_dim, a->scale));
  if (a->block_size < 8 || a->block_size > 1024 || (a->block_size & (a->block_size - 1)) != 0)
    return SVDMLP_ERR_SHAPE_MISMATCH;
  if (a->mask && a->max_tree > 64) return SVDMLP_ERR_SHAPE_MISMATCH;  // a row's mask has a bit for each of 64 tokens
  const int64_t inside = static_cast<int64_t>(a->kv_heads) * a->block_size * a->head_dim;
  if (a->k_block < inside || a->v_block < inside || a->ld_table < a->table_width) return SVDMLP_ERR_SHAPE_MISMATCH;
  if (!rows_aligned(a->q, a->q_token, a->q_head) || !rows_aligned(a->k_cache, a->k_block, 0) ||
      !rows_aligned(a->v_cache, a->v_block, 0) || !rows_aligned(a->out, a->out_token, a->out_head))
    return SVDMLP_ERR_ALIGNMENT;
  if (!a->workspace || (reinterpret_cast<uintptr_t>(a->workspace) & 255u) != 0) return SVDMLP_ERR_INVALID_VALUE;
  if (a->workspace_bytes < svdmlp_tree_workspace_bytes(a->head_dim)) return SVDMLP_ERR_WORKSPACE;
  AttnParams p{};
  common_params(&p, a, a->tokens);
  p.tree = 1;
  const bool pair = static_cast<int64_t>(a->max_tree) * p.gp > 128;
  p.lens = a->lens;
  p.table = a->table;
  p.mask = reinterpret_cast<const long long*>(a->mask);
  p.ld_table = a->ld_table;
  p.block_size = a->block_size;
  for (p.block_shift = 0; (1 << p.block_shift) < a->block_size;) ++p.block_shift;
  p.num_blocks = a->num_blocks;
  p.width = a->table_width;
  p.k = a->k_cache;
  p.v = a->v_cache;
  p.k_token = a->k_block;
  p.v_token = a->v_block;
  const int step = attn_step(pair), box[4] = {64, std::min(a->block_size, step), 1, 1};
  p.snap = kTreeSnap / step;
  int grid = 0, join_rows = 0;
  SVD_CHECK(attn_grid(p, pair, a->tokens, static_cast<int64_t>(a->table_width) * a->block_size,
                      pair ? 256 : static_cast<int64_t>(a->max_tree) * p.gp, &grid, &join_rows));
  CUtensorMap mq, mk, mv;
  SVD_CHECK(query_map(&mq, a->dtype, a->q, a->tokens, a->q_heads, a->head_dim, p.gp, a->q_token, a->q_head));
  const int64_t dims[4] = {a->head_dim, a->block_size, a->kv_heads, a->num_blocks};
  const int64_t head = static_cast<int64_t>(a->block_size) * a->head_dim;
  const int64_t ks[4] = {1, a->head_dim, head, a->k_block}, vs[4] = {1, a->head_dim, head, a->v_block};
  SVD_CHECK(attn_map(&mk, a->dtype, a->k_cache, 4, dims, ks, box));
  SVD_CHECK(attn_map(&mv, a->dtype, a->v_cache, 4, dims, vs, box));
  return pair ? dispatch_attention<true, true>(a->dtype, a->head_dim, mq, mk, mv, p, grid, join_rows, s)
              : dispatch_attention<true, false>(a->dtype, a->head_dim, mq, mk, mv, p, grid, join_rows, s);
}

}  // namespace svdmlp

extern "C" {

int svdmlp_rope(const svdmlp_rope_args* args, void* stream) {
  return svdmlp::rope_impl(args, static_cast<cudaStream_t>(stream));
}

int svdmlp_page_step(const svdmlp_pages_args* args, void* stream) {
  return svdmlp::pages_impl(args, static_cast<cudaStream_t>(stream));
}

int64_t svdmlp_prompt_workspace_bytes(void) { return svdmlp::attn_workspace<128>(); }

int svdmlp_prompt_attention(const svdmlp_prompt_args* args, void* stream) {
  return svdmlp::prompt_impl(args, static_cast<cudaStream_t>(stream));
}

int64_t svdmlp_tree_workspace_bytes(int32_t head_dim) {
  if (head_dim != 64 && head_dim != 128) return SVDMLP_ERR_SHAPE_MISMATCH;
  return head_dim == 128 ? svdmlp::attn_workspace<128>() : svdmlp::attn_workspace<64>();
}

int svdmlp_tree_attention(const svdmlp_tree_args* args, void* stream) {
  return svdmlp::tree_impl(args, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
