// C entries of the 4-bit cache (append, read, decode attention) and of token eviction. Included once, at the end of
// emm_kv.cu, whose contexts, pools and error helpers it uses. Kernels: q4.cuh, attend.cuh, evict.cuh.
#pragma once
#include "attend.cuh"
#include "evict.cuh"
#include "q4.cuh"

namespace {

// Launches, if `early` with programmatic stream serialisation (EMM_OPT_PDL): placed while the kernel before it in the
// stream drains. Every kernel here waits for that one to complete before its first global access.
template <typename... Params, typename... Args>
int launch_after(emm_ctx *ctx, void (*kernel)(Params...), dim3 grid, unsigned block, size_t smem, cudaStream_t st, bool early,
                 const Args &...args) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = early && ctx->pdl ? 1 : 0;
  EMM_CUDA(cudaLaunchKernelEx(&cfg, kernel, args...));
  ctx->launches += 1;
  return EMM_OK;
}

bool q4_dim(int32_t D) { return D == 64 || D == 128 || D == 256; }

// A pool whose rows are 4-bit rows of head_dim channels, in this GPU's memory, every row on a 16-byte boundary.
int check_q4_pool(const emm_pool *p, int32_t head_dim, const char *what) {
  if (!p) return fail(EMM_ERR_BAD_ARG, "%s: null pool", what);
  if (!q4_dim(head_dim)) return fail(EMM_ERR_BAD_ARG, "%s: head dimension %d not in {64, 128, 256}", what, head_dim);
  const emm_pool_desc &d = p->desc;
  if (p->planes != 2 || d.elem_size != 1 || d.head_size != emm::q4_row_bytes(head_dim))
    return fail(EMM_ERR_BAD_ARG, "%s: needs a two-plane pool of bytes with %d bytes per head row, got %d x %d bytes", what,
                emm::q4_row_bytes(head_dim), d.head_size, d.elem_size);
  if (!p->device_local) return fail(EMM_ERR_BAD_ARG, "%s: the pool is not in this GPU's memory", what);
  if (p->align < 16 || d.token_stride % 16 || d.head_stride % 16)
    return fail(EMM_ERR_ALIGN, "%s: rows of the pool must lie on 16-byte boundaries", what);
  return EMM_OK;
}

int check_dtype(int32_t dtype, const char *what) {
  if (dtype != EMM_DTYPE_FP16 && dtype != EMM_DTYPE_BF16)
    return fail(EMM_ERR_BAD_ARG, "%s: dtype %d is neither EMM_DTYPE_FP16 nor EMM_DTYPE_BF16", what, dtype);
  return EMM_OK;
}

constexpr int kSelectSharedMax = 200 * 1024;  // bytes of keys a CTA holds

// log2 of a power of two, else -1.
int32_t shift_of(int32_t v) {
  for (int k = 0; k < 31; ++k)
    if (v == 1 << k) return k;
  return -1;
}

emm::TokenSide token_side(const emm_pool *p) {
  emm::TokenSide s;
  s.layers = p->d_layers;
  s.plane_stride = (uint64_t)p->desc.plane_stride;
  s.block_stride = (uint64_t)p->desc.block_stride;
  s.token_stride = (uint64_t)p->desc.token_stride;
  s.head_stride = (uint64_t)p->desc.head_stride;
  s.num_blocks = (uint32_t)p->desc.num_blocks;
  s.block_size = (uint32_t)p->desc.block_size;
  s.block_shift = shift_of(p->desc.block_size);
  return s;
}

// A single-plane pool of fp32 [NB, H, BS] (accumulated attention weights).
int check_score_pool(const emm_pool *p, const char *what) {
  if (!p) return fail(EMM_ERR_BAD_ARG, "%s: null score pool", what);
  const emm_pool_desc &d = p->desc;
  if (p->planes != 1 || d.elem_size != 4 || p->page_bytes == 0)
    return fail(EMM_ERR_BAD_ARG, "%s: weights are a single-plane pool of fp32 [NB, heads, block size] with dense blocks", what);
  if (!p->device_local) return fail(EMM_ERR_BAD_ARG, "%s: the score pool is not in this GPU's memory", what);
  return EMM_OK;
}

int check_tables(const int32_t *tables, int64_t stride, int32_t width, const int32_t *lens, int32_t B, const char *what) {
  if (B < 0 || width < 0) return fail(EMM_ERR_BAD_ARG, "%s: negative count", what);
  if (B > 0 && (!lens || (width > 0 && !tables))) return fail(EMM_ERR_BAD_ARG, "%s: null pointer", what);
  if (B > 1 && stride < width) return fail(EMM_ERR_BAD_ARG, "%s: table stride smaller than its width", what);
  return EMM_OK;
}

int q4_rows_impl(emm_pool *pool, bool append, int32_t D, int32_t dtype, int32_t layer_begin, int32_t layer_count,
                 const void *key, const void *value, int64_t kls, int64_t kts, int64_t vls, int64_t vts,
                 const int64_t *slots, int32_t T, void *stream) {
  const char *what = append ? "q4_append" : "q4_read";
  if (int rc = check_q4_pool(pool, D, what)) return rc;
  if (int rc = check_dtype(dtype, what)) return rc;
  if (int rc = check_layer_range(pool, layer_begin, layer_count)) return rc;
  if (T < 0) return fail(EMM_ERR_BAD_ARG, "%s: negative token count", what);
  if (T == 0 || layer_count == 0) return EMM_OK;
  if (!key || !value || !slots) return fail(EMM_ERR_BAD_ARG, "%s: null pointer", what);
  const int64_t row = (int64_t)pool->desc.num_kv_heads * D * 2;
  if (kts < row || vts < row)
    return fail(EMM_ERR_BAD_ARG, "%s: token stride smaller than a token row (%lld bytes)", what, (long long)row);
  if (layer_count > 1 && (kls < (int64_t)(T - 1) * kts + row || vls < (int64_t)(T - 1) * vts + row))
    return fail(EMM_ERR_BAD_ARG, "%s: layer stride smaller than one layer of rows", what);
  uint32_t align = 256;
  const uint64_t parts[] = {(uint64_t)key, (uint64_t)value, (uint64_t)kts, (uint64_t)vts,
                            layer_count > 1 ? (uint64_t)kls : 0, layer_count > 1 ? (uint64_t)vls : 0};
  for (uint64_t v : parts) align = std::min(align, pow2_align(v));
  if (align < 2) return fail(EMM_ERR_ALIGN, "%s: key/value not aligned to their elements", what);
  // On 32-byte boundaries (where a projection's output lies) a thread takes a group, else four channels: 4 099 tokens x 32
  // layers x 8 heads written and read back in 252 us, else 966.
  const bool wide = align >= 32;
  const uint64_t rows = (uint64_t)T * (uint64_t)pool->desc.num_kv_heads;
  const uint64_t per_block = wide ? (uint64_t)emm::kRowWarps * (32 / emm::q4_groups(D)) : 256 / (uint64_t)(D / 4);
  const uint64_t blocks = (rows + per_block - 1) / per_block;
  if (rows > 0xffffffffull || blocks > 0x7fffffffull || layer_count > 32767)
    return fail(EMM_ERR_TOO_LARGE, "%s: %d layers x %d tokens", what, layer_count, T);

  emm::Q4RowsArgs a;
  a.pool = token_side(pool);
  a.layer_begin = (uint32_t)layer_begin;
  a.num_tokens = (uint32_t)T;
  a.heads = (uint32_t)pool->desc.num_kv_heads;
  a.key = (uint64_t)key;
  a.value = (uint64_t)value;
  a.key_layer_stride = (uint64_t)kls;
  a.key_token_stride = (uint64_t)kts;
  a.value_layer_stride = (uint64_t)vls;
  a.value_token_stride = (uint64_t)vts;
  a.slots = slots;
  a.status = pool->ctx->d_status;
  DeviceGuard guard(pool->ctx->device);
  if (!guard.ok()) return fail(EMM_ERR_CUDA, "cannot select device %d", pool->ctx->device);
  const dim3 grid((unsigned)blocks, (unsigned)layer_count * 2);
  cudaStream_t st = (cudaStream_t)stream;
  emm_ctx *ctx = pool->ctx;
  const unsigned block = wide ? emm::kRowWarps * 32 : 256;
#define EMM_Q4_ROWS(T_, D_)                                                                                    \
  return append ? launch_after(ctx, wide ? emm::q4_append_rows<T_, D_> : emm::q4_append_units<T_, D_>, grid,   \
                               block, 0, st, true, a)                                                                \
                : launch_after(ctx, wide ? emm::q4_read_rows<T_, D_> : emm::q4_read_units<T_, D_>, grid, block, \
                               0, st, true, a)
  if (dtype == EMM_DTYPE_FP16) {
    if (D == 64) EMM_Q4_ROWS(__half, 64);
    else if (D == 128) EMM_Q4_ROWS(__half, 128);
    else EMM_Q4_ROWS(__half, 256);
  } else {
    if (D == 64) EMM_Q4_ROWS(__nv_bfloat16, 64);
    else if (D == 128) EMM_Q4_ROWS(__nv_bfloat16, 128);
    else EMM_Q4_ROWS(__nv_bfloat16, 256);
  }
#undef EMM_Q4_ROWS
}

// How a call's work is laid out; see attend.cuh. A rule on heads and strides only.
int attend_shape(const emm_pool *pool, int32_t D, int32_t B, int32_t group, int32_t max_len, emm::AttendShape *out,
                 int *smem_out) {
  const emm_pool_desc &d = pool->desc;
  const uint32_t H = (uint32_t)d.num_kv_heads;
  emm::AttendShape s;
  s.ntiles = (uint32_t)(group + 7) / 8;
  // KV heads first (their rows of a token are one copy), in equal shares of at most eight warps, then the tokens of a
  // unit in as many subsets as there are warps left.
  const uint32_t most = std::max(1u, 8u / s.ntiles);
  s.head_groups = (H + most - 1) / most;
  s.heads_cta = (H + s.head_groups - 1) / s.head_groups;
  s.items = (uint32_t)B * s.head_groups;
  const uint64_t sms = (uint64_t)pool->ctx->sm_count;
  s.subsets = std::max(1u, (uint32_t)emm::kAttendWarps / (s.heads_cta * s.ntiles));
  auto units = [&]() {
    const uint32_t tokens = 16 * (uint32_t)emm::attend_tiles(D) * s.subsets;
    return std::max<uint64_t>(1, ((uint64_t)max_len + tokens - 1) / tokens) * s.items;
  };
  // Little work is spread over more, smaller CTAs (577 tokens of one sequence, in a graph: 8.9 us, otherwise 10.0).
  while (s.subsets > 1 && units() < sms) s.subsets /= 2;
  s.tokens = 16 * (uint32_t)emm::attend_tiles(D) * s.subsets;
  s.warps = s.heads_cta * s.ntiles * s.subsets;
  // A tile's offsets within a block take 32 bits.
  s.block_shift = d.token_stride < 1 << 27 && d.block_stride <= 0xffffffffll ? shift_of(d.block_size) : -1;
  s.stages = (uint32_t)emm::attend_stages(D);
  const int merge = (int)((s.subsets - 1) * s.heads_cta * s.ntiles * 8 * (uint32_t)(D + 2) * 4);
  *smem_out = (int)(s.warps * s.stages * (uint32_t)emm::attend_slot_bytes(D)) + merge;
  if (units() + (uint64_t)emm::kItemCost * s.items > 0x7fffffffull)
    return fail(EMM_ERR_TOO_LARGE, "q4_attend: %d sequences of up to %d tokens", B, max_len);
  s.grid = (uint32_t)std::min<uint64_t>(units() + (uint64_t)emm::kItemCost * s.items, sms);
  *out = s;
  return EMM_OK;
}

struct AttendWorkspace {
  uint64_t part_o, part_ml, item_span, cta_item, lse, turns, logits, logit_stride, bytes;
};

AttendWorkspace attend_workspace(const emm::AttendShape &s, int32_t D, int32_t B, int32_t Hq, int32_t group, int32_t max_len,
                                 bool scores) {
  AttendWorkspace w;
  uint64_t at = 0;
  auto take = [&](uint64_t bytes) {
    const uint64_t p = at;
    at += (bytes + 255) / 256 * 256;
    return p;
  };
  const uint64_t rows = 2ull * s.grid * s.heads_cta * (uint32_t)group;
  w.part_o = take(rows * (uint32_t)D * 4);
  w.part_ml = take(rows * 8);
  w.item_span = take((uint64_t)s.items * 8);
  w.cta_item = take((uint64_t)s.grid * 4);
  w.lse = take(scores ? (uint64_t)B * Hq * 4 : 0);
  w.turns = take(scores ? (uint64_t)(B + 1) * 4 : 0);
  w.logit_stride = ((uint64_t)max_len + 7) / 8 * 8;
  w.logits = take(scores ? (uint64_t)B * Hq * w.logit_stride * 4 : 0);
  w.bytes = at;
  return w;
}

// Raises a kernel's dynamic shared memory to the device's limit, once per device. Without it a block's static and dynamic
// shared memory together have 48 KiB, so a kernel whose dynamic part comes near that needs it too.
template <auto kKernel>
int allow_smem(emm_ctx *ctx, int smem, const char *what) {
  const int device = ctx->device;
  static std::atomic<int> limit[kMaxTrackedDevices];
  const bool tracked = device >= 0 && device < kMaxTrackedDevices;
  if (!tracked || limit[device].load(std::memory_order_acquire) < smem) {
    cudaFuncAttributes fa;
    EMM_CUDA(cudaFuncGetAttributes(&fa, kKernel));
    const int most = ctx->max_smem_optin - (int)fa.sharedSizeBytes;
    if (smem > most) return fail(EMM_ERR_TOO_LARGE, "%s: %d bytes of shared memory, the device has %d", what, smem, most);
    EMM_CUDA(cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
    if (tracked) limit[device].store(most, std::memory_order_release);
  }
  return EMM_OK;
}

template <typename T, int D, bool kScores>
int attend_main(emm_ctx *ctx, const emm::AttendArgs &a, int smem, cudaStream_t st) {
  if (int rc = allow_smem<emm::attend_q4<T, D, kScores>>(ctx, smem, "q4_attend")) return rc;
  return launch_after(ctx, emm::attend_q4<T, D, kScores>, dim3(a.sh.grid), a.sh.warps * 32, (size_t)smem, st, true, a);
}

template <typename T, int D>
int attend_launch(emm_ctx *ctx, const emm::AttendArgs &a, int smem, cudaStream_t st) {
  const int rc = a.score_base ? attend_main<T, D, true>(ctx, a, smem, st) : attend_main<T, D, false>(ctx, a, smem, st);
  if (rc) return rc;
  if (a.max_len > a.sh.tokens) {  // else every item is one unit, which no CTA shares
    const bool by_cta = a.sh.items > a.sh.grid;
    const uint32_t rows = a.sh.heads_cta * a.group, x = by_cta ? a.sh.grid : a.sh.items;
    // Few items have many parts each; see attend_join.
    const bool many = x * 8 <= a.sh.grid;
    if (int rc2 = launch_after(ctx, many ? emm::attend_join<T, D, 1> : emm::attend_join<T, D, 8>,
                               dim3(x, many ? rows : (rows + 7) / 8), emm::kJoinWarps * 32, 0, st, true, a, (uint32_t)by_cta))
      return rc2;
  }
  if (a.score_base && a.max_len > 0) {
    const uint32_t chunks = (a.max_len + emm::kScoreTokens - 1) / emm::kScoreTokens;
    const uint64_t turns = (uint64_t)a.num_seqs * a.kv_heads * chunks;
    const unsigned grid = (unsigned)std::min<uint64_t>((turns + 7) / 8, (uint64_t)ctx->sm_count * 6);
    return launch_after(ctx, emm::attend_scores, dim3(grid), 256, 0, st, true, a);
  }
  return EMM_OK;
}

}  // namespace

extern "C" {

int emm_q4_row_bytes(int32_t head_dim) { return q4_dim(head_dim) ? emm::q4_row_bytes(head_dim) : 0; }

int emm_q4_append(emm_pool *pool, int32_t head_dim, int32_t dtype, int32_t layer_begin, int32_t layer_count,
                  const void *d_key, const void *d_value, int64_t key_layer_stride, int64_t key_token_stride,
                  int64_t value_layer_stride, int64_t value_token_stride, const int64_t *d_slot_mapping,
                  int32_t num_tokens, void *stream) {
  return q4_rows_impl(pool, true, head_dim, dtype, layer_begin, layer_count, d_key, d_value, key_layer_stride,
                      key_token_stride, value_layer_stride, value_token_stride, d_slot_mapping, num_tokens, stream);
}

int emm_q4_read(emm_pool *pool, int32_t head_dim, int32_t dtype, int32_t layer_begin, int32_t layer_count, void *d_key,
                void *d_value, int64_t key_layer_stride, int64_t key_token_stride, int64_t value_layer_stride,
                int64_t value_token_stride, const int64_t *d_slot_mapping, int32_t num_tokens, void *stream) {
  return q4_rows_impl(pool, false, head_dim, dtype, layer_begin, layer_count, d_key, d_value, key_layer_stride,
                      key_token_stride, value_layer_stride, value_token_stride, d_slot_mapping, num_tokens, stream);
}

int emm_q4_attend_workspace(emm_pool *pool, int32_t head_dim, int32_t num_seqs, int32_t num_heads, int32_t max_len,
                            int32_t with_scores, uint64_t *bytes) {
  const char *what = "q4_attend_workspace";
  if (!bytes) return fail(EMM_ERR_BAD_ARG, "%s: null argument", what);
  if (int rc = check_q4_pool(pool, head_dim, what)) return rc;
  const int32_t H = pool->desc.num_kv_heads;
  if (num_seqs < 0 || num_heads <= 0 || max_len < 0 || num_heads % H || num_heads / H > EMM_MAX_QUERY_GROUP)
    return fail(EMM_ERR_BAD_ARG, "%s: %d sequences, %d heads, length %d", what, num_seqs, num_heads, max_len);
  emm::AttendShape sh;
  int smem = 0;
  if (int rc = attend_shape(pool, head_dim, num_seqs, num_heads / H, max_len, &sh, &smem)) return rc;
  *bytes = attend_workspace(sh, head_dim, num_seqs, num_heads, num_heads / H, max_len, with_scores != 0).bytes;
  return EMM_OK;
}

int emm_q4_attend(emm_pool *pool, int32_t head_dim, int32_t dtype, int32_t layer, const void *d_query,
                  int64_t query_seq_stride, void *d_out, int64_t out_seq_stride, const int32_t *d_block_tables,
                  int64_t table_stride, int32_t table_width, const int32_t *d_seq_lens, int32_t num_seqs,
                  int32_t num_heads, int32_t max_len, double scale, emm_pool *scores, void *d_workspace,
                  uint64_t workspace_bytes, void *stream) {
  const char *what = "q4_attend";
  if (int rc = check_q4_pool(pool, head_dim, what)) return rc;
  if (int rc = check_dtype(dtype, what)) return rc;
  if (int rc = check_layer_range(pool, layer, 1)) return rc;
  if (int rc = check_tables(d_block_tables, table_stride, table_width, d_seq_lens, num_seqs, what)) return rc;
  const emm_pool_desc &d = pool->desc;
  if (num_heads <= 0 || num_heads % d.num_kv_heads || num_heads / d.num_kv_heads > EMM_MAX_QUERY_GROUP)
    return fail(EMM_ERR_BAD_ARG, "%s: %d query heads on %d KV heads (a multiple of them, at most %d each)", what, num_heads,
                d.num_kv_heads, EMM_MAX_QUERY_GROUP);
  if (max_len < 0 || (int64_t)max_len > (int64_t)table_width * d.block_size)
    return fail(EMM_ERR_LENGTH, "%s: max_len %d needs more than %d blocks of %d tokens", what, max_len, table_width,
                d.block_size);
  if (!(std::fabs(scale) <= 1e38)) return fail(EMM_ERR_BAD_ARG, "%s: the scale is not finite in 32 bits", what);
  if (scores) {
    if (int rc = check_score_pool(scores, what)) return rc;
    if (scores->ctx != pool->ctx) return fail(EMM_ERR_BAD_ARG, "%s: pools of different contexts", what);
    if (scores->desc.num_layers != d.num_layers || scores->desc.num_blocks != d.num_blocks ||
        scores->desc.block_size != d.num_kv_heads || scores->desc.head_size != d.block_size)
      return fail(EMM_ERR_LENGTH, "%s: the score pool must be [%d, %d, %d] in each of %d layers", what, d.num_blocks,
                  d.num_kv_heads, d.block_size, d.num_layers);
  }
  if (num_seqs == 0) return EMM_OK;
  if (!d_query || !d_out) return fail(EMM_ERR_BAD_ARG, "%s: null pointer", what);
  const int64_t row = (int64_t)num_heads * head_dim * 2;
  if (num_seqs > 1 && (query_seq_stride < row || out_seq_stride < row))
    return fail(EMM_ERR_BAD_ARG, "%s: sequence stride smaller than a row of heads (%lld bytes)", what, (long long)row);
  uint32_t align = 256;
  const uint64_t parts[] = {(uint64_t)d_query, (uint64_t)d_out, num_seqs > 1 ? (uint64_t)query_seq_stride : 0,
                            num_seqs > 1 ? (uint64_t)out_seq_stride : 0};
  for (uint64_t v : parts) align = std::min(align, pow2_align(v));
  if (align < 2) return fail(EMM_ERR_ALIGN, "%s: query/out not aligned to their elements", what);
  if ((uint64_t)num_seqs * d.num_kv_heads > 0x7fffffffull) return fail(EMM_ERR_TOO_LARGE, "%s: %d sequences", what, num_seqs);
  const int32_t group = num_heads / d.num_kv_heads;
  emm::AttendArgs a;
  int smem = 0;
  if (int rc = attend_shape(pool, head_dim, num_seqs, group, max_len, &a.sh, &smem)) return rc;
  const AttendWorkspace w = attend_workspace(a.sh, head_dim, num_seqs, num_heads, group, max_len, scores != nullptr);
  if (workspace_bytes < w.bytes || !d_workspace)
    return fail(EMM_ERR_LENGTH, "%s: workspace of %llu bytes, %llu needed", what, (unsigned long long)workspace_bytes,
                (unsigned long long)w.bytes);
  if (pow2_align((uint64_t)d_workspace) < 16) return fail(EMM_ERR_ALIGN, "%s: workspace not on a 16-byte boundary", what);
  const uint64_t ws = (uint64_t)d_workspace;
  a.pool = token_side(pool);
  a.layer_base = pool->h_layers[layer];
  a.query = (uint64_t)d_query;
  a.out = (uint64_t)d_out;
  a.query_seq_stride = (uint64_t)query_seq_stride;
  a.out_seq_stride = (uint64_t)out_seq_stride;
  a.tables = d_block_tables;
  a.table_stride = (uint64_t)table_stride;
  a.lens = d_seq_lens;
  a.num_seqs = (uint32_t)num_seqs;
  a.kv_heads = (uint32_t)d.num_kv_heads;
  a.group = (uint32_t)group;
  a.max_len = (uint32_t)max_len;
  a.scale_log2 = (float)(scale * 1.4426950408889634);
  a.align = align;
  a.score_base = scores ? scores->h_layers[layer] : 0;
  a.score_block_stride = scores ? (uint64_t)scores->desc.block_stride : 0;
  a.part_o = (float *)(ws + w.part_o);
  a.part_ml = (float2 *)(ws + w.part_ml);
  a.item_span = (int2 *)(ws + w.item_span);
  a.cta_item = (int *)(ws + w.cta_item);
  a.lse = (float *)(ws + w.lse);
  a.turns = (uint32_t *)(ws + w.turns);
  a.logits = (float *)(ws + w.logits);
  a.logit_stride = w.logit_stride;
  a.status = pool->ctx->d_status;
  DeviceGuard guard(pool->ctx->device);
  if (!guard.ok()) return fail(EMM_ERR_CUDA, "cannot select device %d", pool->ctx->device);
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == EMM_DTYPE_FP16) {
    if (head_dim == 64) return attend_launch<__half, 64>(pool->ctx, a, smem, st);
    if (head_dim == 128) return attend_launch<__half, 128>(pool->ctx, a, smem, st);
    return attend_launch<__half, 256>(pool->ctx, a, smem, st);
  }
  if (head_dim == 64) return attend_launch<__nv_bfloat16, 64>(pool->ctx, a, smem, st);
  if (head_dim == 128) return attend_launch<__nv_bfloat16, 128>(pool->ctx, a, smem, st);
  return attend_launch<__nv_bfloat16, 256>(pool->ctx, a, smem, st);
}

int emm_select_tokens(emm_pool *scores, const int32_t *d_block_tables, int64_t table_stride, int32_t table_width,
                      const int32_t *d_seq_lens, int32_t num_seqs, int32_t keep, int32_t recent, int32_t sink,
                      int32_t *d_index, int32_t *d_new_lens, void *stream) {
  const char *what = "select_tokens";
  if (int rc = check_score_pool(scores, what)) return rc;
  if (int rc = check_tables(d_block_tables, table_stride, table_width, d_seq_lens, num_seqs, what)) return rc;
  if (keep <= 0 || recent < 0 || sink < 0 || (int64_t)recent + sink > keep)
    return fail(EMM_ERR_BAD_ARG, "%s: keep %d must be positive and cover recent %d + sink %d", what, keep, recent, sink);
  if (num_seqs == 0) return EMM_OK;
  if (!d_index || !d_new_lens) return fail(EMM_ERR_BAD_ARG, "%s: null pointer", what);
  const emm_pool_desc &d = scores->desc;
  if ((uint64_t)num_seqs * d.block_size > 0x7fffffffull || d.num_layers > 65535 ||
      (int64_t)table_width * d.head_size > 0x7fffffffll)
    return fail(EMM_ERR_TOO_LARGE, "%s: %d layers x %d sequences of %d blocks", what, d.num_layers, num_seqs, table_width);
  emm::SelectArgs a;
  a.layers = scores->d_layers;
  a.block_stride = (uint64_t)d.block_stride;
  a.num_blocks = (uint32_t)d.num_blocks;
  a.block_size = (uint32_t)d.head_size;
  a.block_shift = shift_of(d.head_size);
  a.tables = d_block_tables;
  a.table_stride = (uint64_t)table_stride;
  a.table_width = (uint32_t)table_width;
  a.lens = d_seq_lens;
  a.num_seqs = (uint32_t)num_seqs;
  a.heads = (uint32_t)d.block_size;
  a.keep = (uint32_t)keep;
  a.recent = (uint32_t)recent;
  a.sink = (uint32_t)sink;
  a.index = d_index;
  a.new_lens = d_new_lens;
  a.status = scores->ctx->d_status;
  DeviceGuard guard(scores->ctx->device);
  if (!guard.ok()) return fail(EMM_ERR_CUDA, "cannot select device %d", scores->ctx->device);
  const dim3 grid((unsigned)num_seqs * (unsigned)d.block_size, (unsigned)d.num_layers);
  const int64_t most = (int64_t)table_width * d.head_size;
  cudaStream_t st = (cudaStream_t)stream;
  emm_ctx *ctx = scores->ctx;
  // Keys that do not fit shared memory are read again in each pass (8 sequences x 32 layers of 4 096: 795 instead of 748 us).
  if (most * 4 > kSelectSharedMax) return launch_after(ctx, emm::select_tokens<1024, false>, grid, 1024, 0, st, true, a);
  const size_t keys = (size_t)most * 4;
  // Small CTAs where a thread has at most 16 keys: eight CTAs share an SM then, and one's barriers hide behind the others'
  // (2 048 CTAs of 3 000-4 096 keys: 61 us, with 1 024 threads 76; 10 000 keys: 1 024 threads 11 us faster than 256).
  if (most <= 4096) return launch_after(ctx, emm::select_tokens<256, true>, grid, 256, keys, st, true, a);
  if (int rc = allow_smem<emm::select_tokens<1024, true>>(ctx, (int)keys, what)) return rc;
  return launch_after(ctx, emm::select_tokens<1024, true>, grid, 1024, keys, st, true, a);
}

int emm_keep_tokens(emm_pool *pool, const int32_t *d_index, int32_t index_heads, int32_t keep,
                    const int32_t *d_block_tables, int64_t table_stride, int32_t table_width, const int32_t *d_seq_lens,
                    int32_t num_seqs, void *stream) {
  const char *what = "keep_tokens";
  if (!pool) return fail(EMM_ERR_BAD_ARG, "%s: null pool", what);
  if (int rc = check_tables(d_block_tables, table_stride, table_width, d_seq_lens, num_seqs, what)) return rc;
  if (!pool->device_local) return fail(EMM_ERR_BAD_ARG, "%s: the pool is not in this GPU's memory", what);
  if (keep <= 0) return fail(EMM_ERR_BAD_ARG, "%s: keep %d must be positive", what, keep);
  const emm_pool_desc &d = pool->desc;
  emm::KeepArgs a;
  a.pool = token_side(pool);
  if (pool->planes == 1) {
    // A score pool [NB, H, BS]: a token's row of a head is one element.
    if (int rc = check_score_pool(pool, what)) return rc;
    a.heads = (uint32_t)d.block_size;
    a.row_bytes = (uint32_t)d.elem_size;
    a.pool.block_size = (uint32_t)d.head_size;
    a.pool.block_shift = shift_of(d.head_size);
    a.pool.token_stride = (uint64_t)d.elem_size;
    a.pool.head_stride = (uint64_t)d.token_stride;
  } else {
    a.heads = (uint32_t)d.num_kv_heads;
    a.row_bytes = (uint32_t)(d.head_size * d.elem_size);
  }
  if (index_heads != (int32_t)a.heads)
    return fail(EMM_ERR_LENGTH, "%s: index of %d heads, the pool has %u", what, index_heads, a.heads);
  if (num_seqs == 0) return EMM_OK;
  if (!d_index) return fail(EMM_ERR_BAD_ARG, "%s: null pointer", what);
  if ((uint64_t)num_seqs * a.heads * pool->planes > 0x1fffffffull || d.num_layers > 65535 ||
      (int64_t)table_width * a.pool.block_size > 0x7fffffffll)
    return fail(EMM_ERR_TOO_LARGE, "%s: %d layers x %d sequences of %d blocks", what, d.num_layers, num_seqs, table_width);
  a.planes = (uint32_t)pool->planes;
  a.tables = d_block_tables;
  a.table_stride = (uint64_t)table_stride;
  a.table_width = (uint32_t)table_width;
  a.lens = d_seq_lens;
  a.num_seqs = (uint32_t)num_seqs;
  a.keep = (uint32_t)keep;
  a.index = d_index;
  a.status = pool->ctx->d_status;
  uint32_t align = pow2_align(a.row_bytes);
  for (uint64_t p : pool->h_layers) align = std::min(align, pow2_align(p));
  const uint64_t strides[] = {a.pool.plane_stride, a.pool.block_stride, a.pool.token_stride, a.pool.head_stride};
  for (uint64_t v : strides) align = std::min(align, pow2_align(v));
  DeviceGuard guard(pool->ctx->device);
  if (!guard.ok()) return fail(EMM_ERR_CUDA, "cannot select device %d", pool->ctx->device);
  // Two or four CTAs share a row, down to 64 bytes each, where all still fit the GPU at once (four an SM): a CTA's rows
  // come one chunk after the other, so few CTAs cannot keep HBM busy (20 000 -> 10 000 tokens, 4 heads: 4 layers 134
  // instead of 200 us, 16 layers 210 instead of 384).
  a.splits = 1;
  const uint64_t ctas = (uint64_t)num_seqs * a.heads * a.planes * (uint64_t)d.num_layers;
  while (a.splits < 4 && ctas * a.splits * 2 <= 4ull * pool->ctx->sm_count && a.row_bytes % 32 == 0 && a.row_bytes / 2 >= 64) {
    a.splits *= 2;
    a.row_bytes /= 2;
    align = std::min(align, pow2_align(a.row_bytes));
  }
  const dim3 grid((unsigned)num_seqs * a.heads * a.planes * a.splits, (unsigned)d.num_layers);
  cudaStream_t st = (cudaStream_t)stream;
  const uint32_t vec = std::min(align, 16u);
  // 32-bit positions and shifts: 8 sequences x 32 layers in 747 us, with 64 bits and divisions 2 008.
  const bool plain = a.row_bytes / vec <= (uint32_t)emm::kKeepThreads && a.pool.block_shift >= 0 &&
                     std::max(a.pool.block_stride, a.pool.token_stride) <= 0xffffffffull &&
                     (uint64_t)keep < (1ull << 31) - 64 * emm::kKeepThreads;
  emm_ctx *ctx = pool->ctx;
  // CTAs placed while the kernel before them drains are not spread evenly over the SMs. Where they are few, with long
  // chains, that costs more than the start it saves (4 layers: 118 us, and 89 behind a finished kernel).
  const bool early = ctas * a.splits >= 4ull * ctx->sm_count || (uint64_t)keep * a.row_bytes <= 128 * 1024;
#define EMM_KEEP(V_)                                                                                                    \
  return launch_after(ctx, plain ? emm::keep_rows<V_, true> : emm::keep_rows<V_, false>, grid, emm::kKeepThreads, 0, st, \
                      early, a)
  if (vec >= 16) EMM_KEEP(uint4);
  if (vec >= 8) EMM_KEEP(uint2);
  if (vec >= 4) EMM_KEEP(uint32_t);
  if (vec >= 2) EMM_KEEP(uint16_t);
  EMM_KEEP(uint8_t);
#undef EMM_KEEP
}

int emm_reset_scores(emm_pool *scores, const int64_t *d_slot_mapping, int32_t num_tokens, void *stream) {
  const char *what = "reset_scores";
  if (int rc = check_score_pool(scores, what)) return rc;
  if (num_tokens < 0) return fail(EMM_ERR_BAD_ARG, "%s: negative token count", what);
  if (num_tokens == 0) return EMM_OK;
  if (!d_slot_mapping) return fail(EMM_ERR_BAD_ARG, "%s: null pointer", what);
  const emm_pool_desc &d = scores->desc;
  const uint64_t total = (uint64_t)num_tokens * (uint64_t)d.block_size;
  const uint64_t blocks = (total + 255) / 256;
  if (blocks > 0x7fffffffull || d.num_layers > 65535) return fail(EMM_ERR_TOO_LARGE, "%s: %d tokens", what, num_tokens);
  DeviceGuard guard(scores->ctx->device);
  if (!guard.ok()) return fail(EMM_ERR_CUDA, "cannot select device %d", scores->ctx->device);
  return launch_after(scores->ctx, emm::reset_scores, dim3((unsigned)blocks, (unsigned)d.num_layers), 256, 0,
                      (cudaStream_t)stream, true, (const uint64_t *)scores->d_layers, (uint64_t)d.block_stride, (uint32_t)d.num_blocks,
                      (uint32_t)d.head_size, (uint32_t)d.block_size, d_slot_mapping, (uint64_t)num_tokens, scores->ctx->d_status);
}

}  // extern "C"
