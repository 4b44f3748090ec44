// Entry points of the attention operators: checks of the arguments (host only, before any CUDA call), the description of the
// problem, and the choice of the kernel.
#include "attention_common.cuh"
#include "call_checks.cuh"

#include <cmath>

namespace tops {

long long attention_tiles(const AttentionProblem& p, int rows_per_tile) {
    if (!p.page_table) {
        const long long rows = (long long)p.queries * p.group;
        return (long long)p.batch * ((rows + rows_per_tile - 1) / rows_per_tile);
    }
    // each sequence adds at most one partly filled tile, and only if it has a token
    return (long long)p.queries * p.group / rows_per_tile + (p.batch < p.queries ? p.batch : p.queries);
}

int attention_splits(const AttentionProblem& p, long long tiles, int blocks_wanted, int step) {
    long long keys = p.keys;
    if (p.window > 0 && keys > p.window) keys = p.window;
    const long long blocks = tiles * p.kv_heads;
    int splits = 1;
    while (splits < 8 && blocks * splits < blocks_wanted && keys >= (long long)step * splits * 2) splits *= 2;
    return splits;
}

bool launch_attention(const void* kernel, const AttentionProblem& p, int rows_per_tile, int threads, size_t smem, int splits, void** args, const char* name) {
    if (!ensure_dynamic_smem(kernel, smem)) return false;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)splits;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(attention_tiles(p, rows_per_tile) * splits), (unsigned)p.kv_heads);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = current_stream();
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return check_cuda(cudaLaunchKernelExC(&cfg, kernel, args), name);
}

// 16-bit rows of 16-byte pieces on 16-byte boundaries can be copied asynchronously and read as matrix fragments.
static bool whole_pieces(const AttentionProblem& p) {
    const uintptr_t bits = reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.k) | reinterpret_cast<uintptr_t>(p.v) | reinterpret_cast<uintptr_t>(p.y);
    return p.dtype != DTYPE_FLOAT32 && p.dim % 8 == 0 && (bits & 15) == 0;
}

int cache_box_rows(const AttentionProblem& p) {
    if (!p.page_table) return 128;
    if (p.pages == 0) return 0;                              // no cache to describe
    if (p.page_size % 128 == 0) return 128;
    return p.page_size % 8 == 0 && 128 % p.page_size == 0 ? p.page_size : 0;
}

bool make_cache_map(CUtensorMap* map, const AttentionProblem& p, const void* base, int box_rows) {
    const bool paged = p.page_table != nullptr;
    const uint64_t rows = paged ? (uint64_t)p.pages * p.page_size : (uint64_t)p.keys;
    const uint64_t dims[4] = {(uint64_t)p.dim, (uint64_t)p.kv_heads, rows, paged ? 1u : (uint64_t)p.batch};
    const uint64_t strides[3] = {(uint64_t)p.kv_head * 2, (uint64_t)p.kv_token * 2, paged ? rows * (uint64_t)p.kv_token * 2 : (uint64_t)p.kv_batch * 2};
    const uint32_t box[4] = {64, 1, (uint32_t)box_rows, 1};
    return make_tensor_map(map, base, 2, false, p.dtype == DTYPE_FLOAT16, 4, dims, strides, box, nullptr);
}

// The kernel, by the rows of a sequence (tokens times heads per key head, on average: the host does not know each length).  Measured, us, few-rows kernel / many-rows
// kernel, 8 sequences of 4000 keys and 8 key heads: dim 128, 16 rows 39 / 43, 20 rows 52 / 44, 32 rows 62 / 47; dim 64, 16 rows 30 / 37.  One sequence of 16000 keys, dim 128:
// 16 rows 31 / 37, 20 rows 40 / 37, 32 rows 45 / 38.  Heads above 128 and scales that are not positive stay with the few-rows kernel (dim 256, 64 rows: 135, mma.sync
// kernel 409); pages that no copy box fits go to the mma.sync kernel.
static bool run_attention(const AttentionProblem& p) {
    if (!whole_pieces(p)) return attention_fma(p);
    if (cache_box_rows(p) > 0) {
        const long long rows = (long long)p.queries * p.group / (p.page_table ? p.batch : 1);
        const bool few = rows <= 16;
        if (attention_step_fits(p) && (few || !attention_chunk_takes(p))) return attention_step(p);
        if (attention_chunk_takes(p)) return attention_chunk(p);
    }
    return attention_rows(p);
}

static bool attention_dtype(int dt) { return dt == DTYPE_FLOAT16 || dt == DTYPE_BFLOAT16 || dt == DTYPE_FLOAT32; }

// Limits that both operators share: head sizes, grid and index ranges.
static const char* common_limits(const AttentionProblem& p) {
    if (p.dim < 1 || p.dim > 256) return "heads of 1 to 256 elements";
    if (p.kv_heads < 1 || p.kv_heads > 65535 || p.heads % p.kv_heads != 0) return "query heads a multiple of 1 to 65535 key heads";
    if ((long long)p.queries * p.heads >= 0x7FFFFFFFll / 8 || (long long)p.batch * p.queries * p.heads >= 0x7FFFFFFFll / 8) return "fewer than 2^28 query rows";
    return nullptr;
}

}  // namespace tops

using namespace tops;

TOPS_API int tops_paged_attention_forward(const PagedAttentionCall* call) {
    const char* name = "tops_paged_attention_forward";
    if (!call) return call_fail(name, TOPS_ERR_INVALID, "null call", {});
    const PagedAttentionCall& c = *call;
    Tensor* y = c.y;
    const OutputList outs = {y, c.q, c.key_cache, c.value_cache, c.page_table, c.query_start, c.kv_length};
    for (const Tensor* t : {c.q, c.key_cache, c.value_cache, c.page_table, c.query_start, c.kv_length, (const Tensor*)y})
        if (!tensor_given(t)) return call_fail(name, TOPS_ERR_INVALID, "q, key_cache, value_cache, page_table, query_start, kv_length and y are required", outs);
    if (c.q->ndim != 3 || !same_shape(c.q, y)) return call_fail(name, TOPS_ERR_INVALID, "q and y are [tokens, heads, dim]", outs);
    if (c.key_cache->ndim != 4 || !same_shape(c.key_cache, c.value_cache) || c.key_cache->shape[3] != c.q->shape[2])
        return call_fail(name, TOPS_ERR_INVALID, "key_cache and value_cache are [pages, page_size, kv_heads, dim] with q's dim", outs);
    if (!attention_dtype(c.q->dtype) || c.key_cache->dtype != c.q->dtype || c.value_cache->dtype != c.q->dtype || y->dtype != c.q->dtype)
        return call_fail(name, TOPS_ERR_UNSUPPORTED, "q, caches and y share one of float16, bfloat16, float32", outs);
    if (c.page_table->dtype != DTYPE_INT32 || c.query_start->dtype != DTYPE_INT32 || c.kv_length->dtype != DTYPE_INT32)
        return call_fail(name, TOPS_ERR_INVALID, "page_table, query_start and kv_length are int32", outs);
    if (c.page_table->ndim != 2 || c.kv_length->size != (size_t)c.page_table->shape[0] || c.query_start->size != c.kv_length->size + 1)
        return call_fail(name, TOPS_ERR_INVALID, "page_table [batch, width], query_start [batch + 1], kv_length [batch]", outs);
    if (!std::isfinite(c.scale) || c.window < 0) return call_fail(name, TOPS_ERR_INVALID, "a finite scale and a window of 0 or more", outs);
    for (const Tensor* t : {c.q, c.key_cache, c.value_cache, c.page_table, c.query_start, c.kv_length})
        if (overlap(t, y)) return call_fail(name, TOPS_ERR_INVALID, "y shares memory with an operand", outs);
    AttentionProblem p;
    p.queries = c.q->shape[0];
    p.heads = c.q->shape[1];
    p.dim = c.q->shape[2];
    p.pages = c.key_cache->shape[0];
    p.page_size = c.key_cache->shape[1];
    p.kv_heads = c.key_cache->shape[2];
    p.batch = c.page_table->shape[0];
    p.table_width = c.page_table->shape[1];
    const char* limit = common_limits(p);
    if (!limit && p.page_size < 1) limit = "pages of at least one token";
    if (!limit && ((long long)p.pages * p.page_size >= 0x7FFFFFFFll || (long long)p.table_width * p.page_size >= 0x40000000ll))
        limit = "fewer than 2^31 tokens in the cache and 2^30 in one row of the page table";
    if (!limit && p.heads < 1) limit = "at least one head";
    if (limit) return call_fail(name, TOPS_ERR_UNSUPPORTED, limit, outs);
    if (!on_current_device({c.q, c.key_cache, c.value_cache, c.page_table, c.query_start, c.kv_length, y}))
        return call_fail(name, TOPS_ERR_INVALID, "a tensor belongs to another device than the current one", {});
    if (!acquire_device()) return tops_last_error();
    if (p.queries == 0 || p.batch == 0) return TOPS_OK;
    p.q = c.q->data; p.k = c.key_cache->data; p.v = c.value_cache->data; p.y = y->data;
    p.q_token = (long long)p.heads * p.dim;
    p.q_head = p.dim;
    p.kv_token = (long long)p.kv_heads * p.dim;
    p.kv_head = p.dim;
    p.keys = p.table_width * p.page_size;
    p.group = p.heads / p.kv_heads;
    p.group_div.set((uint32_t)p.group);
    p.page_table = reinterpret_cast<const int*>(c.page_table->data);
    p.page_div.set((uint32_t)p.page_size);
    p.query_start = reinterpret_cast<const int*>(c.query_start->data);
    p.kv_length = reinterpret_cast<const int*>(c.kv_length->data);
    p.scale_log2 = c.scale * kLog2E;
    p.window = c.window < p.keys ? c.window : 0;             // a window that no sequence can outgrow is none
    p.dtype = c.q->dtype;
    p.status = device_status_word();
    if (!run_attention(p)) return tops_last_error();
    finish_op();
    return TOPS_OK;
}

TOPS_API int tops_cross_attention_forward(const CrossAttentionCall* call) {
    const char* name = "tops_cross_attention_forward";
    if (!call) return call_fail(name, TOPS_ERR_INVALID, "null call", {});
    const CrossAttentionCall& c = *call;
    Tensor* y = c.y;
    const OutputList outs = {y, c.q, c.k, c.v, c.key_length, c.mask};
    for (const Tensor* t : {c.q, c.k, c.v, (const Tensor*)y})
        if (!tensor_given(t)) return call_fail(name, TOPS_ERR_INVALID, "q, k, v and y are required", outs);
    for (const Tensor* t : {c.key_length, c.mask})
        if (t && !tensor_given(t)) return call_fail(name, TOPS_ERR_INVALID, "key_length or mask without data", outs);
    if (c.q->ndim != 4 || !same_shape(c.q, y)) return call_fail(name, TOPS_ERR_INVALID, "q and y are [batch, queries, heads, dim] or, heads_first, [batch, heads, queries, dim]", outs);
    if (c.k->ndim != 4 || !same_shape(c.k, c.v) || c.k->shape[0] != c.q->shape[0] || c.k->shape[3] != c.q->shape[3])
        return call_fail(name, TOPS_ERR_INVALID, "k and v have one shape with q's batch and dim", outs);
    if (!attention_dtype(c.q->dtype) || c.k->dtype != c.q->dtype || c.v->dtype != c.q->dtype || y->dtype != c.q->dtype)
        return call_fail(name, TOPS_ERR_UNSUPPORTED, "q, k, v and y share one of float16, bfloat16, float32", outs);
    if (!std::isfinite(c.scale)) return call_fail(name, TOPS_ERR_INVALID, "a finite scale", outs);
    AttentionProblem p;
    const int tokens_at = c.heads_first ? 2 : 1, heads_at = c.heads_first ? 1 : 2;
    p.batch = c.q->shape[0];
    p.queries = c.q->shape[tokens_at];
    p.heads = c.q->shape[heads_at];
    p.dim = c.q->shape[3];
    p.keys = c.k->shape[tokens_at];
    p.kv_heads = c.k->shape[heads_at];
    if (c.key_length && (c.key_length->dtype != DTYPE_INT32 || c.key_length->size != (size_t)p.batch))
        return call_fail(name, TOPS_ERR_INVALID, "key_length is int32 [batch]", outs);
    if (c.mask) {
        const int dt = c.mask->dtype;
        if (c.mask->size != (size_t)p.batch * (size_t)p.keys) return call_fail(name, TOPS_ERR_INVALID, "mask has batch * keys elements (one per key, the same for all heads and queries)", outs);
        if (dt == DTYPE_UINT8 || dt == DTYPE_INT8) p.mask_kind = kMaskBytes;
        else if (dt == DTYPE_FLOAT32) p.mask_kind = kMaskF32;
        else if (dt == c.q->dtype) p.mask_kind = dt == DTYPE_FLOAT16 ? kMaskF16 : kMaskBF16;
        else return call_fail(name, TOPS_ERR_UNSUPPORTED, "mask is uint8, int8, float32 or of q's type", outs);
    }
    const char* limit = common_limits(p);
    if (!limit && p.heads < 1) limit = "at least one head";
    if (!limit && p.keys >= 0x40000000) limit = "fewer than 2^30 keys";
    if (limit) return call_fail(name, TOPS_ERR_UNSUPPORTED, limit, outs);
    for (const Tensor* t : {c.q, c.k, c.v, c.key_length, c.mask})
        if (overlap(t, y)) return call_fail(name, TOPS_ERR_INVALID, "y shares memory with an operand", outs);
    if (!on_current_device({c.q, c.k, c.v, c.key_length, c.mask, y}))
        return call_fail(name, TOPS_ERR_INVALID, "a tensor belongs to another device than the current one", {});
    if (!acquire_device()) return tops_last_error();
    if (y->size == 0) return TOPS_OK;
    if (p.keys == 0) { zero_fill(y); finish_op(); return TOPS_OK; }
    p.q = c.q->data; p.k = c.k->data; p.v = c.v->data; p.y = y->data;
    p.q_batch = (long long)p.queries * p.heads * p.dim;
    p.q_token = c.heads_first ? p.dim : (long long)p.heads * p.dim;
    p.q_head = c.heads_first ? (long long)p.queries * p.dim : p.dim;
    p.kv_batch = (long long)p.keys * p.kv_heads * p.dim;
    p.kv_token = c.heads_first ? p.dim : (long long)p.kv_heads * p.dim;
    p.kv_head = c.heads_first ? (long long)p.keys * p.dim : p.dim;
    p.group = p.heads / p.kv_heads;
    p.group_div.set((uint32_t)p.group);
    p.kv_length = c.key_length ? reinterpret_cast<const int*>(c.key_length->data) : nullptr;
    p.mask = c.mask ? c.mask->data : nullptr;
    p.scale_log2 = c.scale * kLog2E;
    p.dtype = c.q->dtype;
    p.status = device_status_word();
    if (!run_attention(p)) return tops_last_error();
    finish_op();
    return TOPS_OK;
}
