// What the attention kernels share: the description of a call, the mapping from a block to its rows and keys, and the
// join of partial results inside a thread-block cluster.
//
//   y = softmax(scale * q K^T + mask) V,   one softmax per (token, head)
//
// All kernels walk the keys once and keep, per row, the running maximum m of the scores (in units of log2), the running sum
// l of exp2(score - m) and the accumulator o = sum exp2(score - m) V.  Two partial results over disjoint keys join exactly:
//   m = max(m1, m2),  l = l1 2^(m1 - m) + l2 2^(m2 - m),  o likewise;  y = o / l, and 0 where no key was seen (l = 0).
//
// The `group` query heads that share a key head are rows of one problem: row r of a sequence is token r / group, head r % group
// of the key head.  So the keys are read once for the whole group, and a single new token still fills `group` rows.
#pragma once

#include "common.cuh"
#include "umma.cuh"

namespace tops {

enum MaskKind { kMaskNone = 0, kMaskBytes = 1, kMaskF32 = 2, kMaskF16 = 3, kMaskBF16 = 4 };

struct AttentionProblem {
    const void* q = nullptr;
    const void* k = nullptr;
    const void* v = nullptr;
    void* y = nullptr;
    long long q_batch = 0, q_token = 0, q_head = 0;       // element strides of q and of y
    long long kv_batch = 0, kv_token = 0, kv_head = 0;    // element strides of k and of v; paged: kv_token walks cache rows
    int batch = 0;
    int queries = 0;             // dense: per batch row; paged: rows of q over all sequences
    int keys = 0;                // dense: extent of k; paged: table width * page size
    int heads = 0, kv_heads = 0, group = 1, dim = 0;
    FastDiv group_div;
    const int* page_table = nullptr;      // null: dense
    int table_width = 0, page_size = 1, pages = 0;
    FastDiv page_div;
    const int* query_start = nullptr;     // paged only
    const int* kv_length = nullptr;       // paged: required; dense: may be null
    const void* mask = nullptr;           // dense only, [batch, keys]
    int mask_kind = kMaskNone;
    float scale_log2 = 0.0f;              // scale * log2(e): scores are kept in units of log2
    int window = 0;                       // paged only; 0 none
    int dtype = DTYPE_FLOAT32;
    int* status = nullptr;
};

constexpr float kLog2E = 1.44269504088896340736f;

// One block's rows: `rows` rows from row `row0` of sequence `seq`, and the keys [key_begin, key_end) that any of them sees.
struct RowTile {
    int seq = 0, row0 = 0, rows = 0;
    int token0 = 0;              // first token of the sequence in q (paged); 0 for dense
    int first_position = 0;      // paged: position of the sequence's first new token, may be negative
    int length = 0;              // keys of the sequence
    int key_begin = 0, key_end = 0;
};

__device__ __forceinline__ void report_bad_index(const AttentionProblem& p) {
    if (p.status) atomicExch(p.status, kStatusBadIndex);
}

// Finds tile number `index`, counting tiles of `rows_per_tile` rows through the sequences; false past the last one.
// Called by whole warps; every warp of a block gets the same answer.  Paged: the tile counts of 32 sequences at a time are
// added up by a warp scan (the host does not know them: query_start lives in device memory).
__device__ __forceinline__ bool locate_tile(const AttentionProblem& p, int index, int rows_per_tile, RowTile& t) {
    const int lane = threadIdx.x & 31;
    int tokens = p.queries;
    if (!p.page_table) {
        const int per_batch = (p.queries * p.group + rows_per_tile - 1) / rows_per_tile;
        t.seq = index / per_batch;
        if (t.seq >= p.batch) return false;
        t.row0 = (index - t.seq * per_batch) * rows_per_tile;
        t.length = p.keys;
        if (p.kv_length) t.length = min(max(p.kv_length[t.seq], 0), p.keys);
        t.key_begin = 0;
        t.key_end = t.length;
    } else {
        int before = 0;
        bool found = false;
        for (int base = 0; base < p.batch; base += 32) {
            const int b = base + lane;
            int start = 0, end = 0, length = 0;
            if (b < p.batch) {
                const int s = p.query_start[b], e = p.query_start[b + 1];
                length = p.kv_length[b];                     // fetched along with the bounds: one round trip less
                start = min(max(s, 0), p.queries);
                end = min(max(e, start), p.queries);
                if (start != s || end != e) report_bad_index(p);
            }
            const int tiles = ((end - start) * p.group + rows_per_tile - 1) / rows_per_tile;
            int sum = tiles;
            #pragma unroll
            for (int d = 1; d < 32; d <<= 1) { const int o = __shfl_up_sync(~0u, sum, d); if (lane >= d) sum += o; }
            const unsigned past = __ballot_sync(~0u, index < before + sum);
            if (past) {
                const int at = __ffs(past) - 1;
                t.seq = base + at;
                t.token0 = __shfl_sync(~0u, start, at);
                tokens = __shfl_sync(~0u, end, at) - t.token0;
                t.row0 = (index - before - __shfl_sync(~0u, sum - tiles, at)) * rows_per_tile;
                t.length = __shfl_sync(~0u, length, at);
                found = true;
                break;
            }
            before += __shfl_sync(~0u, sum, 31);
        }
        if (!found) return false;
        const int length = t.length;
        t.length = min(max(length, 0), p.keys);
        if (length != t.length) report_bad_index(p);
        t.first_position = t.length - tokens;
    }
    t.rows = min(rows_per_tile, tokens * p.group - t.row0);
    if (p.page_table) {
        const int first = t.first_position + (int)p.group_div.div((uint32_t)t.row0);
        const int last = t.first_position + (int)p.group_div.div((uint32_t)(t.row0 + t.rows - 1));
        t.key_end = min(t.length, last + 1);
        t.key_begin = p.window > 0 ? max(0, first - p.window + 1) : 0;
    }
    if (t.key_end < t.key_begin) t.key_end = t.key_begin;
    return true;
}

// Row of the cache (paged) or of the batch row (dense) that holds key j of the sequence, -1 when its page is not in the cache.
__device__ __forceinline__ int key_row(const AttentionProblem& p, int seq, int j) {
    if (!p.page_table) return j;
    const int column = (int)p.page_div.div((uint32_t)j);
    const int page = p.page_table[(long long)seq * p.table_width + column];
    if ((unsigned)page >= (unsigned)p.pages) { report_bad_index(p); return -1; }
    return page * p.page_size + (j - column * p.page_size);
}

// What the mask adds to key j's scores, in units of log2; -Inf excludes the key (the type's lowest value does too, so that
// a row that is masked throughout is empty rather than a softmax over rounding errors).
__device__ __forceinline__ float mask_value(uint8_t x) { return x ? 0.0f : -INFINITY; }
__device__ __forceinline__ float mask_value(float x) { return x <= -3.402823466e+38f ? -INFINITY : x * kLog2E; }
__device__ __forceinline__ float mask_value(__half h) { const float x = __half2float(h); return x <= -65504.0f ? -INFINITY : x * kLog2E; }
__device__ __forceinline__ float mask_value(__nv_bfloat16 h) { const float x = __bfloat162float(h); return x <= -3.3895313892515355e+38f ? -INFINITY : x * kLog2E; }

__device__ __forceinline__ float key_bias(const AttentionProblem& p, int seq, int j) {
    const long long at = (long long)seq * p.keys + j;
    switch (p.mask_kind) {
        case kMaskBytes: return mask_value(reinterpret_cast<const uint8_t*>(p.mask)[at]);
        case kMaskF32:   return mask_value(reinterpret_cast<const float*>(p.mask)[at]);
        case kMaskF16:   return mask_value(reinterpret_cast<const __half*>(p.mask)[at]);
        case kMaskBF16:  return mask_value(reinterpret_cast<const __nv_bfloat16*>(p.mask)[at]);
        default:         return 0.0f;
    }
}
// Keys j, j + 32, j + 64 and j + 96 at once, as they lie in memory (looked at later by mask_values) ...
__device__ __forceinline__ void load_mask(const AttentionProblem& p, int seq, int j, int key_end, uint32_t (&raw)[4]) {
    const long long at = (long long)seq * p.keys + j;
    #pragma unroll
    for (int e = 0; e < 4; e++) {
        if (j + e * 32 >= key_end) continue;
        if (p.mask_kind == kMaskBytes) raw[e] = reinterpret_cast<const uint8_t*>(p.mask)[at + e * 32];
        else if (p.mask_kind == kMaskF32) raw[e] = reinterpret_cast<const uint32_t*>(p.mask)[at + e * 32];
        else raw[e] = reinterpret_cast<const uint16_t*>(p.mask)[at + e * 32];
    }
}
// ... and what they add; -Inf from key_end on.
__device__ __forceinline__ void mask_values(const AttentionProblem& p, const uint32_t (&raw)[4], int j, int key_end, float (&b)[4]) {
    #pragma unroll
    for (int e = 0; e < 4; e++) {
        float x;
        if (p.mask_kind == kMaskBytes) x = mask_value((uint8_t)raw[e]);
        else if (p.mask_kind == kMaskF32) x = mask_value(__uint_as_float(raw[e]));
        else if (p.mask_kind == kMaskF16) x = mask_value(__ushort_as_half((unsigned short)raw[e]));
        else x = mask_value(__ushort_as_bfloat16((unsigned short)raw[e]));
        b[e] = j + e * 32 < key_end ? x : -INFINITY;
    }
}

// Drops the 128-key tiles of [lo, lo + n) at either end whose keys the mask excludes altogether: padding is not copied.  A whole warp, `n` > 0.
__device__ __forceinline__ void trim_masked(const AttentionProblem& p, int seq, int key_end, int& lo, int& n) {
    const int lane = threadIdx.x & 31;
    auto kept = [&](int tile) {
        uint32_t raw[4] = {0u, 0u, 0u, 0u};
        float b[4];
        load_mask(p, seq, tile * 128 + lane, key_end, raw);
        mask_values(p, raw, tile * 128 + lane, key_end, b);
        return __any_sync(~0u, b[0] != -INFINITY || b[1] != -INFINITY || b[2] != -INFINITY || b[3] != -INFINITY) != 0;
    };
    while (n > 0 && !kept(lo + n - 1)) n--;
    while (n > 0 && !kept(lo)) { lo++; n--; }
}

// Element offset of row r of the tile's sequence in q and y (without the dimension).
__device__ __forceinline__ long long row_offset(const AttentionProblem& p, const RowTile& t, int kv_head, int r) {
    const int token = (int)p.group_div.div((uint32_t)r), head = kv_head * p.group + (r - token * p.group);
    const long long batch = p.page_table ? 0 : (long long)t.seq * p.q_batch;
    return batch + (long long)(t.token0 + token) * p.q_token + (long long)head * p.q_head;
}

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 2^(m - top) for a partial result with maximum m: 0 when it has seen no key.
__device__ __forceinline__ float partial_weight(float m, float top) { return m == -INFINITY ? 0.0f : exp2_approx(m - top); }

template <typename T> __device__ __forceinline__ float to_float(T x);
template <> __device__ __forceinline__ float to_float<float>(float x) { return x; }
template <> __device__ __forceinline__ float to_float<__half>(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ float from_float<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
// Two floats as one 32-bit word of 16-bit values, the first in the low half.
template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// Four neighbouring results; `aligned`: the row start and dim are multiples of four elements.
template <typename T> __device__ __forceinline__ void store4(T* to, const float (&x)[4], int left, bool aligned) {
    if (aligned) {
        if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(to) = make_float4(x[0], x[1], x[2], x[3]);
        else *reinterpret_cast<uint2*>(to) = make_uint2(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]));
    } else {
        for (int i = 0; i < left && i < 4; i++) to[i] = from_float<T>(x[i]);
    }
}

// ---- the warp-level building blocks of the 16-bit kernels ---------------------------------------------------------------
// 16 bytes global -> shared without a register, zeros when `bytes` is 0 (nothing is read then).
__device__ __forceinline__ void copy_async_16(uint32_t to, const void* from, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void load_matrix4(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void load_matrix4_trans(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
// c[16 x 8] += a[16 x 16] b[16 x 8], float32 accumulators.
template <typename T> __device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// ---- clusters --------------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_size() { uint32_t n; asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(n)); return n; }
__device__ __forceinline__ uint32_t cluster_rank() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t peer_address(uint32_t shared_address, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(shared_address), "r"(rank));
    return a;
}
__device__ __forceinline__ float4 load_peer_f4(uint32_t a) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ float2 load_peer_f2(uint32_t a) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(a) : "memory");
    return v;
}

// Every block of the cluster holds o[rows][PITCH] and stats[rows] = (m, l) over its share of the keys, complete in shared memory
// for the whole block (the caller has synchronised it).  The blocks read one another's partials through distributed shared
// memory and each writes every n-th group of four results, in a fixed order of the partials: the result does not depend on timing, and no
// workspace or second launch is needed.  Called by all THREADS threads of all blocks of the cluster.
template <typename T, int PITCH, int THREADS>
__device__ __forceinline__ void join_and_store(const AttentionProblem& p, const RowTile& t, int kv_head, const float* o, const float2* stats) {
    const uint32_t ranks = cluster_size(), rank = cluster_rank();
    const uint32_t o_at = (uint32_t)__cvta_generic_to_shared(o), stats_at = (uint32_t)__cvta_generic_to_shared(stats);
    const bool aligned = (p.dim & 3) == 0 && (reinterpret_cast<uintptr_t>(p.y) & (4 * sizeof(T) - 1)) == 0;
    const int quads = (p.dim + 3) >> 2;
    if (ranks > 1) cluster_sync();
    for (int i = threadIdx.x + (int)rank * THREADS; i < t.rows * quads; i += THREADS * (int)ranks) {
        const int r = i / quads, d = (i - r * quads) * 4;
        float x[4];
        if (ranks == 1) {
            const float2 s = stats[r];
            const float inv = s.y == 0.0f ? 0.0f : 1.0f / s.y;
            const float4 v = *reinterpret_cast<const float4*>(o + (size_t)r * PITCH + d);
            x[0] = v.x * inv; x[1] = v.y * inv; x[2] = v.z * inv; x[3] = v.w * inv;
            if (s.y == 0.0f) x[0] = x[1] = x[2] = x[3] = 0.0f;
        } else {
            float top = -INFINITY, l = 0.0f;
            for (uint32_t c = 0; c < ranks; c++) top = fmaxf(top, load_peer_f2(peer_address(stats_at + r * 8, c)).x);
            x[0] = x[1] = x[2] = x[3] = 0.0f;
            for (uint32_t c = 0; c < ranks; c++) {
                const float2 s = load_peer_f2(peer_address(stats_at + r * 8, c));
                const float w = partial_weight(s.x, top);
                const float4 v = load_peer_f4(peer_address(o_at + ((uint32_t)r * PITCH + d) * 4, c));
                if (s.x != -INFINITY) {
                    l = __fmaf_rn(s.y, w, l);
                    x[0] = __fmaf_rn(v.x, w, x[0]); x[1] = __fmaf_rn(v.y, w, x[1]);
                    x[2] = __fmaf_rn(v.z, w, x[2]); x[3] = __fmaf_rn(v.w, w, x[3]);
                }
            }
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            #pragma unroll
            for (int e = 0; e < 4; e++) x[e] *= inv;
        }
        store4(reinterpret_cast<T*>(p.y) + row_offset(p, t, kv_head, t.row0 + r) + d, x, p.dim - d, aligned);
    }
    if (ranks > 1) cluster_sync();                         // nobody leaves while a peer still reads its shared memory
}

// ---- launch ----------------------------------------------------------------------------------------------------------
// How many blocks share one row tile's keys.  `tiles` row tiles (an upper bound), `step` keys is the least share worth a
// block; a cluster spans at most eight blocks.
int attention_splits(const AttentionProblem& p, long long tiles, int blocks_wanted, int step);
// Upper bound of the row tiles over all sequences.
long long attention_tiles(const AttentionProblem& p, int rows_per_tile);
bool launch_attention(const void* kernel, const AttentionProblem& p, int rows_per_tile, int threads, size_t smem, int splits, void** args, const char* name);

// Tensor map over k or v: (dim, head, row, batch) in boxes of 64 x 1 x box_rows x 1, 128-byte swizzle; dims past the head are zeros.
bool make_cache_map(CUtensorMap* map, const AttentionProblem& p, const void* base, int box_rows);
// Rows of a box that stay inside a page (dense: 128): a divisor of 128 that is a multiple of the 8-row swizzle group; 0 if there is none.
int cache_box_rows(const AttentionProblem& p);

bool attention_chunk_takes(const AttentionProblem& p);
bool attention_chunk(const AttentionProblem& p);     // 16-bit types, dim <= 128, cache_box_rows > 0, scale > 0: 256 rows per block, tcgen05
bool attention_step_fits(const AttentionProblem& p);
bool attention_step(const AttentionProblem& p);      // 16-bit types, cache_box_rows > 0: up to 64 rows per block, tcgen05
bool attention_fma(const AttentionProblem& p);       // any type, any dim up to 256
bool attention_rows(const AttentionProblem& p);      // 16-bit types, dim % 8 == 0: 16 rows per block, mma.sync

}  // namespace tops
