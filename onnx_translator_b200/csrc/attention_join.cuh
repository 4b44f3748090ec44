// Items that several blocks share: where the partial results lie, and the kernel that joins them.
//
// Block c of the main kernel works on the c-th share of all work; slot 2 c holds the partial result of its first item, slot 2 c + 1 that of its last one.
// An item that begins in share c and ends in share c + k - 1 has its k parts in c's slot and in slots 2 (c + 1), 2 (c + 2), ...: block c leaves a
// job that says so.  The parts are joined in the order of the keys, so the result does not depend on timing.
#pragma once

#include "attention_common.cuh"

#include <cstdlib>

namespace tops {

struct JoinJob {
    RowTile t;
    int kv_head = 0;
    int parts = 0;               // 0: no item of this share goes on in the next
    int slot = 0;                // of the first part
};

struct PartialResults {          // scratch of one call, from the stream-ordered pool
    float* o = nullptr;          // [2 * blocks][N][DIMS]
    float2* stats = nullptr;     // [2 * blocks][N]: maximum, sum of weights
    JoinJob* jobs = nullptr;     // [blocks]
};

// One launch attribute (a kernel is scheduled while its predecessor drains), or none with TOPS_PDL=0.
inline unsigned overlap_launches() {
    static const unsigned on = [] { const char* e = getenv("TOPS_PDL"); return e && e[0] == '0' ? 0u : 1u; }();
    return on;
}

inline bool allocate_partials(PartialResults& parts, int blocks, int rows, int dims, cudaStream_t stream) {
    const size_t o_bytes = (size_t)2 * blocks * rows * dims * sizeof(float), stat_bytes = (size_t)2 * blocks * rows * sizeof(float2);
    char* scratch = nullptr;
    if (!TOPS_CUDA_OK(cudaMallocAsync((void**)&scratch, o_bytes + stat_bytes + (size_t)blocks * sizeof(JoinJob), stream))) return false;
    parts.o = reinterpret_cast<float*>(scratch);
    parts.stats = reinterpret_cast<float2*>(scratch + o_bytes);
    parts.jobs = reinterpret_cast<JoinJob*>(scratch + o_bytes + stat_bytes);
    return true;
}

// Block (c, q): `rows` rows of job c, eight warps.  With few parts a warp joins whole rows by itself, all loads in flight together; with many (a few long sequences
// over all SMs) the warps take every eighth part of a row and meet in shared memory.
constexpr int kJoinThreads = 256;
template <typename T, int N, int DIMS>
__global__ void __launch_bounds__(kJoinThreads) attention_join(const __grid_constant__ AttentionProblem p, const PartialResults parts, const int rows) {
    constexpr int WARPS = kJoinThreads / 32, QUADS = DIMS / 4, PER_LANE = (QUADS + 31) / 32;
    __shared__ float4 partial[WARPS][QUADS];
    __shared__ float partial_l[WARPS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const JoinJob job = parts.jobs[blockIdx.x];
    const int row_begin = (int)blockIdx.y * rows, row_end = min(row_begin + rows, job.t.rows);
    if (job.parts == 0 || row_begin >= row_end) return;
    auto slot = [&](int k) { return k == 0 ? job.slot : 2 * ((int)blockIdx.x + k); };
    const bool aligned = (p.dim & 3) == 0 && (reinterpret_cast<uintptr_t>(p.y) & (4 * sizeof(T) - 1)) == 0;
    if (job.parts <= 8) {
        #pragma unroll 1
        for (int r = row_begin + warp; r < row_end; r += WARPS) {
            float2 s = make_float2(-INFINITY, 0.0f);
            if (lane < job.parts) s = parts.stats[(long long)slot(lane) * N + r];
            float4 v[8][PER_LANE];
            #pragma unroll
            for (int k = 0; k < 8; k++)
                #pragma unroll
                for (int e = 0; e < PER_LANE; e++)
                    if (k < job.parts && lane + e * 32 < QUADS) v[k][e] = *reinterpret_cast<const float4*>(parts.o + ((long long)slot(k) * N + r) * DIMS + (lane + e * 32) * 4);
            const float top = fmaxf(fmaxf(fmaxf(__shfl_sync(~0u, s.x, 0), __shfl_sync(~0u, s.x, 1)), fmaxf(__shfl_sync(~0u, s.x, 2), __shfl_sync(~0u, s.x, 3))),
                                    fmaxf(fmaxf(__shfl_sync(~0u, s.x, 4), __shfl_sync(~0u, s.x, 5)), fmaxf(__shfl_sync(~0u, s.x, 6), __shfl_sync(~0u, s.x, 7))));
            const float w = partial_weight(s.x, top), weighted = s.x == -INFINITY ? 0.0f : s.y * w;
            float l = 0.0f;
            float x[PER_LANE][4] = {};
            #pragma unroll
            for (int k = 0; k < 8; k++) {
                const float wk = __shfl_sync(~0u, w, k), mk = __shfl_sync(~0u, s.x, k);
                l += __shfl_sync(~0u, weighted, k);
                if (k < job.parts && mk != -INFINITY)          // a part without a key holds nothing
                    #pragma unroll
                    for (int e = 0; e < PER_LANE; e++) {
                        if (lane + e * 32 >= QUADS) continue;
                        x[e][0] = __fmaf_rn(v[k][e].x, wk, x[e][0]); x[e][1] = __fmaf_rn(v[k][e].y, wk, x[e][1]);
                        x[e][2] = __fmaf_rn(v[k][e].z, wk, x[e][2]); x[e][3] = __fmaf_rn(v[k][e].w, wk, x[e][3]);
                    }
            }
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            T* to = reinterpret_cast<T*>(p.y) + row_offset(p, job.t, job.kv_head, job.t.row0 + r);
            #pragma unroll
            for (int e = 0; e < PER_LANE; e++) {
                const int d = (lane + e * 32) * 4;
                #pragma unroll
                for (int k = 0; k < 4; k++) x[e][k] *= inv;
                if (d < p.dim && lane + e * 32 < QUADS) store4(to + d, x[e], p.dim - d, aligned);
            }
        }
        return;
    }
    for (int r = row_begin; r < row_end; r++) {
        float top = -INFINITY;
        for (int k = lane; k < job.parts; k += 32) top = fmaxf(top, parts.stats[(long long)slot(k) * N + r].x);
        #pragma unroll
        for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
        float l = 0.0f;
        float4 sum[PER_LANE];
        #pragma unroll
        for (int e = 0; e < PER_LANE; e++) sum[e] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        #pragma unroll 4
        for (int k = warp; k < job.parts; k += WARPS) {
            const long long row = (long long)slot(k) * N + r;
            const float2 s = parts.stats[row];
            const float w = partial_weight(s.x, top);
            if (s.x != -INFINITY) l = __fmaf_rn(s.y, w, l);
            #pragma unroll
            for (int e = 0; e < PER_LANE; e++) {
                const int quad = lane + e * 32;
                if (quad < QUADS) {
                    const float4 v = *reinterpret_cast<const float4*>(parts.o + row * DIMS + quad * 4);
                    if (s.x != -INFINITY) {                    // a part without a key holds nothing
                        sum[e].x = __fmaf_rn(v.x, w, sum[e].x); sum[e].y = __fmaf_rn(v.y, w, sum[e].y);
                        sum[e].z = __fmaf_rn(v.z, w, sum[e].z); sum[e].w = __fmaf_rn(v.w, w, sum[e].w);
                    }
                }
            }
        }
        #pragma unroll
        for (int e = 0; e < PER_LANE; e++) if (lane + e * 32 < QUADS) partial[warp][lane + e * 32] = sum[e];
        if (lane == 0) partial_l[warp] = l;
        __syncthreads();
        for (int quad = threadIdx.x; quad < QUADS; quad += kJoinThreads) {
            float all = 0.0f, x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            #pragma unroll
            for (int w = 0; w < WARPS; w++) {
                const float4 v = partial[w][quad];
                all += partial_l[w];
                x[0] += v.x; x[1] += v.y; x[2] += v.z; x[3] += v.w;
            }
            const float inv = all == 0.0f ? 0.0f : 1.0f / all;
            #pragma unroll
            for (int e = 0; e < 4; e++) x[e] *= inv;
            if (quad * 4 < p.dim) store4(reinterpret_cast<T*>(p.y) + row_offset(p, job.t, job.kv_head, job.t.row0 + r) + quad * 4, x, p.dim - quad * 4, aligned);
        }
        __syncthreads();
    }
}

// Enqueues the join (when the main kernel was launched: `ok`) and gives the scratch back in stream order.  `items` (an upper bound) tells how many parts an item has about: with
// many, rows are the longer work and are spread over more blocks (256 rows, 18 parts each: 83 us with 32 rows a block, 44 with 8); with few, blocks without work
// cost more (13 ragged windows: 47 against 50 us).
template <typename T, int N, int DIMS>
bool join_partials(const AttentionProblem& p, const PartialResults& parts, int blocks, long long items, cudaStream_t stream, bool ok) {
    if (ok) {
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cudaLaunchConfig_t cfg = {};
        int rows = N < 64 ? 4 : blocks >= 6 * items ? 8 : 32;
        cfg.gridDim = dim3((unsigned)blocks, (unsigned)(N / rows));
        cfg.blockDim = dim3(kJoinThreads);
        cfg.stream = stream;
        cfg.attrs = attr;
        cfg.numAttrs = overlap_launches();
        AttentionProblem copy = p;
        PartialResults copy_parts = parts;
        void* args[] = {&copy, &copy_parts, &rows};
        ok = check_cuda(cudaLaunchKernelExC(&cfg, (const void*)attention_join<T, N, DIMS>, args), "attention_join");
    }
    return TOPS_CUDA_OK(cudaFreeAsync(parts.o, stream)) && ok;
}

}  // namespace tops
