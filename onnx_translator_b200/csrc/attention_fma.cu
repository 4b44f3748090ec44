// Attention in float32 arithmetic on the FMA units: float32 tensors, and 16-bit ones whose head size or alignment the
// tensor-core kernels do not take.
//
// A block owns R rows (8 for single tokens, 32 for longer chunks) of one key head and walks its share of the keys in tiles of C.
// Operands are widened to float32 on the way into shared memory.  Scores: a thread owns a small rows x keys patch (2 x 4 for
// R = 32) and reads both operands as 16-byte vectors, so one shared-memory read feeds about three multiply-adds.  Softmax: 256 / R
// threads per row.  Product with V: a thread owns four neighbouring dimensions of a few rows.
//
// Measured: 25 TFLOP/s on a prompt of 8192 tokens, dim 128 (R = 32); 27 us for 2 x 1023 queries over 77 keys, 8 heads of 40, where each block's two key tiles are a chain of
// latencies.
#include "attention_common.cuh"

namespace tops {

constexpr int kFmaThreads = 256;

template <typename T, int R, int DP, int C>
__global__ void __launch_bounds__(kFmaThreads) attention_fma_kernel(const __grid_constant__ AttentionProblem p, const int tiles) {
    constexpr int KP = DP + 4;                              // pitch of a key row: neighbouring keys start four banks apart
    extern __shared__ __align__(16) float smem[];
    float* qs = smem;                                       // [R][DP]
    float* ks = qs + R * DP;                                // [C][KP]
    float* vs = ks + C * KP;                                // [C][DP]
    float* ss = vs + C * DP;                                // [R][C + 1]
    float2* stats = reinterpret_cast<float2*>(ss + ((R * (C + 1) + 3) & ~3));   // [R] running (m, l)
    float* fade = reinterpret_cast<float*>(stats + R);      // [R] factor of the accumulator
    int* rows_of = reinterpret_cast<int*>(fade + R);        // [C] cache row of each key of the tile, -1: not there
    float* bias = reinterpret_cast<float*>(rows_of + C);    // [C]

    const int splits = (int)cluster_size(), rank = (int)cluster_rank();
    RowTile t;
    if (!locate_tile(p, tiles - 1 - (int)(blockIdx.x / (unsigned)splits), R, t)) return;    // the whole cluster leaves
    const int kv_head = blockIdx.y, tid = threadIdx.x;
    const int dim = p.dim;

    // this block's keys
    const int all = t.key_end - t.key_begin;
    const int share = ((all + splits - 1) / splits + C - 1) / C * C;
    const int lo = min(t.key_begin + rank * share, t.key_end), hi = min(lo + share, t.key_end);

    const T* q = reinterpret_cast<const T*>(p.q);
    for (int i = tid; i < R * DP / 4; i += kFmaThreads) {
        const int r = i / (DP / 4), d = (i - r * (DP / 4)) * 4;
        const T* row = q + (r < t.rows ? row_offset(p, t, kv_head, t.row0 + r) : 0);
        #pragma unroll
        for (int e = 0; e < 4; e++) qs[r * DP + d + e] = r < t.rows && d + e < dim ? to_float(row[d + e]) : 0.0f;
    }
    if (tid < R) stats[tid] = make_float2(-INFINITY, 0.0f);

    constexpr int QUADS = DP / 4;
    constexpr int GROUPS = kFmaThreads / QUADS;             // row groups of the product with V
    constexpr int RPT = R >= GROUPS ? R / GROUPS : 1;
    const int dq = tid % QUADS, rg = tid / QUADS;
    float acc[RPT][4];
    #pragma unroll
    for (int i = 0; i < RPT; i++) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.0f;

    const long long kv_base = (p.page_table ? 0 : (long long)t.seq * p.kv_batch) + (long long)kv_head * p.kv_head;
    const T* kp = reinterpret_cast<const T*>(p.k) + kv_base;
    const T* vp = reinterpret_cast<const T*>(p.v) + kv_base;
    const bool vec = (dim & 3) == 0 && ((reinterpret_cast<uintptr_t>(p.k) | reinterpret_cast<uintptr_t>(p.v)) & (4 * sizeof(T) - 1)) == 0;

    for (int j0 = lo; j0 < hi; j0 += C) {
        __syncthreads();
        if (tid < C) {
            const int j = j0 + tid;
            int row = -1;
            float b = -INFINITY;
            if (j < hi) {
                b = key_bias(p, t.seq, j);
                if (b != -INFINITY) row = key_row(p, t.seq, j);
            }
            rows_of[tid] = row;
            bias[tid] = b;
        }
        __syncthreads();
        if (vec) {
            for (int i = tid; i < C * QUADS; i += kFmaThreads) {
                const int c = i / QUADS, d = (i - c * QUADS) * 4;
                const int row = rows_of[c];
                float4 a = make_float4(0, 0, 0, 0), b = a;
                if (row >= 0 && d < dim) {
                    const long long at = (long long)row * p.kv_token + d;
                    if constexpr (sizeof(T) == 4) {
                        a = *reinterpret_cast<const float4*>(kp + at);
                        b = *reinterpret_cast<const float4*>(vp + at);
                    } else {
                        const uint2 x = *reinterpret_cast<const uint2*>(kp + at), y = *reinterpret_cast<const uint2*>(vp + at);
                        const T* xt = reinterpret_cast<const T*>(&x);
                        const T* yt = reinterpret_cast<const T*>(&y);
                        a = make_float4(to_float(xt[0]), to_float(xt[1]), to_float(xt[2]), to_float(xt[3]));
                        b = make_float4(to_float(yt[0]), to_float(yt[1]), to_float(yt[2]), to_float(yt[3]));
                    }
                }
                *reinterpret_cast<float4*>(ks + c * KP + d) = a;
                *reinterpret_cast<float4*>(vs + c * DP + d) = b;
            }
        } else {
            for (int i = tid; i < C * DP; i += kFmaThreads) {
                const int c = i / DP, d = i - c * DP;
                const int row = rows_of[c];
                const bool there = row >= 0 && d < dim;
                const long long at = (long long)row * p.kv_token + d;
                ks[c * KP + d] = there ? to_float(kp[at]) : 0.0f;
                vs[c * DP + d] = there ? to_float(vp[at]) : 0.0f;
            }
        }
        __syncthreads();
        {   // scores
            constexpr int RI = R == 32 ? 16 : 8, KI = kFmaThreads / RI, RQ = R / RI, KQ = C / KI;
            const int ri = tid / KI, ki = tid % KI;
            float s[RQ][KQ];
            #pragma unroll
            for (int a = 0; a < RQ; a++)
                #pragma unroll
                for (int b = 0; b < KQ; b++) s[a][b] = 0.0f;
            for (int d = 0; d < dim; d += 4) {
                float4 qv[RQ], kv[KQ];
                #pragma unroll
                for (int a = 0; a < RQ; a++) qv[a] = *reinterpret_cast<const float4*>(qs + (ri * RQ + a) * DP + d);
                #pragma unroll
                for (int b = 0; b < KQ; b++) kv[b] = *reinterpret_cast<const float4*>(ks + (ki + KI * b) * KP + d);
                #pragma unroll
                for (int a = 0; a < RQ; a++)
                    #pragma unroll
                    for (int b = 0; b < KQ; b++) {
                        s[a][b] = __fmaf_rn(qv[a].x, kv[b].x, s[a][b]);
                        s[a][b] = __fmaf_rn(qv[a].y, kv[b].y, s[a][b]);
                        s[a][b] = __fmaf_rn(qv[a].z, kv[b].z, s[a][b]);
                        s[a][b] = __fmaf_rn(qv[a].w, kv[b].w, s[a][b]);
                    }
            }
            #pragma unroll
            for (int a = 0; a < RQ; a++) {
                const int r = ri * RQ + a;
                const int position = t.first_position + (int)p.group_div.div((uint32_t)(t.row0 + r));
                #pragma unroll
                for (int b = 0; b < KQ; b++) {
                    const int c = ki + KI * b, j = j0 + c;
                    bool seen = bias[c] != -INFINITY;
                    if (p.page_table) seen = seen && j <= position && (p.window == 0 || j > position - p.window);
                    ss[r * (C + 1) + c] = seen ? __fmaf_rn(s[a][b], p.scale_log2, bias[c]) : -INFINITY;
                }
            }
        }
        __syncthreads();
        {   // running maximum and sum
            constexpr int PER_ROW = kFmaThreads / R;
            const int r = tid / PER_ROW, l0 = tid % PER_ROW;
            const float2 old = stats[r];
            float m = old.x;
            for (int c = l0; c < C; c += PER_ROW) m = fmaxf(m, ss[r * (C + 1) + c]);
            #pragma unroll
            for (int d = PER_ROW / 2; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, d, PER_ROW));
            const float base = m == -INFINITY ? 0.0f : m;
            float sum = 0.0f;
            for (int c = l0; c < C; c += PER_ROW) {
                const float w = exp2f(ss[r * (C + 1) + c] - base);
                ss[r * (C + 1) + c] = w;
                sum += w;
            }
            #pragma unroll
            for (int d = PER_ROW / 2; d > 0; d >>= 1) sum += __shfl_xor_sync(~0u, sum, d, PER_ROW);
            const float f = old.x == -INFINITY ? 0.0f : exp2f(old.x - base);
            __syncwarp();
            if (l0 == 0) { fade[r] = f; stats[r] = make_float2(m, __fmaf_rn(old.y, f, sum)); }
        }
        __syncthreads();
        if (rg * RPT < R) {   // product with V
            #pragma unroll
            for (int i = 0; i < RPT; i++) {
                const float f = fade[rg * RPT + i];
                acc[i][0] *= f; acc[i][1] *= f; acc[i][2] *= f; acc[i][3] *= f;
            }
            const int n = min(C, hi - j0);
            for (int c = 0; c < n; c++) {
                const float4 v = *reinterpret_cast<const float4*>(vs + c * DP + dq * 4);
                #pragma unroll
                for (int i = 0; i < RPT; i++) {
                    const float w = ss[(rg * RPT + i) * (C + 1) + c];
                    acc[i][0] = __fmaf_rn(w, v.x, acc[i][0]); acc[i][1] = __fmaf_rn(w, v.y, acc[i][1]);
                    acc[i][2] = __fmaf_rn(w, v.z, acc[i][2]); acc[i][3] = __fmaf_rn(w, v.w, acc[i][3]);
                }
            }
        }
    }
    __syncthreads();
    if (rg * RPT < R)                                        // the queries are done with: their room holds the accumulator
        #pragma unroll
        for (int i = 0; i < RPT; i++)
            *reinterpret_cast<float4*>(qs + (rg * RPT + i) * DP + dq * 4) = make_float4(acc[i][0], acc[i][1], acc[i][2], acc[i][3]);
    __syncthreads();
    join_and_store<T, DP, kFmaThreads>(p, t, kv_head, qs, stats);
}

template <typename T, int R, int DP, int C> static bool launch_fma(const AttentionProblem& p) {
    const size_t smem = sizeof(float) * (size_t)(R * DP + C * (DP + 4) + C * DP + ((R * (C + 1) + 3) & ~3) + 3 * R + 2 * C);
    const int tiles = (int)attention_tiles(p, R);
    const int splits = attention_splits(p, tiles, 4 * kNumSMs, 2 * C);
    int count = tiles;
    AttentionProblem copy = p;
    void* args[] = {&copy, &count};
    return launch_attention((const void*)attention_fma_kernel<T, R, DP, C>, p, R, kFmaThreads, smem, splits, args, "attention_fma");
}

template <typename T, int R> static bool launch_fma_dim(const AttentionProblem& p) {
    if (p.dim <= 64) return launch_fma<T, R, 64, 64>(p);
    if (p.dim <= 128) return launch_fma<T, R, 128, 64>(p);
    return launch_fma<T, R, 256, 32>(p);
}

template <typename T> static bool launch_fma_rows(const AttentionProblem& p) {
    // rows per sequence on average: a single token's group does not fill 32
    const long long rows = (long long)p.queries * p.group / (p.page_table ? p.batch : 1);
    return rows <= 8 ? launch_fma_dim<T, 8>(p) : launch_fma_dim<T, 32>(p);
}

bool attention_fma(const AttentionProblem& p) {
    switch (p.dtype) {
        case DTYPE_FLOAT16:  return launch_fma_rows<__half>(p);
        case DTYPE_BFLOAT16: return launch_fma_rows<__nv_bfloat16>(p);
        default:             return launch_fma_rows<float>(p);
    }
}

}  // namespace tops
