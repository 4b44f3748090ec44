// Attention for 16-bit types whose cache the copy engine's boxes do not fit (pages that are neither a multiple of 8 that divides 128 nor a multiple of 128): keys are
// fetched row by row instead.
//
// A block owns 16 rows (token, head-of-the-group) of one key head: one m16 tile of mma.sync.m16n8k16.  With so few rows the tensor
// instruction is there to spare registers and issue slots, not for its rate: per KT keys a warp issues KT * dim / 64 of them, a
// tenth of what the load of the same keys takes.  Each of the four warps walks its own tiles of KT keys with a private ring
// of STAGES cp.async buffers -- no block-wide barrier in the loop --, keeps its own (m, l, o), and the warps, then the blocks of
// the cluster that share the sequence, join at the end.
//
// Measured (dim 128, 8 sequences of 4000 keys, 8 key heads, 16 rows each): 43 us, 3.0 TB/s.  Bound by the chain copy -> ldmatrix -> mma -> softmax of each warp with eight
// warps on an SM (ncu: issue slots 34 % busy); copies alone run at twice that.
#include "attention_common.cuh"

namespace tops {

constexpr int kRowsThreads = 128;
constexpr int kRowsWarps = kRowsThreads / 32;

template <typename T, int DP, int KT, int STAGES, bool MASKED>
__global__ void __launch_bounds__(kRowsThreads) attention_rows_kernel(const __grid_constant__ AttentionProblem p, const int tiles) {
    constexpr int CHUNKS = DP / 8;                          // 16-byte pieces of a padded row
    constexpr int ROW_BYTES = DP * 2;
    constexpr int TILE_BYTES = KT * ROW_BYTES;              // of K, and of V
    constexpr int PITCH = DP + 8;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ float2 warp_stats[kRowsWarps][16];
    __shared__ float2 stats[16];

    const int splits = (int)cluster_size(), rank = (int)cluster_rank();
    RowTile t;
    if (!locate_tile(p, tiles - 1 - (int)(blockIdx.x / (unsigned)splits), 16, t)) return;   // the whole cluster leaves
    const int kv_head = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int dim = p.dim;

    const int first = t.key_begin / KT, count = (t.key_end + KT - 1) / KT - first;
    const int share = (count + splits - 1) / splits;
    const int lo = first + min(rank * share, count), hi = first + min((rank + 1) * share, count);

    const long long kv_base = (p.page_table ? 0 : (long long)t.seq * p.kv_batch) + (long long)kv_head * p.kv_head;
    const T* kp = reinterpret_cast<const T*>(p.k) + kv_base;
    const T* vp = reinterpret_cast<const T*>(p.v) + kv_base;
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + (uint32_t)warp * (STAGES * 2 * TILE_BYTES);

    // cache row of the lane's key of a tile; -1 where nothing is to be read
    auto rows_of = [&](int tile) {
        const int j = tile * KT + lane;
        if (lane >= KT || tile >= hi || j < t.key_begin || j >= t.key_end) return -1;    // pages in front of a window may be gone
        if constexpr (MASKED) if (key_bias(p, t.seq, j) == -INFINITY) return -1;
        return key_row(p, t.seq, j);
    };
    const int my_chunk = lane % CHUNKS;
    const bool chunk_there = my_chunk * 8 < dim;
    auto issue = [&](int stage, int rows) {
        const uint32_t base = ring + (uint32_t)stage * (2 * TILE_BYTES);
        #pragma unroll
        for (int i = 0; i < KT * CHUNKS / 32; i++) {
            const int r = i * (32 / CHUNKS) + lane / CHUNKS;
            const int row = __shfl_sync(~0u, rows, r);
            const bool there = row >= 0 && chunk_there;
            const long long at = there ? (long long)row * p.kv_token + my_chunk * 8 : 0;
            const uint32_t to = base + (uint32_t)(r * ROW_BYTES + ((my_chunk ^ (r & 7)) << 4));
            copy_async_16(to, kp + at, there ? 16u : 0u);
            copy_async_16(to + TILE_BYTES, vp + at, there ? 16u : 0u);
        }
    };

    int next = lo + warp;
    #pragma unroll
    for (int s = 0; s < STAGES - 1; s++) {
        if (next < hi) issue(s, rows_of(next));
        copy_async_commit();
        next += kRowsWarps;
    }
    int next_rows = rows_of(next);

    // queries: the A fragments of every 16 dimensions
    const int r0 = lane >> 2, r1 = r0 + 8, pair = (lane & 3) * 2;
    uint32_t qf[DP / 16][4];
    {
        const T* q0 = r0 < t.rows ? reinterpret_cast<const T*>(p.q) + row_offset(p, t, kv_head, t.row0 + r0) : nullptr;
        const T* q1 = r1 < t.rows ? reinterpret_cast<const T*>(p.q) + row_offset(p, t, kv_head, t.row0 + r1) : nullptr;
        #pragma unroll
        for (int ks = 0; ks < DP / 16; ks++) {
            const int d = ks * 16 + pair;
            qf[ks][0] = q0 && d < dim ? *reinterpret_cast<const uint32_t*>(q0 + d) : 0u;
            qf[ks][1] = q1 && d < dim ? *reinterpret_cast<const uint32_t*>(q1 + d) : 0u;
            qf[ks][2] = q0 && d + 8 < dim ? *reinterpret_cast<const uint32_t*>(q0 + d + 8) : 0u;
            qf[ks][3] = q1 && d + 8 < dim ? *reinterpret_cast<const uint32_t*>(q1 + d + 8) : 0u;
        }
    }
    // keys each of the two rows sees: [low, high); rows past the tile's last compute on zeros and are not stored
    int high0 = t.key_end, high1 = t.key_end, low0 = 0, low1 = 0, all_low = 0, all_high = t.key_end;
    if (p.page_table) {
        auto position = [&](int r) { return t.first_position + (int)p.group_div.div((uint32_t)(t.row0 + min(r, t.rows - 1))); };
        high0 = position(r0) + 1;
        high1 = position(r1) + 1;
        all_high = position(0) + 1;
        if (p.window > 0) {
            low0 = high0 - p.window;
            low1 = high1 - p.window;
            all_low = position(15) + 1 - p.window;
        }
    }

    float o[DP / 8][4];
    #pragma unroll
    for (int i = 0; i < DP / 8; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f;

    int stage = 0;
    for (int tile = lo + warp; tile < hi; tile += kRowsWarps) {
        copy_async_wait<STAGES - 2>();
        __syncwarp();                                       // all lanes' pieces have landed, and the oldest buffer is read out
        if (next < hi) issue(stage == 0 ? STAGES - 1 : stage - 1, next_rows);
        copy_async_commit();
        next += kRowsWarps;
        next_rows = rows_of(next);

        const uint32_t ks_at = ring + (uint32_t)stage * (2 * TILE_BYTES), vs_at = ks_at + TILE_BYTES;
        float s[KT / 8][4];
        #pragma unroll
        for (int n = 0; n < KT / 8; n++) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
        #pragma unroll
        for (int ks = 0; ks < DP / 16; ks++) {
            if (ks * 16 < dim) {
                #pragma unroll
                for (int n = 0; n < KT / 16; n++) {
                    const int key = n * 16 + (lane >> 4) * 8 + (lane & 7), chunk = ks * 2 + ((lane >> 3) & 1);
                    uint32_t b[4];
                    load_matrix4(b, ks_at + (uint32_t)(key * ROW_BYTES + ((chunk ^ (key & 7)) << 4)));
                    mma16816<T>(s[2 * n], qf[ks], b[0], b[1]);
                    mma16816<T>(s[2 * n + 1], qf[ks], b[2], b[3]);
                }
            }
        }
        const int j0 = tile * KT;
        float top0 = -INFINITY, top1 = -INFINITY;
        #pragma unroll
        for (int n = 0; n < KT / 8; n++)
            #pragma unroll
            for (int e = 0; e < 4; e++) s[n][e] *= p.scale_log2;
        if (MASKED || j0 < all_low || j0 + KT > all_high) {
            float my_bias = 0.0f;
            if constexpr (MASKED) my_bias = lane < KT && j0 + lane < t.key_end ? key_bias(p, t.seq, j0 + lane) : -INFINITY;
            #pragma unroll
            for (int n = 0; n < KT / 8; n++)
                #pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int c = n * 8 + pair + e, j = j0 + c;
                    float bias = 0.0f;
                    if constexpr (MASKED) bias = __shfl_sync(~0u, my_bias, c);
                    const bool out = MASKED && bias == -INFINITY;
                    s[n][e] = j < high0 && j >= low0 && !out ? s[n][e] + bias : -INFINITY;
                    s[n][2 + e] = j < high1 && j >= low1 && !out ? s[n][2 + e] + bias : -INFINITY;
                }
        }
        #pragma unroll
        for (int n = 0; n < KT / 8; n++) {
            top0 = fmaxf(top0, fmaxf(s[n][0], s[n][1]));
            top1 = fmaxf(top1, fmaxf(s[n][2], s[n][3]));
        }
        top0 = fmaxf(top0, __shfl_xor_sync(~0u, top0, 1)); top0 = fmaxf(top0, __shfl_xor_sync(~0u, top0, 2));
        top1 = fmaxf(top1, __shfl_xor_sync(~0u, top1, 1)); top1 = fmaxf(top1, __shfl_xor_sync(~0u, top1, 2));
        if (__any_sync(~0u, top0 > m0 || top1 > m1)) {
            const float n0 = fmaxf(m0, top0), n1 = fmaxf(m1, top1);
            const float f0 = partial_weight(m0, n0), f1 = partial_weight(m1, n1);
            #pragma unroll
            for (int i = 0; i < DP / 8; i++) { o[i][0] *= f0; o[i][1] *= f0; o[i][2] *= f1; o[i][3] *= f1; }
            l0 *= f0; l1 *= f1;
            m0 = n0; m1 = n1;
        }
        const float base0 = m0 == -INFINITY ? 0.0f : m0, base1 = m1 == -INFINITY ? 0.0f : m1;
        uint32_t pf[KT / 16][4];                            // weights as A fragments; the sums keep the unrounded weights
        #pragma unroll
        for (int n = 0; n < KT / 8; n++) {
            const float a = exp2_approx(s[n][0] - base0), b = exp2_approx(s[n][1] - base0);
            const float c = exp2_approx(s[n][2] - base1), d = exp2_approx(s[n][3] - base1);
            l0 += a + b;
            l1 += c + d;
            pf[n >> 1][(n & 1) * 2] = pack2<T>(a, b);
            pf[n >> 1][(n & 1) * 2 + 1] = pack2<T>(c, d);
        }
        #pragma unroll
        for (int dn = 0; dn < DP / 16; dn++) {
            if (dn * 16 < dim) {
                #pragma unroll
                for (int n = 0; n < KT / 16; n++) {
                    const int key = n * 16 + ((lane >> 3) & 1) * 8 + (lane & 7), chunk = dn * 2 + (lane >> 4);
                    uint32_t b[4];
                    load_matrix4_trans(b, vs_at + (uint32_t)(key * ROW_BYTES + ((chunk ^ (key & 7)) << 4)));
                    mma16816<T>(o[2 * dn], pf[n], b[0], b[1]);
                    mma16816<T>(o[2 * dn + 1], pf[n], b[2], b[3]);
                }
            }
        }
        stage = stage == STAGES - 1 ? 0 : stage + 1;
    }

    // join the warps
    l0 += __shfl_xor_sync(~0u, l0, 1); l0 += __shfl_xor_sync(~0u, l0, 2);
    l1 += __shfl_xor_sync(~0u, l1, 1); l1 += __shfl_xor_sync(~0u, l1, 2);
    copy_async_wait<0>();
    __syncthreads();                                        // every warp has left its ring
    float* partial = reinterpret_cast<float*>(smem);        // [warps][16][PITCH]
    {
        float* mine = partial + warp * 16 * PITCH;
        if ((lane & 3) == 0) { warp_stats[warp][r0] = make_float2(m0, l0); warp_stats[warp][r1] = make_float2(m1, l1); }
        #pragma unroll
        for (int i = 0; i < DP / 8; i++) {
            *reinterpret_cast<float2*>(mine + r0 * PITCH + i * 8 + pair) = make_float2(o[i][0], o[i][1]);
            *reinterpret_cast<float2*>(mine + r1 * PITCH + i * 8 + pair) = make_float2(o[i][2], o[i][3]);
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < t.rows * (DP / 4); i += kRowsThreads) {
        const int r = i / (DP / 4), d = (i - r * (DP / 4)) * 4;
        float top = -INFINITY, l = 0.0f;
        #pragma unroll
        for (int w = 0; w < kRowsWarps; w++) top = fmaxf(top, warp_stats[w][r].x);
        float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        #pragma unroll
        for (int w = 0; w < kRowsWarps; w++) {
            const float f = partial_weight(warp_stats[w][r].x, top);
            const float4 x = *reinterpret_cast<const float4*>(partial + (w * 16 + r) * PITCH + d);
            l = __fmaf_rn(warp_stats[w][r].y, f, l);
            sum.x = __fmaf_rn(x.x, f, sum.x); sum.y = __fmaf_rn(x.y, f, sum.y); sum.z = __fmaf_rn(x.z, f, sum.z); sum.w = __fmaf_rn(x.w, f, sum.w);
        }
        *reinterpret_cast<float4*>(partial + r * PITCH + d) = sum;      // nobody else reads warp 0's element
        if (d == 0) stats[r] = make_float2(top, l);
    }
    __syncthreads();
    join_and_store<T, PITCH, kRowsThreads>(p, t, kv_head, partial, stats);
}

template <typename T, int DP, int KT, int STAGES> static bool launch_rows(const AttentionProblem& p) {
    const size_t smem = (size_t)kRowsWarps * STAGES * 2 * KT * DP * 2;
    int tiles = (int)attention_tiles(p, 16);
    const int splits = attention_splits(p, tiles, 8 * kNumSMs, 4 * kRowsWarps * KT);
    AttentionProblem copy = p;
    void* args[] = {&copy, &tiles};
    const bool masked = p.mask_kind != kMaskNone;
    const void* kernel = masked ? (const void*)attention_rows_kernel<T, DP, KT, STAGES, true> : (const void*)attention_rows_kernel<T, DP, KT, STAGES, false>;
    return launch_attention(kernel, p, 16, kRowsThreads, smem, splits, args, "attention_rows");
}

template <typename T> static bool launch_rows_dim(const AttentionProblem& p) {
    if (p.dim <= 64) return launch_rows<T, 64, 32, 3>(p);
    if (p.dim <= 128) return launch_rows<T, 128, 16, 3>(p);
    return launch_rows<T, 256, 16, 3>(p);
}

bool attention_rows(const AttentionProblem& p) {
    return p.dtype == DTYPE_FLOAT16 ? launch_rows_dim<__half>(p) : launch_rows_dim<__nv_bfloat16>(p);
}

}  // namespace tops
