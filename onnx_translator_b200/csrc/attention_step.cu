// Attention of few rows per key head (single new tokens, small groups of them) on the 5th-generation tensor cores.  HBM bound: the keys and
// values of a sequence are read once and nothing else may take as long.
//
// The scores are computed transposed, so that the many keys fill the 128 rows of the instruction and the few queries its N columns:
//   S^T[128 keys x N] = K[128 x dim] Q^T,      O^T[dim x N] += V^T[dim x 128] P^T
// K is the A operand as it lies in memory; V, [keys][dim], is A seen MN-major; Q and P are K-major B operands of N rows.  Both
// products take N = 16 columns for up to 16 rows: an eighth of the tensor time of a tile whose rows are the queries, and a thread
// of the softmax owns one key -- its mask, its visibility -- with the N scores of that key in registers.
//
// The maximum of a row would have to be taken across the threads.  Instead all rows keep a running reference m, and a tile only checks
// (one predicate, or-reduced by the barrier it needs anyway) that no score exceeds m by more than 8 in log2: the weights stay below
// 2^8, the sums are float32, and the quotient o / l does not depend on m.  When the check fails, about ln(tiles) times per row, the block
// takes the true maximum and rescales o and l.  Sums of weights stay per thread (per key) until the end.
//
// Rows are worked on four at a time: the columns between t.rows and the next multiple of four hold scores of zero queries and are dropped
// at the end (a branch per row cost more than the arithmetic of three idle ones).
//
// Warps 0-3 softmax, warp 4 copies (TMA, page by page, 128 keys of K or V per ring slot), warp 5 issues the MMAs.  Blocks of a cluster share a
// sequence's keys and join at the end; tensor memory is given back before that, so a block that waits for its peers holds none.
#include "attention_common.cuh"

#include <type_traits>

namespace tops {

void count_tensor_core_launch();

constexpr int kStepThreads = 192;
constexpr int kStepKeys = 128;

template <int DB, int N, int SLOTS> struct StepLayout {
    static constexpr int kSlotBytes = kStepKeys * 128 * DB;
    static constexpr int kQBytes = N * 128 * DB;
    static constexpr int kPBytes = N * 128 * 2;               // one of the two buffers
    static constexpr int kPitch = DB * 64 + 4;
    static constexpr int kSmem = SLOTS * kSlotBytes + kQBytes + 2 * kPBytes + 1024;   // and room to align
    static constexpr int kOAccs = DB > 2 ? 2 : 1;             // accumulators of 128 dimensions
    static constexpr uint32_t kColumns = (2 + kOAccs) * N <= 64 ? 64 : (2 + kOAccs) * N <= 128 ? 128 : 256;
    static_assert(SLOTS <= 8, "a slot's release is read from barriers of the last four tiles");
    static_assert(N * kPitch * 4 <= SLOTS * kSlotBytes, "the partial result reuses the ring");
};

// True for all 128 softmax threads if it is for one.
__device__ __forceinline__ bool any_of_softmax(bool x) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %1, 0;\n\t"
        "barrier.cta.red.or.pred p, 1, 128, q;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r) : "r"((uint32_t)x) : "memory");
    return r != 0;
}
__device__ __forceinline__ void softmax_sync() { asm volatile("barrier.cta.sync 1, 128;" ::: "memory"); }

template <int N> __device__ __forceinline__ void tmem_load_columns(uint32_t at, float (&x)[N]) {
    if constexpr (N == 16) {
        uint32_t r[16];
        umma::tmem_load_32x16(at, r);
        umma::tmem_load_wait();
        #pragma unroll
        for (int i = 0; i < 16; i++) x[i] = __uint_as_float(r[i]);
    } else {
        #pragma unroll
        for (int c = 0; c < N; c += 32) {
            uint32_t r[32];
            umma::tmem_load_32x32(at + c, r);
            umma::tmem_load_wait();
            #pragma unroll
            for (int i = 0; i < 32; i++) x[c + i] = __uint_as_float(r[i]);
        }
    }
}
// The N columns of one accumulator times the rows' factors.
template <int N> __device__ __forceinline__ void tmem_scale_columns(uint32_t at, const float* factor) {
    constexpr int W = N == 16 ? 16 : 32;
    #pragma unroll
    for (int c = 0; c < N; c += W) {
        uint32_t r[W];
        if constexpr (W == 16) umma::tmem_load_32x16(at + c, r); else umma::tmem_load_32x32(at + c, r);
        umma::tmem_load_wait();
        #pragma unroll
        for (int i = 0; i < W; i++) r[i] = __float_as_uint(__uint_as_float(r[i]) * factor[c + i]);
        if constexpr (W == 16) umma::tmem_store_32x16(at + c, r); else umma::tmem_store_32x32(at + c, r);
    }
    umma::tmem_store_wait();
}

constexpr float kNoMaximum = -3.402823466e+38f;               // finite, so that score - m is never Inf - Inf
constexpr float kMaximumSlack = 8.0f;

template <typename T, int DB, int N, int SLOTS>
__global__ void __launch_bounds__(kStepThreads)
attention_step_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                      const __grid_constant__ AttentionProblem p, const int tiles, const int box_rows) {
    using L = StepLayout<DB, N, SLOTS>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t full[SLOTS], s_full[4], p_ready[2], pv_done[4], drained;
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_word, drain_word;
    __shared__ float warp_top[4][N], fade[N], warp_sum[4][N];
    __shared__ int high[N];
    __shared__ float2 stats[N];
    uint8_t* ring = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t* q_tile = ring + SLOTS * L::kSlotBytes;
    uint8_t* p_tile = q_tile + L::kQBytes;

    const int splits = (int)cluster_size(), rank = (int)cluster_rank();
    const int kv_head = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    RowTile t;
    if (!locate_tile(p, tiles - 1 - (int)(blockIdx.x / (unsigned)splits), N, t)) return;    // the whole cluster leaves

    if (warp == 5) umma::tmem_alloc(&tmem_slot, L::kColumns);
    volatile int* abort_flag = &abort_word;

    const int first = t.key_begin / kStepKeys, count = (t.key_end + kStepKeys - 1) / kStepKeys - first;
    const int share = (count + splits - 1) / splits;
    const int lo = first + min(rank * share, count), hi = first + min((rank + 1) * share, count), n = hi - lo;

    // Copies (warp 4): load number g is the keys (g even) or values (g odd) of tile g / 2 of this block, into ring slot g % SLOTS.  The first SLOTS
    // of them need no slot to be given back and are started before the block has even met.
    int g = 0, box_row = -1, next_page = 0;
    uint32_t load_slot = 0, load_phase = 0;
    // A tile's pages are fetched a tile ahead and looked at only when the tile's turn comes, so that the copies never wait for the table.
    auto box_needed = [&](int tile, int j) { return tile < hi && lane * box_rows < kStepKeys && j < t.key_end; };
    auto fetch_page = [&](int tile) {
        const int j = tile * kStepKeys + lane * box_rows;
        const bool needed = p.page_table && box_needed(tile, j) && j + box_rows > t.key_begin;     // pages in front of a window may be gone
        return needed ? p.page_table[(long long)t.seq * p.table_width + (int)p.page_div.div((uint32_t)j)] : 0;
    };
    auto page_row = [&](int tile, int page) {                  // cache row of this lane's box of a tile; -1: nothing to copy
        const int j = tile * kStepKeys + lane * box_rows;
        if (!box_needed(tile, j)) return -1;
        if (!p.page_table) return j;
        const int outside = p.pages * p.page_size;             // a row outside the map reads as zeros
        if (j + box_rows <= t.key_begin) return outside;
        if ((unsigned)page >= (unsigned)p.pages) { report_bad_index(p); return outside; }
        return page * p.page_size + (j - (int)p.page_div.div((uint32_t)j) * p.page_size);
    };
    auto load = [&] {                                          // the whole warp; false when the block gives up
        if (g >= SLOTS) {                                      // the slot's last contents: keys are read out with their scores, values with their product
            const int old = g - SLOTS, i = old >> 1;
            if (!__all_sync(~0u, umma::mbar_wait((old & 1) ? &pv_done[i & 3] : &s_full[i & 3], (uint32_t)(i >> 2) & 1u, abort_flag))) return false;
        }
        const int boxes = __popc(__ballot_sync(~0u, box_row >= 0));
        uint8_t* to = ring + load_slot * L::kSlotBytes;
        const CUtensorMap* map = (g & 1) ? &v_map : &k_map;
        const int batch = p.page_table ? 0 : t.seq;
        if (umma::elect_one()) umma::mbar_expect_tx(&full[load_slot], (uint32_t)(boxes * box_rows) * 128u * DB);
        __syncwarp();
        for (int x = 0; x < boxes; x++) {
            const int row = __shfl_sync(~0u, box_row, x);
            if (umma::elect_one()) {
                #pragma unroll
                for (int b = 0; b < DB; b++) umma::tma_load_4d(to + b * (kStepKeys * 128) + x * box_rows * 128, map, &full[load_slot], b * 64, kv_head, row, batch);
            }
            __syncwarp();
        }
        if (g & 1) {
            box_row = page_row(lo + (g >> 1) + 1, next_page);
            next_page = fetch_page(lo + (g >> 1) + 2);
        }
        g++;
        if (++load_slot == SLOTS) { load_slot = 0; load_phase ^= 1u; }
        return true;
    };
    if (warp == 4) {
        if (lane == 0) {
            for (int s = 0; s < SLOTS; s++) umma::mbar_init(&full[s], 1);
            for (int b = 0; b < 4; b++) { umma::mbar_init(&s_full[b], 1); umma::mbar_init(&pv_done[b], 1); }
            for (int b = 0; b < 2; b++) umma::mbar_init(&p_ready[b], 128);
            umma::mbar_init(&drained, 1);
            abort_word = drain_word = 0;
            umma::mbar_fence_init();
        }
        __syncwarp();
        box_row = fetch_page(lo);
        next_page = fetch_page(lo + 1);
        box_row = page_row(lo, box_row);
        while (g < 2 * n && g < SLOTS) load();
    }

    // queries and zeroed weights into shared memory, the N rows 128 bytes each, 16-byte pieces XORed with the row as the swizzle wants
    for (int i = threadIdx.x; i < N * DB * 8; i += kStepThreads) {
        const int r = i / (DB * 8), c = i - r * (DB * 8);
        uint4 x = make_uint4(0, 0, 0, 0);
        if (r < t.rows && c * 8 < p.dim) x = *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.q) + row_offset(p, t, kv_head, t.row0 + r) + c * 8);
        *reinterpret_cast<uint4*>(q_tile + (c >> 3) * (N * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = x;
    }
    if (threadIdx.x < N) fade[threadIdx.x] = 1.0f;            // of the columns that no row uses
    for (int i = threadIdx.x; i < 2 * L::kPBytes / 16; i += kStepThreads) reinterpret_cast<uint4*>(p_tile)[i] = make_uint4(0, 0, 0, 0);
    if (threadIdx.x < N)
        high[threadIdx.x] = p.page_table ? t.first_position + (int)p.group_div.div((uint32_t)(t.row0 + min((int)threadIdx.x, t.rows - 1))) + 1 : t.key_end;
    umma::fence_proxy_async_smem();
    umma::fence_before_sync();
    __syncthreads();
    umma::fence_after_sync();
    const uint32_t tmem = tmem_slot, tmem_o = tmem + 2 * N;

    if (warp == 4) {
        while (g < 2 * n && load()) {}
        if (lane == 0) {                                       // no copy of this block is in flight when it leaves
            for (int k = min(g, SLOTS); k > 0; k--) {
                if (load_slot == 0) { load_slot = SLOTS; load_phase ^= 1u; }
                load_slot--;
                umma::mbar_wait(&full[load_slot], load_phase, &drain_word);
            }
        }
    } else if (warp == 5) {
        // ---- products: the whole warp waits, one elected lane issues --------------------------------------------------------
        constexpr uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
        constexpr uint32_t idesc_s = umma::instr_desc(fmt, fmt, 128, N), idesc_o = idesc_s | umma::kInstrAMnMajor;
        uint32_t slot = 0, phase = 0;
        auto wait = [&](uint64_t* bar, uint32_t parity) { return (bool)__all_sync(~0u, umma::mbar_wait(bar, parity, abort_flag)); };
        auto scores = [&](int i) {                             // S^T of tile i
            if (!wait(&full[slot], phase)) return false;
            umma::fence_after_sync();
            const uint64_t da = umma::smem_desc_k_major_sw128(ring + slot * L::kSlotBytes), db = umma::smem_desc_k_major_sw128(q_tile);
            if (umma::elect_one()) {
                #pragma unroll
                for (int b = 0; b < DB; b++)
                    #pragma unroll
                    for (int k = 0; k < 4; k++)
                        umma::mma_ss<false>(tmem + (i & 1) * N, da + (uint64_t)(b * (kStepKeys * 128 >> 4) + 2 * k), db + (uint64_t)(b * (N * 128 >> 4) + 2 * k), idesc_s, (uint32_t)(b | k));
                umma::mma_commit(&s_full[i & 3]);
            }
            __syncwarp();
            return true;
        };
        auto step = [&] { if (++slot == SLOTS) { slot = 0; phase ^= 1u; } };
        bool ok = n > 0 ? scores(0) : true;
        for (int i = 0; i < n && ok; i++) {
            step();                                            // this tile's values
            const uint32_t v_slot = slot, v_phase = phase;
            step();                                            // the next tile's keys
            ok = (i + 1 == n || scores(i + 1)) && wait(&p_ready[i & 1], (uint32_t)(i >> 1) & 1u) && wait(&full[v_slot], v_phase);
            if (!ok) break;
            umma::fence_after_sync();
            const uint64_t da = umma::smem_desc_mn_major_sw128(ring + v_slot * L::kSlotBytes, DB == 1 ? 0u : (uint32_t)(kStepKeys * 128));
            const uint64_t db = umma::smem_desc_k_major_sw128(p_tile + (i & 1) * L::kPBytes);
            if (umma::elect_one()) {
                #pragma unroll
                for (int a = 0; a < L::kOAccs; a++)
                    #pragma unroll
                    for (int k = 0; k < 8; k++)
                        umma::mma_ss<false>(tmem_o + a * N, da + (uint64_t)(a * 2 * (kStepKeys * 128 >> 4) + k * (2048 >> 4)),
                                            db + (uint64_t)((k >> 2) * (N * 128 >> 4) + 2 * (k & 3)), idesc_o, (uint32_t)(i | k));
                umma::mma_commit(&pv_done[i & 3]);
            }
            __syncwarp();
        }
        if (!ok) {
            if (umma::elect_one()) umma::mma_commit(&drained);
            __syncwarp();
            umma::mbar_wait(&drained, 0, &drain_word);
        }
    } else {
        // ---- softmax: a thread per key -------------------------------------------------------------------------------------
        const int key = threadIdx.x;
        const uint32_t lanes = (uint32_t)warp << 21;           // this warp's quarter of tensor memory
        int all_high = t.key_end, all_low = 0;
        if (p.page_table) {
            all_high = high[0];
            if (p.window > 0) all_low = high[N - 1] - p.window;
        }
        const bool masked = p.mask_kind != kMaskNone;
        float m[N], l[N];
        #pragma unroll
        for (int r = 0; r < N; r++) { m[r] = kNoMaximum; l[r] = 0.0f; }
        uint32_t slot = 0, phase = 0;
        bool ok = true;
        for (int i = 0; i < n; i++) {
            const int j0 = (lo + i) * kStepKeys, j = j0 + key;
            if (++slot == SLOTS) { slot = 0; phase ^= 1u; }    // the slot of this tile's values
            const bool edge = masked || j0 < all_low || j0 + kStepKeys > all_high;
            bool dead = false;                                 // a key that no row sees: its value must not reach the product
            float bias = 0.0f;
            if (edge) {
                dead = j >= t.key_end;
                if (masked && !dead) { bias = key_bias(p, t.seq, j); dead = bias == -INFINITY; }
            }
            if (!umma::mbar_wait(&s_full[i & 3], (uint32_t)(i >> 2) & 1u, abort_flag)) ok = false;
            umma::fence_after_sync();
            float z[N];
            tmem_load_columns<N>(tmem + lanes + (i & 1) * N, z);
            float over = -INFINITY;
            if (!edge) {
                #pragma unroll
                for (int c = 0; c < N; c += 4)
                    if (c < t.rows)
                        #pragma unroll
                        for (int r = c; r < c + 4; r++) { z[r] *= p.scale_log2; over = fmaxf(over, z[r] - m[r]); }
            } else {
                #pragma unroll
                for (int c = 0; c < N; c += 4)
                    if (c < t.rows)
                        #pragma unroll
                        for (int r = c; r < c + 4; r++) {
                            const bool seen = !dead && j < high[r] && (p.window == 0 || j >= high[r] - p.window);
                            z[r] = seen ? __fmaf_rn(z[r], p.scale_log2, bias) : -INFINITY;
                            over = fmaxf(over, z[r] - m[r]);
                        }
            }
            if (any_of_softmax(over > kMaximumSlack)) {
                #pragma unroll
                for (int c = 0; c < N; c += 4)
                    if (c < t.rows)
                        #pragma unroll
                        for (int r = c; r < c + 4; r++) {
                            float top = z[r];
                            #pragma unroll
                            for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
                            if (lane == 0) warp_top[warp][r] = top;
                        }
                softmax_sync();
                #pragma unroll
                for (int c = 0; c < N; c += 4)
                    if (c < t.rows)
                        #pragma unroll
                        for (int r = c; r < c + 4; r++) {
                            const float top = fmaxf(m[r], fmaxf(fmaxf(warp_top[0][r], warp_top[1][r]), fmaxf(warp_top[2][r], warp_top[3][r])));
                            const float f = exp2_approx(m[r] - top);
                            l[r] *= f;
                            m[r] = top;
                            if (key == r) fade[r] = f;
                        }
                softmax_sync();
                if (i > 0) {
                    if (!umma::mbar_wait(&pv_done[(i - 1) & 3], (uint32_t)((i - 1) >> 2) & 1u, abort_flag)) ok = false;
                    umma::fence_after_sync();
                    #pragma unroll
                    for (int a = 0; a < L::kOAccs; a++) tmem_scale_columns<N>(tmem_o + lanes + a * N, fade);
                }
            }
            if (i > 1 && !umma::mbar_wait(&pv_done[(i - 2) & 3], (uint32_t)((i - 2) >> 2) & 1u, abort_flag)) ok = false;    // the weights of tile i - 2 are read
            uint8_t* to = p_tile + (i & 1) * L::kPBytes + (key >> 6) * (N * 128) + (key & 7) * 2;
            #pragma unroll
            for (int c = 0; c < N; c += 4)
                if (c < t.rows)
                    #pragma unroll
                    for (int r = c; r < c + 4; r++) {
                        const float w = exp2_approx(z[r] - m[r]);
                        l[r] += w;
                        *reinterpret_cast<T*>(to + r * 128 + ((((key & 63) >> 3) ^ (r & 7)) << 4)) = from_float<T>(w);
                    }
            if (dead) {                                        // a weight of zero times a NaN would still be one
                if (!umma::mbar_wait(&full[slot], phase, abort_flag)) ok = false;
                uint8_t* row = ring + slot * L::kSlotBytes + key * 128;
                #pragma unroll
                for (int b = 0; b < DB; b++)
                    #pragma unroll
                    for (int c = 0; c < 8; c++) *reinterpret_cast<uint4*>(row + b * (kStepKeys * 128) + c * 16) = make_uint4(0, 0, 0, 0);
            }
            umma::fence_proxy_async_smem();
            umma::fence_before_sync();
            umma::mbar_arrive(&p_ready[i & 1]);
            if (++slot == SLOTS) { slot = 0; phase ^= 1u; }
            if (!ok) break;
        }
        if (n > 0) {
            if (ok) ok = umma::mbar_wait(&pv_done[(n - 1) & 3], (uint32_t)((n - 1) >> 2) & 1u, abort_flag);
            umma::fence_after_sync();
        }
        // o[r][d] into the ring (everything in it has been read), the sums of weights across the keys
        float* o = reinterpret_cast<float*>(ring);
        __syncwarp();
        if (n > 0) {
            #pragma unroll
            for (int a = 0; a < L::kOAccs; a++) {
                float x[N];
                tmem_load_columns<N>(tmem_o + lanes + a * N, x);
                const int d = a * 128 + key;
                if (d < DB * 64)
                    #pragma unroll
                    for (int r = 0; r < N; r++) if (r < t.rows) o[r * L::kPitch + d] = x[r];
            }
        }
        #pragma unroll
        for (int r = 0; r < N; r++) {
            if (r < t.rows) {
                float sum = l[r];
                #pragma unroll
                for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(~0u, sum, d);
                if (lane == 0) warp_sum[warp][r] = sum;
            }
        }
        softmax_sync();
        #pragma unroll
        for (int r = 0; r < N; r++)
            if (key == r && r < t.rows) {
                const float sum = (warp_sum[0][r] + warp_sum[1][r]) + (warp_sum[2][r] + warp_sum[3][r]);
                stats[r] = make_float2(sum == 0.0f ? -INFINITY : m[r], sum);
            }
    }
    umma::fence_before_sync();
    __syncthreads();
    if (threadIdx.x == 0 && abort_word && p.status) atomicExch(p.status, 1);
    if (warp == 5) {
        umma::fence_after_sync();
        umma::tmem_dealloc(tmem, L::kColumns);
    }
    join_and_store<T, L::kPitch, kStepThreads>(p, t, kv_head, reinterpret_cast<const float*>(ring), stats);
}

template <typename T, int DB, int N, int SLOTS> static bool launch_step(const AttentionProblem& p) {
    using L = StepLayout<DB, N, SLOTS>;
    int box_rows = cache_box_rows(p);
    CUtensorMap k_map, v_map;
    if (!make_cache_map(&k_map, p, p.k, box_rows) || !make_cache_map(&v_map, p, p.v, box_rows)) {
        set_error(TOPS_ERR_CUDA, "attention_step: the tensor map was refused");
        return false;
    }
    int tiles = (int)attention_tiles(p, N);
    const int splits = attention_splits(p, tiles, 8 * kNumSMs, kStepKeys);
    AttentionProblem copy = p;
    void* args[] = {&k_map, &v_map, &copy, &tiles, &box_rows};
    if (!launch_attention((const void*)attention_step_kernel<T, DB, N, SLOTS>, p, N, kStepThreads, L::kSmem, splits, args, "attention_step")) return false;
    count_tensor_core_launch();
    return true;
}

template <typename T> static bool launch_step_size(const AttentionProblem& p) {
    const long long rows = (long long)p.queries * p.group / (p.page_table ? p.batch : 1);
    if (p.dim <= 64) return rows <= 16 ? launch_step<T, 1, 16, 6>(p) : rows <= 32 ? launch_step<T, 1, 32, 6>(p) : launch_step<T, 1, 64, 8>(p);
    if (p.dim <= 128) return rows <= 16 ? launch_step<T, 2, 16, 3>(p) : rows <= 32 ? launch_step<T, 2, 32, 5>(p) : launch_step<T, 2, 64, 5>(p);
    return rows <= 16 ? launch_step<T, 4, 16, 3>(p) : launch_step<T, 4, 32, 2>(p);
}

bool attention_step(const AttentionProblem& p) {
    return p.dtype == DTYPE_FLOAT16 ? launch_step_size<__half>(p) : launch_step_size<__nv_bfloat16>(p);
}

}  // namespace tops
