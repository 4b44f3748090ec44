// Attention of many rows per key head (prompts, chunks of them, whole targets) on the 5th-generation tensor cores.  Tensor bound for dim 128, with the
// exponentials close behind: per 128 x 128 scores the two products take 2 * 4 * dim cycles of the tensor pipe and the 16384 exponentials 1024 cycles of
// the special-function units.
//
// A block works on two tiles of 128 rows (token, head of the group) of one key head against the same keys.  Per 128 keys and tile:
//   S[128 x 128] = Q[128 x dim] K^T      both operands K-major in shared memory, S in tensor memory
//   P = exp2(S * scale - m)              a thread per row: no exchange between threads; P goes back over S, as 16-bit, two to a column
//   O[128 x dim] += P V                  P is read from tensor memory, V is [keys][dim], an MN-major B operand, as it lies in memory
// The tiles alternate: while one is in its softmax the tensor pipe works for the other.  m is a running reference: it only follows the row maximum
// when that has grown by more than 8 in log2 (weights up to 2^8 are exact enough in 16 bits, sums are float32), so O is rarely rescaled; a row's threads do
// that themselves.
//
// As in the kernel for few rows the work is split evenly: all items -- (two row tiles, key head) with their keys -- stand in one row, weighted by the keys
// they see, and each of the 148 blocks takes an equal piece of it; pieces of items are joined by a second kernel.
//
// Measured (bf16, dim 128, 32 heads over 8 key heads): 2048 tokens over 32768 keys before them 1010 us, 1.12 PFLOP/s (0.67 of a cuBLAS burst), 1213 us when the card is at
// its power limit (0.93 PFLOP/s; cuBLAS 1.38 there); a prompt of 8192 tokens 500 us, 1.10 PFLOP/s.  A pair of tiles takes about 3450 cycles: a tile's softmax (2050:
// exponentials 1300, maximum 400, tensor memory and barriers 350) and its two products (1024, and more while both tiles compete) follow one another, and the other tile fills
// the gaps.  Tried and not kept: a quarter of the exponentials as a polynomial on the multiply-add units (1066 us), the product begun on the first 96 keys' weights (1040 us).
//
// Warps 0-3 and 4-7 softmax of the two tiles, warp 8 copies keys and values (TMA, page by page), warp 9 issues the MMAs, warp 10 finds the next item and
// copies its queries.
#include "attention_join.cuh"

#include <type_traits>

namespace tops {

void count_tensor_core_launch();

constexpr int kChunkThreads = 384;                          // three warpgroups: the last warp has no role
constexpr int kChunkKeys = 128;
constexpr int kChunkRows = 256;                               // row capacity of an item: two tiles

template <int DB, int SLOTS> struct ChunkLayout {
    static constexpr int kSlotBytes = kChunkKeys * 128 * DB;
    static constexpr int kQBytes = 128 * 128 * DB;            // one of the two tiles
    static constexpr int kDims = DB * 64;
    static constexpr int kSmem = SLOTS * kSlotBytes + 2 * kQBytes + 1024;
};

// ---- the row of all items ------------------------------------------------------------------------------------------------
// Sequence b has `count` items per key head; item i weighs base + slope * (i + 1): the keys it sees and kItemKeys for what an item costs besides
// (fetching queries, filling the pipeline, storing: as long as 400 keys, measured on items of 12 tiles).  Exactness only matters for the balance.
// All weights of a sequence have a closed sum, so a place in the row is found without walking the items.
constexpr int kItemKeys = 448;
struct ChunkSequence { int start, tokens, length, count, base, slope; };

__device__ __forceinline__ ChunkSequence chunk_sequence(const AttentionProblem& p, int b, int item_tokens) {
    ChunkSequence w = {0, 0, 0, 0, 0, 0};
    if (b >= p.batch) return w;
    if (p.page_table) {
        const int s = p.query_start[b], e = p.query_start[b + 1], length = p.kv_length[b];
        w.start = min(max(s, 0), p.queries);
        const int end = min(max(e, w.start), p.queries);
        w.tokens = end - w.start;
        w.length = min(max(length, 0), p.keys);
        if (w.start != s || end != e || w.length != length) report_bad_index(p);
        if (p.window > 0) w.base = max(1, (int)min((long long)w.length, (long long)p.window + item_tokens));
        else { w.base = max(0, w.length - w.tokens); w.slope = item_tokens; }
    } else {
        w.tokens = p.queries;
        w.length = p.kv_length ? min(max(p.kv_length[b], 0), p.keys) : p.keys;
        w.base = max(1, w.length);
    }
    w.base += kItemKeys;
    w.count = (w.tokens + item_tokens - 1) / item_tokens;
    return w;
}
__device__ __forceinline__ long long weight_of_first(const ChunkSequence& w, long long n) { return n * w.base + (long long)w.slope * (n * (n + 1) / 2); }

__device__ __forceinline__ long long chunk_total(const AttentionProblem& p, int item_tokens, const ChunkSequence& head) {     // head: the lane's own of the first 32, fetched before
    long long sum = 0;
    for (int b = threadIdx.x & 31; b < p.batch; b += 32) {
        const ChunkSequence w = b < 32 ? head : chunk_sequence(p, b, item_tokens);
        sum += weight_of_first(w, w.count);
    }
    #pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(~0u, sum, d);
    return sum * p.kv_heads;
}

struct ChunkPlace { ChunkSequence w; int seq, item, kv_head; long long offset, weight; };

__device__ __forceinline__ ChunkPlace chunk_place(const AttentionProblem& p, long long x, int item_tokens, const ChunkSequence& head) {
    const int lane = threadIdx.x & 31;
    ChunkPlace at = {};
    long long before = 0;
    for (int base = 0; base < p.batch; base += 32) {
        const ChunkSequence w = base == 0 ? head : chunk_sequence(p, base + lane, item_tokens);
        const long long mine = weight_of_first(w, w.count) * p.kv_heads;
        long long sum = mine;
        #pragma unroll
        for (int d = 1; d < 32; d <<= 1) { const long long o = __shfl_up_sync(~0u, sum, d); if (lane >= d) sum += o; }
        const unsigned past = __ballot_sync(~0u, x < before + sum);
        if (past) {
            const int l = __ffs(past) - 1;
            at.seq = base + l;
            at.w.start = __shfl_sync(~0u, w.start, l);
            at.w.tokens = __shfl_sync(~0u, w.tokens, l);
            at.w.length = __shfl_sync(~0u, w.length, l);
            at.w.count = __shfl_sync(~0u, w.count, l);
            at.w.base = __shfl_sync(~0u, w.base, l);
            at.w.slope = __shfl_sync(~0u, w.slope, l);
            const long long inside = x - before - __shfl_sync(~0u, sum - mine, l);
            int lo = 0, hi = at.w.count - 1;                   // the last item whose predecessors weigh no more than `inside`
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if (weight_of_first(at.w, mid) * p.kv_heads <= inside) lo = mid; else hi = mid - 1;
            }
            at.item = lo;
            at.weight = (long long)at.w.base + (long long)at.w.slope * (lo + 1);
            const long long rest = inside - weight_of_first(at.w, lo) * p.kv_heads;
            at.kv_head = (int)(rest / at.weight);
            at.offset = rest - at.kv_head * at.weight;
            break;
        }
        before += __shfl_sync(~0u, sum, 31);
    }
    return at;
}

__device__ __forceinline__ RowTile chunk_rows(const AttentionProblem& p, const ChunkPlace& at, int item_tokens) {
    RowTile t;
    t.seq = at.seq;
    const int first = at.item * item_tokens, tokens = min(item_tokens, at.w.tokens - first);
    t.row0 = first * p.group;
    t.rows = tokens * p.group;
    t.token0 = at.w.start;
    t.length = t.key_end = at.w.length;
    t.key_begin = 0;
    if (p.page_table) {
        t.first_position = at.w.length - at.w.tokens;
        t.key_end = max(0, min(t.length, t.first_position + first + tokens));
        if (p.window > 0) t.key_begin = min(max(0, t.first_position + first - p.window + 1), t.key_end);
    }
    return t;
}

struct ChunkSegment {
    RowTile t;
    int kv_head;
    int lo, n;                   // 128-key tiles lo .. lo + n - 1; n < 0: no more segments
    int part;                    // scratch slot of the partial result, -1: the item is whole
    int second;                  // whether the second row tile has rows
    int pages[16];               // pages of tile lo
};

// Two floats at a time: x * scale + base, and running sums.
__device__ __forceinline__ void fma2(float& x0, float& x1, float scale, float base) {
    asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %2};\n\tmov.b64 c, {%3, %3};\n\t"
        "fma.rn.f32x2 a, a, b, c;\n\tmov.b64 {%0, %1}, a;\n\t}" : "+f"(x0), "+f"(x1) : "f"(scale), "f"(base));
}
__device__ __forceinline__ void add2(float& s0, float& s1, float x0, float x1) {
    asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %3};\n\tadd.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}"
        : "+f"(s0), "+f"(s1) : "f"(x0), "f"(x1));
}

constexpr float kChunkSlack = 8.0f;

template <typename T, int DB, int SLOTS, bool MASKED>
__global__ void __launch_bounds__(kChunkThreads, 1)
attention_chunk_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                       const __grid_constant__ AttentionProblem p, const int box_rows, const int tile_tokens, const PartialResults parts) {
    using L = ChunkLayout<DB, SLOTS>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t full[SLOTS], empty[SLOTS], q_full, q_empty, s_full[2], p_ready[2], pv_done[2], o_full[2], seg_full[2], seg_empty[2], drained;
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_word, drain_word;
    __shared__ __align__(16) unsigned char segment_memory[2 * sizeof(ChunkSegment)];
    __shared__ __align__(16) float warp_bias[MASKED ? 8 : 1][MASKED ? kChunkKeys : 4];    // every softmax warp its own: warps never wait for one another
    ChunkSegment* segments = reinterpret_cast<ChunkSegment*>(segment_memory);
    uint8_t* q_tiles = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t* ring = q_tiles + 2 * L::kQBytes;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    volatile int* abort_flag = &abort_word;
    const int item_tokens = 2 * tile_tokens, tile_rows = tile_tokens * p.group;

    if (threadIdx.x == 0) {
        for (int s = 0; s < SLOTS; s++) { umma::mbar_init(&full[s], 1); umma::mbar_init(&empty[s], 1); }
        umma::mbar_init(&q_full, 1);
        umma::mbar_init(&q_empty, 1);
        for (int b = 0; b < 2; b++) {
            umma::mbar_init(&s_full[b], 1); umma::mbar_init(&p_ready[b], 128); umma::mbar_init(&pv_done[b], 1); umma::mbar_init(&o_full[b], 1);
            umma::mbar_init(&seg_full[b], 1); umma::mbar_init(&seg_empty[b], 10);      // copies, products, eight softmax warps
        }
        umma::mbar_init(&drained, 1);
        abort_word = drain_word = 0;
        umma::mbar_fence_init();
    }
    if (warp == 8 && lane == 0) { umma::tma_prefetch_desc(&k_map); umma::tma_prefetch_desc(&v_map); umma::tma_prefetch_desc(&q_map); }
    asm volatile("griddepcontrol.wait;" ::: "memory");         // nothing so far has touched global or tensor memory
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    ChunkSequence head = {0, 0, 0, 0, 0, 0};
    if (warp == 10) head = chunk_sequence(p, lane, item_tokens);
    if (warp == 9) umma::tmem_alloc(&tmem_slot, 512);
    umma::fence_before_sync();
    __syncthreads();
    umma::fence_after_sync();
    const uint32_t tmem = tmem_slot;                           // S / P of the two tiles at columns 0 and 128, O at 256 and 384
    auto wait = [&](uint64_t* bar, uint32_t parity) { return (bool)__all_sync(~0u, umma::mbar_wait(bar, parity, abort_flag)); };   // a whole warp

    // 384 threads start with 168 registers each, 64512 in all; 2 * 128 * 208 + 128 * 80 = 63488 of them go to where the scores are held
    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
        if (warp == 10) {
            // ---- items and their queries ------------------------------------------------------------------------------------
            const long long total = chunk_total(p, item_tokens, head);
            const long long share = (total + gridDim.x - 1) / gridDim.x;
            const long long x0 = min((long long)blockIdx.x * share, total), x1 = min(x0 + share, total);
            long long x = x0;
            JoinJob job;
            int loaded = 0;                                        // items whose queries were copied
            for (int s = 0;; s++) {
                const int buf = s & 1;
                ChunkSegment seg;
                seg.n = -1;
                int page = 0, item_first = 0;
                if (x < x1) {
                    const ChunkPlace at = chunk_place(p, x, item_tokens, head);
                    seg.t = chunk_rows(p, at, item_tokens);
                    item_first = at.item * item_tokens;
                    seg.kv_head = at.kv_head;
                    seg.second = seg.t.rows > tile_rows;
                    const long long take = min(at.weight - at.offset, x1 - x);
                    const int first = seg.t.key_begin / kChunkKeys;
                    const int all = seg.t.key_end > seg.t.key_begin ? (seg.t.key_end + kChunkKeys - 1) / kChunkKeys - first : 0;
                    // a place inside the item's weight as a number of its tiles; the item's end is all of them
                    auto tiles_at = [&](long long o) { return o >= at.weight ? all : (int)min((long long)all, max(o - kItemKeys + kChunkKeys - 1, 0ll) / kChunkKeys); };
                    const int from = tiles_at(at.offset), to = tiles_at(at.offset + take);
                    seg.lo = first + from;
                    seg.n = to - from;
                    if constexpr (MASKED) trim_masked(p, seg.t.seq, seg.t.key_end, seg.lo, seg.n);
                    seg.part = at.offset == 0 && take == at.weight ? -1 : (int)blockIdx.x * 2 + (x == x0 ? 0 : 1);
                    if (seg.part >= 0 && at.offset <= x - x0 && x - at.offset + at.weight > x1)
                        job = JoinJob{seg.t, seg.kv_head, (int)((x - at.offset + at.weight - 1) / share) - (int)blockIdx.x + 1, seg.part};
                    x += take;
                    const int j = seg.lo * kChunkKeys + lane * box_rows;
                    if (p.page_table && seg.n > 0 && lane * box_rows < kChunkKeys && j < seg.t.key_end && j + box_rows > seg.t.key_begin)
                        page = p.page_table[(long long)seg.t.seq * p.table_width + (int)p.page_div.div((uint32_t)j)];
                }
                if (s > 1 && !wait(&seg_empty[buf], (uint32_t)((s >> 1) - 1) & 1u)) break;
                if (lane < 16) segments[buf].pages[lane] = page;
                if (lane == 0) {
                    segments[buf].t = seg.t;
                    segments[buf].kv_head = seg.kv_head;
                    segments[buf].lo = seg.lo;
                    segments[buf].n = seg.n;
                    segments[buf].part = seg.part;
                    segments[buf].second = seg.second;
                    asm volatile("fence.acq_rel.cta;" ::: "memory");
                }
                __syncwarp();
                if (lane == 0) umma::mbar_arrive(&seg_full[buf]);
                if (seg.n < 0) break;
                if (seg.n > 0) {
                    if (loaded > 0 && !wait(&q_empty, (uint32_t)(loaded - 1) & 1u)) break;       // the last item's scores are all there
                    const int tiles = seg.second ? 2 : 1, token = (p.page_table ? seg.t.token0 : 0) + item_first, batch = p.page_table ? 0 : seg.t.seq;
                    if (umma::elect_one()) umma::mbar_expect_tx(&q_full, (uint32_t)(tiles * tile_rows) * 128u * DB);
                    __syncwarp();
                    for (int q = 0; q < tiles; q++)
                        if (umma::elect_one()) {
                            #pragma unroll
                            for (int b = 0; b < DB; b++)
                                umma::tma_load_5d(q_tiles + q * L::kQBytes + b * (128 * 128), &q_map, &q_full, b * 64, 0, seg.kv_head, token + q * tile_tokens, batch);
                        }
                    __syncwarp();
                    loaded++;
                }
            }
            if (lane == 0) parts.jobs[blockIdx.x] = job;
            if (loaded > 0 && lane == 0) umma::mbar_wait(&q_full, (uint32_t)(loaded - 1) & 1u, &drain_word);     // none of its copies is in flight when the block leaves
        } else if (warp == 8) {
            // ---- keys and values: load number g is the keys (g even) or values (g odd) of this block's tile g / 2, into ring slot g % SLOTS ----
            int g = 0;
            uint32_t slot = 0, phase = 0;
            bool alive = true;
            for (int s = 0; alive; s++) {
                if (!wait(&seg_full[s & 1], (uint32_t)(s >> 1) & 1u)) break;
                const ChunkSegment& seg = segments[s & 1];
                const int n = seg.n, lo = seg.lo, key_begin = seg.t.key_begin, key_end = seg.t.key_end, kv_head = seg.kv_head, sequence = seg.t.seq;
                const int batch = p.page_table ? 0 : sequence;
                int page = seg.pages[lane & 15];
                __syncwarp();
                if (n < 0) break;
                auto box_needed = [&](int j) { return lane * box_rows < kChunkKeys && j < key_end; };
                for (int i = 0; i < n && alive; i++) {
                    const int j = (lo + i) * kChunkKeys + lane * box_rows;
                    int row = -1;                                  // cache row of this lane's box; -1: nothing to copy
                    if (box_needed(j)) {
                        row = j;
                        if (p.page_table) {
                            row = p.pages * p.page_size;           // a row outside the map reads as zeros
                            if (j + box_rows > key_begin) {        // pages in front of a window may be gone
                                if ((unsigned)page < (unsigned)p.pages) row = page * p.page_size + (j - (int)p.page_div.div((uint32_t)j) * p.page_size);
                                else report_bad_index(p);
                            }
                        }
                    }
                    const int next_j = j + kChunkKeys;             // the next tile's pages, looked at when its turn comes
                    if (p.page_table && i + 1 < n && box_needed(next_j) && next_j + box_rows > key_begin)
                        page = p.page_table[(long long)sequence * p.table_width + (int)p.page_div.div((uint32_t)next_j)];
                    const int boxes = __popc(__ballot_sync(~0u, row >= 0));
                    #pragma unroll 1
                    for (int kv = 0; kv < 2; kv++, g++) {
                        if (g >= SLOTS && !wait(&empty[slot], phase ^ 1u)) { alive = false; break; }
                        uint8_t* to = ring + slot * L::kSlotBytes;
                        const CUtensorMap* map = kv ? &v_map : &k_map;
                        if (umma::elect_one()) umma::mbar_expect_tx(&full[slot], (uint32_t)(boxes * box_rows) * 128u * DB);
                        __syncwarp();
                        for (int x = 0; x < boxes; x++) {
                            const int box_row = __shfl_sync(~0u, row, x);
                            if (umma::elect_one()) {
                                #pragma unroll
                                for (int b = 0; b < DB; b++) umma::tma_load_4d(to + b * (kChunkKeys * 128) + x * box_rows * 128, map, &full[slot], b * 64, kv_head, box_row, batch);
                            }
                            __syncwarp();
                        }
                        if (++slot == SLOTS) { slot = 0; phase ^= 1u; }
                    }
                }
                if (lane == 0) umma::mbar_arrive(&seg_empty[s & 1]);
            }
            if (lane == 0) {                                       // no copy of this block is in flight when it leaves
                for (int k = min(g, SLOTS); k > 0; k--) {
                    if (slot == 0) { slot = SLOTS; phase ^= 1u; }
                    slot--;
                    umma::mbar_wait(&full[slot], phase, &drain_word);
                }
            }
        } else if (warp == 9) {
            // ---- products: the whole warp waits, one elected lane issues ------------------------------------------------------
            constexpr uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
            constexpr uint32_t idesc_s = umma::instr_desc(fmt, fmt, 128, kChunkKeys), idesc_o = umma::instr_desc(fmt, fmt, 128, L::kDims) | umma::kInstrBMnMajor;
            uint32_t slot = 0, phase = 0;
            auto step = [&] { if (++slot == SLOTS) { slot = 0; phase ^= 1u; } };
            int items = 0;
            uint32_t weights_of[2] = {0u, 0u};                     // tiles of weights read so far, per row tile
            bool ok = true;
            // scores of row tile q against the keys in k_slot
            auto scores = [&](int q, uint32_t k_slot, bool frees_keys, bool frees_queries) {
                const uint64_t da = umma::smem_desc_k_major_sw128(q_tiles + q * L::kQBytes), db = umma::smem_desc_k_major_sw128(ring + k_slot * L::kSlotBytes);
                if (umma::elect_one()) {
                    #pragma unroll
                    for (int b = 0; b < DB; b++)
                        #pragma unroll
                        for (int k = 0; k < 4; k++)
                            umma::mma_ss<false>(tmem + q * 128, da + (uint64_t)(b * (128 * 128 >> 4) + 2 * k), db + (uint64_t)(b * (kChunkKeys * 128 >> 4) + 2 * k), idesc_s, (uint32_t)(b | k));
                    umma::mma_commit(&s_full[q]);
                    if (frees_keys) umma::mma_commit(&empty[k_slot]);
                    if (frees_queries) umma::mma_commit(&q_empty);
                }
                __syncwarp();
            };
            for (int s = 0; ok; s++) {
                if (!wait(&seg_full[s & 1], (uint32_t)(s >> 1) & 1u)) { ok = false; break; }
                const int n = segments[s & 1].n, tiles = segments[s & 1].second ? 2 : 1;
                __syncwarp();
                if (n < 0) break;
                if (lane == 0) umma::mbar_arrive(&seg_empty[s & 1]);
                if (n == 0) continue;
                ok = wait(&q_full, (uint32_t)items & 1u) && wait(&full[slot], phase);
                if (!ok) break;
                items++;
                umma::fence_after_sync();
                for (int q = 0; q < tiles; q++) scores(q, slot, q == tiles - 1, n == 1 && q == tiles - 1);
                step();
                for (int i = 0; i < n && ok; i++) {
                    const uint32_t v_slot = slot;
                    if (!wait(&full[slot], phase)) { ok = false; break; }
                    step();
                    const uint32_t k_slot = slot, k_phase = phase;
                    if (i + 1 < n) step();
                    const uint64_t db = umma::smem_desc_mn_major_sw128(ring + v_slot * L::kSlotBytes, (uint32_t)(kChunkKeys * 128));
                    for (int q = 0; q < tiles; q++) {
                        if (!wait(&p_ready[q], weights_of[q] & 1u)) { ok = false; break; }
                        weights_of[q]++;
                        umma::fence_after_sync();
                        if (umma::elect_one()) {
                            #pragma unroll
                            for (int k = 0; k < 8; k++)
                                umma::mma_ts_f16(tmem + 256 + q * 128, tmem + q * 128 + k * 8, db + (uint64_t)(k * (2048 >> 4)), idesc_o, (uint32_t)(i | k));
                            umma::mma_commit(&pv_done[q]);
                            if (i == n - 1) umma::mma_commit(&o_full[q]);
                            if (q == tiles - 1) umma::mma_commit(&empty[v_slot]);
                        }
                        __syncwarp();
                        if (i + 1 < n) {
                            if (q == 0) {
                                if (!wait(&full[k_slot], k_phase)) { ok = false; break; }
                                umma::fence_after_sync();
                            }
                            scores(q, k_slot, q == tiles - 1, i + 2 == n && q == tiles - 1);
                        }
                    }
                }
            }
            if (!ok) {
                if (umma::elect_one()) umma::mma_commit(&drained);
                __syncwarp();
                umma::mbar_wait(&drained, 0, &drain_word);
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        // ---- softmax: a thread per row -------------------------------------------------------------------------------------
        const int group = warp >> 2, quarter = warp & 3, row = quarter * 32 + lane;
        const uint32_t lanes = (uint32_t)quarter << 21;        // this warp's quarter of tensor memory
        const uint32_t s_at = tmem + lanes + group * 128, o_at = tmem + lanes + 256 + group * 128;
        const float scale = p.scale_log2, per_scale = 1.0f / p.scale_log2;
        uint32_t slot = 0, phase = 0;                          // of the ring, both row tiles use every tile of keys
        uint32_t mine = 0, items = 0;                          // tiles of scores and items of this row tile so far
        bool ok = true;
        for (int s = 0; ok; s++) {
            ok = wait(&seg_full[s & 1], (uint32_t)(s >> 1) & 1u);
            if (!ok) break;
            const ChunkSegment& seg = segments[s & 1];
            const int n = seg.n;
            if (n < 0) break;
            const RowTile t = seg.t;
            const int lo = seg.lo, part = seg.part, kv_head = seg.kv_head, used = group == 0 || seg.second;
            __syncwarp();
            if (lane == 0) umma::mbar_arrive(&seg_empty[s & 1]);
            if (!used) {
                const uint32_t moved = slot + 2u * (uint32_t)n;
                slot = moved % SLOTS;
                phase ^= (moved / SLOTS) & 1u;
                continue;
            }
            const int r = group * tile_rows + row;             // row of the item
            const bool valid = row < tile_rows && r < t.rows;
            int high = t.key_end, low = 0, all_high = t.key_end, all_low = 0;
            if (p.page_table) {
                high = t.first_position + (int)p.group_div.div((uint32_t)(t.row0 + min(r, t.rows - 1))) + 1;
                all_high = __reduce_min_sync(~0u, high);
                if (p.window > 0) { low = high - p.window; all_low = __reduce_max_sync(~0u, low); }
            }
            uint32_t mask_raw[4] = {0u, 0u, 0u, 0u};
            if constexpr (MASKED) if (n > 0) load_mask(p, t.seq, lo * kChunkKeys + lane, t.key_end, mask_raw);
            float m = -INFINITY, l0 = 0.0f, l1 = 0.0f;          // m in units of the raw score
            for (int i = 0; i < n; i++) {
                const int j0 = (lo + i) * kChunkKeys;
                if (++slot == SLOTS) { slot = 0; phase ^= 1u; }    // the slot of this tile's values
                bool dead = j0 + row >= t.key_end;             // a key that no row sees: its value must not reach the product
                bool biased = false;
                if constexpr (MASKED) {
                    __syncwarp();                              // the last tile's biases have been read
                    bool some = false;
                    float four[4];
                    mask_values(p, mask_raw, j0 + lane, t.key_end, four);
                    load_mask(p, t.seq, j0 + kChunkKeys + lane, i + 1 < n ? t.key_end : 0, mask_raw);      // the next tile's, on their way during this one
                    #pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float b = four[e];
                        warp_bias[warp][e * 32 + lane] = b * per_scale;       // in units of the raw score
                        some = some || b != 0.0f;
                        if (e == quarter) dead = b == -INFINITY;
                    }
                    __syncwarp();
                    biased = __any_sync(~0u, some);
                }
                ok = wait(&s_full[group], mine & 1u);
                if (!ok) break;
                umma::fence_after_sync();
                float x[128];
                #pragma unroll
                for (int c = 0; c < 128; c += 32) umma::tmem_load_32x32(s_at + c, *reinterpret_cast<uint32_t (*)[32]>(x + c));
                umma::tmem_load_wait();
                if (MASKED && biased) {
                    #pragma unroll
                    for (int c = 0; c < 128; c += 4) {
                        const float4 b = *reinterpret_cast<const float4*>(&warp_bias[warp][c]);
                        const float bias[4] = {b.x, b.y, b.z, b.w};
                        #pragma unroll
                        for (int e = 0; e < 4; e++) x[c + e] = bias[e] == -INFINITY ? -INFINITY : x[c + e] + bias[e];
                    }
                }
                if (!MASKED && (j0 < all_low || j0 + kChunkKeys > all_high)) {
                    const int to = high - j0, from = low - j0;
                    #pragma unroll
                    for (int c = 0; c < 128; c++) x[c] = c < to && c >= from ? x[c] : -INFINITY;
                }
                float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                #pragma unroll
                for (int c = 0; c < 128; c += 8)
                    #pragma unroll
                    for (int e = 0; e < 4; e++) top[e] = fmaxf(top[e], fmaxf(x[c + 2 * e], x[c + 2 * e + 1]));
                const float most = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
                if (__any_sync(~0u, valid && (most - m) * scale > kChunkSlack)) {
                    const float next = fmaxf(m, most);
                    const float f = m == -INFINITY ? 0.0f : exp2_approx((m - next) * scale);
                    m = next;
                    l0 *= f; l1 *= f;
                    if (i > 0) {
                        ok = wait(&pv_done[group], (mine - 1) & 1u);
                        if (!ok) break;
                        umma::fence_after_sync();
                        #pragma unroll 1
                        for (int c = 0; c < L::kDims; c += 32) {
                            uint32_t o[32];
                            umma::tmem_load_32x32(o_at + c, o);
                            umma::tmem_load_wait();
                            #pragma unroll
                            for (int e = 0; e < 32; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                            umma::tmem_store_32x32(o_at + c, o);
                        }
                    }
                }
                const float base = m == -INFINITY ? 0.0f : -m * scale;
                if (dead) {                                    // a weight of zero times a NaN would still be one
                    if (!umma::mbar_wait(&full[slot], phase, abort_flag)) ok = false;
                    uint8_t* key = ring + slot * L::kSlotBytes + row * 128;
                    #pragma unroll
                    for (int b = 0; b < DB; b++)
                        #pragma unroll
                        for (int c = 0; c < 8; c++) *reinterpret_cast<uint4*>(key + b * (kChunkKeys * 128) + c * 16) = make_uint4(0, 0, 0, 0);
                    umma::fence_proxy_async_smem();
                }
                #pragma unroll
                for (int c = 0; c < 128; c += 64) {
                    uint32_t w[32];
                    #pragma unroll
                    for (int e = 0; e < 64; e += 2) {
                        float &a = x[c + e], &b = x[c + e + 1];
                        fma2(a, b, scale, base);
                        a = exp2_approx(a);
                        b = exp2_approx(b);
                        add2(l0, l1, a, b);
                        w[e / 2] = pack2<T>(a, b);
                    }
                    umma::tmem_store_32x32(s_at + c / 2, w);
                }
                umma::tmem_store_wait();
                __syncwarp();
                umma::fence_before_sync();
                umma::mbar_arrive(&p_ready[group]);
                mine++;
                if (++slot == SLOTS) { slot = 0; phase ^= 1u; }
            }
            ok = __all_sync(~0u, ok);
            if (!ok) break;
            // the item's (or its part's) result
            const float l = l0 + l1;
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            if (n > 0) {
                ok = wait(&o_full[group], items & 1u);
                if (!ok) break;
                items++;
                umma::fence_after_sync();
            }
            if (part >= 0) {
                if (valid) parts.stats[(long long)part * kChunkRows + r] = make_float2(l == 0.0f ? -INFINITY : m * scale, l);
                float* to = parts.o + ((long long)part * kChunkRows + r) * L::kDims;
                #pragma unroll 1
                for (int c = 0; c < L::kDims; c += 32) {
                    uint32_t o[32];
                    umma::tmem_load_32x32(o_at + c, o);
                    umma::tmem_load_wait();
                    if (valid && n > 0)
                        #pragma unroll
                        for (int e = 0; e < 32; e += 4) *reinterpret_cast<uint4*>(to + c + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                }
            } else {
                T* to = valid ? reinterpret_cast<T*>(p.y) + row_offset(p, t, kv_head, t.row0 + r) : nullptr;
                #pragma unroll 1
                for (int c = 0; c < L::kDims; c += 32) {
                    uint32_t o[32];
                    umma::tmem_load_32x32(o_at + c, o);
                    umma::tmem_load_wait();
                    if (valid)
                        #pragma unroll
                        for (int e = 0; e < 32; e += 8) {
                            if (c + e >= p.dim) break;         // dim is a multiple of eight
                            float y[8];
                            #pragma unroll
                            for (int k = 0; k < 8; k++) y[k] = inv == 0.0f ? 0.0f : __uint_as_float(o[e + k]) * inv;
                            *reinterpret_cast<uint4*>(to + c + e) = make_uint4(pack2<T>(y[0], y[1]), pack2<T>(y[2], y[3]), pack2<T>(y[4], y[5]), pack2<T>(y[6], y[7]));
                        }
                }
            }
            umma::fence_before_sync();                         // the next item's first weights are only published after these loads
        }
    }
    umma::fence_before_sync();
    __syncthreads();
    if (threadIdx.x == 0 && abort_word && p.status) atomicExch(p.status, 1);
    if (warp == 9) {
        umma::fence_after_sync();
        umma::tmem_dealloc(tmem, 512);
    }
}

// Map over q: (dim, head of the group, key head, token, batch) in boxes of 64 x group x 1 x tile_tokens x 1.
static bool make_query_map(CUtensorMap* map, const AttentionProblem& p, int tile_tokens) {
    const uint64_t dims[5] = {(uint64_t)p.dim, (uint64_t)p.group, (uint64_t)p.kv_heads, (uint64_t)p.queries, p.page_table ? 1u : (uint64_t)p.batch};
    const uint64_t whole = (uint64_t)p.queries * p.heads * p.dim * 2;
    const uint64_t strides[4] = {(uint64_t)p.q_head * 2, (uint64_t)p.q_head * p.group * 2, (uint64_t)p.q_token * 2, whole};
    const uint32_t box[5] = {64, (uint32_t)p.group, 1, (uint32_t)tile_tokens, 1};
    return make_tensor_map(map, p.q, 2, false, p.dtype == DTYPE_FLOAT16, 5, dims, strides, box, nullptr);
}

template <typename T, int DB, int SLOTS> static bool launch_chunk(const AttentionProblem& p) {
    using L = ChunkLayout<DB, SLOTS>;
    DeviceState* st = acquire_device();
    if (!st) return false;
    int box_rows = cache_box_rows(p), tile_tokens = 128 / p.group;
    CUtensorMap q_map, k_map, v_map;
    if (!make_query_map(&q_map, p, tile_tokens) || !make_cache_map(&k_map, p, p.k, box_rows) || !make_cache_map(&v_map, p, p.v, box_rows)) {
        set_error(TOPS_ERR_CUDA, "attention_chunk: the tensor map was refused");
        return false;
    }
    const bool masked = p.mask_kind != kMaskNone;
    const void* kernel = masked ? (const void*)attention_chunk_kernel<T, DB, SLOTS, true> : (const void*)attention_chunk_kernel<T, DB, SLOTS, false>;
    if (!ensure_dynamic_smem(kernel, L::kSmem)) return false;
    const long long items = attention_tiles(p, 2 * tile_tokens * p.group) * p.kv_heads, most = items * (p.keys > 0 ? (p.keys + kChunkKeys - 1) / kChunkKeys : 1);
    const int blocks = (int)(most < (long long)st->sm_count ? most : (long long)st->sm_count);
    cudaStream_t stream = current_stream();
    PartialResults parts;
    if (!allocate_partials(parts, blocks, kChunkRows, L::kDims, stream)) return false;
    AttentionProblem copy = p;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(kChunkThreads);
    cfg.dynamicSmemBytes = L::kSmem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = overlap_launches();
    void* args[] = {&q_map, &k_map, &v_map, &copy, &box_rows, &tile_tokens, &parts};
    bool ok = check_cuda(cudaLaunchKernelExC(&cfg, kernel, args), "attention_chunk");
    ok = join_partials<T, kChunkRows, L::kDims>(copy, parts, blocks, items, stream, ok);
    if (ok) count_tensor_core_launch();
    return ok;
}

// A whole group of heads has to fit a tile.  Maximum and mask are applied to the scores before they are scaled: the scale has to be positive, and not
// so small that a mask divided by it overflows.
bool attention_chunk_takes(const AttentionProblem& p) {
    return p.dim <= 128 && p.group <= 128 && p.scale_log2 > (p.mask_kind == kMaskNone ? 0.0f : 1e-4f) && cache_box_rows(p) > 0;
}

bool attention_chunk(const AttentionProblem& p) {
    if (p.dtype == DTYPE_FLOAT16) return p.dim <= 64 ? launch_chunk<__half, 1, 8>(p) : launch_chunk<__half, 2, 4>(p);
    return p.dim <= 64 ? launch_chunk<__nv_bfloat16, 1, 8>(p) : launch_chunk<__nv_bfloat16, 2, 4>(p);
}

}  // namespace tops
