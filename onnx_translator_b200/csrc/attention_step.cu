// Attention of few rows per key head (single new tokens, small groups of them) on the 5th-generation tensor cores.  HBM bound: the keys and
// values of a sequence are read once and nothing else may take as long.
//
// The scores are computed transposed, so that the many keys fill the 128 rows of the instruction and the few queries its N columns:
//   S^T[128 keys x N] = K[128 x dim] Q^T,      O^T[dim x N] += V^T[dim x 128] P^T
// K is the A operand as it lies in memory; V, [keys][dim], is A seen MN-major; Q and P are K-major B operands of N rows.  A thread of the softmax owns
// one key -- its mask, its visibility -- with the N scores of that key in registers.
//
// The maximum of a row would have to be taken across the threads.  Instead all rows keep a running reference m, and a tile only checks
// (one predicate, or-reduced by the barrier it needs anyway) that no score exceeds m by more than 8 in log2: the weights stay below
// 2^8, the sums are float32, and the quotient o / l does not depend on m.  When the check fails, about ln(tiles) times per row, the block
// takes the true maximum and rescales o and l.  Sums of weights stay per thread (per key) until the end.
// Rows are worked on four at a time: the columns between t.rows and the next multiple of four hold scores of zero queries and are dropped
// at the end (a branch per row cost more than the arithmetic of three idle ones).
//
// Work is split evenly whatever the lengths: all 128-key tiles of all (sequence, key head) items stand in one row, and block c takes the c-th share of
// it, possibly the end of one item, some whole items and the beginning of another.  The pipeline runs on across items.  An item that lies inside one share
// is stored at once; of an item that spans several, each block leaves (m, l, o) in scratch memory, at most two per block, and a
// second small kernel joins them in the order of the keys.  (Clusters that join through distributed shared memory were measured first: the GPU
// holds only 15 clusters of eight such blocks at a time, 120 of 148 SMs, and 16 items then took two rounds: 235 us where this takes 151.)
//
// Warps 0-3 and 8-11: two softmax groups that take the items in turn -- one finishes its item (sums, tensor memory, stores) while the other
// is in the next item's tiles.  Warp 4 copies (TMA, page by page, 128 keys of K or V per ring slot), warp 5 issues the MMAs, warp 6 finds the next
// item and brings its queries.
//
// Measured (dim 128, 32 heads over 8 key heads): one new token for 64 sequences of 300 to 8192 keys 127 us, 6.1 TB/s; for two of 131072 and 100003 keys 151 us, 6.4 TB/s (a
// plain copy: 6.57); for one of 511 keys 10 us, a chain of latencies: finding the item, four tiles of 0.9 us, the result.  A tile costs the MMA warp about 1650 cycles
// (sixteen instructions of 39 and the barriers between), copying it 2600.
#include "attention_join.cuh"

#include <type_traits>

namespace tops {

void count_tensor_core_launch();

constexpr int kStepThreads = 384;
constexpr int kStepKeys = 128;

template <int DB, int N, int SLOTS> struct StepLayout {
    static constexpr int kSlotBytes = kStepKeys * 128 * DB;
    static constexpr int kQBytes = N * 128 * DB;              // one of the two buffers
    static constexpr int kPBytes = N * 128 * 2;               // one of the two buffers
    static constexpr int kDims = DB * 64;
    static constexpr int kSmem = SLOTS * kSlotBytes + 2 * kQBytes + 2 * kPBytes + 1024;   // and room to align
    static constexpr int kOAccs = DB > 2 ? 2 : 1;             // accumulators of 128 dimensions
    static constexpr uint32_t kUsed = (2 + 2 * kOAccs) * N, kColumns = kUsed <= 64 ? 64 : kUsed <= 128 ? 128 : kUsed <= 256 ? 256 : 512;
    static_assert(SLOTS <= 8, "a slot's release is read from barriers of the last four tiles");
};

// ---- the row of all tiles ------------------------------------------------------------------------------------------------
// Sequence b has tiles_of_rows row tiles of N rows; each of them, for each key head, counts `units` 128-key tiles (at least one, so that
// rows without a key are visited as well).
struct SequenceWork { int start, tokens, length, units, row_tiles; };

template <int N> __device__ __forceinline__ SequenceWork sequence_work(const AttentionProblem& p, int b, bool whole) {
    SequenceWork w = {0, 0, 0, 0, 0};
    if (b >= p.batch) return w;
    int first_key = 0;
    if (p.page_table) {
        const int s = p.query_start[b], e = p.query_start[b + 1], length = p.kv_length[b];
        w.start = min(max(s, 0), p.queries);
        const int end = min(max(e, w.start), p.queries);
        w.tokens = end - w.start;
        w.length = min(max(length, 0), p.keys);
        if (w.start != s || end != e || w.length != length) report_bad_index(p);
        if (p.window > 0) first_key = max(0, w.length - w.tokens - p.window + 1);
    } else {
        w.tokens = p.queries;
        w.length = p.kv_length ? min(max(p.kv_length[b], 0), p.keys) : p.keys;
    }
    w.row_tiles = (w.tokens * p.group + N - 1) / N;
    w.units = whole ? 1 : max(1, (w.length + kStepKeys - 1) / kStepKeys - first_key / kStepKeys);
    return w;
}

// Where a unit of that row lies: row tile, key head and unit inside them.
struct UnitPlace { SequenceWork w; int seq, row_tile, kv_head, unit; };

// All units; called by whole warps.  `head` is the lane's own of the first 32 sequences, fetched before.
template <int N> __device__ __forceinline__ int total_units(const AttentionProblem& p, bool whole, const SequenceWork& head) {
    int sum = 0;
    for (int b = threadIdx.x & 31; b < p.batch; b += 32) {
        const SequenceWork w = b < 32 ? head : sequence_work<N>(p, b, whole);
        sum += w.row_tiles * w.units;
    }
    #pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(~0u, sum, d);
    return sum * p.kv_heads;
}

template <int N> __device__ __forceinline__ UnitPlace place_unit(const AttentionProblem& p, int x, bool whole, const SequenceWork& head) {
    const int lane = threadIdx.x & 31;
    UnitPlace at = {};
    int before = 0;
    for (int base = 0; base < p.batch; base += 32) {
        const SequenceWork w = base == 0 ? head : sequence_work<N>(p, base + lane, whole);
        const int mine = w.row_tiles * w.units * p.kv_heads;
        int sum = mine;
        #pragma unroll
        for (int d = 1; d < 32; d <<= 1) { const int o = __shfl_up_sync(~0u, sum, d); if (lane >= d) sum += o; }
        const unsigned past = __ballot_sync(~0u, x < before + sum);
        if (past) {
            const int l = __ffs(past) - 1;
            at.seq = base + l;
            at.w.start = __shfl_sync(~0u, w.start, l);
            at.w.tokens = __shfl_sync(~0u, w.tokens, l);
            at.w.length = __shfl_sync(~0u, w.length, l);
            at.w.units = __shfl_sync(~0u, w.units, l);
            at.w.row_tiles = __shfl_sync(~0u, w.row_tiles, l);
            const int inside = x - before - __shfl_sync(~0u, sum - mine, l);
            const int item = inside / at.w.units;
            at.unit = inside - item * at.w.units;
            at.row_tile = item / p.kv_heads;
            at.kv_head = item - at.row_tile * p.kv_heads;
            break;
        }
        before += __shfl_sync(~0u, sum, 31);
    }
    return at;
}

template <int N> __device__ __forceinline__ RowTile row_tile_of(const AttentionProblem& p, const UnitPlace& at) {
    RowTile t;
    t.seq = at.seq;
    t.row0 = at.row_tile * N;
    t.rows = min(N, at.w.tokens * p.group - t.row0);
    t.token0 = at.w.start;
    t.length = t.key_end = at.w.length;
    t.key_begin = 0;
    if (p.page_table) {
        t.first_position = at.w.length - at.w.tokens;
        const int first = t.first_position + (int)p.group_div.div((uint32_t)t.row0);
        const int last = t.first_position + (int)p.group_div.div((uint32_t)(t.row0 + t.rows - 1));
        t.key_end = max(0, min(t.length, last + 1));
        if (p.window > 0) t.key_begin = min(max(0, first - p.window + 1), t.key_end);
    }
    return t;
}

// First 128-key tile of an item's units.
__device__ __forceinline__ int first_tile_of(const AttentionProblem& p, const UnitPlace& at) {
    return p.window > 0 && p.page_table ? max(0, at.w.length - at.w.tokens - p.window + 1) / kStepKeys : 0;
}

struct Segment {
    RowTile t;
    int kv_head;
    int lo, n;                   // 128-key tiles lo .. lo + n - 1; n < 0: no more segments
    int part;                    // scratch slot of the partial result, -1: the item is whole
    int pages[16];               // pages of tile lo
};

// True for all 128 threads of a softmax group if it is for one.
__device__ __forceinline__ bool any_of_softmax(int group, bool x) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %1, 0;\n\t"
        "barrier.cta.red.or.pred p, %2, 128, q;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r) : "r"((uint32_t)x), "r"(1 + group) : "memory");
    return r != 0;
}
__device__ __forceinline__ void softmax_sync(int group) { asm volatile("barrier.cta.sync %0, 128;" ::"r"(1 + group) : "memory"); }

template <int W> __device__ __forceinline__ void tmem_load_some(uint32_t at, uint32_t (&r)[W]) {
    if constexpr (W == 4) umma::tmem_load_32x4(at, r);
    else if constexpr (W == 8) umma::tmem_load_32x8(at, r);
    else if constexpr (W == 16) umma::tmem_load_32x16(at, r);
    else umma::tmem_load_32x32(at, r);
}
// The first R columns of one accumulator.
template <int R> __device__ __forceinline__ void tmem_load_columns(uint32_t at, float (&x)[R]) {
    uint32_t r[R];
    tmem_load_some<R>(at, r);
    umma::tmem_load_wait();
    #pragma unroll
    for (int i = 0; i < R; i++) x[i] = __uint_as_float(r[i]);
}
// The same times the rows' factors, in place.
template <int R> __device__ __forceinline__ void tmem_scale_columns(uint32_t at, const float* factor) {
    uint32_t r[R];
    tmem_load_some<R>(at, r);
    umma::tmem_load_wait();
    #pragma unroll
    for (int i = 0; i < R; i++) r[i] = __float_as_uint(__uint_as_float(r[i]) * factor[i]);
    if constexpr (R == 4) umma::tmem_store_32x4(at, r);
    else if constexpr (R == 8) umma::tmem_store_32x8(at, r);
    else if constexpr (R == 16) umma::tmem_store_32x16(at, r);
    else umma::tmem_store_32x32(at, r);
    umma::tmem_store_wait();
}

constexpr float kNoMaximum = -3.402823466e+38f;               // finite, so that score - m is never Inf - Inf
constexpr float kMaximumSlack = 8.0f;

template <typename T, int DB, int R, int SLOTS>
__global__ void __launch_bounds__(kStepThreads)
attention_step_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                      const __grid_constant__ AttentionProblem p, const int box_rows, const PartialResults parts) {
    constexpr int N = R > 16 ? 32 : 16;                       // columns of the instructions; rows beyond R are zero queries whose results nobody reads
    using L = StepLayout<DB, N, SLOTS>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t full[SLOTS], s_full[4], p_ready[2], pv_done[4], seg_full[2], seg_empty[2], o_full[2], turn[2], drained;
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_word, drain_word;
    __shared__ __align__(16) unsigned char segment_memory[2 * sizeof(Segment)];
    Segment* segments = reinterpret_cast<Segment*>(segment_memory);
    __shared__ __align__(16) float group_floats[2][7 * R];    // per softmax group: warp_top[4], fade, top_of, sums
    __shared__ int group_high[2][R];
    uint8_t* ring = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t* q_tiles = ring + SLOTS * L::kSlotBytes;
    uint8_t* p_tile = q_tiles + 2 * L::kQBytes;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    volatile int* abort_flag = &abort_word;

    if (threadIdx.x == 0) {
        for (int s = 0; s < SLOTS; s++) umma::mbar_init(&full[s], 1);
        for (int b = 0; b < 4; b++) { umma::mbar_init(&s_full[b], 1); umma::mbar_init(&pv_done[b], 1); }
        for (int b = 0; b < 2; b++) { umma::mbar_init(&p_ready[b], 128); umma::mbar_init(&seg_full[b], 1); umma::mbar_init(&seg_empty[b], 7); umma::mbar_init(&o_full[b], 1); umma::mbar_init(&turn[b], 4); }
        umma::mbar_init(&drained, 1);
        abort_word = drain_word = 0;
        umma::mbar_fence_init();
    }
    if (threadIdx.x < 2 * R) group_floats[threadIdx.x / R][4 * R + threadIdx.x % R] = 1.0f;      // fade of the columns that no row uses
    if (warp == 4 && lane == 0) { umma::tma_prefetch_desc(&k_map); umma::tma_prefetch_desc(&v_map); }
    // Scheduled while the previous kernel of the stream drains; nothing so far has touched global or tensor memory.  The join in turn may be scheduled early: it
    // waits for this grid before it reads.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const bool whole = parts.o == nullptr;                     // the unit is the item: nothing is split, nothing joined
    SequenceWork head = {0, 0, 0, 0, 0};
    if (warp == 6) head = sequence_work<R>(p, lane, whole);
    if (warp == 5) umma::tmem_alloc(&tmem_slot, L::kColumns);
    umma::fence_before_sync();
    __syncthreads();
    umma::fence_after_sync();
    const uint32_t tmem = tmem_slot, tmem_o = tmem + 2 * N;
    auto wait = [&](uint64_t* bar, uint32_t parity) { return (bool)__all_sync(~0u, umma::mbar_wait(bar, parity, abort_flag)); };   // a whole warp

    if (warp == 6) {
        // ---- items: what this block works on, and its queries ---------------------------------------------------------------
        const int total = total_units<R>(p, whole, head);
        const int share = (total + (int)gridDim.x - 1) / (int)gridDim.x;
        const int x0 = min((int)blockIdx.x * share, total), x1 = min(x0 + share, total);
        int x = x0, s = 0;
        JoinJob job;                                           // the item that begins in this share and ends behind it
        for (;; s++) {
            const int buf = s & 1;
            UnitPlace at = {};
            Segment seg;
            seg.n = -1;
            int page = 0;
            if (x < x1) {
                at = place_unit<R>(p, x, whole, head);
                seg.t = row_tile_of<R>(p, at);
                seg.kv_head = at.kv_head;
                const int take = min(at.w.units - at.unit, x1 - x), first = first_tile_of(p, at);
                // the units counted for the sequence may reach past the keys of this row tile
                seg.lo = max(first + at.unit, seg.t.key_begin / kStepKeys);
                const int all = (seg.t.key_end + kStepKeys - 1) / kStepKeys, hi = whole ? all : min(first + at.unit + take, all);
                seg.n = seg.t.key_end > seg.t.key_begin ? max(hi - seg.lo, 0) : 0;
                if (p.mask_kind != kMaskNone) trim_masked(p, seg.t.seq, seg.t.key_end, seg.lo, seg.n);
                seg.part = at.unit == 0 && take == at.w.units ? -1 : (int)blockIdx.x * 2 + (x == x0 ? 0 : 1);
                if (seg.part >= 0 && x - at.unit >= x0 && x - at.unit + at.w.units > x1)
                    job = JoinJob{seg.t, seg.kv_head, (x - at.unit + at.w.units - 1) / share - (int)blockIdx.x + 1, seg.part};
                x += take;
                const int j = seg.lo * kStepKeys + lane * box_rows;
                if (p.page_table && seg.n > 0 && lane * box_rows < kStepKeys && j < seg.t.key_end && j + box_rows > seg.t.key_begin)
                    page = p.page_table[(long long)seg.t.seq * p.table_width + (int)p.page_div.div((uint32_t)j)];
            }
            // sixteen-byte pieces of the rows, XORed with the row as the swizzle wants; loaded before the buffer is free
            constexpr int PIECES = N * DB * 8 / 32;
            constexpr int BATCH = PIECES < 16 ? PIECES : 16;
            bool alive = true;
            #pragma unroll 1
            for (int base = 0; base < PIECES; base += BATCH) {
                uint4 piece[BATCH];
                #pragma unroll
                for (int k = 0; k < BATCH; k++) {
                    const int i = (base + k) * 32 + lane, r = i / (DB * 8), c = i - r * (DB * 8);
                    piece[k] = make_uint4(0, 0, 0, 0);
                    if (seg.n > 0 && r < seg.t.rows && c * 8 < p.dim)
                        piece[k] = *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.q) + row_offset(p, seg.t, seg.kv_head, seg.t.row0 + r) + c * 8);
                }
                if (base == 0 && s > 1) alive = wait(&seg_empty[buf], (uint32_t)((s >> 1) - 1) & 1u);
                if (!alive) break;
                uint8_t* q_tile = q_tiles + buf * L::kQBytes;
                #pragma unroll
                for (int k = 0; k < BATCH; k++) {
                    const int i = (base + k) * 32 + lane, r = i / (DB * 8), c = i - r * (DB * 8);
                    *reinterpret_cast<uint4*>(q_tile + (c >> 3) * (N * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = piece[k];
                }
            }
            if (!alive) break;
            if (lane < 16) segments[buf].pages[lane] = page;
            if (lane == 0) {
                segments[buf].t = seg.t;
                segments[buf].kv_head = seg.kv_head;
                segments[buf].lo = seg.lo;
                segments[buf].n = seg.n;
                segments[buf].part = seg.part;
            }
            umma::fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) umma::mbar_arrive(&seg_full[buf]);
            if (seg.n < 0) break;
        }
        if (!whole && lane == 0) parts.jobs[blockIdx.x] = job;
    } else if (warp == 4) {
        // ---- copies: load number g is the keys (g even) or values (g odd) of this block's tile g / 2, into ring slot g % SLOTS ----------
        int g = 0;
        uint32_t slot = 0, phase = 0;
        bool alive = true;
        for (int s = 0; alive; s++) {
            if (!wait(&seg_full[s & 1], (uint32_t)(s >> 1) & 1u)) break;
            const Segment& seg = segments[s & 1];
            const int n = seg.n, lo = seg.lo, key_begin = seg.t.key_begin, key_end = seg.t.key_end, kv_head = seg.kv_head, sequence = seg.t.seq;
            const int batch = p.page_table ? 0 : sequence;
            int page = seg.pages[lane & 15];
            __syncwarp();
            if (n < 0) break;
            auto box_needed = [&](int j) { return lane * box_rows < kStepKeys && j < key_end; };
            for (int i = 0; i < n && alive; i++) {
                const int j = (lo + i) * kStepKeys + lane * box_rows;
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
                // the next tile's pages, looked at when its turn comes: the copies never wait for the table
                const int next_j = j + kStepKeys;
                if (p.page_table && i + 1 < n && box_needed(next_j) && next_j + box_rows > key_begin)
                    page = p.page_table[(long long)sequence * p.table_width + (int)p.page_div.div((uint32_t)next_j)];
                const int boxes = __popc(__ballot_sync(~0u, row >= 0));
                #pragma unroll 1
                for (int kv = 0; kv < 2; kv++, g++) {
                    if (g >= SLOTS) {                          // the slot's last contents: keys are read out with their scores, values with their product
                        const int old = g - SLOTS, tile = old >> 1;
                        if (!wait((old & 1) ? &pv_done[tile & 3] : &s_full[tile & 3], (uint32_t)(tile >> 2) & 1u)) { alive = false; break; }
                    }
                    uint8_t* to = ring + slot * L::kSlotBytes;
                    const CUtensorMap* map = kv ? &v_map : &k_map;
                    if (umma::elect_one()) umma::mbar_expect_tx(&full[slot], (uint32_t)(boxes * box_rows) * 128u * DB);
                    __syncwarp();
                    for (int x = 0; x < boxes; x++) {
                        const int box_row = __shfl_sync(~0u, row, x);
                        if (umma::elect_one()) {
                            #pragma unroll
                            for (int b = 0; b < DB; b++) umma::tma_load_4d(to + b * (kStepKeys * 128) + x * box_rows * 128, map, &full[slot], b * 64, kv_head, box_row, batch);
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
    } else if (warp == 5) {
        // ---- products: the whole warp waits, one elected lane issues; the scores of the next tile, which may belong to the next item, go out before this
        // tile's product with V, so that the softmax always has work -------------------------------------------------------------------
        constexpr uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
        constexpr uint32_t idesc_s = umma::instr_desc(fmt, fmt, 128, N), idesc_o = idesc_s | umma::kInstrAMnMajor;
        uint32_t slot = 0, phase = 0;
        auto step = [&] { if (++slot == SLOTS) { slot = 0; phase ^= 1u; } };
        int s = -1, left = 0, tile = 0;                        // segment, tiles of it whose scores are still to come, number of the next tile
        bool ok = true, fresh = false;
        // Advances to the next tile, no further than segment `limit`, and issues its scores.  The segment behind an empty one is only published when the one before
        // has been stored, so with a tile's product still to issue the look ahead ends at the next segment.
        enum { kEnd, kIssued, kLater };
        auto scores = [&](int limit) {
            fresh = false;
            while (left == 0) {
                if (s >= limit) return kLater;
                s++;
                if (!wait(&seg_full[s & 1], (uint32_t)(s >> 1) & 1u)) { ok = false; return kEnd; }
                left = segments[s & 1].n;
                __syncwarp();
                if (left < 0) return kEnd;
                fresh = true;
                if (left == 0 && lane == 0) umma::mbar_arrive(&seg_empty[s & 1]);
            }
            if (!wait(&full[slot], phase)) { ok = false; return kEnd; }
            umma::fence_after_sync();
            left--;
            const uint64_t da = umma::smem_desc_k_major_sw128(ring + slot * L::kSlotBytes), db = umma::smem_desc_k_major_sw128(q_tiles + (s & 1) * L::kQBytes);
            if (umma::elect_one()) {
                #pragma unroll
                for (int b = 0; b < DB; b++)
                    #pragma unroll
                    for (int k = 0; k < 4; k++)
                        umma::mma_ss<false>(tmem + (tile & 1) * N, da + (uint64_t)(b * (kStepKeys * 128 >> 4) + 2 * k), db + (uint64_t)(b * (N * 128 >> 4) + 2 * k), idesc_s, (uint32_t)(b | k));
                umma::mma_commit(&s_full[tile & 3]);
                if (left == 0) umma::mma_commit(&seg_empty[s & 1]);      // the queries have been read
            }
            __syncwarp();
            tile++;
            step();                                            // on to this tile's values
            return kIssued;
        };
        constexpr int kNoLimit = 0x7FFFFFFF;
        int more = scores(kNoLimit);
        while (more == kIssued && ok) {
            const int i = tile - 1;
            const bool first = fresh;
            const uint32_t o_at = tmem_o + (uint32_t)((s & 1) * L::kOAccs * N);
            const int of = s;
            const bool last = left == 0;
            const uint32_t v_slot = slot, v_phase = phase;
            step();
            more = scores(of + 1);
            if (!ok) break;
            ok = wait(&p_ready[i & 1], (uint32_t)(i >> 1) & 1u) && wait(&full[v_slot], v_phase);
            if (!ok) break;
            umma::fence_after_sync();
            const uint64_t da = umma::smem_desc_mn_major_sw128(ring + v_slot * L::kSlotBytes, DB == 1 ? 0u : (uint32_t)(kStepKeys * 128));
            const uint64_t db = umma::smem_desc_k_major_sw128(p_tile + (i & 1) * L::kPBytes);
            if (umma::elect_one()) {
                #pragma unroll
                for (int a = 0; a < L::kOAccs; a++)
                    #pragma unroll
                    for (int k = 0; k < 8; k++)
                        umma::mma_ss<false>(o_at + a * N, da + (uint64_t)(a * 2 * (kStepKeys * 128 >> 4) + k * (2048 >> 4)),
                                            db + (uint64_t)((k >> 2) * (N * 128 >> 4) + 2 * (k & 3)), idesc_o, first ? (uint32_t)k : 1u);
                umma::mma_commit(&pv_done[i & 3]);
                if (last) umma::mma_commit(&o_full[of & 1]);   // a barrier of its own: the other group's tiles may be far ahead when this one is looked at
            }
            __syncwarp();
            if (more == kLater) more = scores(kNoLimit);
        }
        if (!ok) {
            if (umma::elect_one()) umma::mma_commit(&drained);
            __syncwarp();
            umma::mbar_wait(&drained, 0, &drain_word);
        }
    } else if (warp != 7) {
        // ---- softmax: a thread per key -------------------------------------------------------------------------------------
        const int group = warp >> 3, quarter = warp & 3, key = quarter * 32 + lane;
        const uint32_t lanes = (uint32_t)quarter << 21;        // this warp's quarter of tensor memory
        float (*warp_top)[R] = reinterpret_cast<float (*)[R]>(group_floats[group]);
        float *fade = group_floats[group] + 4 * R, *top_of = fade + R, *sums = top_of + R;
        int* high = group_high[group];
        const bool masked = p.mask_kind != kMaskNone;
        uint32_t slot = 0, phase = 0, o_phase = 0;             // o_phase counts this group's items that had a key
        bool ok = true;
        int i = 0;                                             // number of the tile
        for (int s = 0;; s++) {
            if (any_of_softmax(group, !ok)) break;
            ok = umma::mbar_wait(&seg_full[s & 1], (uint32_t)(s >> 1) & 1u, abort_flag);
            const Segment& seg = segments[s & 1];
            const int n = seg.n;
            const uint32_t my_o = tmem_o + lanes + (uint32_t)((s & 1) * L::kOAccs * N);
            if (any_of_softmax(group, !ok)) { ok = false; break; }
            if (n < 0) break;
            if ((s & 1) != group) {                            // the other group's item: only the ring and the tile count move on
                i += n;
                const uint32_t moved = slot + 2u * (uint32_t)n;
                slot = moved % SLOTS;
                phase ^= (moved / SLOTS) & 1u;
                softmax_sync(group);                           // all have read n
                if (key == 0) umma::mbar_arrive(&seg_empty[s & 1]);
                // and this group's tiles begin when the other's end: barriers that count tiles tell two neighbouring phases apart, no more
                ok = umma::mbar_wait(&turn[s & 1], (uint32_t)(s >> 1) & 1u, abort_flag);
                continue;
            }
            const int rows = seg.t.rows, key_end = seg.t.key_end, lo = seg.lo;
            if (key < R) {
                high[key] = p.page_table ? seg.t.first_position + (int)p.group_div.div((uint32_t)(seg.t.row0 + min(key, rows - 1))) + 1 : key_end;
                top_of[key] = kNoMaximum;
            }
            softmax_sync(group);
            int all_high = key_end, all_low = 0;
            if (p.page_table) {
                all_high = high[0];
                if (p.window > 0) all_low = high[R - 1] - p.window;
            }
            float l[R];
            #pragma unroll
            for (int r = 0; r < R; r++) l[r] = 0.0f;
            for (int it = 0; it < n; it++, i++) {
                const int j0 = (lo + it) * kStepKeys, j = j0 + key;
                if (++slot == SLOTS) { slot = 0; phase ^= 1u; }    // the slot of this tile's values
                const bool edge = masked || j0 < all_low || j0 + kStepKeys > all_high;
                bool dead = false;                             // a key that no row sees: its value must not reach the product
                float bias = 0.0f;
                if (edge) {
                    dead = j >= key_end;
                    if (masked && !dead) { bias = key_bias(p, seg.t.seq, j); dead = bias == -INFINITY; }
                }
                if (!umma::mbar_wait(&s_full[i & 3], (uint32_t)(i >> 2) & 1u, abort_flag)) ok = false;
                umma::fence_after_sync();
                float z[R];
                __syncwarp();
                tmem_load_columns<R>(tmem + lanes + (i & 1) * N, z);
                float over = -INFINITY;
                #pragma unroll
                for (int c = 0; c < R; c += 4)
                    if (c < rows) {
                        const float4 m = *reinterpret_cast<const float4*>(top_of + c);
                        const float mr[4] = {m.x, m.y, m.z, m.w};
                        #pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const int r = c + e;
                            if (!edge) z[r] *= p.scale_log2;
                            else {
                                const bool seen = !dead && j < high[r] && (p.window == 0 || j >= high[r] - p.window);
                                z[r] = seen ? __fmaf_rn(z[r], p.scale_log2, bias) : -INFINITY;
                            }
                            over = fmaxf(over, z[r] - mr[e]);
                        }
                    }
                if (any_of_softmax(group, over > kMaximumSlack || !ok)) {
                    if (any_of_softmax(group, !ok)) { ok = false; break; }        // a wait has run out: all leave
                    #pragma unroll
                    for (int c = 0; c < R; c += 4)
                        if (c < rows)
                            #pragma unroll
                            for (int r = c; r < c + 4; r++) {
                                float top = z[r];
                                #pragma unroll
                                for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
                                if (lane == 0) warp_top[quarter][r] = top;
                            }
                    softmax_sync(group);
                    if (key < R && (key & ~3) < rows) {
                        const float old = top_of[key];
                        const float top = fmaxf(old, fmaxf(fmaxf(warp_top[0][key], warp_top[1][key]), fmaxf(warp_top[2][key], warp_top[3][key])));
                        fade[key] = exp2_approx(old - top);
                        top_of[key] = top;
                    }
                    softmax_sync(group);
                    #pragma unroll
                    for (int c = 0; c < R; c += 4)
                        if (c < rows) {
                            const float4 f = *reinterpret_cast<const float4*>(fade + c);
                            l[c] *= f.x; l[c + 1] *= f.y; l[c + 2] *= f.z; l[c + 3] *= f.w;
                        }
                    if (it > 0) {
                        if (!umma::mbar_wait(&pv_done[(i - 1) & 3], (uint32_t)((i - 1) >> 2) & 1u, abort_flag)) ok = false;
                        umma::fence_after_sync();
                        __syncwarp();
                        #pragma unroll
                        for (int a = 0; a < L::kOAccs; a++) tmem_scale_columns<R>(my_o + a * N, fade);
                    }
                }
                if (i > 1 && !umma::mbar_wait(&pv_done[(i - 2) & 3], (uint32_t)((i - 2) >> 2) & 1u, abort_flag)) ok = false;    // the weights of tile i - 2 are read
                uint8_t* to = p_tile + (i & 1) * L::kPBytes + (key >> 6) * (N * 128) + (key & 7) * 2;
                #pragma unroll
                for (int c = 0; c < R; c += 4)
                    if (c < rows) {
                        const float4 m = *reinterpret_cast<const float4*>(top_of + c);
                        const float mr[4] = {m.x, m.y, m.z, m.w};
                        #pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const int r = c + e;
                            const float w = exp2_approx(z[r] - mr[e]);
                            l[r] += w;
                            *reinterpret_cast<T*>(to + r * 128 + ((((key & 63) >> 3) ^ (r & 7)) << 4)) = from_float<T>(w);
                        }
                    }
                if (dead) {                                    // a weight of zero times a NaN would still be one
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
            }
            if (any_of_softmax(group, !ok)) { ok = false; break; }
            if (lane == 0) umma::mbar_arrive(&turn[s & 1]);
            // the item's (or its part's) result
            if (n > 0) {
                if (!umma::mbar_wait(&o_full[group], o_phase, abort_flag)) ok = false;
                umma::fence_after_sync();
                o_phase ^= 1u;
            }
            __syncwarp();
            float x[L::kOAccs][R];
            #pragma unroll
            for (int a = 0; a < L::kOAccs; a++) tmem_load_columns<R>(my_o + a * N, x[a]);
            // sums of weights over the keys
            #pragma unroll
            for (int c = 0; c < R; c += 4)
                if (c < rows)
                    #pragma unroll
                    for (int r = c; r < c + 4; r++) {
                        float sum = l[r];
                        #pragma unroll
                        for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(~0u, sum, d);
                        if (lane == 0) warp_top[quarter][r] = sum;
                    }
            softmax_sync(group);
            if (key < rows) {
                const float sum = (warp_top[0][key] + warp_top[1][key]) + (warp_top[2][key] + warp_top[3][key]);
                sums[key] = sum == 0.0f ? 0.0f : 1.0f / sum;
                if (seg.part >= 0) parts.stats[(long long)seg.part * R + key] = make_float2(sum == 0.0f ? -INFINITY : top_of[key], sum);
            }
            softmax_sync(group);
            if (seg.part >= 0) {
                #pragma unroll
                for (int a = 0; a < L::kOAccs; a++) {
                    const int d = a * 128 + key;
                    if (d < L::kDims)
                        #pragma unroll
                        for (int r = 0; r < R; r++) if (r < rows) parts.o[((long long)seg.part * R + r) * L::kDims + d] = x[a][r];
                }
            } else {
                #pragma unroll
                for (int a = 0; a < L::kOAccs; a++) {
                    const int d = a * 128 + key;
                    if (d < p.dim)
                        #pragma unroll
                        for (int r = 0; r < R; r++)
                            if (r < rows) reinterpret_cast<T*>(p.y)[row_offset(p, seg.t, seg.kv_head, seg.t.row0 + r) + d] = from_float<T>(sums[r] == 0.0f ? 0.0f : x[a][r] * sums[r]);
                }
            }
            umma::fence_before_sync();
            softmax_sync(group);                                    // sums, weights and the segment have been read by all
            if (lane == 0) umma::mbar_arrive(&seg_empty[s & 1]);
        }
    }
    umma::fence_before_sync();
    __syncthreads();
    if (threadIdx.x == 0 && abort_word && p.status) atomicExch(p.status, 1);
    if (warp == 5) {
        umma::fence_after_sync();
        umma::tmem_dealloc(tmem, L::kColumns);
    }
}

template <typename T, int DB, int R, int SLOTS> static bool launch_step(const AttentionProblem& p) {
    constexpr int N = R > 16 ? 32 : 16;
    using L = StepLayout<DB, N, SLOTS>;
    DeviceState* st = acquire_device();
    if (!st) return false;
    int box_rows = cache_box_rows(p);
    CUtensorMap k_map, v_map;
    if (!make_cache_map(&k_map, p, p.k, box_rows) || !make_cache_map(&v_map, p, p.v, box_rows)) {
        set_error(TOPS_ERR_CUDA, "attention_step: the tensor map was refused");
        return false;
    }
    const void* kernel = (const void*)attention_step_kernel<T, DB, R, SLOTS>;
    if (!ensure_dynamic_smem(kernel, L::kSmem)) return false;
    // One block per SM (two of the small ones: with heads of 64 a tile is half as long to copy but not to work on), but none that cannot get a tile.  Where an item cannot have more than four tiles (512 keys), a block takes it whole: the join costs as much as
    // three tiles in a row.
    const long long units = (p.keys + kStepKeys - 1) / kStepKeys, items = attention_tiles(p, R) * p.kv_heads;
    const bool whole = units <= 4;
    const long long most = whole ? items : items * units;
    const long long room = (long long)st->sm_count * (DB == 1 && N == 16 ? 2 : 1);
    const int blocks = (int)(most < room ? most : room);
    cudaStream_t stream = current_stream();
    PartialResults parts;
    if (!whole && !allocate_partials(parts, blocks, R, L::kDims, stream)) return false;
    AttentionProblem copy = p;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(kStepThreads);
    cfg.dynamicSmemBytes = L::kSmem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = overlap_launches();
    void* args[] = {&k_map, &v_map, &copy, &box_rows, &parts};
    bool ok = check_cuda(cudaLaunchKernelExC(&cfg, kernel, args), "attention_step");
    if (!whole) ok = join_partials<T, R, L::kDims>(copy, parts, blocks, items, stream, ok);
    if (ok) count_tensor_core_launch();
    return ok;
}

// Room for 4, 8, 16 or 32 rows, by the rows of a sequence on average (longer sequences take several row tiles): the softmax and its code shrink with it.  Ring
// slots: as many as shared memory holds with one block per SM -- for heads of 64 with two blocks.
template <typename T, int DB, int SLOTS, int SLOTS32> static bool launch_step_rows(const AttentionProblem& p) {
    const long long rows = (long long)p.queries * p.group / (p.page_table ? p.batch : 1);
    if (rows <= 4) return launch_step<T, DB, 4, SLOTS>(p);
    if (rows <= 8) return launch_step<T, DB, 8, SLOTS>(p);
    return rows <= 16 ? launch_step<T, DB, 16, SLOTS>(p) : launch_step<T, DB, 32, SLOTS32>(p);
}

template <typename T> static bool launch_step_size(const AttentionProblem& p) {
    if (p.dim <= 64) return launch_step_rows<T, 1, 5, 8>(p);
    if (p.dim <= 128) return launch_step_rows<T, 2, 5, 5>(p);
    return launch_step_rows<T, 4, 3, 2>(p);
}

// The units of the whole problem are counted in 32 bits.
bool attention_step_fits(const AttentionProblem& p) {
    return attention_tiles(p, 4) * p.kv_heads * ((p.keys + kStepKeys - 1) / kStepKeys + 1) < 0x40000000ll;
}

bool attention_step(const AttentionProblem& p) {
    return p.dtype == DTYPE_FLOAT16 ? launch_step_size<__half>(p) : launch_step_size<__nv_bfloat16>(p);
}

}  // namespace tops
