// RMS norm of every query and key head, the rotary position embedding, and the append of keys and values to a paged cache, in
// one pass over the projection.
//
//   n = x * rsqrt(mean(x^2) + epsilon) * weight;   (a, b) -> (a cos - b sin, a sin + b cos)
//
// Each element is read once and written once (HBM bound); norms and rotations are float32, rounded once when stored.
#include "attention_common.cuh"
#include "call_checks.cuh"

#include <cmath>

namespace tops {

struct HeadsView {                           // strides in elements
    const void* in = nullptr;
    void* out = nullptr;                     // null: not written here
    void* cache = nullptr;                   // null: not appended
    const void* weight = nullptr;            // null: no norm
    int weight_f32 = 0;
    int heads = 0;
    int rotate = 0;
    long long in_batch = 0, in_token = 0, in_head = 0;
    long long out_batch = 0, out_token = 0, out_head = 0;
};

struct NormRotaryProblem {
    HeadsView part[3];                       // queries, keys, values
    int blocks[3] = {0, 0, 0};               // head blocks of each part
    int tokens = 0, seq = 1;                 // tokens in all; per batch row (heads_first)
    FastDiv seq_div, block_div;
    int dim = 0, half = 0;                   // half = rotary_dim / 2
    int interleaved = 0;
    float epsilon = 0.0f, inv_dim = 0.0f;
    const float* cos_table = nullptr;
    const float* sin_table = nullptr;
    int table_rows = 0;
    const void* positions = nullptr;
    int positions_64 = 0;
    const void* slots = nullptr;
    int slots_64 = 0;
    long long cache_rows = 0;
    int cache_heads = 0;
    int* status = nullptr;
};

__device__ __forceinline__ long long read_index(const void* p, int is64, int i) {
    return is64 ? reinterpret_cast<const long long*>(p)[i] : (long long)reinterpret_cast<const int*>(p)[i];
}

// Where a token's rows go: its table row (-1: none) and cache slot (-1: not stored).
struct TokenPlace { int batch, in_row, table_row; long long slot; bool bad_position; };

__device__ __forceinline__ TokenPlace place_token(const NormRotaryProblem& p, int token, bool positioned, bool append) {
    TokenPlace at;
    at.batch = (int)p.seq_div.div((uint32_t)token);
    at.in_row = token - at.batch * p.seq;
    at.table_row = -1;
    at.slot = -1;
    at.bad_position = false;
    if (positioned) {
        const long long pos = read_index(p.positions, p.positions_64, token);
        if (pos >= 0 && pos < p.table_rows) at.table_row = (int)pos;
        else { at.bad_position = true; if (p.status) atomicExch(p.status, kStatusBadIndex); }
    }
    if (append) {
        at.slot = read_index(p.slots, p.slots_64, token);
        if (at.slot >= p.cache_rows) { at.slot = -1; if (p.status) atomicExch(p.status, kStatusBadIndex); }
    }
    return at;
}

template <typename T> __device__ __forceinline__ float read_weight(const HeadsView& h, int d) {
    return h.weight_f32 ? reinterpret_cast<const float*>(h.weight)[d] : to_float(reinterpret_cast<const T*>(h.weight)[d]);
}

// General form: a warp per (token, head), elements strided over the lanes, the normalised head staged in shared memory so that
// any pairing of elements can be read back.  Takes every head size, alignment and rotary extent.
template <typename T>
__global__ void __launch_bounds__(128) norm_rotary_general(const __grid_constant__ NormRotaryProblem p) {
    extern __shared__ float staged[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float* mine = staged + warp * p.dim;
    const int per_token = p.part[0].heads + p.part[1].heads + p.part[2].heads;
    const long long items = (long long)p.tokens * per_token;
    for (long long item = (long long)blockIdx.x * 4 + warp; item < items; item += (long long)gridDim.x * 4) {
        const int token = (int)(item / per_token);
        int head = (int)(item - (long long)token * per_token), which = 0;
        while (head >= p.part[which].heads) head -= p.part[which++].heads;
        const HeadsView& h = p.part[which];
        const TokenPlace at = place_token(p, token, p.positions != nullptr, h.cache != nullptr);
        const T* in = reinterpret_cast<const T*>(h.in) + at.batch * h.in_batch + at.in_row * h.in_token + head * h.in_head;
        float sum = 0.0f;
        for (int d = lane; d < p.dim; d += 32) {
            const float x = to_float(in[d]);
            mine[d] = x;
            sum = __fmaf_rn(x, x, sum);
        }
        #pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
        const float factor = rsqrtf(__fmaf_rn(sum, p.inv_dim, p.epsilon));
        __syncwarp();
        if (h.weight) for (int d = lane; d < p.dim; d += 32) mine[d] = mine[d] * factor * read_weight<T>(h, d);
        __syncwarp();
        T* out = h.out ? reinterpret_cast<T*>(h.out) + at.batch * h.out_batch + at.in_row * h.out_token + head * h.out_head : nullptr;
        T* cache = h.cache && at.slot >= 0 && !at.bad_position ? reinterpret_cast<T*>(h.cache) + (at.slot * p.cache_heads + head) * p.dim : nullptr;
        for (int d = lane; d < p.dim; d += 32) {
            float y = mine[d];
            if (h.rotate && d < 2 * p.half && at.table_row >= 0) {
                const bool second = p.interleaved ? (d & 1) : d >= p.half;
                const int pair = p.interleaved ? d >> 1 : (second ? d - p.half : d);
                const float other = mine[p.interleaved ? d ^ 1 : (second ? d - p.half : d + p.half)];
                const float c = p.cos_table[(long long)at.table_row * p.half + pair], s = p.sin_table[(long long)at.table_row * p.half + pair];
                y = second ? __fmaf_rn(other, s, y * c) : __fmaf_rn(y, c, -(other * s));
            }
            if (at.bad_position) y = 0.0f;
            if (out) out[d] = from_float<T>(y);
            if (cache) cache[d] = from_float<T>(y);
        }
        __syncwarp();
    }
}

template <typename T> static bool launch_general(const NormRotaryProblem& p) {
    DeviceState* st = acquire_device();
    if (!st) return false;
    const long long items = (long long)p.tokens * (p.part[0].heads + p.part[1].heads + p.part[2].heads);
    const int blocks = grid_for((size_t)items, 4, st->sm_count, 16);
    norm_rotary_general<T><<<blocks, 128, 4 * sizeof(float) * (size_t)p.dim, current_stream()>>>(p);
    return TOPS_CHECK_LAUNCH("norm_rotary_general");
}

// Vector form: dim a multiple of 8 up to 256, 16-byte aligned rows.  LPH lanes hold a head, eight elements each, and work through HB heads of one token, whose
// cosines and sines are read once for them; all HB loads are in flight while position, slot and table row are looked up.  Issue slots bound it next to HBM:
// arithmetic is two floats to an instruction, and 64 registers a thread keep 32 warps on an SM (112 us with 80 of them, 94 us with 64: 4.4 TB/s).  (Fetching the next item ahead was measured and is not done: its registers cost more warps than it hid, 166 against 122 us
// for 16384 tokens of 32 + 2 * 8 heads of 128.)
// Three layouts of a head over the lanes: eight neighbours with interleaved pairs; four and four elements half a head apart where
// the whole head is turned in pairs (i, i + half), so that a lane holds both elements of its pairs; eight neighbours and a shuffle to the partner's lane
// where only part of the head is turned.
enum RotaryLayout { kLayoutInterleaved = 0, kLayoutPaired = 1, kLayoutShuffled = 2 };

// Eight elements as they lie in memory: at d and d + 4, or (paired) four at each of two places.
template <typename T> struct Raw8 { uint4 w[sizeof(T) / 2]; };
template <typename T, bool PAIRED> __device__ __forceinline__ Raw8<T> load_raw8(const T* first, int apart) {
    Raw8<T> r;
    if constexpr (PAIRED && sizeof(T) == 2) {
        const uint2 a = *reinterpret_cast<const uint2*>(first), b = *reinterpret_cast<const uint2*>(first + apart);
        r.w[0] = make_uint4(a.x, a.y, b.x, b.y);
    } else if constexpr (PAIRED) {
        r.w[0] = *reinterpret_cast<const uint4*>(first);
        r.w[1] = *reinterpret_cast<const uint4*>(first + apart);
    } else {
        #pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; i++) r.w[i] = reinterpret_cast<const uint4*>(first)[i];
    }
    return r;
}
template <typename T> __device__ __forceinline__ void widen8(const Raw8<T>& r, float (&x)[8]) {
    const T* t = reinterpret_cast<const T*>(&r);
    #pragma unroll
    for (int i = 0; i < 8; i++) x[i] = to_float(t[i]);
}
template <typename T, bool PAIRED> __device__ __forceinline__ void load8(const T* first, int apart, float (&x)[8]) { widen8(load_raw8<T, PAIRED>(first, apart), x); }
template <typename T, bool PAIRED> __device__ __forceinline__ void store8(T* to, int apart, const float (&x)[8]) {
    if constexpr (sizeof(T) == 4) {
        reinterpret_cast<float4*>(to)[0] = make_float4(x[0], x[1], x[2], x[3]);
        *reinterpret_cast<float4*>(to + (PAIRED ? apart : 4)) = make_float4(x[4], x[5], x[6], x[7]);
    } else if constexpr (PAIRED) {
        *reinterpret_cast<uint2*>(to) = make_uint2(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]));
        *reinterpret_cast<uint2*>(to + apart) = make_uint2(pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7]));
    } else {
        *reinterpret_cast<uint4*>(to) = make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7]));
    }
}

// r = a * b (+ c) for two floats in one instruction.
__device__ __forceinline__ void mul_pair(float& r0, float& r1, float a0, float a1, float b0, float b1) {
    asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmul.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}"
        : "=f"(r0), "=f"(r1) : "f"(a0), "f"(a1), "f"(b0), "f"(b1));
}
__device__ __forceinline__ void fma_pair(float& r0, float& r1, float a0, float a1, float b0, float b1, float c0, float c1) {
    asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\tfma.rn.f32x2 a, a, b, c;\n\tmov.b64 {%0, %1}, a;\n\t}"
        : "=f"(r0), "=f"(r1) : "f"(a0), "f"(a1), "f"(b0), "f"(b1), "f"(c0), "f"(c1));
}

constexpr int kNormThreads = 128;

template <typename T, int LPH, int HB, int LAYOUT>
__global__ void __launch_bounds__(kNormThreads, sizeof(T) == 2 ? 8 : 6) norm_rotary_vector(const __grid_constant__ NormRotaryProblem p, const uint32_t items) {
    constexpr int PER_WARP = 32 / LPH;
    constexpr bool PAIRED = LAYOUT == kLayoutPaired;
    const int lane = threadIdx.x & 31, in_head = lane % LPH, group = lane / LPH;
    const uint32_t warp = blockIdx.x * (kNormThreads / 32) + (threadIdx.x >> 5), warps = gridDim.x * (kNormThreads / 32);
    const int half = p.half, d = in_head * (PAIRED ? 4 : 8);
    const bool mine = in_head * 8 < p.dim;
    // shuffled: the lane that holds the other elements of this lane's pairs
    const bool second = LAYOUT == kLayoutShuffled && d >= half;
    const int partner = LAYOUT == kLayoutShuffled ? (lane - in_head) + (d < 2 * half ? (second ? d - half : d + half) / 8 : in_head) : lane;

    for (uint32_t base = warp * PER_WARP; base < items; base += warps * PER_WARP) {
        const uint32_t item = base + group;
        const bool there = item < items;
        const uint32_t token = p.block_div.div(there ? item : 0u);
        int block = (int)((there ? item : 0u) - token * p.block_div.d), which = 0;
        if (block >= p.blocks[0]) { block -= p.blocks[0]; which = 1; if (block >= p.blocks[1]) { block -= p.blocks[1]; which = 2; } }
        const HeadsView& h = p.part[which];
        const int head0 = block * HB, batch = (int)p.seq_div.div(token), in_row = (int)token - batch * p.seq;
        const T* in = reinterpret_cast<const T*>(h.in) + batch * h.in_batch + in_row * h.in_token + head0 * h.in_head + d;
        Raw8<T> raw[HB];
        #pragma unroll
        for (int i = 0; i < HB; i++) if (there && mine && head0 + i < h.heads) raw[i] = load_raw8<T, PAIRED>(in + i * h.in_head, half);
        const bool normed = h.weight && mine;
        float w[8];
        if (normed) {
            if (h.weight_f32) load8<float, PAIRED>(reinterpret_cast<const float*>(h.weight) + d, half, w);
            else load8<T, PAIRED>(reinterpret_cast<const T*>(h.weight) + d, half, w);
        }
        const TokenPlace at = place_token(p, (int)token, p.positions != nullptr, h.cache != nullptr);
        constexpr int N = LAYOUT == kLayoutShuffled ? 8 : 4;
        float c[N], s[N];
        const bool turned = h.rotate && at.table_row >= 0 && (PAIRED ? mine : d < 2 * half);
        if (turned) {
            const long long row = (long long)at.table_row * half + (LAYOUT == kLayoutInterleaved ? d / 2 : (second ? d - half : d));
            #pragma unroll
            for (int e = 0; e < N; e += 4) {
                const float4 cv = *reinterpret_cast<const float4*>(p.cos_table + row + e), sv = *reinterpret_cast<const float4*>(p.sin_table + row + e);
                c[e] = cv.x; c[e + 1] = cv.y; c[e + 2] = cv.z; c[e + 3] = cv.w;
                s[e] = sv.x; s[e + 1] = sv.y; s[e + 2] = sv.z; s[e + 3] = sv.w;
            }
        }
        T* out = h.out ? reinterpret_cast<T*>(h.out) + batch * h.out_batch + in_row * h.out_token + head0 * h.out_head + d : nullptr;
        T* cache = h.cache && at.slot >= 0 && !at.bad_position ? reinterpret_cast<T*>(h.cache) + (at.slot * p.cache_heads + head0) * p.dim + d : nullptr;
        const bool any_normed = __any_sync(~0u, normed);     // the groups of a warp may be in different parts: all of them reduce, or none
        #pragma unroll
        for (int i = 0; i < HB; i++) {
            const bool here = there && mine && head0 + i < h.heads;
            float x[8];
            if (here) widen8(raw[i], x);
            else {
                #pragma unroll
                for (int e = 0; e < 8; e++) x[e] = 0.0f;
            }
            if (any_normed) {
                float sum0 = 0.0f, sum1 = 0.0f;
                #pragma unroll
                for (int e = 0; e < 8; e += 2) fma_pair(sum0, sum1, x[e], x[e + 1], x[e], x[e + 1], sum0, sum1);
                float sum = sum0 + sum1;
                #pragma unroll
                for (int o = LPH / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
                const float factor = rsqrtf(__fmaf_rn(sum, p.inv_dim, p.epsilon));
                if (normed)
                    #pragma unroll
                    for (int e = 0; e < 8; e += 2) {
                        mul_pair(x[e], x[e + 1], x[e], x[e + 1], factor, factor);
                        mul_pair(x[e], x[e + 1], x[e], x[e + 1], w[e], w[e + 1]);
                    }
            }
            if constexpr (LAYOUT == kLayoutShuffled) {
                #pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float other = __shfl_sync(~0u, x[e], partner);
                    if (turned) x[e] = second ? __fmaf_rn(other, s[e], x[e] * c[e]) : __fmaf_rn(x[e], c[e], -(other * s[e]));
                }
            } else if (turned) {
                #pragma unroll
                for (int e = 0; e < 4; e += 2) {
                    const int a0 = PAIRED ? e : 2 * e, a1 = PAIRED ? e + 1 : 2 * e + 2, b0 = PAIRED ? e + 4 : 2 * e + 1, b1 = PAIRED ? e + 5 : 2 * e + 3;
                    float t0, t1, u0, u1;
                    mul_pair(t0, t1, x[b0], x[b1], -s[e], -s[e + 1]);
                    mul_pair(u0, u1, x[b0], x[b1], c[e], c[e + 1]);
                    fma_pair(x[b0], x[b1], x[a0], x[a1], s[e], s[e + 1], u0, u1);
                    fma_pair(x[a0], x[a1], x[a0], x[a1], c[e], c[e + 1], t0, t1);
                }
            }
            if (here) {
                if (at.bad_position)
                    #pragma unroll
                    for (int e = 0; e < 8; e++) x[e] = 0.0f;
                if (out) store8<T, PAIRED>(out + i * h.out_head, half, x);
                if (cache) store8<T, PAIRED>(cache + (long long)i * p.dim, half, x);
            }
        }
    }
}

// Whether every row that the vector form reads or writes starts on a 16-byte boundary, and pairs are met lane by lane.
static bool vector_form(const NormRotaryProblem& p) {
    if (p.dim % 8 != 0 || p.dim > 256 || p.half % 4 != 0 || (!p.interleaved && 2 * p.half != p.dim && p.half % 8 != 0)) return false;
    uintptr_t bits = reinterpret_cast<uintptr_t>(p.cos_table) | reinterpret_cast<uintptr_t>(p.sin_table);
    for (const HeadsView& h : p.part)
        for (const void* a : {h.in, (const void*)h.out, (const void*)h.cache, h.weight}) bits |= reinterpret_cast<uintptr_t>(a);
    return (bits & 15) == 0;
}

template <typename T, int LPH, int HB> static bool launch_vector(NormRotaryProblem p) {
    DeviceState* st = acquire_device();
    if (!st) return false;
    int blocks = 0;
    for (int i = 0; i < 3; i++) blocks += p.blocks[i] = (p.part[i].heads + HB - 1) / HB;
    p.block_div.set((uint32_t)blocks);
    const uint32_t items = (uint32_t)p.tokens * (uint32_t)blocks;
    const int grid = grid_for(items, kNormThreads / LPH, st->sm_count, 16);
    if (p.interleaved || p.half == 0) norm_rotary_vector<T, LPH, HB, kLayoutInterleaved><<<grid, kNormThreads, 0, current_stream()>>>(p, items);
    else if (2 * p.half == p.dim) norm_rotary_vector<T, LPH, HB, kLayoutPaired><<<grid, kNormThreads, 0, current_stream()>>>(p, items);
    else norm_rotary_vector<T, LPH, HB, kLayoutShuffled><<<grid, kNormThreads, 0, current_stream()>>>(p, items);
    return TOPS_CHECK_LAUNCH("norm_rotary_vector");
}

template <typename T, int LPH> static bool launch_vector_heads(const NormRotaryProblem& p) {
    // four heads per group share a token's table row (measured 94 us, two 121, eight 149 for 16384 tokens of 48 heads of 128); with too few heads to give every SM 512
    // threads that way, one each spreads them further
    const long long heads = (long long)p.tokens * (p.part[0].heads + p.part[1].heads + p.part[2].heads);
    return heads * LPH >= (long long)kNumSMs * 512 * 4 ? launch_vector<T, LPH, 4>(p) : launch_vector<T, LPH, 1>(p);
}

template <typename T> static bool launch_any(const NormRotaryProblem& p) {
    if (!vector_form(p)) return launch_general<T>(p);
    if (p.dim <= 64) return launch_vector_heads<T, 8>(p);
    if (p.dim <= 128) return launch_vector_heads<T, 16>(p);
    return launch_vector_heads<T, 32>(p);
}

static bool run_norm_rotary(const NormRotaryProblem& p, int dtype) {
    switch (dtype) {
        case DTYPE_FLOAT16:  return launch_any<__half>(p);
        case DTYPE_BFLOAT16: return launch_any<__nv_bfloat16>(p);
        default:             return launch_any<float>(p);
    }
}

// Strides of a dense [..., S, H, D] or, heads_first, [B, H, S, D] tensor with `heads_in_memory` heads.
static void strides_of(long long& batch, long long& token, long long& head, bool heads_first, long long seq, long long heads_in_memory, long long dim) {
    batch = seq * heads_in_memory * dim;
    token = heads_first ? dim : heads_in_memory * dim;
    head = heads_first ? seq * dim : dim;
}

}  // namespace tops

using namespace tops;

TOPS_API int tops_qk_norm_rotary_forward(const QKNormRotaryCall* call) {
    const char* name = "tops_qk_norm_rotary_forward";
    if (!call) return call_fail(name, TOPS_ERR_INVALID, "null call", {});
    const QKNormRotaryCall& c = *call;
    OutputList outs;
    for (const Tensor* t : {(const Tensor*)c.q_out, (const Tensor*)c.k_out}) if (t) outs.tensors[outs.count++] = t;
    outs.outputs = outs.count;
    for (const Tensor* t : {c.q, c.k, c.v, c.q_weight, c.k_weight, c.cos_table, c.sin_table, c.positions, (const Tensor*)c.key_cache, (const Tensor*)c.value_cache, c.slots})
        outs.tensors[outs.count++] = t;
    auto fail = [&](int code, const char* what) { return call_fail(name, code, what, outs); };
    for (int i = 0; i < outs.count; i++)
        if (outs.tensors[i] && !outs.tensors[i]->data) return fail(TOPS_ERR_INVALID, "a tensor without data");
    if (!c.q || !c.q_out) return fail(TOPS_ERR_INVALID, "q and q_out are required");
    const bool packed = c.packed_kv_heads > 0, first = c.heads_first != 0, cached = c.key_cache != nullptr;
    if (c.packed_kv_heads < 0 || (packed && (c.k || c.v || first))) return fail(TOPS_ERR_INVALID, "packed keys and values come inside q: k and v NULL, not heads_first");
    if (c.q->ndim < 2 || (first && c.q->ndim != 4)) return fail(TOPS_ERR_INVALID, "q is [..., tokens, heads, dim] or, heads_first, [batch, heads, tokens, dim]");
    const int nd = c.q->ndim, dim = c.q->shape[nd - 1], heads_at = first ? 1 : nd - 2;
    const int heads = c.q->shape[heads_at] - (packed ? 2 * c.packed_kv_heads : 0);
    if (dim < 1 || dim > 1024) return fail(TOPS_ERR_UNSUPPORTED, "heads of 1 to 1024 elements");
    if (heads < 1) return fail(TOPS_ERR_INVALID, "no query heads");
    const int dt = c.q->dtype;
    if (dt != DTYPE_FLOAT16 && dt != DTYPE_BFLOAT16 && dt != DTYPE_FLOAT32) return fail(TOPS_ERR_UNSUPPORTED, "float16, bfloat16 or float32");
    const size_t token_count = c.q->size / ((size_t)c.q->shape[heads_at] * (size_t)dim);
    if (token_count >= 0x7FFFFFFFull / 64) return fail(TOPS_ERR_UNSUPPORTED, "fewer than 2^25 tokens");
    // shapes of the outputs: q's with its own heads
    auto shaped = [&](const Tensor* t, int want_heads) {
        if (t->ndim != nd || t->dtype != dt) return false;
        for (int i = 0; i < nd; i++) if (t->shape[i] != (i == heads_at ? want_heads : c.q->shape[i])) return false;
        return true;
    };
    if (!shaped(c.q_out, heads)) return fail(TOPS_ERR_INVALID, "q_out has q's shape (packed: with the query heads alone) and type");
    int kv_heads = packed ? c.packed_kv_heads : 0;
    if (c.k) {
        if (c.k->ndim != nd) return fail(TOPS_ERR_INVALID, "k has q's rank");
        kv_heads = c.k->shape[heads_at];
        if (kv_heads < 1 || !shaped(c.k, kv_heads)) return fail(TOPS_ERR_INVALID, "k has q's shape but for the heads, and its type");
    }
    const bool keys = packed || c.k;
    if ((unsigned long long)token_count * (unsigned long long)((long long)heads + 2ll * kv_heads) >= 0x7FFFFFFFull / 4) return fail(TOPS_ERR_UNSUPPORTED, "fewer than 2^29 heads over all tokens");
    if (c.v && (!c.k || !shaped(c.v, kv_heads))) return fail(TOPS_ERR_INVALID, "v has k's shape and type");
    if (c.k_out && (!keys || !shaped(c.k_out, kv_heads))) return fail(TOPS_ERR_INVALID, "k_out has the key heads' shape and type");
    if (keys && !c.k_out && !cached) return fail(TOPS_ERR_INVALID, "keys need k_out or a cache to go to");
    if (cached != (c.value_cache != nullptr) || cached != (c.slots != nullptr) || (cached && (!keys || (!packed && !c.v))))
        return fail(TOPS_ERR_INVALID, "key_cache, value_cache and slots come together, with keys and values to store");
    if (!cached && c.v) return fail(TOPS_ERR_INVALID, "v is only read for a cache");
    if (cached) {
        const Tensor* kc = c.key_cache;
        if (kc->ndim != 4 || !same_shape(kc, c.value_cache) || kc->dtype != dt || c.value_cache->dtype != dt || kc->shape[2] != kv_heads || kc->shape[3] != dim)
            return fail(TOPS_ERR_INVALID, "key_cache and value_cache are [pages, page_size, kv_heads, dim] of q's type");
        if ((c.slots->dtype != DTYPE_INT32 && c.slots->dtype != DTYPE_INT64) || c.slots->size != token_count)
            return fail(TOPS_ERR_INVALID, "slots is int32 or int64 with one entry per token");
    }
    for (const Tensor* w : {c.q_weight, c.k_weight})
        if (w && (w->size != (size_t)dim || (w->dtype != dt && w->dtype != DTYPE_FLOAT32))) return fail(TOPS_ERR_INVALID, "weights have dim elements of q's type or float32");
    if (c.k_weight && !keys) return fail(TOPS_ERR_INVALID, "k_weight without keys");
    if ((c.q_weight || c.k_weight) && !(std::isfinite(c.epsilon) && c.epsilon >= 0.0f)) return fail(TOPS_ERR_INVALID, "epsilon is finite and not negative");
    const bool rotate = c.cos_table != nullptr;
    if (rotate != (c.sin_table != nullptr) || rotate != (c.positions != nullptr)) return fail(TOPS_ERR_INVALID, "cos_table, sin_table and positions come together");
    if (rotate) {
        if (c.cos_table->ndim != 2 || !same_shape(c.cos_table, c.sin_table) || c.cos_table->dtype != DTYPE_FLOAT32 || c.sin_table->dtype != DTYPE_FLOAT32 ||
            c.cos_table->shape[1] < 1 || 2 * (long long)c.cos_table->shape[1] > dim)
            return fail(TOPS_ERR_INVALID, "the tables are float32 [positions, rotary_dim / 2] with rotary_dim at most dim");
        if ((c.positions->dtype != DTYPE_INT32 && c.positions->dtype != DTYPE_INT64) || c.positions->size != token_count)
            return fail(TOPS_ERR_INVALID, "positions is int32 or int64 with one entry per token");
    }
    // an output may be its own operand, element for element, and nothing else
    for (int i = 0; i < outs.outputs; i++)
        for (int j = i + 1; j < outs.count; j++) {
            const Tensor *o = outs.tensors[i], *t = outs.tensors[j];
            const bool itself = !packed && ((o == c.q_out && t == c.q) || (o == c.k_out && t == c.k)) && o->data == t->data;
            if (!itself && overlap(o, t)) return fail(TOPS_ERR_INVALID, "an output shares memory with another tensor of the call");
        }
    if (cached && overlap(c.key_cache, c.value_cache)) return fail(TOPS_ERR_INVALID, "the two caches share memory");
    if (cached)
        for (const Tensor* cache : {c.key_cache, c.value_cache})
            for (int j = outs.outputs; j < outs.count; j++)
                if (outs.tensors[j] != c.key_cache && outs.tensors[j] != c.value_cache && overlap(cache, outs.tensors[j])) return fail(TOPS_ERR_INVALID, "a cache shares memory with another tensor of the call");
    for (int i = 0; i < outs.count; i++)
        if (!on_current_device({outs.tensors[i]})) return call_fail(name, TOPS_ERR_INVALID, "a tensor belongs to another device than the current one", {});
    if (!acquire_device()) return tops_last_error();
    if (token_count == 0) return TOPS_OK;

    NormRotaryProblem p;
    const long long size = dtype_bytes(dt);
    p.tokens = (int)token_count;
    p.seq = first ? c.q->shape[2] : p.tokens;
    p.seq_div.set((uint32_t)p.seq);
    p.dim = dim;
    p.half = rotate ? c.cos_table->shape[1] : 0;
    p.interleaved = c.interleaved != 0;
    p.epsilon = c.epsilon;
    p.inv_dim = 1.0f / (float)dim;
    if (rotate) {
        p.cos_table = reinterpret_cast<const float*>(c.cos_table->data);
        p.sin_table = reinterpret_cast<const float*>(c.sin_table->data);
        p.table_rows = c.cos_table->shape[0];
        p.positions = c.positions->data;
        p.positions_64 = c.positions->dtype == DTYPE_INT64;
    }
    if (cached) {
        p.slots = c.slots->data;
        p.slots_64 = c.slots->dtype == DTYPE_INT64;
        p.cache_rows = (long long)c.key_cache->shape[0] * c.key_cache->shape[1];
        p.cache_heads = kv_heads;
    }
    p.status = device_status_word();
    HeadsView& q = p.part[0];
    q.in = c.q->data;
    q.out = c.q_out->data;
    q.weight = c.q_weight ? c.q_weight->data : nullptr;
    q.weight_f32 = c.q_weight && c.q_weight->dtype == DTYPE_FLOAT32;
    q.heads = heads;
    q.rotate = rotate;
    strides_of(q.in_batch, q.in_token, q.in_head, first, p.seq, c.q->shape[heads_at], dim);
    strides_of(q.out_batch, q.out_token, q.out_head, first, p.seq, heads, dim);
    if (keys) {
        HeadsView& k = p.part[1];
        k = q;
        k.in = packed ? (const char*)c.q->data + (long long)heads * dim * size : (const char*)c.k->data;
        k.out = c.k_out ? c.k_out->data : nullptr;
        k.cache = cached ? c.key_cache->data : nullptr;
        k.weight = c.k_weight ? c.k_weight->data : nullptr;
        k.weight_f32 = c.k_weight && c.k_weight->dtype == DTYPE_FLOAT32;
        k.heads = kv_heads;
        if (!packed) strides_of(k.in_batch, k.in_token, k.in_head, first, p.seq, kv_heads, dim);
        strides_of(k.out_batch, k.out_token, k.out_head, first, p.seq, kv_heads, dim);
        if (cached) {
            HeadsView& v = p.part[2];
            v = k;
            v.in = packed ? (const char*)k.in + (long long)kv_heads * dim * size : (const char*)c.v->data;
            v.out = nullptr;
            v.cache = c.value_cache->data;
            v.weight = nullptr;
            v.rotate = 0;
        }
    }
    if (!run_norm_rotary(p, dt)) return tops_last_error();
    finish_op();
    return TOPS_OK;
}
