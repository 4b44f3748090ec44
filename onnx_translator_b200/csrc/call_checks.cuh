// Host-side argument checks shared by the operators whose calls are structs of many tensors.
#pragma once

#include "common.cuh"

#include <initializer_list>

namespace tops {

inline bool tensor_given(const Tensor* t) { return t && t->data; }

inline bool same_shape(const Tensor* a, const Tensor* b) {
    if (a->ndim != b->ndim) return false;
    for (int i = 0; i < a->ndim; i++) if (a->shape[i] != b->shape[i]) return false;
    return true;
}

// Whether two tensors share a byte of memory (null and empty tensors share nothing).
inline bool overlap(const Tensor* a, const Tensor* b) {
    if (!tensor_given(a) || !tensor_given(b) || a->size == 0 || b->size == 0) return false;
    const uintptr_t a0 = reinterpret_cast<uintptr_t>(a->data), b0 = reinterpret_cast<uintptr_t>(b->data);
    return a0 < b0 + b->size * (size_t)dtype_bytes((int)b->dtype) && b0 < a0 + a->size * (size_t)dtype_bytes((int)a->dtype);
}

inline bool on_current_device(std::initializer_list<const Tensor*> tensors) {
    const int device = tops_get_device();
    for (const Tensor* t : tensors) if (t && tensor_device(t) != device) return false;
    return true;
}

// A rejected call: records the error and zero-fills the outputs (the first `n_outs` tensors) that share no memory with an operand.
struct OutputList {
    static constexpr int kMost = 16;
    const Tensor* tensors[kMost] = {nullptr};
    int outputs = 0, count = 0;
    OutputList() = default;
    // one output, then the operands
    OutputList(std::initializer_list<const Tensor*> list) { outputs = 1; for (const Tensor* t : list) if (count < kMost) tensors[count++] = t; }
};

inline int call_fail(const char* name, int code, const char* what, const OutputList& list) {
    set_error(code, "%s: %s", name, what);
    for (int i = 0; i < list.outputs; i++) {
        const Tensor* out = list.tensors[i];
        bool shared = !tensor_given(out) || tensor_device(out) != tops_get_device();
        for (int j = list.outputs; j < list.count && !shared; j++) shared = overlap(out, list.tensors[j]);
        if (!shared) zero_fill(const_cast<Tensor*>(out));
    }
    return tops_last_error();
}

}  // namespace tops
