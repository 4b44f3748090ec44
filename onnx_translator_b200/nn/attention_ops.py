"""Graph nodes of a decoder with cached keys and values: norms and rotation of the heads with the append to the cache, attention of
new tokens over a paged cache, attention to an encoder's states.  The reference has no attention operator; its graphs spell
it out as MatMul, Softmax and element-wise nodes (nn/Operators.py:1361-1432, 671-704).  The nodes have the interface of the operator classes in
Operators.py and one C call each (include/tensor_ops_b200.h documents shapes, types and refusals)."""
from __future__ import annotations

import ctypes

from . import Ops, Tensor, Tensor_
from .. import capi
from ..capi import CCrossAttentionCall, CPagedAttentionCall, CQKNormRotaryCall
from ..device import DeviceArray


class _StructCall(Ops):
    """Fills a call struct with tensor handles and runs it; operands stay on the device (a cache is updated where it lives)."""

    def _new_output(self, shape, dtype):
        """Zero-filled: rows that belong to no sequence are not written by the kernels."""
        out = DeviceArray.empty(shape, dtype, zero=True, lib=self.lib)
        handle, out.handle = out.handle, None
        return handle

    def _run(self, entry, call, operands, outputs):
        """``operands``: struct member -> Tensor or None; ``outputs``: struct member -> (shape, dtype)."""
        handles, made = [], {}
        try:
            for member, t in operands.items():
                if t is not None:
                    handles.append(self._numpy_to_ctensor(t.to_device().data, t.dtype))
                    setattr(call, member, ctypes.cast(handles[-1], ctypes.c_void_p))
            for member, (shape, dtype) in outputs.items():
                made[member] = self._new_output(shape, dtype)
                setattr(call, member, ctypes.cast(made[member], ctypes.c_void_p))
            rc = getattr(self.lib, entry)(ctypes.byref(call))
        except Exception:
            for h in list(made.values()):
                self.lib.free_tensor(h)
            raise
        finally:
            for h in handles:
                self.lib.free_tensor(h)
        if rc:
            for h in made.values():
                self.lib.free_tensor(h)
            capi.check(self.lib)
            raise capi.TensorOpsError(f"{entry} failed with code {rc}")
        results = [self._finish([], made[m], shape, dtype) for m, (shape, dtype) in outputs.items()]
        return results[0] if len(results) == 1 else results


class QKNormRotary(_StructCall):
    """RMS norm per head, rotary position embedding and the append to a paged cache, in one pass.

    inputs: [q, k or "", v or "", q_weight or "", k_weight or "", cos or "", sin or "", positions or "", key_cache or "",
    value_cache or "", slots or ""].  With ``packed_kv_heads`` q is the whole projection [..., tokens, heads + 2 * packed_kv_heads, dim].
    outputs: [rotated queries] or [rotated queries, rotated keys] (always the latter where there are keys and no cache).  The cache tensors
    are written in place."""

    def __init__(self, inputs, outputs, packed_kv_heads=0, heads_first=False, interleaved=False, epsilon=1e-6, dtype="bfloat16", version="17"):
        super().__init__(inputs, outputs)
        self.packed_kv_heads, self.heads_first, self.interleaved = int(packed_kv_heads), bool(heads_first), bool(interleaved)
        self.epsilon, self.dtype, self.version = float(epsilon), dtype, version

    def _shapes(self, q_shape, k_shape, cached):
        at = 1 if self.heads_first else len(q_shape) - 2
        heads = q_shape[at] - 2 * self.packed_kv_heads
        kv_heads = self.packed_kv_heads or (k_shape[at] if k_shape is not None else 0)
        with_heads = lambda n: tuple(n if i == at else s for i, s in enumerate(q_shape))  # noqa: E731
        shapes = [with_heads(heads)]
        if kv_heads and (len(self.outputs) == 2 or not cached):
            shapes.append(with_heads(kv_heads))
        return shapes

    def forward(self, q: Tensor, k: Tensor = None, v: Tensor = None, q_weight: Tensor = None, k_weight: Tensor = None, cos: Tensor = None,
                sin: Tensor = None, positions: Tensor = None, key_cache: Tensor = None, value_cache: Tensor = None, slots: Tensor = None) -> dict:
        call = CQKNormRotaryCall(packed_kv_heads=self.packed_kv_heads, heads_first=int(self.heads_first), epsilon=self.epsilon,
                                 interleaved=int(self.interleaved))
        shapes = self._shapes(self._shape_of(q), None if k is None else self._shape_of(k), key_cache is not None)
        outs = dict(zip(("q_out", "k_out"), ((s, q.dtype) for s in shapes)))
        return self._publish(self._run("tops_qk_norm_rotary_forward", call, {
            "q": q, "k": k, "v": v, "q_weight": q_weight, "k_weight": k_weight, "cos_table": cos, "sin_table": sin, "positions": positions,
            "key_cache": key_cache, "value_cache": value_cache, "slots": slots}, outs))

    def forward_(self, q: Tensor_, k: Tensor_ = None, v=None, q_weight=None, k_weight=None, cos=None, sin=None, positions=None,
                 key_cache=None, value_cache=None, slots=None) -> dict:
        shapes = self._shapes(tuple(q.size), None if k is None else tuple(k.size), key_cache is not None)
        outs = [Tensor_(*s, dtype=q.dtype) for s in shapes]
        return self._publish(outs[0] if len(outs) == 1 else outs)


class PagedAttention(_StructCall):
    """A ragged batch of new tokens attends, causally, over a paged cache that holds their keys and values already.

    inputs: [q, key_cache, value_cache, page_table, query_start, kv_length]; ``scale`` None is 1 / sqrt(dim).  Rows of the result that
    belong to no sequence are zeros; in a recorded plan, which reuses its tensors, they keep what the last run that owned them left."""

    def __init__(self, inputs, outputs, scale=None, window=0, dtype="bfloat16", version="17"):
        super().__init__(inputs, outputs)
        self.scale, self.window, self.dtype, self.version = scale, int(window), dtype, version

    def forward(self, q: Tensor, key_cache: Tensor, value_cache: Tensor, page_table: Tensor, query_start: Tensor, kv_length: Tensor) -> dict:
        shape = self._shape_of(q)
        call = CPagedAttentionCall(scale=shape[-1] ** -0.5 if self.scale is None else float(self.scale), window=self.window)
        return self._publish(self._run("tops_paged_attention_forward", call, {
            "q": q, "key_cache": key_cache, "value_cache": value_cache, "page_table": page_table, "query_start": query_start,
            "kv_length": kv_length}, {"y": (shape, q.dtype)}))

    def forward_(self, q: Tensor_, *_) -> dict:
        return self._publish(Tensor_(*q.size, dtype=q.dtype))


class CrossAttention(_StructCall):
    """Queries attend to an encoder's states of another length, without causality.

    inputs: [q, k, v, key_length or "", mask or ""]; ``scale`` None is 1 / sqrt(dim)."""

    def __init__(self, inputs, outputs, scale=None, heads_first=False, dtype="bfloat16", version="17"):
        super().__init__(inputs, outputs)
        self.scale, self.heads_first, self.dtype, self.version = scale, bool(heads_first), dtype, version

    def forward(self, q: Tensor, k: Tensor, v: Tensor, key_length: Tensor = None, mask: Tensor = None) -> dict:
        shape = self._shape_of(q)
        call = CCrossAttentionCall(scale=shape[-1] ** -0.5 if self.scale is None else float(self.scale), heads_first=int(self.heads_first))
        return self._publish(self._run("tops_cross_attention_forward", call, {"q": q, "k": k, "v": v, "key_length": key_length, "mask": mask},
                                       {"y": (shape, q.dtype)}))

    def forward_(self, q: Tensor_, *_) -> dict:
        return self._publish(Tensor_(*q.size, dtype=q.dtype))
