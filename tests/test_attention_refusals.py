"""Calls of the attention operators that are refused.  The checks run on the host before any CUDA call, so they are tested without a GPU, on
tensors that describe memory nobody touches."""
import ctypes

import numpy as np
import pytest

from onnx_translator_b200 import capi, nn
from onnx_translator_b200.nn.attention_ops import CrossAttention, PagedAttention, QKNormRotary


@pytest.fixture(scope="module")
def lib():
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is present: a refused call would clear outputs that do not exist")
    return capi.load()


_next = [1 << 40]


def T(lib, *shape, dtype="bfloat16", at=None):
    """A tensor at an address of its own (or `at`); never dereferenced."""
    arr, nd = capi.shape_array(shape)
    if at is None:
        _next[0] += 1 << 44
        at = _next[0]
    return lib.tops_wrap(at, arr, nd, capi.DTYPE_MAP[dtype])


def _try(lib, entry, struct, tensors, **scalars):
    call = struct(**scalars)
    for name, t in tensors.items():
        setattr(call, name, None if t is None else ctypes.cast(t, ctypes.c_void_p))
    lib.tops_clear_error()
    rc = getattr(lib, entry)(ctypes.byref(call))
    message = lib.tops_last_error_message().decode()
    lib.tops_clear_error()
    return rc, message


INVALID, NO_DEVICE, UNSUPPORTED = 1, 3, 5
NO_GPU = (2, 3)          # what an accepted call ends with here


def _paged(lib, change=None, **scalars):
    t = {"q": T(lib, 6, 8, 64), "key_cache": T(lib, 10, 16, 2, 64), "value_cache": T(lib, 10, 16, 2, 64), "page_table": T(lib, 3, 5, dtype="int32"),
         "query_start": T(lib, 4, dtype="int32"), "kv_length": T(lib, 3, dtype="int32"), "y": T(lib, 6, 8, 64)}
    t.update(change(t) if callable(change) else change or {})
    return _try(lib, "tops_paged_attention_forward", capi.CPagedAttentionCall, t, **{"scale": 0.125, "window": 0, **scalars})


def test_paged_attention_accepts_and_refuses(lib):
    assert _paged(lib)[0] in NO_GPU
    for name in ("q", "key_cache", "value_cache", "page_table", "query_start", "kv_length", "y"):
        assert _paged(lib, {name: None})[0] == INVALID
        assert _paged(lib, lambda t: {name: T(lib, *[t[name].contents.shape[i] for i in range(t[name].contents.ndim)],
                                              dtype=capi.CODE_TO_DTYPE[t[name].contents.dtype], at=0)})[0] == INVALID
    cases = [({"y": T(lib, 6, 8, 32)}, INVALID), ({"y": T(lib, 6, 8, 64, dtype="float16")}, UNSUPPORTED), ({"q": T(lib, 6, 512), "y": T(lib, 6, 512)}, INVALID),
             ({"key_cache": T(lib, 10, 16, 2, 32)}, INVALID), ({"value_cache": T(lib, 9, 16, 2, 64)}, INVALID),
             ({"key_cache": T(lib, 10, 16, 2, 64, dtype="float16")}, UNSUPPORTED),
             ({"key_cache": T(lib, 10, 16, 3, 64), "value_cache": T(lib, 10, 16, 3, 64)}, UNSUPPORTED),
             ({"key_cache": T(lib, 10, 16, 0, 64), "value_cache": T(lib, 10, 16, 0, 64)}, UNSUPPORTED),
             ({"key_cache": T(lib, 10, 0, 2, 64), "value_cache": T(lib, 10, 0, 2, 64)}, UNSUPPORTED),
             ({"page_table": T(lib, 3, 5, dtype="int64")}, INVALID), ({"query_start": T(lib, 4, dtype="int64")}, INVALID),
             ({"kv_length": T(lib, 3, dtype="int64")}, INVALID), ({"query_start": T(lib, 3, dtype="int32")}, INVALID),
             ({"kv_length": T(lib, 4, dtype="int32")}, INVALID), ({"page_table": T(lib, 15, dtype="int32")}, INVALID)]
    for change, code in cases:
        rc, message = _paged(lib, change)
        assert rc == code and "tops_paged_attention_forward" in message, (change, rc, message)
    for dtype in ("float64", "int8", "float8_e4m3"):
        assert _paged(lib, {n: T(lib, *s, dtype=dtype) for n, s in (("q", (6, 8, 64)), ("y", (6, 8, 64)), ("key_cache", (10, 16, 2, 64)),
                                                                   ("value_cache", (10, 16, 2, 64)))})[0] == UNSUPPORTED
    big = {"q": T(lib, 6, 8, 264), "y": T(lib, 6, 8, 264), "key_cache": T(lib, 10, 16, 2, 264), "value_cache": T(lib, 10, 16, 2, 264)}
    assert _paged(lib, big)[0] == UNSUPPORTED
    huge = {"key_cache": T(lib, 1 << 20, 1 << 12, 2, 64), "value_cache": T(lib, 1 << 20, 1 << 12, 2, 64)}
    assert _paged(lib, huge)[0] == UNSUPPORTED
    assert _paged(lib, {"page_table": T(lib, 3, 1 << 27, dtype="int32")})[0] == UNSUPPORTED
    for scale in (float("nan"), float("inf")):
        assert _paged(lib, scale=scale)[0] == INVALID
    assert _paged(lib, window=-1)[0] == INVALID
    for name in ("q", "key_cache", "value_cache"):                   # y on top of an operand, or reaching into it
        assert _paged(lib, lambda t: {"y": T(lib, 6, 8, 64, at=t[name].contents.data)})[0] == INVALID
        assert _paged(lib, lambda t: {"y": T(lib, 6, 8, 64, at=t[name].contents.data - 2 * 6 * 8 * 64 + 2)})[0] == INVALID
        assert _paged(lib, lambda t: {"y": T(lib, 6, 8, 64, at=t[name].contents.data - 2 * 6 * 8 * 64)})[0] in NO_GPU
    assert lib.tops_paged_attention_forward(None) == INVALID
    lib.tops_clear_error()


def _cross(lib, change=None, **scalars):
    t = {"q": T(lib, 2, 5, 4, 64), "k": T(lib, 2, 9, 2, 64), "v": T(lib, 2, 9, 2, 64), "y": T(lib, 2, 5, 4, 64)}
    t.update(change(t) if callable(change) else change or {})
    return _try(lib, "tops_cross_attention_forward", capi.CCrossAttentionCall, t, **{"scale": 0.125, **scalars})


def test_cross_attention_accepts_and_refuses(lib):
    assert _cross(lib)[0] in NO_GPU
    assert _cross(lib, {"key_length": T(lib, 2, dtype="int32"), "mask": T(lib, 2, 1, 1, 9, dtype="float32")})[0] in NO_GPU
    for dtype in ("uint8", "int8", "bfloat16"):
        assert _cross(lib, {"mask": T(lib, 2, 9, dtype=dtype)})[0] in NO_GPU
    for name in ("q", "k", "v", "y"):
        assert _cross(lib, {name: None})[0] == INVALID
    cases = [({"y": T(lib, 2, 4, 4, 64)}, INVALID), ({"k": T(lib, 2, 9, 2, 32)}, INVALID), ({"v": T(lib, 2, 8, 2, 64)}, INVALID),
             ({"k": T(lib, 3, 9, 2, 64), "v": T(lib, 3, 9, 2, 64)}, INVALID), ({"k": T(lib, 2, 9, 3, 64), "v": T(lib, 2, 9, 3, 64)}, UNSUPPORTED),
             ({"k": T(lib, 2, 9, 2, 64, dtype="float16")}, UNSUPPORTED), ({"key_length": T(lib, 2, dtype="int64")}, INVALID),
             ({"key_length": T(lib, 3, dtype="int32")}, INVALID), ({"mask": T(lib, 2, 5, 9, dtype="uint8")}, INVALID),
             ({"mask": T(lib, 2, 9, dtype="float16")}, UNSUPPORTED), ({"mask": T(lib, 2, 9, dtype="int32")}, UNSUPPORTED),
             ({"mask": T(lib, 2, 9, dtype="uint8", at=0)}, INVALID)]
    for change, code in cases:
        rc, message = _cross(lib, change)
        assert rc == code and "tops_cross_attention_forward" in message, (change, rc, message)
    assert _cross(lib, scale=float("inf"))[0] == INVALID
    # the same shapes read as [batch, heads, tokens, dim]: 5 query heads over 9 key heads
    assert _cross(lib, heads_first=1)[0] == UNSUPPORTED
    for name in ("q", "k", "v"):
        assert _cross(lib, lambda t: {"y": T(lib, 2, 5, 4, 64, at=t[name].contents.data + 16)})[0] == INVALID
    assert lib.tops_cross_attention_forward(None) == INVALID
    lib.tops_clear_error()


def _rotary(lib, change=None, **scalars):
    t = {"q": T(lib, 6, 8, 64), "k": T(lib, 6, 2, 64), "v": T(lib, 6, 2, 64), "q_weight": T(lib, 64), "k_weight": T(lib, 64, dtype="float32"),
         "cos_table": T(lib, 100, 16, dtype="float32"), "sin_table": T(lib, 100, 16, dtype="float32"), "positions": T(lib, 6, dtype="int64"),
         "q_out": T(lib, 6, 8, 64), "k_out": None, "key_cache": T(lib, 10, 16, 2, 64), "value_cache": T(lib, 10, 16, 2, 64), "slots": T(lib, 6, dtype="int32")}
    t.update(change(t) if callable(change) else change or {})
    return _try(lib, "tops_qk_norm_rotary_forward", capi.CQKNormRotaryCall, t, **{"epsilon": 1e-6, **scalars})


def test_qk_norm_rotary_accepts_and_refuses(lib):
    nothing = {"key_cache": None, "value_cache": None, "slots": None, "v": None}
    assert _rotary(lib)[0] in NO_GPU
    assert _rotary(lib, {"k_out": T(lib, 6, 2, 64)})[0] in NO_GPU
    assert _rotary(lib, lambda t: {**nothing, "q_out": t["q"], "k_out": t["k"]})[0] in NO_GPU
    assert _rotary(lib, {**nothing, "k": None, "k_weight": None})[0] in NO_GPU
    assert _rotary(lib, {"k": None, "v": None, "q": T(lib, 6, 12, 64)}, packed_kv_heads=2)[0] in NO_GPU
    cases = [({"q": None}, INVALID), ({"q_out": None}, INVALID), ({"q_out": T(lib, 6, 7, 64)}, INVALID), ({"q_out": T(lib, 6, 8, 64, dtype="float32")}, INVALID),
             ({"k": T(lib, 6, 3, 64)}, INVALID), ({"k": T(lib, 5, 2, 64)}, INVALID), ({"v": None}, INVALID), ({"v": T(lib, 6, 1, 64)}, INVALID),
             ({"slots": None}, INVALID), ({"value_cache": None}, INVALID), ({"key_cache": None}, INVALID), ({"slots": T(lib, 5, dtype="int32")}, INVALID),
             ({"slots": T(lib, 6, dtype="int16")}, INVALID), ({"key_cache": T(lib, 10, 16, 2, 32), "value_cache": T(lib, 10, 16, 2, 32)}, INVALID),
             ({"positions": None}, INVALID), ({"cos_table": None}, INVALID), ({"positions": T(lib, 7, dtype="int32")}, INVALID),
             ({"cos_table": T(lib, 100, 33, dtype="float32"), "sin_table": T(lib, 100, 33, dtype="float32")}, INVALID),
             ({"cos_table": T(lib, 100, 16), "sin_table": T(lib, 100, 16)}, INVALID), ({"q_weight": T(lib, 63)}, INVALID),
             ({"q_weight": T(lib, 64, dtype="float16")}, INVALID), ({"key_cache": None, "value_cache": None, "slots": None}, INVALID),
             ({**nothing}, INVALID), ({"k_out": T(lib, 6, 8, 64)}, INVALID), ({"q": T(lib, 64), "q_out": T(lib, 64)}, INVALID)]
    for change, code in cases:
        rc, message = _rotary(lib, change)
        assert rc == code and "tops_qk_norm_rotary_forward" in message, (change, rc, message)
    f64 = {n: T(lib, *s, dtype="float64") for n, s in (("q", (6, 8, 64)), ("k", (6, 2, 64)), ("v", (6, 2, 64)), ("q_out", (6, 8, 64)))}
    assert _rotary(lib, f64)[0] == UNSUPPORTED
    assert _rotary(lib, {**nothing, "k": None, "k_weight": None, "q_weight": None, "q": T(lib, 6, 1, 2048), "q_out": T(lib, 6, 1, 2048)})[0] == UNSUPPORTED
    for epsilon in (-1.0, float("nan"), float("inf")):
        assert _rotary(lib, epsilon=epsilon)[0] == INVALID
    assert _rotary(lib, packed_kv_heads=2)[0] == INVALID                       # k and v given as well
    assert _rotary(lib, {"k": None, "v": None}, packed_kv_heads=4)[0] == INVALID   # no query head left
    assert _rotary(lib, packed_kv_heads=-1)[0] == INVALID
    assert _rotary(lib, heads_first=1)[0] == INVALID                           # three dimensions
    assert _rotary(lib, lambda t: {"q_out": T(lib, 6, 8, 64, at=t["q"].contents.data + 2)})[0] == INVALID      # shifted onto itself
    assert _rotary(lib, lambda t: {"k_out": T(lib, 6, 2, 64, at=t["q_out"].contents.data)})[0] == INVALID
    assert _rotary(lib, lambda t: {"k_out": T(lib, 6, 2, 64, at=t["value_cache"].contents.data)})[0] == INVALID
    assert _rotary(lib, lambda t: {"value_cache": t["key_cache"]})[0] == INVALID
    assert _rotary(lib, lambda t: {"v": T(lib, 6, 2, 64, at=t["key_cache"].contents.data)})[0] == INVALID
    assert lib.tops_qk_norm_rotary_forward(None) == INVALID
    lib.tops_clear_error()


def test_nodes_infer_shapes():
    t = nn.Tensor_
    q, k, v = t(2, 5, 12, 64, dtype="float16"), t(2, 7, 2, 64, dtype="float16"), t(2, 7, 2, 64, dtype="float16")
    assert CrossAttention([], []).forward_(q, k, v)["tensor"].size == (2, 5, 12, 64)
    assert PagedAttention([], []).forward_(t(9, 4, 64, dtype="float16"))["tensor"].size == (9, 4, 64)
    packed = QKNormRotary([], ["q"], packed_kv_heads=2).forward_(q, key_cache=t(3, 16, 2, 64))["tensor"]
    assert packed.size == (2, 5, 8, 64) and packed.dtype == "float16"
    both = QKNormRotary([], ["q", "k"], heads_first=True).forward_(t(2, 8, 5, 64), t(2, 2, 5, 64))["tensor"]
    assert [o.size for o in both] == [(2, 8, 5, 64), (2, 2, 5, 64)]
