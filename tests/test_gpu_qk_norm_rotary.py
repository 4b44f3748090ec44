"""RMS norm per head, rotation and append to the paged cache, against float64."""
import ctypes
import zlib

import numpy as np
import pytest

from attention_ref import HALF_STEP, assert_close, device, exact, fill
from datagen import to_f64

pytestmark = pytest.mark.gpu


def _rng(*what):
    return np.random.default_rng(zlib.crc32(repr(what).encode()))


def _reference(x, weight, epsilon, cos, sin, positions, interleaved, dtype):
    """x [T, H, D] -> (y, tolerance).  The norm's factor is off by at most (D / 2 + 8) 2^-24 of itself (a float32 sum of D squares, halved by
    the root; reciprocal root 2 ulp; three products); a rotation adds two products and a sum, 3 * 2^-24 of |a| + |b|; one rounding at the end."""
    dim = x.shape[-1]
    n = x.copy()
    relative = 0.0
    if weight is not None:
        n = x / np.sqrt((x * x).mean(-1, keepdims=True) + epsilon) * weight
        relative = (dim / 2 + 8) * 2.0 ** -24
    size = np.abs(n)
    y = n.copy()
    if cos is not None:
        half = cos.shape[1]
        c, s = cos[positions][:, None], sin[positions][:, None]
        first = (slice(0, 2 * half, 2) if interleaved else slice(0, half))
        second = (slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half))
        a, b = n[..., first], n[..., second]
        y[..., first], y[..., second] = a * c - b * s, a * s + b * c
        size[..., first] = size[..., second] = np.abs(a) + np.abs(b)
        relative = relative + 3 * 2.0 ** -24
    return y, relative * size + HALF_STEP[dtype] * np.abs(y) + (2.0 ** -24 if dtype == "float16" else 0.0)


class Problem:
    def __init__(self, seed, dtype, tokens, heads, kv_heads, dim, rotary, interleaved=False, source="separate", batch=1, page=0, norm=True,
                 k_out=None, weight_dtype=None, index="int32"):
        rng = _rng(seed, dtype, tokens, heads, kv_heads, dim, rotary, source)
        self.dtype, self.source, self.batch, self.page, self.interleaved, self.index = dtype, source, batch, page, interleaved, index
        self.tokens, self.heads, self.kv_heads, self.dim = tokens, heads, kv_heads, dim
        self.weight_dtype = weight_dtype or dtype
        self.q, self.k, self.v = (exact(rng, (tokens, h, dim), dtype, 3.0) for h in (heads, kv_heads, kv_heads))
        self.qw, self.kw = (exact(rng, (dim,), self.weight_dtype) if norm else None for _ in range(2))
        self.cos = self.sin = self.positions = None
        if rotary:
            angle = rng.uniform(0, 2 * np.pi, (50, rotary // 2))
            self.cos, self.sin = np.cos(angle).astype(np.float32).astype(np.float64), np.sin(angle).astype(np.float32).astype(np.float64)
            self.positions = rng.integers(0, 50, tokens)
        self.slots = None
        if page:
            pages = -(-tokens // page) + 1
            self.cache_shape = (pages, page, kv_heads, dim)
            self.slots = rng.permutation(pages * page)[:tokens]
            if tokens > 3:
                self.slots[1] = -1
        self.k_out = (not page) if k_out is None else k_out

    def _laid(self, x):
        """[T, H, D] in the layout of the call."""
        if self.source == "heads_first":
            return np.ascontiguousarray(x.reshape(self.batch, -1, *x.shape[1:]).transpose(0, 2, 1, 3))
        return x.reshape(self.batch, -1, *x.shape[1:]) if self.batch > 1 else x

    def _flat(self, y, heads):
        if self.source == "heads_first":
            y = y.transpose(0, 2, 1, 3)
        return y.reshape(-1, heads, self.dim)

    def run(self, in_place=False, expect=0):
        from onnx_translator_b200 import capi
        lib = capi.load()
        lib.tops_clear_error()
        packed = self.source == "packed"
        tensors = {"q": device(self._laid(np.concatenate([self.q, self.k, self.v], 1) if packed else self.q), self.dtype)}
        if not packed:
            tensors["k"] = device(self._laid(self.k), self.dtype)
            tensors["v"] = device(self._laid(self.v), self.dtype) if self.page else None
        for name, w in (("q_weight", self.qw), ("k_weight", self.kw)):
            tensors[name] = None if w is None else device(w, self.weight_dtype)
        if self.cos is not None:
            tensors.update(cos_table=device(self.cos, "float32"), sin_table=device(self.sin, "float32"),
                           positions=device(self.positions.astype(self.index), self.index))
        tensors["q_out"] = tensors["q"] if in_place else device(self._laid(np.full(self.q.shape, 7.0)), self.dtype)
        if self.k_out:
            tensors["k_out"] = tensors["k"] if in_place else device(self._laid(np.full(self.k.shape, 7.0)), self.dtype)
        if self.page:
            tensors.update(key_cache=device(np.full(self.cache_shape, 5.0), self.dtype), value_cache=device(np.full(self.cache_shape, 5.0), self.dtype),
                           slots=device(self.slots.astype(self.index), self.index))
        call = fill(capi.CQKNormRotaryCall(packed_kv_heads=self.kv_heads if packed else 0, heads_first=int(self.source == "heads_first"), epsilon=1e-5,
                                           interleaved=int(self.interleaved)), **tensors)
        assert lib.tops_qk_norm_rotary_forward(ctypes.byref(call)) == 0, lib.tops_last_error_message()
        assert lib.tops_sync() == expect
        lib.tops_clear_error()
        return {name: to_f64(t.numpy(), self.dtype) for name, t in tensors.items() if name in ("q_out", "k_out", "key_cache", "value_cache")}

    def check(self, got):
        yq, tq = _reference(self.q, self.qw, 1e-5, self.cos, self.sin, self.positions, self.interleaved, self.dtype)
        yk, tk = _reference(self.k, self.kw, 1e-5, self.cos, self.sin, self.positions, self.interleaved, self.dtype)
        assert_close(self._flat(got["q_out"], self.heads), yq, tq, "queries")
        if self.k_out:
            assert_close(self._flat(got["k_out"], self.kv_heads), yk, tk, "keys")
        if self.page:
            for name, y, t in (("key_cache", yk, tk), ("value_cache", self.v, np.zeros_like(self.v))):
                rows = got[name].reshape(-1, self.kv_heads, self.dim)
                stored = self.slots >= 0
                assert_close(rows[self.slots[stored]], y[stored], t[stored], name)
                rest = np.ones(len(rows), bool)
                rest[self.slots[stored]] = False
                assert np.all(rows[rest] == 5.0), name + ": rows without a token changed"


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("source", ["separate", "packed", "heads_first"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("sizes", [(1, 1, 1, 64, 64), (6, 8, 2, 128, 128), (33, 5, 5, 80, 40), (12, 3, 1, 96, 96), (10, 4, 2, 256, 256), (8, 2, 1, 40, 24),
                                   (4, 2, 2, 33, 10), (9, 2, 1, 6, 6), (6, 16, 2, 128, 64), (150, 7, 3, 64, 32), (3, 2, 1, 520, 512)],
                         ids=lambda s: "t%d_h%d_kv%d_d%d_r%d" % s)
def test_norm_and_rotation(dtype, source, interleaved, sizes):
    batch = 3 if sizes[0] % 3 == 0 and source != "packed" else 1
    p = Problem(1, dtype, *sizes, interleaved=interleaved, source=source, batch=batch)
    p.check(p.run())
    p = Problem(2, dtype, *sizes, interleaved=interleaved, source=source, batch=batch, page=4, index="int64")
    p.check(p.run())


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_parts_that_are_left_out(dtype):
    for kw in ({"rotary": 0}, {"norm": False}, {"weight_dtype": "float32"}, {"page": 16, "k_out": True}, {"rotary": 0, "norm": False, "page": 16}):
        rotary = kw.pop("rotary", 64)
        p = Problem(3, dtype, 20, 6, 2, 64, rotary, **kw)
        p.check(p.run())


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("dim", [128, 33, 80])
def test_in_place(dtype, dim):
    for source in ("separate", "heads_first"):
        p = Problem(4, dtype, 30, 5, 5, dim, 2 * (dim // 4), source=source)
        p.check(p.run(in_place=True))


def test_zero_rows_and_large_values():
    """A row of zeros normalises to zeros; squares of float16's largest values stay in float32's range."""
    p = Problem(5, "float16", 8, 4, 2, 128, 128)
    p.q[0] = 0.0
    p.q[1] = 60000.0
    p.k[2] = -60000.0
    p.check(p.run())


def test_many_tokens():
    p = Problem(6, "bfloat16", 5000, 12, 4, 128, 128, source="packed", page=64)
    p.check(p.run())


@pytest.mark.parametrize("dim", [128, 33])
def test_indices_outside_their_tables(dim):
    """A position outside the tables: the token's heads are zero and not stored; a slot outside the cache: not stored.  Both are reported."""
    for bad in (-1, 50, 2 ** 31 - 1):
        p = Problem(7, "bfloat16", 12, 4, 2, dim, 32, page=4, k_out=True)
        p.positions[5] = bad
        got = p.run(expect=1)
        assert np.all(got["q_out"][5] == 0.0) and np.all(got["k_out"][5] == 0.0)
        slot = p.slots[5]
        for name in ("key_cache", "value_cache"):
            assert np.all(got[name].reshape(-1, 2, dim)[slot] == 5.0)
    p = Problem(8, "bfloat16", 12, 4, 2, dim, 32, page=4, index="int64")
    free = sorted(set(range(p.cache_shape[0] * 4)) - set(p.slots.tolist()))
    p.slots[7] = 2 ** 40
    got = p.run(expect=1)
    assert np.all(got["key_cache"].reshape(-1, 2, dim)[free] == 5.0)
