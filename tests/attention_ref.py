"""Attention operators in float64 with the error that float32 / 16-bit arithmetic may add, for the tests; and thin callers of the C entry
points.  Activations are float64 arrays whose values are exact in the type under test."""
from __future__ import annotations

import ctypes

import numpy as np

from datagen import from_f64, to_f64

# Half a step of each type relative to the value: one rounding to the nearest.
HALF_STEP = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8, "float32": 2.0 ** -24}
LOWEST = {"float16": -65504.0, "bfloat16": -3.3895313892515355e38, "float32": -3.4028234663852886e38}
LOG2E = 1.4426950408889634


def exact(rng, shape, dtype, spread=1.0):
    """Random values that the type represents exactly, as float64."""
    return to_f64(from_f64(rng.normal(0.0, spread, shape), dtype), dtype)


def attention(q, k, v, seen, scale, dtype, bias=None):
    """q [n, H, D], k and v [L, Hk, D], seen [n, L] -> (y, tolerance), both [n, H, D].

    The tolerance, term by term, with p the weights and A = sum_j p_j |v_j|:
    * the result is rounded once: half a step of |y| (and of the smallest normal, for results near zero);
    * the weights enter the product with V rounded to the type (16-bit types): half a step of A;
    * a score is a float32 sum of D exact products, each partial sum off by at most 2^-23 of the sum of magnitudes (tensor cores
      may truncate): (D + 2) 2^-23 S with S = scale sum_d |q_d k_d|; twice, for the numerator and the denominator;
    * exp2 of a float32 argument z: 2^-22 from the function and |z| 2^-23 from rounding z and the maximum, again twice;
    * sums of L weights in float32: L 2^-24 for numerator and denominator each."""
    n, heads, dim = q.shape
    length, kv_heads = k.shape[0], k.shape[1]
    group = heads // kv_heads
    y, tol = np.zeros((n, heads, dim)), np.zeros((n, heads, dim))
    if n == 0:
        return y, tol
    for h in range(heads):
        kh, vh = k[:, h // group], v[:, h // group]
        z = q[:, h] @ kh.T * scale
        size = np.abs(q[:, h]) @ np.abs(kh).T * abs(scale)
        if bias is not None:
            z, size = z + bias, size + np.abs(bias)
        z = np.where(seen, z, -np.inf)
        top = z.max(axis=1, initial=-np.inf)
        top = np.where(np.isfinite(top), top, 0.0)[:, None]
        w = np.exp(z - top)
        total = w.sum(axis=1, keepdims=True)
        p = np.divide(w, total, out=np.zeros_like(w), where=total > 0)
        y[:, h] = p @ vh
        a = p @ np.abs(vh)
        worst = np.where(seen, size, 0.0).max(axis=1, initial=0.0)[:, None]
        relative = 2 * ((dim + 2) * 2.0 ** -23 * worst + 2.0 ** -22 + LOG2E * worst * 2.0 ** -22) + 2 * length * 2.0 ** -24
        relative += 0.0 if dtype == "float32" else HALF_STEP[dtype]
        tol[:, h] = relative * a + HALF_STEP[dtype] * np.abs(y[:, h]) + (2.0 ** -24 if dtype == "float16" else 0.0)
    return y, tol


def assert_close(got, want, tol, what=""):
    bad = ~(np.abs(got - want) <= tol)
    if bad.any():
        at = tuple(int(i[0]) for i in np.nonzero(bad))
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.size} outside, first at {at}: got {got[at]!r} want {want[at]!r} tolerance {tol[at]:.3g}")


def device(array, dtype):
    from onnx_translator_b200.device import DeviceArray
    return DeviceArray.from_numpy(from_f64(array, dtype) if dtype in HALF_STEP else np.ascontiguousarray(array), dtype)


def fill(call, **tensors):
    """Stores the handles of DeviceArrays in the struct; keeps them alive with it."""
    call.kept = tensors
    for name, t in tensors.items():
        setattr(call, name, None if t is None else ctypes.cast(t.handle, ctypes.c_void_p))
    return call


class Paged:
    """A ragged paged problem: ``pairs`` holds (new tokens, keys) per sequence; the caches hold NaN wherever no key lies."""

    def __init__(self, rng, dtype, heads, kv_heads, dim, page, pairs, window=0, extra_rows=0, spread=1.0):
        self.dtype, self.page, self.window, self.pairs, self.scale = dtype, page, window, pairs, dim ** -0.5
        self.kv_heads, self.dim = kv_heads, dim
        total = sum(n for n, _ in pairs)
        self.q = exact(rng, (total + extra_rows, heads, dim), dtype, spread)
        counts = [-(-length // page) for _, length in pairs]
        width = max(max(counts, default=0), 1) + 1
        pages = sum(counts) + 2
        order = rng.permutation(pages)
        self.table = np.full((len(pairs), width), -7, np.int32)
        self.keys, self.values = [], []
        self.key_cache = np.full((pages, page, kv_heads, dim), np.nan)
        self.value_cache = np.full((pages, page, kv_heads, dim), np.nan)
        used = 0
        for b, (_, length) in enumerate(pairs):
            mine = order[used:used + counts[b]]
            used += counts[b]
            self.table[b, :counts[b]] = mine
            k, v = exact(rng, (length, kv_heads, dim), dtype, spread), exact(rng, (length, kv_heads, dim), dtype)
            self.keys.append(k)
            self.values.append(v)
            j = np.arange(length)
            self.key_cache[mine[j // page], j % page] = k
            self.value_cache[mine[j // page], j % page] = v
        self.query_start = np.concatenate([[0], np.cumsum([n for n, _ in pairs])]).astype(np.int32)
        self.kv_length = np.array([length for _, length in pairs], np.int32)

    def want(self):
        ys, tols = [], []
        at = 0
        for (n, length), k, v in zip(self.pairs, self.keys, self.values):
            place = (length - n + np.arange(n))[:, None]
            j = np.arange(length)[None, :]
            seen = j <= place
            if self.window:
                seen &= j > place - self.window
            y, tol = attention(self.q[at:at + n], k, v, seen, self.scale, self.dtype)
            ys.append(y)
            tols.append(tol)
            at += n
        return np.concatenate(ys), np.concatenate(tols)

    def call(self, fill_value=7.0):
        from onnx_translator_b200 import capi
        return fill(capi.CPagedAttentionCall(scale=self.scale, window=self.window), q=device(self.q, self.dtype),
                    key_cache=device(self.key_cache, self.dtype), value_cache=device(self.value_cache, self.dtype),
                    page_table=device(self.table, "int32"), query_start=device(self.query_start, "int32"), kv_length=device(self.kv_length, "int32"),
                    y=device(np.full(self.q.shape, fill_value), self.dtype))


def run_paged(problem):
    from onnx_translator_b200 import capi
    lib = capi.load()
    call = problem.call()
    rc = lib.tops_paged_attention_forward(ctypes.byref(call))
    capi.check(lib)
    assert rc == 0
    got = to_f64(call.kept["y"].numpy(), problem.dtype)
    capi.check(lib)
    return got


def run_cross(q, k, v, dtype, scale, key_length=None, mask=None, mask_dtype="uint8", heads_first=False):
    from onnx_translator_b200 import capi
    lib = capi.load()
    call = fill(capi.CCrossAttentionCall(scale=scale, heads_first=int(heads_first)), q=device(q, dtype), k=device(k, dtype), v=device(v, dtype),
                key_length=None if key_length is None else device(np.asarray(key_length, np.int32), "int32"),
                mask=None if mask is None else device(mask, mask_dtype), y=device(np.full(q.shape, 7.0), dtype))
    rc = lib.tops_cross_attention_forward(ctypes.byref(call))
    capi.check(lib)
    assert rc == 0
    got = to_f64(call.kept["y"].numpy(), dtype)
    capi.check(lib)
    return got
