"""The attention operators together, as a decoder uses them: a layer that appends to its cache and attends over it, token by token, node by
node and as one captured graph.  Every attention node is compared with float64 on the very values it was given."""
import zlib

import numpy as np
import pytest

from attention_ref import assert_close, attention, exact
from datagen import from_f64, to_f64

pytestmark = pytest.mark.gpu


def _inputs(nn, rng, dtype, batch, width, table, lengths, page_size, enc):
    """One step: every sequence gets its token number lengths[b] (0-based)."""
    t = lambda a, d: nn.Tensor(*np.shape(a), dtype=d, data=np.ascontiguousarray(a))  # noqa: E731
    slots = table[np.arange(batch), lengths // page_size] * page_size + lengths % page_size
    return [t(from_f64(exact(rng, (batch, width), dtype), dtype), dtype), t(lengths.astype(np.int32), "int32"), t(slots.astype(np.int32), "int32"),
            t(table, "int32"), t(np.arange(batch + 1, dtype=np.int32), "int32"), t((lengths + 1).astype(np.int32), "int32"),
            t(from_f64(enc[0], dtype), dtype), t(from_f64(enc[1], dtype), dtype), t(enc[2], "int32")]


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
def test_decoding_steps_node_by_node_and_captured(dtype):
    from onnx_translator_b200 import nn
    batch, heads, kv_heads, dim, page_size, steps, keys = 3, 8, 2, 64, 8, 21, 45
    rng = np.random.default_rng(zlib.crc32(dtype.encode()))
    make = lambda: nn.cached_decoder_layer(batch, heads, kv_heads, dim, pages=16, page_size=page_size, seed=3, dtype=dtype)  # noqa: E731
    graph, replayed = make(), make()
    table = rng.permutation(16)[:12].reshape(batch, 4).astype(np.int32)
    enc = (exact(rng, (batch, keys, kv_heads, dim), dtype), exact(rng, (batch, keys, kv_heads, dim), dtype), np.array([45, 17, 1], np.int32))
    plan = None
    stored = [([], []) for _ in range(batch)]
    for step in range(steps):
        lengths = np.array([step, step + 2, step + 9])
        if step == 0:
            lengths_before = lengths.copy()
        inputs = _inputs(nn, rng, dtype, batch, heads * dim, table, lengths, page_size, enc)
        outs = graph.forward(*inputs)
        y, qkv, q, seen, cross_q, crossed = (to_f64(o.numpy(), dtype) for o in outs)
        # what the cache holds now, from the cache itself
        caches = [to_f64(graph.initializers[n].numpy(), dtype).reshape(-1, kv_heads, dim) for n in ("key_cache", "value_cache")]
        for b in range(batch):
            j = np.arange(lengths[b] + 1)
            rows = table[b, j // page_size] * page_size + j % page_size
            k, v = caches[0][rows], caches[1][rows]
            stored[b][0].append(k[-1])
            stored[b][1].append(v[-1])
            assert np.array_equal(v[-1], qkv[b, heads + kv_heads:])                # the value as projected
            first = lengths_before[b]
            assert np.array_equal(k[first:], np.stack(stored[b][0])) and np.array_equal(v[first:], np.stack(stored[b][1]))   # older rows stay
            want, tol = attention(q[b:b + 1], k, v, np.ones((1, len(j)), bool), dim ** -0.5, dtype)
            assert_close(seen[b:b + 1], want, tol, f"step {step} sequence {b}")
            n = enc[2][b]
            want, tol = attention(cross_q[b], enc[0][b], enc[1][b], np.broadcast_to(np.arange(keys) < n, (1, keys)), dim ** -0.5, dtype)
            assert_close(crossed[b], want, tol, f"step {step} cross {b}")
        assert np.isfinite(y).all()
        # the same step as one recorded plan, captured from the second step on
        if plan is None:
            plan = replayed.plan(*inputs)
            again = plan.outputs
        else:
            again = plan.run(*inputs)
            if step == 1:
                assert plan.capture()
        for a, b in zip(outs, again):
            assert np.array_equal(a.numpy().view(np.uint8), b.numpy().view(np.uint8)), f"step {step}: the plan differs"
    assert plan.captured
    plan.close()


def test_prompt_then_steps_equal_one_prompt():
    """A prompt in two chunks and single tokens gives, at the last token, the same cache and (up to rounding of the weights) the same result as one prompt."""
    from attention_ref import Paged, run_paged
    problem = Paged(np.random.default_rng(5), "bfloat16", 8, 2, 128, 16, [(300, 300)])
    whole = run_paged(problem)
    _, tol = problem.want()
    for n, length in ((200, 200), (99, 299), (1, 300)):
        part = Paged(np.random.default_rng(5), "bfloat16", 8, 2, 128, 16, [(300, 300)])
        part.q = problem.q[length - n:length]
        part.query_start = np.array([0, n], np.int32)
        part.kv_length = np.array([length], np.int32)
        assert_close(run_paged(part), whole[length - n:length], 2 * tol[length - n:length])


def test_node_on_a_padded_batch_gives_zeros_behind_the_last_sequence():
    from onnx_translator_b200 import nn
    from attention_ref import Paged
    problem = Paged(np.random.default_rng(6), "float16", 4, 2, 64, 16, [(2, 40), (1, 17)], extra_rows=5)
    t = lambda a, d: nn.Tensor(*np.shape(a), dtype=d, data=np.ascontiguousarray(from_f64(a, d) if d == "float16" else a))  # noqa: E731
    node = nn.PagedAttention([], [], dtype="float16")
    y = to_f64(node.forward(t(problem.q, "float16"), t(problem.key_cache, "float16"), t(problem.value_cache, "float16"), t(problem.table, "int32"),
                            t(problem.query_start, "int32"), t(problem.kv_length, "int32"))["tensor"].numpy(), "float16")
    want, tol = problem.want()
    assert_close(y[:3], want, tol)
    assert np.all(y[3:] == 0.0)
