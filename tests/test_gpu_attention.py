"""Paged and cross attention against a float64 evaluation of their definition, at the sizes, masks and layouts where kernels go wrong.
attention_ref.attention derives the tolerances."""
import ctypes
import zlib

import numpy as np
import pytest

from attention_ref import HALF_STEP, LOWEST, Paged, assert_close, attention, device, exact, fill, run_cross, run_paged
from datagen import to_f64

pytestmark = pytest.mark.gpu

TYPES = ("bfloat16", "float16", "float32")


def _rng(*what):
    return np.random.default_rng(zlib.crc32(repr(what).encode()))


# (new tokens, keys) of each sequence
BATCHES = {
    "one_key": [(1, 1)], "no_key": [(1, 0)], "one": [(1, 511)], "steps": [(1, 17), (1, 1), (1, 300), (1, 16), (1, 129)],
    "chunks": [(5, 5), (3, 40), (1, 64), (16, 33)], "longer_than_its_keys": [(4, 2), (2, 2)], "no_token": [(0, 30), (2, 9), (0, 0), (3, 3)],
    "prompt": [(131, 131)], "chunk_over_past": [(70, 389), (1, 200)], "long": [(1, 3000), (2, 2111)],
}


@pytest.mark.parametrize("batch", BATCHES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(4, 4, 64, 16), (8, 2, 128, 16), (6, 2, 80, 32), (7, 1, 256, 64), (3, 1, 64, 7), (2, 2, 33, 5)],
                         ids=lambda s: "h%d_kv%d_d%d_page%d" % s)
def test_paged(dtype, shape, batch):
    heads, kv_heads, dim, page = shape
    problem = Paged(_rng(dtype, shape, batch), dtype, heads, kv_heads, dim, page, BATCHES[batch])
    want, tol = problem.want()
    assert_close(run_paged(problem), want, tol, batch)


@pytest.mark.parametrize("window", [1, 5, 16, 100, 4096, 2 ** 31 - 1])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
def test_paged_window(dtype, window, dim):
    problem = Paged(_rng(dtype, window), dtype, 6, 2, dim, 16, [(1, 300), (40, 40), (150, 333), (3, 2), (1, 1)], window=window)
    want, tol = problem.want()
    assert_close(run_paged(problem), want, tol)


@pytest.mark.parametrize("group", [1, 2, 5, 16, 17, 40])
@pytest.mark.parametrize("dim", [8, 40, 96, 128])
def test_paged_groups_of_heads(group, dim):
    problem = Paged(_rng(group, dim), "bfloat16", 2 * group, 2, dim, 16, [(1, 90), (3, 50), (21, 77)])
    want, tol = problem.want()
    assert_close(run_paged(problem), want, tol)


@pytest.mark.parametrize("page", [1, 2, 8, 24, 48, 64, 128, 200, 256, 384])
@pytest.mark.parametrize("tokens", [1, 150])
def test_paged_page_sizes(page, tokens):
    problem = Paged(_rng(page, tokens), "float16", 4, 2, 64, page, [(tokens, 411), (tokens, 150), (tokens, 777)])
    want, tol = problem.want()
    assert_close(run_paged(problem), want, tol)


@pytest.mark.parametrize("dtype", ("bfloat16", "float16"))
@pytest.mark.parametrize("shape", [(8, 2, 128, 64), (3, 3, 64, 16), (6, 1, 40, 128)], ids=lambda s: "h%d_kv%d_d%d_page%d" % s)
def test_paged_longer_prompts(dtype, shape):
    heads, kv_heads, dim, page = shape
    problem = Paged(_rng(dtype, shape), dtype, heads, kv_heads, dim, page, [(600, 600), (257, 1500), (1, 900), (0, 64), (129, 129), (300, 4000)])
    want, tol = problem.want()
    assert_close(run_paged(problem), want, tol)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [1, 200])
def test_rows_behind_the_last_sequence_stay(dtype, tokens):
    problem = Paged(_rng(dtype, tokens), dtype, 4, 2, 64, 16, [(tokens, 210), (tokens, 230)], extra_rows=9)
    got = run_paged(problem)
    want, tol = problem.want()
    assert_close(got[:2 * tokens], want, tol)
    assert np.all(got[2 * tokens:] == 7.0)


def test_many_tiles_per_block():
    """Long enough that every block works through tens of 128-key tiles of one item and goes on to the next."""
    problem = Paged(_rng("many tiles"), "bfloat16", 4, 2, 64, 128, [(1, 70001), (3, 60011), (1, 65)])
    want, tol = problem.want()
    assert_close(run_paged(problem), want, tol)
    problem = Paged(_rng("many tiles", 128), "float16", 1, 1, 128, 64, [(1, 200003)])
    want, tol = problem.want()
    assert_close(run_paged(problem), want, tol)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [1, 200])
def test_large_scores(dtype, tokens):
    """Scores of several hundred: the maximum has to be taken off before the exponential, and moves from tile to tile."""
    problem = Paged(_rng(dtype, tokens, "large"), dtype, 4, 2, 64, 16, [(tokens, 700)], spread=6.0)
    want, tol = problem.want()
    assert_close(run_paged(problem), want, tol)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [1, 200])
def test_nan_and_infinity_in_real_keys_show(dtype, tokens):
    """A NaN in a key that a row sees makes that row NaN, wherever in a tile the key stands; rows that do not see its tile stay as they are."""
    for at in (0, 1, 2, 3, 5, 6, 7, 37, 126, 130):
        problem = Paged(_rng(dtype, tokens, "nan"), dtype, 4, 2, 64, 16, [(tokens, 300), (tokens, 260)])
        page, offset = problem.table[0, at // 16], at % 16
        problem.key_cache[page, offset, 0, 5] = np.nan
        got = run_paged(problem)
        want, tol = problem.want()
        if tokens <= 300 - at:
            sees = np.arange(tokens) + 300 - tokens >= at
            assert np.isnan(got[:tokens][sees, :2]).all()
        assert_close(got[:, 2:], want[:, 2:], tol[:, 2:])
        assert_close(got[tokens:], want[tokens:], tol[tokens:])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scale", [0.0, -0.3, 1e-6, 3.0])
def test_scales(dtype, scale):
    """No scale, a negative one, a tiny and a large one."""
    for tokens in (2, 140):
        problem = Paged(_rng(dtype, tokens, "scale"), dtype, 4, 2, 64, 16, [(tokens, 300)])
        problem.scale = scale
        want, tol = problem.want()
        assert_close(run_paged(problem), want, tol)


@pytest.mark.parametrize("tokens", [1, 200])
def test_ascending_scores(tokens):
    """Every tile has a larger maximum than all before it."""
    problem = Paged(_rng("ascending", tokens), "bfloat16", 2, 1, 64, 16, [(tokens, 900)])
    problem.q[:] = 0.0
    problem.q[..., 0] = 8.0
    ramp = to_f64(_codes(np.arange(900) / 8.0, "bfloat16"), "bfloat16")
    problem.keys[0][:, :, 0] = ramp[:, None]
    for j in range(900):
        problem.key_cache[problem.table[0, j // 16], j % 16] = problem.keys[0][j]
    want, tol = problem.want()
    assert_close(run_paged(problem), want, tol)


def _codes(x, dtype):
    from datagen import from_f64
    return from_f64(x, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [1, 140])
def test_a_page_outside_the_cache_is_not_followed(dtype, tokens):
    from onnx_translator_b200 import capi
    lib = capi.load()
    for bad in (-1, 10 ** 6):
        problem = Paged(_rng(dtype, "bad page", tokens), dtype, 4, 2, 64, 16, [(tokens, 200), (tokens, 180)])
        problem.table[0, 3] = bad
        problem.keys[0][48:64] = 0.0
        problem.values[0][48:64] = 0.0
        want, tol = problem.want()
        call = problem.call()
        lib.tops_clear_error()
        assert lib.tops_paged_attention_forward(ctypes.byref(call)) == 0
        assert lib.tops_sync() == 1 and b"outside its table" in lib.tops_last_error_message()
        lib.tops_clear_error()
        assert_close(to_f64(call.kept["y"].numpy(), dtype), want, tol)
        capi.check(lib)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [1, 150])
def test_a_page_table_without_columns(dtype, tokens):
    """No sequence can have a key: zeros for the sequences' rows, nothing else is touched; a length is cut and reported."""
    from onnx_translator_b200 import capi
    lib = capi.load()
    for length, status in ((0, 0), (5, 1)):
        problem = Paged(_rng(dtype, "no columns"), dtype, 4, 2, 64, 16, [(tokens, 0)], extra_rows=2)
        problem.table = np.zeros((1, 0), np.int32)
        problem.kv_length[:] = length
        call = problem.call()
        lib.tops_clear_error()
        assert lib.tops_paged_attention_forward(ctypes.byref(call)) == 0, lib.tops_last_error_message()
        assert lib.tops_sync() == status
        lib.tops_clear_error()
        got = to_f64(call.kept["y"].numpy(), dtype)
        assert np.all(got[:tokens] == 0.0) and np.all(got[tokens:] == 7.0)


def test_inconsistent_tables_stay_in_bounds():
    """Sequence bounds past the rows of q and lengths past the table are cut and reported."""
    from onnx_translator_b200 import capi
    lib = capi.load()
    for tokens in (2, 150):
        problem = Paged(_rng("tables"), "bfloat16", 4, 2, 64, 16, [(tokens, 200)])
        call = problem.call()
        for name, values in (("query_start", [0, 10 ** 9]), ("query_start", [-5, tokens]), ("kv_length", [10 ** 9]), ("kv_length", [-3])):
            kept = call.kept[name]
            changed = device(np.array(values, np.int32), "int32")
            if name == "kv_length" and values[0] > 0:
                table = np.zeros_like(problem.table)
                call.kept["full_table"] = device(table, "int32")
                call.page_table = ctypes.cast(call.kept["full_table"].handle, ctypes.c_void_p)
            setattr(call, name, ctypes.cast(changed.handle, ctypes.c_void_p))
            lib.tops_clear_error()
            assert lib.tops_paged_attention_forward(ctypes.byref(call)) == 0
            assert lib.tops_sync() == 1
            lib.tops_clear_error()
            setattr(call, name, ctypes.cast(kept.handle, ctypes.c_void_p))
            call.page_table = ctypes.cast(call.kept["page_table"].handle, ctypes.c_void_p)


# ---- cross attention -----------------------------------------------------------------------------------------------------
def _cross(dtype, batch, queries, keys, heads, kv_heads, dim, heads_first=False, lengths=None, mask=None, mask_dtype="uint8", poison=True):
    rng = _rng(dtype, batch, queries, keys, heads, kv_heads, dim, mask_dtype)
    scale = dim ** -0.5
    q = exact(rng, (batch, queries, heads, dim), dtype)
    k, v = exact(rng, (batch, keys, kv_heads, dim), dtype), exact(rng, (batch, keys, kv_heads, dim), dtype)
    kept = np.ones((batch, keys), bool)
    if lengths is not None:
        kept &= np.arange(keys) < np.asarray(lengths)[:, None]
    bias = None
    if mask is not None:
        kept &= (mask != 0) if mask_dtype in ("uint8", "int8") else mask > LOWEST[mask_dtype]
        bias = None if mask_dtype in ("uint8", "int8") else np.where(kept, mask, 0.0)
    want, tol = zip(*(attention(q[b], k[b], v[b], np.broadcast_to(kept[b], (queries, keys)), scale, dtype, None if bias is None else bias[b])
                      for b in range(batch)))
    want, tol = np.stack(want), np.stack(tol)
    if poison:                                   # excluded keys hold what must not matter
        for b in range(batch):
            k[b][~kept[b]] = np.nan
            v[b][~kept[b]] = np.where(np.arange(dim) % 2, np.inf, np.nan)
    if heads_first:
        q, k, v = (np.ascontiguousarray(x.transpose(0, 2, 1, 3)) for x in (q, k, v))
    got = run_cross(q, k, v, dtype, scale, lengths, mask, mask_dtype, heads_first)
    if heads_first:
        got = got.transpose(0, 2, 1, 3)
    assert_close(got, want, tol)
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads_first", [False, True])
@pytest.mark.parametrize("sizes", [(1, 1, 1, 1, 1, 64), (3, 1, 333, 4, 4, 64), (2, 5, 77, 6, 2, 40), (1, 130, 200, 4, 1, 128), (2, 300, 257, 2, 2, 64),
                                   (2, 17, 500, 3, 3, 96), (1, 260, 1030, 2, 1, 128), (1, 3, 50, 2, 2, 7), (1, 140, 90, 2, 2, 256), (2, 1, 5000, 2, 2, 128)],
                         ids=lambda s: "b%d_q%d_k%d_h%d_kv%d_d%d" % s)
def test_cross(dtype, heads_first, sizes):
    _cross(dtype, *sizes, heads_first=heads_first)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("queries", [1, 150])
def test_cross_lengths(dtype, queries):
    got = _cross(dtype, 5, queries, 300, 4, 2, 64, lengths=[300, 0, 1, 129, 255])
    assert np.all(got[1] == 0.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("queries", [1, 150])
@pytest.mark.parametrize("mask_dtype", ["uint8", "int8", "float32", "same"])
def test_cross_masks(dtype, queries, mask_dtype):
    """Random holes, a row masked throughout, -Inf and the type's lowest value, with and without lengths."""
    mask_dtype = dtype if mask_dtype == "same" else mask_dtype
    rng = _rng(dtype, queries, mask_dtype, "mask")
    keep = rng.random((4, 290)) < 0.7
    keep[1] = False
    keep[2] = False
    keep[2, 200] = True
    if mask_dtype in ("uint8", "int8"):
        mask = np.where(keep, rng.integers(1, 100, keep.shape), 0).astype(mask_dtype)
    else:
        mask = np.where(keep, exact(rng, keep.shape, mask_dtype), np.where(rng.random(keep.shape) < 0.5, -np.inf, LOWEST[mask_dtype]))
    got = _cross(dtype, 4, queries, 290, 4, 2, 64, mask=mask, mask_dtype=mask_dtype)
    assert np.all(got[1] == 0.0)
    _cross(dtype, 4, queries, 290, 2, 2, 128, lengths=[290, 100, 201, 33], mask=mask, mask_dtype=mask_dtype, heads_first=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("queries", [1, 150])
def test_cross_padding_of_whole_tiles(dtype, queries):
    """Padding in front, behind and in the middle that is longer than a tile of keys; one row without any key."""
    mask = np.ones((5, 1111), np.uint8)
    mask[0, 300:] = 0
    mask[1, :900] = 0
    mask[2, 130:1000] = 0
    mask[3] = 0
    mask[4, :1110] = 0
    got = _cross(dtype, 5, queries, 1111, 4, 2, 64, mask=mask)
    assert np.all(got[3] == 0.0)


def test_no_keys_at_all_gives_zeros():
    from onnx_translator_b200 import capi
    q = exact(_rng("none"), (2, 3, 4, 64), "bfloat16")
    assert np.all(run_cross(q, np.zeros((2, 0, 4, 64)), np.zeros((2, 0, 4, 64)), "bfloat16", 0.125) == 0.0)
    assert run_cross(np.zeros((2, 0, 4, 64)), np.zeros((2, 5, 4, 64)), np.zeros((2, 5, 4, 64)), "bfloat16", 0.125).size == 0


# ---- streams, captures, devices -------------------------------------------------------------------------------------------
@pytest.mark.parametrize("tokens", [1, 150])
def test_captured_and_replayed_with_new_lengths(tokens):
    """One captured call serves other lengths and pages: they are read on the device at every launch."""
    from onnx_translator_b200 import capi
    lib = capi.load()
    first = Paged(_rng("capture", tokens), "bfloat16", 8, 2, 128, 16, [(tokens, 1000), (tokens, 160)])
    second = Paged(_rng("replay", tokens), "bfloat16", 8, 2, 128, 16, [(tokens, 160), (tokens, 995)])
    call = first.call()
    assert lib.tops_paged_attention_forward(ctypes.byref(call)) == 0
    assert lib.tops_capture_begin() == 0
    assert lib.tops_paged_attention_forward(ctypes.byref(call)) == 0
    graph = lib.tops_capture_end()
    assert graph
    assert lib.tops_capture_launch(graph) == 0
    want, tol = first.want()
    assert_close(to_f64(call.kept["y"].numpy(), "bfloat16"), want, tol)
    other = second.call()
    assert first.table.shape == second.table.shape and first.key_cache.shape == second.key_cache.shape
    for name in ("q", "key_cache", "value_cache", "page_table", "query_start", "kv_length"):
        lib.flatten_forward(other.kept[name].handle, call.kept[name].handle)
    assert lib.tops_capture_launch(graph) == 0
    want, tol = second.want()
    assert_close(to_f64(call.kept["y"].numpy(), "bfloat16"), want, tol)
    lib.tops_capture_free(graph)
    capi.check(lib)


@pytest.mark.parametrize("tokens", [1, 150])
def test_two_captured_calls_on_two_streams(tokens):
    """Two graphs of the same operator run at once: nothing is shared between calls."""
    import torch
    from onnx_translator_b200 import capi
    lib = capi.load()
    problems = [Paged(_rng("streams", i, tokens), "float16", 8, 2, 128, 16, [(tokens, 2000 + i), (tokens, 800)]) for i in range(2)]
    calls = [p.call() for p in problems]
    lib.tops_sync()
    streams = [torch.cuda.Stream() for _ in range(2)]
    graphs = []
    try:
        for call, stream in zip(calls, streams):
            lib.tops_set_stream(stream.cuda_stream)
            assert lib.tops_capture_begin() == 0
            assert lib.tops_paged_attention_forward(ctypes.byref(call)) == 0
            graphs.append(lib.tops_capture_end())
        for _ in range(20):
            for graph, stream in zip(graphs, streams):
                lib.tops_set_stream(stream.cuda_stream)
                assert lib.tops_capture_launch(graph) == 0
        torch.cuda.synchronize()
    finally:
        lib.tops_set_stream(None)
    for problem, call in zip(problems, calls):
        want, tol = problem.want()
        assert_close(to_f64(call.kept["y"].numpy(), "float16"), want, tol)
    for graph in graphs:
        lib.tops_capture_free(graph)
    capi.check(lib)


@pytest.mark.parametrize("tokens", [1, 333])
def test_same_call_same_bits(tokens):
    """Partial results are joined in a fixed order."""
    problem = Paged(_rng("bits", tokens), "bfloat16", 8, 1, 128, 16, [(tokens, 6000)])
    a, b = run_paged(problem), run_paged(problem)
    assert np.array_equal(a, b)


def test_unaligned_operands():
    """Heads of eight elements read from an address that is only two-byte aligned."""
    import torch
    from onnx_translator_b200 import capi
    lib = capi.load()
    for tokens in (1, 140):
        problem = Paged(_rng("unaligned", tokens), "float16", 4, 2, 64, 16, [(tokens, 300)])
        call = problem.call()
        moved = {}
        for name in ("q", "key_cache", "value_cache", "y"):
            t = call.kept[name]
            room = torch.empty(t.size + 1, dtype=torch.float16, device="cuda")
            shape, nd = capi.shape_array(t.shape)
            handle = lib.tops_wrap(room.data_ptr() + 2, shape, nd, capi.DTYPE_MAP["float16"])
            lib.flatten_forward(t.handle, handle)
            moved[name] = (room, handle)
            setattr(call, name, ctypes.cast(handle, ctypes.c_void_p))
        assert lib.tops_paged_attention_forward(ctypes.byref(call)) == 0
        lib.flatten_forward(moved["y"][1], call.kept["y"].handle)
        want, tol = problem.want()
        assert_close(to_f64(call.kept["y"].numpy(), "float16"), want, tol)
        for _, handle in moved.values():
            lib.free_tensor(handle)
        capi.check(lib)


@pytest.mark.parametrize("dtype,page,tokens", [("bfloat16", 64, 1), ("bfloat16", 64, 200), ("bfloat16", 40, 1), ("float16", 16, 12), ("float32", 64, 2)])
def test_offsets_past_32_bits(dtype, page, tokens):
    """Pages whose elements lie more than 2^31 from the start of the cache, filled by the append and read by attention."""
    import torch
    from onnx_translator_b200 import capi
    lib = capi.load()
    torch_type = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}[dtype]
    heads, kv_heads, dim, keys = 16, 8, 128, 300
    pages = (2 ** 31 // (kv_heads * dim)) // page + 40
    rng = _rng("far", dtype, page, tokens)
    q, k, v = exact(rng, (tokens, heads, dim), dtype), exact(rng, (keys, kv_heads, dim), dtype), exact(rng, (keys, kv_heads, dim), dtype)
    caches = [torch.zeros((pages, page, kv_heads, dim), dtype=torch_type, device="cuda") for _ in range(2)]
    torch.cuda.synchronize()
    shape, nd = capi.shape_array(caches[0].shape)
    handles = [lib.tops_wrap(c.data_ptr(), shape, nd, capi.DTYPE_MAP[dtype]) for c in caches]
    table = (pages - 1 - np.arange(-(-keys // page))).astype(np.int32)[None]
    j = np.arange(keys)
    slots = table[0, j // page].astype(np.int64) * page + j % page
    append = fill(capi.CQKNormRotaryCall(), q=device(np.zeros((keys, heads, dim)), dtype), k=device(k, dtype), v=device(v, dtype),
                  q_out=device(np.zeros((keys, heads, dim)), dtype), slots=device(slots.astype(np.int32), "int32"))
    call = fill(capi.CPagedAttentionCall(scale=dim ** -0.5), q=device(q, dtype), page_table=device(table, "int32"),
                query_start=device(np.array([0, tokens], np.int32), "int32"), kv_length=device(np.array([keys], np.int32), "int32"),
                y=device(np.full(q.shape, 7.0), dtype))
    for c in (append, call):
        c.key_cache, c.value_cache = (ctypes.cast(h, ctypes.c_void_p) for h in handles)
    assert lib.tops_qk_norm_rotary_forward(ctypes.byref(append)) == 0, lib.tops_last_error_message()
    assert lib.tops_paged_attention_forward(ctypes.byref(call)) == 0, lib.tops_last_error_message()
    seen = j[None, :] <= (keys - tokens + np.arange(tokens))[:, None]
    want, tol = attention(q, k, v, seen, dim ** -0.5, dtype)
    got = to_f64(call.kept["y"].numpy(), dtype)
    capi.check(lib)
    assert_close(got, want, tol)
    for h in handles:
        lib.free_tensor(h)
    del caches
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", TYPES)
def test_cross_attention_on_another_stream_and_captured(dtype):
    """The caller's stream carries the call; one captured call serves new contents and lengths."""
    import torch
    from onnx_translator_b200 import capi
    lib = capi.load()
    for queries in (1, 150):
        rng = _rng("stream", dtype, queries)
        sets = [(exact(rng, (2, queries, 4, 64), dtype), exact(rng, (2, 700, 2, 64), dtype), exact(rng, (2, 700, 2, 64), dtype),
                 np.array([n, 700 - n], np.int32)) for n in (650, 33)]
        call = fill(capi.CCrossAttentionCall(scale=0.125), q=device(sets[0][0], dtype), k=device(sets[0][1], dtype), v=device(sets[0][2], dtype),
                    key_length=device(sets[0][3], "int32"), y=device(np.full(sets[0][0].shape, 7.0), dtype))
        others = [device(x, dtype) for x in sets[1][:3]] + [device(sets[1][3], "int32")]
        lib.tops_sync()
        stream = torch.cuda.Stream()
        lib.tops_set_stream(stream.cuda_stream)
        try:
            assert lib.tops_capture_begin() == 0
            assert lib.tops_cross_attention_forward(ctypes.byref(call)) == 0
            graph = lib.tops_capture_end()
            for which in (0, 1):
                if which:
                    for name, other in zip(("q", "k", "v", "key_length"), others):
                        lib.flatten_forward(other.handle, call.kept[name].handle)
                assert lib.tops_capture_launch(graph) == 0
                got = to_f64(call.kept["y"].numpy(), dtype)
                q, k, v, lengths = sets[which]
                for b in range(2):
                    want, tol = attention(q[b], k[b], v[b], np.broadcast_to(np.arange(700) < lengths[b], (queries, 700)), 0.125, dtype)
                    assert_close(got[b], want, tol)
            lib.tops_capture_free(graph)
        finally:
            lib.tops_set_stream(None)
        capi.check(lib)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("most", [1, 2, 30])
def test_hundreds_of_short_sequences(dtype, most):
    """More sequences than lanes and than SMs, many of them without keys or without tokens: every block goes through dozens of items."""
    rng = _rng("hundreds", dtype, most)
    pairs = []
    for b in range(333):
        n = int(rng.integers(0, most + 1)) if most > 1 else 1
        pairs.append((n, 0 if b % 7 == 3 else n + int(rng.integers(0, 200 if b % 5 else 700))))
    problem = Paged(rng, dtype, 8, 2, 64, 16, pairs, extra_rows=3)
    want, tol = problem.want()
    got = run_paged(problem)
    assert_close(got[:len(want)], want, tol)
    assert np.all(got[len(want):] == 7.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("queries", [1, 100])
def test_hundreds_of_short_sources(dtype, queries):
    rng = _rng("sources", dtype, queries)
    _cross(dtype, 101, queries, 150, 4, 2, 64, lengths=rng.integers(0, 151, 101), mask=(rng.random((101, 150)) < 0.8).astype(np.uint8))
