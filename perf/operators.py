"""The attention operators that are measured: their plain forms, the calls a user makes of them, and their definition in 64 bits.

Three operators that run one after the other in a decoder with cached keys and values:

qk_norm_rotary    RMS norm of every query and key head, the position rotation, and the append of keys and values to a paged cache
paged_attention   a ragged batch of new tokens (one each, or chunks) attends over the cache
cross_attention   decoder tokens attend to an encoder's states of another length, with a padding mask

With ``own`` false ``run`` computes them with elementary torch operations in 32 bits; with ``own`` true it calls the library.
"""
import ctypes
import math
import random

import torch

own = False

_TYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}


# ---- the cases ---------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one decoding step of eight sequences, grouped heads: latency
        {"name": "norm_rotary_step", "op": "qk_norm_rotary", "type": "bfloat16", "tokens": 8, "heads": 32, "kv_heads": 8, "dim": 128,
         "rotary": 128, "interleaved": False, "source": "packed", "cache": True, "page": 16},
        # a long prompt's projection, rotated and stored in one go: the largest copy-like call
        {"name": "norm_rotary_prompt", "op": "qk_norm_rotary", "type": "bfloat16", "tokens": 16384, "heads": 32, "kv_heads": 8, "dim": 128,
         "rotary": 128, "interleaved": False, "source": "packed", "cache": True, "page": 64},
        # an exported graph's layout [batch, heads, tokens, dim], half of each head rotated in pairs, an odd head size, no cache
        {"name": "norm_rotary_heads_first", "op": "qk_norm_rotary", "type": "float16", "tokens": 3 * 517, "batch": 3, "heads": 20, "kv_heads": 20,
         "dim": 80, "rotary": 40, "interleaved": True, "source": "heads_first", "cache": False, "page": 16},
        # one token of one conversation of 511: the smallest attention call
        {"name": "decode_one", "op": "paged_attention", "type": "bfloat16", "batch": 1, "q_min": 1, "q_max": 1, "kv_min": 511, "kv_max": 511,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "window": 0, "spread": 1},
        # one token each of a full serving batch with lengths of all sizes
        {"name": "decode_batch", "op": "paged_attention", "type": "bfloat16", "batch": 64, "q_min": 1, "q_max": 1, "kv_min": 300, "kv_max": 8192,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "window": 0, "spread": 2},
        # two very long documents, one token each: few rows, the long axis has to be split
        {"name": "decode_long", "op": "paged_attention", "type": "float16", "batch": 2, "q_min": 1, "q_max": 1, "kv_min": 100003, "kv_max": 131072,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "window": 0, "spread": 3},
        # a prompt of 8192 without a past: causal attention at its densest
        {"name": "prompt_whole", "op": "paged_attention", "type": "bfloat16", "batch": 1, "q_min": 8192, "q_max": 8192, "kv_min": 8192, "kv_max": 8192,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "window": 0, "spread": 4},
        # the next 2048 tokens of a long prompt over a cache of 32768 before them
        {"name": "prompt_chunk", "op": "paged_attention", "type": "bfloat16", "batch": 1, "q_min": 2048, "q_max": 2048, "kv_min": 34816, "kv_max": 34816,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 128, "window": 0, "spread": 5},
        # ragged chunks over caches of odd lengths, heads of 64 in groups of three, a sliding window
        {"name": "mixed_window", "op": "paged_attention", "type": "float16", "batch": 13, "q_min": 1, "q_max": 513, "kv_min": 700, "kv_max": 5001,
         "heads": 12, "kv_heads": 4, "dim": 64, "page": 16, "window": 1024, "spread": 6},
        # one decoder token per sequence against encoder states, padded to the longest
        {"name": "cross_step", "op": "cross_attention", "type": "float16", "batch": 16, "queries": 1, "keys": 1500, "heads": 20, "kv_heads": 20,
         "dim": 64, "heads_first": True, "mask": "lengths", "spread": 7},
        # a batch of whole targets against long sources under a padding mask
        {"name": "cross_batch", "op": "cross_attention", "type": "bfloat16", "batch": 8, "queries": 1024, "keys": 4096, "heads": 16, "kv_heads": 16,
         "dim": 128, "heads_first": False, "mask": "bool", "spread": 8},
        # a latent grid against 77 text states in float32: odd lengths
        {"name": "cross_float32", "op": "cross_attention", "type": "float32", "batch": 2, "queries": 1023, "keys": 77, "heads": 8, "kv_heads": 8,
         "dim": 40, "heads_first": False, "mask": "additive", "spread": 9},
    ]


def _log(rng, low, high):
    """A whole number between low and high, evenly spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _draw_once(rng):
    op = rng.choice(["qk_norm_rotary", "paged_attention", "paged_attention", "cross_attention"])
    kv_heads = rng.choice([1, 2, 4, 5, 8, 12, 16])
    heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 7, 8])
    half = rng.choice(["float16", "bfloat16"])
    if op == "qk_norm_rotary":
        dim = rng.choice([40, 64, 80, 96, 128, 128, 256])
        source = rng.choice(["packed", "separate", "heads_first"])
        batch = rng.choice([1, 2, 3, 5]) if source == "heads_first" else 1
        return {"op": op, "type": rng.choice([half, half, "float32"]), "tokens": batch * _log(rng, 1, 16384 // batch), "batch": batch, "heads": heads,
                "kv_heads": kv_heads, "dim": dim, "rotary": rng.choice([dim, dim, dim // 2]), "interleaved": rng.random() < 0.4, "source": source,
                "cache": rng.random() < 0.6, "page": rng.choice([16, 32, 64, 128])}
    if op == "paged_attention":
        decode = rng.random() < 0.5
        kv_max = _log(rng, 1, 131072 if decode else 34816)
        q_max = 1 if decode else min(kv_max, _log(rng, 2, 8192))
        return {"op": op, "type": half if rng.random() < 0.85 else "float32", "batch": _log(rng, 1, 128 if decode else 32),
                "q_min": rng.randint(1, q_max), "q_max": q_max, "kv_min": rng.randint(max(1, min(q_max, kv_max)), kv_max), "kv_max": kv_max,
                "heads": heads, "kv_heads": kv_heads, "dim": rng.choice([64, 64, 80, 96, 128, 128, 128, 256]), "page": rng.choice([16, 32, 64, 128]),
                "window": rng.choice([0, 0, 0, _log(rng, 16, 4096)]), "spread": rng.randrange(1 << 30)}
    return {"op": op, "type": half if rng.random() < 0.8 else "float32", "batch": _log(rng, 1, 64), "queries": _log(rng, 1, 4096), "keys": _log(rng, 1, 8192),
            "heads": heads, "kv_heads": kv_heads, "dim": rng.choice([40, 64, 64, 80, 128, 128]), "heads_first": rng.random() < 0.5,
            "mask": rng.choice(["none", "lengths", "bool", "additive"]), "spread": rng.randrange(1 << 30)}


def draw(rng):
    while True:
        case = _draw_once(rng)
        cost, size = work(case), _plain_elements(case)
        # no dearer than the largest listed call in arithmetic or bytes (float32 runs on far slower units), and the plain form's temporaries fit
        if cost["flops"] <= (5.0e11 if case["type"] != "float32" else 2.5e10) and cost["bytes"] <= 1.6e9 and size <= 2.3e9:
            return case


def _lengths(case):
    """Query and key counts of a paged case's sequences: a function of the case, the longest of each among them."""
    rng = random.Random(case["spread"])
    kv = [_log(rng, case["kv_min"], case["kv_max"]) for _ in range(case["batch"])]
    kv[rng.randrange(len(kv))] = case["kv_max"]
    q = [min(k, _log(rng, case["q_min"], case["q_max"])) for k in kv]
    q[kv.index(case["kv_max"])] = case["q_max"]
    return q, kv


def _key_lengths(case):
    rng = random.Random(case["spread"])
    lengths = [rng.randint(max(1, case["keys"] // 2), case["keys"]) for _ in range(case["batch"])]
    lengths[rng.randrange(len(lengths))] = case["keys"]
    return lengths if case["mask"] != "none" else [case["keys"]] * case["batch"]


def _visible(q, kv, window):
    """Sum over the q newest of kv tokens of the keys each sees."""
    def up_to(n):                       # sum of min(p, window) for p in 1..n
        if not window or n <= window:
            return n * (n + 1) // 2
        return window * (window + 1) // 2 + (n - window) * window
    return up_to(kv) - up_to(kv - q)


def _plain_elements(case):
    """Scores or gathered keys that the plain form holds at once."""
    if case["op"] == "paged_attention":
        q, kv = _lengths(case)
        return case["batch"] * max(kv) * max(max(q) * case["heads"], case["kv_heads"] * case["dim"])
    if case["op"] == "cross_attention":
        return case["batch"] * case["heads"] * case["queries"] * case["keys"]
    return 0


def work(case):
    size = 4 if case["type"] == "float32" else 2
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "qk_norm_rotary":
        rows = case["tokens"]
        copied = kv_heads if case["cache"] else 0
        values = rows * (heads + kv_heads + copied) * dim
        tables = 4 * rows * case["rotary"] + 4 * rows * (2 if case["cache"] else 1)
        return {"bytes": 2 * values * size + tables + 2 * dim * size, "flops": rows * (heads + kv_heads) * (4 * dim + 3 * case["rotary"])}
    if case["op"] == "paged_attention":
        q, kv = _lengths(case)
        window = case["window"]
        seen = [min(k, n + window - 1) if window else k for n, k in zip(q, kv)]
        pages = sum(-(-s // case["page"]) for s in seen)
        pairs = sum(_visible(n, k, window) for n, k in zip(q, kv))
        return {"bytes": size * dim * (2 * heads * sum(q) + 2 * kv_heads * sum(seen)) + 4 * (pages + 2 * len(q)), "flops": 4 * dim * heads * pairs}
    lengths = _key_lengths(case)
    batch, queries = case["batch"], case["queries"]
    mask = {"none": 0, "lengths": 4 * batch, "bool": batch * case["keys"], "additive": 4 * batch * case["keys"]}[case["mask"]]
    return {"bytes": size * dim * (2 * heads * batch * queries + 2 * kv_heads * sum(lengths)) + mask, "flops": 4 * dim * heads * queries * sum(lengths)}


# ---- inputs ------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    dtype = _TYPES[case["type"]]
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]

    def normal(*shape, spread=1.0):
        out = torch.empty(shape, dtype=dtype, device=dev)
        return out.normal_(0.0, spread, generator=gen)

    s = {"case": dict(case)}
    if case["op"] == "qk_norm_rotary":
        tokens, rotary = case["tokens"], case["rotary"]
        batch = case.get("batch", 1)
        if case["source"] == "packed":
            s["q"], s["k"], s["v"] = normal(tokens, heads + 2 * kv_heads, dim, spread=3.0), None, None
        else:
            lead = (batch, heads, tokens // batch) if case["source"] == "heads_first" else (tokens, heads)
            lead_kv = (batch, kv_heads, tokens // batch) if case["source"] == "heads_first" else (tokens, kv_heads)
            s["q"], s["k"], s["v"] = normal(*lead, dim, spread=3.0), normal(*lead_kv, dim, spread=3.0), normal(*lead_kv, dim)
        s["q_weight"] = (1.0 + 0.2 * torch.randn(dim, device=dev, generator=gen)).to(dtype)
        s["k_weight"] = (1.0 + 0.2 * torch.randn(dim, device=dev, generator=gen)).to(dtype)
        reach = 40000
        angle = torch.arange(reach, device=dev, dtype=torch.float64)[:, None] * (10000.0 ** (-torch.arange(0, rotary, 2, device=dev, dtype=torch.float64) / rotary))
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        s["positions"] = (torch.arange(tokens, device=dev) + int(torch.randint(0, reach - tokens, (1,), device=dev, generator=gen))).to(torch.int32)
        s["q_out"] = torch.empty(_qk_shapes(case)[0], dtype=dtype, device=dev)
        s["k_out"] = None if case["cache"] else torch.empty(_qk_shapes(case)[1], dtype=dtype, device=dev)
        s["key_cache"] = s["value_cache"] = s["slots"] = None
        if case["cache"]:
            pages = -(-tokens // case["page"]) + 2
            s["key_cache"], s["value_cache"] = normal(pages, case["page"], kv_heads, dim), normal(pages, case["page"], kv_heads, dim)
            order = torch.randperm(pages, device=dev, generator=gen)
            at = torch.arange(tokens, device=dev)
            s["slots"] = (order[at // case["page"]] * case["page"] + at % case["page"]).to(torch.int32)
        return s
    s["scale"] = 1.0 / math.sqrt(dim)
    if case["op"] == "paged_attention":
        q, kv = _lengths(case)
        width = max(-(-k // case["page"]) for k in kv)
        pages = sum(-(-k // case["page"]) for k in kv)
        s["q"] = normal(sum(q), heads, dim, spread=1.5)
        s["key_cache"], s["value_cache"] = normal(pages, case["page"], kv_heads, dim), normal(pages, case["page"], kv_heads, dim)
        order = torch.randperm(pages, device=dev, generator=gen).to(torch.int32)
        used = torch.tensor([-(-k // case["page"]) for k in kv], device=dev)
        first = torch.cumsum(used, 0) - used
        column = torch.arange(width, device=dev)
        s["page_table"] = torch.where(column < used[:, None], order[(first[:, None] + column).clamp(max=pages - 1)], -1).to(torch.int32)
        s["query_start"] = torch.tensor([0] + q, device=dev).cumsum(0).to(torch.int32)
        s["kv_length"] = torch.tensor(kv, device=dev, dtype=torch.int32)
        s["q_longest"], s["kv_longest"] = max(q), max(kv)
    else:
        batch, queries, keys = case["batch"], case["queries"], case["keys"]
        first = case["heads_first"]
        s["q"] = normal(*((batch, heads, queries) if first else (batch, queries, heads)), dim, spread=1.5)
        s["k"] = normal(*((batch, kv_heads, keys) if first else (batch, keys, kv_heads)), dim)
        s["v"] = normal(*((batch, kv_heads, keys) if first else (batch, keys, kv_heads)), dim)
        lengths = torch.tensor(_key_lengths(case), device=dev, dtype=torch.int32)
        kept = torch.arange(keys, device=dev) < lengths[:, None]
        s["key_length"] = lengths if case["mask"] == "lengths" else None
        s["mask"] = None
        if case["mask"] == "bool":
            s["mask"] = kept.to(torch.uint8)
        elif case["mask"] == "additive":
            s["mask"] = torch.where(kept, torch.randn(batch, keys, device=dev, generator=gen), torch.finfo(torch.float32).min)
    s["y"] = torch.empty_like(s["q"])
    return s


def _qk_shapes(case):
    """Shapes of the rotated queries and keys."""
    batch, tokens = case.get("batch", 1), case["tokens"]
    if case["source"] == "heads_first":
        return [(batch, h, tokens // batch, case["dim"]) for h in (case["heads"], case["kv_heads"])]
    return [(tokens, h, case["dim"]) for h in (case["heads"], case["kv_heads"])]


# ---- one pass ----------------------------------------------------------------------------------------------------------
def run(state):
    return _run_own(state) if own else _PLAIN[state["case"]["op"]](state)


def _rms(x, weight):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * weight.float()


def _rotate(x, cos, sin, interleaved):
    half = cos.shape[-1]
    turned, rest = x[..., :2 * half], x[..., 2 * half:]
    a, b = (turned[..., 0::2], turned[..., 1::2]) if interleaved else (turned[..., :half], turned[..., half:])
    lo, hi = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack((lo, hi), -1).flatten(-2) if interleaved else torch.cat((lo, hi), -1)
    return torch.cat((turned, rest), -1)


def _plain_qk_norm_rotary(s):
    case, dtype = s["case"], s["q"].dtype
    heads, kv_heads = case["heads"], case["kv_heads"]
    q, k, v = s["q"], s["k"], s["v"]
    if k is None:
        q, k, v = q[:, :heads], q[:, heads:heads + kv_heads], q[:, heads + kv_heads:]
    at = s["positions"].long()
    cos, sin = s["cos"][at], s["sin"][at]
    if case["source"] == "heads_first":
        cos, sin = (t.view(case["batch"], 1, -1, t.shape[-1]) for t in (cos, sin))
    else:
        cos, sin = cos[:, None], sin[:, None]
    q = _rotate(_rms(q.float(), s["q_weight"]), cos, sin, case["interleaved"]).to(dtype)
    k = _rotate(_rms(k.float(), s["k_weight"]), cos, sin, case["interleaved"]).to(dtype)
    if not case["cache"]:
        return {"q": q, "k": k}
    if case["source"] == "heads_first":
        k, v = (t.transpose(1, 2).reshape(-1, kv_heads, case["dim"]) for t in (k, v))
    slots = s["slots"].long()
    s["key_cache"].view(-1, kv_heads, case["dim"])[slots] = k
    s["value_cache"].view(-1, kv_heads, case["dim"])[slots] = v
    return {"q": q, "key_cache": s["key_cache"], "value_cache": s["value_cache"]}


def _softmax_product(scores, seen, values):
    """softmax over the seen scores, times values; a row that sees nothing gives zeros."""
    scores = torch.where(seen, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = weights.sum(-1, keepdim=True)
    return (weights @ values) / torch.where(total == 0, 1.0, total)


def _plain_paged_attention(s):
    case, q = s["case"], s["q"]
    heads, kv_heads, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    longest, dev = s["q_longest"], q.device
    start, kv = s["query_start"].long(), s["kv_length"].long()
    batch, total, group = kv.numel(), q.shape[0], heads // kv_heads
    count = start[1:] - start[:-1]
    table = s["page_table"].long().clamp(min=0)
    column = torch.arange(table.shape[1] * page, device=dev)
    held = (column < kv[:, None])[:, :, None, None]
    keys = torch.where(held, s["key_cache"][table].view(batch, -1, kv_heads, dim).float(), 0.0).permute(0, 2, 3, 1)
    values = torch.where(held, s["value_cache"][table].view(batch, -1, kv_heads, dim).float(), 0.0).permute(0, 2, 1, 3)
    row = torch.arange(longest, device=dev)
    rows = q[(start[:-1, None] + row).clamp(max=total - 1)].float().view(batch, longest, kv_heads, group, dim).permute(0, 2, 3, 1, 4)
    scores = (rows.reshape(batch, kv_heads, group * longest, dim) @ keys).view(batch, kv_heads, group, longest, -1) * s["scale"]
    position = (kv - count)[:, None] + row
    seen = (column <= position[..., None]) & (column < kv[:, None, None])
    if case["window"]:
        seen = seen & (column > position[..., None] - case["window"])
    out = _softmax_product(scores, seen[:, None, None], values[:, :, None])
    out = out.permute(0, 3, 1, 2, 4).reshape(batch, longest, heads, dim)
    token = torch.arange(total, device=dev)
    which = torch.searchsorted(start, token, right=True) - 1
    return {"y": out[which, token - start[which]].to(q.dtype)}


def _plain_cross_attention(s):
    case, q, k, v = s["case"], s["q"].float(), s["k"].float(), s["v"].float()
    if not case["heads_first"]:
        q, k, v = q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2)
    group = case["heads"] // case["kv_heads"]
    q = q.reshape(case["batch"], case["kv_heads"], group * case["queries"], case["dim"])
    scores = (q @ k.transpose(-1, -2)) * s["scale"]
    seen = torch.ones(case["batch"], case["keys"], dtype=torch.bool, device=q.device)
    if case["mask"] == "lengths":
        seen = torch.arange(case["keys"], device=q.device) < s["key_length"][:, None]
    elif case["mask"] == "bool":
        seen = s["mask"] != 0
    elif case["mask"] == "additive":
        seen = s["mask"] > torch.finfo(torch.float32).min
        scores = scores + torch.where(seen, s["mask"], 0.0)[:, None, None]
    v = torch.where(seen[:, None, :, None], v, 0.0)
    out = _softmax_product(scores, seen[:, None, None], v).view(case["batch"], case["heads"], case["queries"], case["dim"])
    return {"y": (out if case["heads_first"] else out.transpose(1, 2)).contiguous().to(s["q"].dtype)}


_PLAIN = {"qk_norm_rotary": _plain_qk_norm_rotary, "paged_attention": _plain_paged_attention, "cross_attention": _plain_cross_attention}


# ---- the framework's calls ---------------------------------------------------------------------------------------------
def _wrap(lib, capi, tensor):
    """The library's description of a torch tensor's memory, None for None."""
    if tensor is None:
        return None
    name = {torch.float16: "float16", torch.bfloat16: "bfloat16", torch.float32: "float32", torch.int32: "int32", torch.uint8: "uint8"}[tensor.dtype]
    shape, ndim = capi.shape_array(tensor.shape)
    return ctypes.cast(lib.tops_wrap(tensor.data_ptr(), shape, ndim, capi.DTYPE_MAP[name]), ctypes.c_void_p)


def _describe(state):
    """The call's struct, filled in once for the buffers that a serving program keeps."""
    from onnx_translator_b200 import capi
    lib, case = capi.load(), state["case"]
    t = lambda name: _wrap(lib, capi, state.get(name))  # noqa: E731
    if case["op"] == "qk_norm_rotary":
        call = capi.CQKNormRotaryCall(q=t("q"), k=t("k"), v=t("v") if case["cache"] else None,
                                      packed_kv_heads=case["kv_heads"] if state["k"] is None else 0,
                                      heads_first=int(case["source"] == "heads_first"), q_weight=t("q_weight"), k_weight=t("k_weight"), epsilon=1e-6,
                                      cos_table=t("cos"), sin_table=t("sin"), positions=t("positions"), interleaved=int(case["interleaved"]),
                                      q_out=t("q_out"), k_out=t("k_out"), key_cache=t("key_cache"), value_cache=t("value_cache"), slots=t("slots"))
        outputs = {"q": state["q_out"]}
        outputs.update({"key_cache": state["key_cache"], "value_cache": state["value_cache"]} if case["cache"] else {"k": state["k_out"]})
        entry = lib.tops_qk_norm_rotary_forward
    elif case["op"] == "paged_attention":
        call = capi.CPagedAttentionCall(q=t("q"), key_cache=t("key_cache"), value_cache=t("value_cache"), page_table=t("page_table"),
                                        query_start=t("query_start"), kv_length=t("kv_length"), scale=state["scale"], window=case["window"], y=t("y"))
        outputs, entry = {"y": state["y"]}, lib.tops_paged_attention_forward
    else:
        call = capi.CCrossAttentionCall(q=t("q"), k=t("k"), v=t("v"), key_length=t("key_length"), mask=t("mask"), scale=state["scale"],
                                        heads_first=int(case["heads_first"]), y=t("y"))
        outputs, entry = {"y": state["y"]}, lib.tops_cross_attention_forward
    return lib, entry, call, outputs


def _run_own(state):
    if "call" not in state:
        state["call"] = _describe(state)
    lib, entry, call, outputs = state["call"]
    lib.tops_set_stream(torch.cuda.current_stream().cuda_stream or 1)       # 1: CUDA's name for the default stream
    if entry(ctypes.byref(call)):
        raise RuntimeError(lib.tops_last_error_message().decode())
    return outputs


# ---- the definition in 64 bits -----------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    group = heads // kv_heads
    if case["op"] == "qk_norm_rotary":
        if case["source"] == "packed":
            q, k, v = s["q"].split([heads, kv_heads, kv_heads], dim=1)
        elif case["source"] == "heads_first":
            q, k, v = (x.permute(0, 2, 1, 3).flatten(0, 1) for x in (s["q"], s["k"], s["v"]))
        else:
            q, k, v = s["q"], s["k"], s["v"]
        turn = torch.complex(s["cos"].double(), s["sin"].double())[s["positions"].long()].unsqueeze(1)
        done = []
        for x, weight in ((q, s["q_weight"]), (k, s["k_weight"])):
            x = x.double()
            x = x / (x.pow(2).sum(-1, keepdim=True) / dim + 1e-6).sqrt() * weight.double()
            pairs = x[..., :case["rotary"]]
            pairs = pairs.unflatten(-1, (-1, 2)) if case["interleaved"] else pairs.unflatten(-1, (2, -1)).transpose(-1, -2)
            z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
            z = z.flatten(-2) if case["interleaved"] else z.transpose(-1, -2).flatten(-2)
            done.append(torch.cat([z, x[..., case["rotary"]:]], -1))
        if case["source"] == "heads_first":
            done = [x.unflatten(0, (case["batch"], -1)).transpose(1, 2) for x in done]
        if not case["cache"]:
            return {"q": done[0], "k": done[1]}
        k = done[1].transpose(1, 2).flatten(0, 1) if case["source"] == "heads_first" else done[1]
        caches = []
        for cache, new in ((s["key_cache"], k), (s["value_cache"], v.double())):
            rows = cache.double().flatten(0, 1)
            rows.index_copy_(0, s["slots"].long(), new.contiguous())
            caches.append(rows.view(cache.shape))
        return {"q": done[0], "key_cache": caches[0], "value_cache": caches[1]}
    if work(case)["flops"] > 2e12:
        return None
    y = torch.zeros(s["y"].shape, dtype=torch.float64, device=s["y"].device)
    if case["op"] == "paged_attention":
        counts, lengths = _lengths(case)
        begin = 0
        for b, (n, length) in enumerate(zip(counts, lengths)):
            pages = s["page_table"][b, :-(-length // case["page"])].long()
            place = torch.arange(length - n, length, device=y.device)[:, None]
            key = torch.arange(length, device=y.device)
            hidden = (key > place) | ((place - key >= case["window"]) if case["window"] else False)
            for h in range(kv_heads):
                k = s["key_cache"][pages, :, h].flatten(0, 1)[:length].double()
                v = s["value_cache"][pages, :, h].flatten(0, 1)[:length].double()
                for g in range(h * group, (h + 1) * group):
                    score = s["q"][begin:begin + n, g].double() @ k.T * s["scale"]
                    y[begin:begin + n, g] = torch.softmax(score.masked_fill(hidden, -math.inf), -1) @ v
            begin += n
        return {"y": y}
    lengths = _key_lengths(case)
    heads_axis = 1 if case["heads_first"] else 2
    for b, length in enumerate(lengths):
        for h in range(heads):
            q = s["q"][b].select(heads_axis - 1, h).double()
            k, v = (s[n][b].select(heads_axis - 1, h // group)[:length].double() for n in ("k", "v"))
            score = q @ k.T * s["scale"]
            if case["mask"] == "additive":
                score = score + s["mask"][b, :length].double()
            y[b].select(heads_axis - 1, h).copy_(torch.softmax(score, -1) @ v)
    return {"y": y}
