"""What answering from packed codes takes, as cases to measure.

``op`` says which operator of the package a case is about:

``linear``  ``packed_linear.packed_linear``: the product of activations with a matrix held as packed 4-bit codes, with low-rank
            adapters of many requests beside it;
``append``  ``packed_cache.append_packed``: new keys and values into a paged cache of 4-bit codes, and ``read_packed``: the values that
            it holds for them;
``attend``  ``packed_cache.attend_packed``: attention of one query per sequence, or of whole prompts, over such a cache.

Inputs.  Matrices are Gaussian (sigma 0.02), rounded to the nearest code under abs-max scales per row, or under scales and integer
zero points per group of columns.  Activations are Gaussian with channel scales of their own.  Keys and values are Gaussian, a tenth of
their channels larger.  Pages of a sequence lie anywhere in the cache.  Sequences of a ragged batch differ in length, some are empty,
some have no query in this step.
"""
import math
import os
import random
import sys

import torch

own = False
DEVICE = "cuda"
DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16}


def listed():
    return [
        # a key projection of the smallest width in use here, one token of one request with an adapter: launches and latency
        {"name": "linear 1024x4096 t1 r16", "op": "linear", "dtype": "float16", "m": 1024, "n": 4096, "tokens": 1, "group": 0, "adapters": 4, "rank": 16},
        # a decoding step of sixteen requests, each with an adapter of its own
        {"name": "linear 8192x8192 t16 r16", "op": "linear", "dtype": "bfloat16", "m": 8192, "n": 8192, "tokens": 16, "group": 0, "adapters": 32, "rank": 16},
        # a wider step, INT4 with scale and zero point per group of 128 columns, a pruned layer with an odd number of rows
        {"name": "linear 14333x4096 t61 g128 r8", "op": "linear", "dtype": "float16", "m": 14333, "n": 4096, "tokens": 61, "group": 128, "adapters": 24, "rank": 8},
        # prompts of several requests through the largest matrix of a block
        {"name": "linear 8192x28672 t2048 r32", "op": "linear", "dtype": "bfloat16", "m": 8192, "n": 28672, "tokens": 2048, "group": 0, "adapters": 8, "rank": 32},
        # a decoding step of a few sequences
        {"name": "append b8 q1 h8 d128", "op": "append", "dtype": "bfloat16", "kv_heads": 8, "head_dim": 128, "page": 64, "batch": 8, "queries": 1, "length": 1000, "ragged": False},
        # prompts of different lengths, some of them on top of what is in the cache
        {"name": "append b7 q2039 h8 d128", "op": "append", "dtype": "float16", "kv_heads": 8, "head_dim": 128, "page": 16, "batch": 7, "queries": 2039, "length": 4100, "ragged": True},
        # the first steps of one sequence
        {"name": "attend b1 q1 137 h8/8 d64", "op": "attend", "dtype": "float16", "heads": 8, "kv_heads": 8, "head_dim": 64, "page": 16, "batch": 1, "queries": 1, "length": 137, "ragged": False,
         "causal": True, "softcap": 0.0, "slopes": False, "prefix": 0},
        # a decoding step of a full batch, sequences of all lengths, grouped heads
        {"name": "attend b48 q1 8191 h64/8 d128", "op": "attend", "dtype": "bfloat16", "heads": 64, "kv_heads": 8, "head_dim": 128, "page": 64, "batch": 48, "queries": 1, "length": 8191, "ragged": True,
         "causal": True, "softcap": 0.0, "slopes": False, "prefix": 0},
        # one sequence, very long: the work lies along one axis only
        {"name": "attend b1 q1 131072 h64/8 d128", "op": "attend", "dtype": "bfloat16", "heads": 64, "kv_heads": 8, "head_dim": 128, "page": 128, "batch": 1, "queries": 1, "length": 131072, "ragged": False,
         "causal": True, "softcap": 0.0, "slopes": False, "prefix": 0},
        # four drafted tokens at once, capped scores and a bias by distance
        {"name": "attend b16 q4 2000 cap bias", "op": "attend", "dtype": "float16", "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 32, "batch": 16, "queries": 4, "length": 2000, "ragged": False,
         "causal": True, "softcap": 30.0, "slopes": True, "prefix": 0},
        # prompts of different lengths, partly in the cache already, under a prefix that all may see
        {"name": "attend b5 q1500 2500 prefix", "op": "attend", "dtype": "float16", "heads": 32, "kv_heads": 8, "head_dim": 64, "page": 64, "batch": 5, "queries": 1500, "length": 2500, "ragged": True,
         "causal": True, "softcap": 0.0, "slopes": False, "prefix": 300},
        # a long prompt on top of an equally long one
        {"name": "attend b1 q4096 8192 h32/8 d128", "op": "attend", "dtype": "bfloat16", "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64, "batch": 1, "queries": 4096, "length": 8192, "ragged": False,
         "causal": True, "softcap": 0.0, "slopes": False, "prefix": 0},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("linear", "linear", "append", "attend", "attend", "attend"))
    dtype = rng.choice(sorted(DTYPES))
    if op == "linear":
        m, n = _log(rng, 64, 28672), 32 * _log(rng, 8, 896)
        while m * n > 8192 * 28672:
            m, n = _log(rng, 64, 28672), 32 * _log(rng, 8, 896)
        groups = [g for g in (64, 128, 256) if n % g == 0]
        return {"op": op, "dtype": dtype, "m": m, "n": n, "tokens": _log(rng, 1, min(4096, 2048 * 8192 * 28672 // (m * n))), "group": rng.choice([0] + groups),
                "adapters": rng.choice((0, 1, 5, 16, 32)), "rank": rng.choice((8, 16, 32, 64))}
    page, head_dim = rng.choice((16, 32, 64, 128)), rng.choice((64, 128))
    if op == "append":
        return {"op": op, "dtype": dtype, "kv_heads": rng.choice((1, 4, 5, 8, 16)), "head_dim": head_dim, "page": page, "batch": _log(rng, 1, 16), "queries": _log(rng, 1, 1024),
                "length": _log(rng, 1024, 4096), "ragged": rng.random() < 0.5}
    heads, kv_heads = rng.choice(((8, 8), (12, 12), (8, 1), (32, 8), (64, 8), (40, 8), (28, 4), (32, 2)))
    batch, queries = (_log(rng, 1, 48), rng.choice((1, 1, 2, 5))) if rng.random() < 0.6 else (_log(rng, 1, 6), _log(rng, 6, 1500))
    length = max(queries, _log(rng, 64, 131072 // batch if queries < 6 else 6144))
    while batch * queries * heads * length > 1 << 30 or batch * length > 262144:
        length = max(queries, length // 2)
        batch = max(1, batch - 1)
    return {"op": op, "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "batch": batch, "queries": queries, "length": length,
            "ragged": rng.random() < 0.5, "causal": rng.random() < 0.8, "softcap": rng.choice((0.0, 0.0, 20.0, 50.0)), "slopes": rng.random() < 0.25, "prefix": rng.choice((0, 0, 17, 400))}


def _sequences(case):
    """(length with this step's tokens, this step's tokens) of every sequence: a part of the case, not of the seed."""
    if not case["ragged"]:
        return [(case["length"], case["queries"])] * case["batch"]
    rng = random.Random(case["batch"] * 7919 + case["queries"] * 104729 + case["length"])
    out = [(case["length"], case["queries"])]
    for _ in range(case["batch"] - 1):
        length = rng.randint(0, case["length"])
        queries = min(length, case["queries"] if case["queries"] < 6 else rng.randint(0, case["queries"]))
        out.append((length, 0 if rng.random() < 0.06 else queries))
    return out


def _visible(case):
    """(row, key) pairs of one head that the masks leave."""
    total = 0
    for length, queries in _sequences(case):
        for p in range(length - queries, length):
            total += min(length, max(p + 1, case["prefix"])) if case["causal"] else length
    return total


def work(case):
    if case["op"] == "linear":
        m, n, t, r = case["m"], case["n"], case["tokens"], case["rank"]
        groups = n // case["group"] if case["group"] else 1
        used = min(t, case["adapters"])
        return {"bytes": m * n // 2 + 8 * m * groups + 2 * t * (m + n) + (2 * used * r * (m + n)), "flops": 2 * t * m * n + (2 * t * r * (m + n) if used else 0)}
    tokens = sum(q for _, q in _sequences(case))
    h, d = case["kv_heads"], case["head_dim"]
    if case["op"] == "append":
        return {"bytes": 2 * tokens * h * (2 * d + 2 * (d // 2 + 2) + 2 * d), "flops": 8 * tokens * h * d}
    keys = sum(length for length, q in _sequences(case) if q)
    return {"bytes": keys * h * (d + 4) + 4 * tokens * case["heads"] * d, "flops": 4 * d * case["heads"] * _visible(case)}


# ---- inputs ----------------------------------------------------------------------------------------------------------------------

def _pack(codes):
    """Codes -8..7 [..., d] (whole numbers in any type) as bytes: entry 2 i in the lower half of byte i."""
    fields = (codes + 8).to(torch.uint8)
    return (fields[..., 0::2] | (fields[..., 1::2] << 4)).contiguous()


def _fields(packed):
    """The fields 0..15 of packed bytes, in order."""
    return torch.stack((packed & 15, packed >> 4), -1).flatten(-2)


def _round_rows(v):
    """Abs-max scale per row, rounded to float16 through float32 (1 for a row of zeros), and the codes under it."""
    v = v.float()
    scale = (v.abs().amax(-1, keepdim=True) / 7.5).to(torch.float16)
    scale = torch.where(scale == 0, torch.ones_like(scale), scale)
    return torch.clamp(torch.round(v / scale.float()), -8, 7), scale


def _linear_inputs(case, gen):
    m, n, t, r, a, dtype = case["m"], case["n"], case["tokens"], case["rank"], case["adapters"], DTYPES[case["dtype"]]
    randn = lambda *shape: torch.randn(*shape, generator=gen, device=DEVICE)  # noqa: E731
    w = randn(m, n).mul_(0.02)
    if case["group"]:
        w = w.view(m, n // case["group"], case["group"])
        low, high = w.amin(-1, keepdim=True), w.amax(-1, keepdim=True)
        scale = (high - low) / 15
        zero = torch.round(-low / scale)
        codes = torch.clamp(torch.round(w / scale + zero), 0, 15).sub_(8).view(m, n)
        scale, zero, qmin = scale.squeeze(-1).contiguous(), zero.squeeze(-1).contiguous(), 0
    else:
        codes, scale = _round_rows(w)
        scale, zero, qmin = scale.float(), torch.zeros(1, 1, device=DEVICE), -8
    state = {"codes": _pack(codes), "scale": scale, "zero": zero, "qmin": qmin, "x": (randn(t, n) * torch.exp(0.5 * randn(n))).to(dtype)}
    if a:
        state["down"] = (randn(a, r, n) / math.sqrt(n)).to(dtype)
        state["up"] = (randn(a, m, r) * 0.1).to(dtype)
        state["scaling"] = 0.5 + torch.rand(a, generator=gen, device=DEVICE)
        # a step has an adapter per request in any order; the tokens of a prompt stand together
        ids = torch.randint(-1, a, (min(t, 64),), generator=gen, device=DEVICE, dtype=torch.int32)
        state["index"] = ids.repeat_interleave(-(-t // ids.numel()))[:t].contiguous()
    return state


def _cache_inputs(case, gen):
    seqs, page, h, d, dtype = _sequences(case), case["page"], case["kv_heads"], case["head_dim"], DTYPES[case["dtype"]]
    per = -(-max(length for length, _ in seqs) // page)
    pages = case["batch"] * per + 3
    order = torch.randperm(pages, generator=gen, device=DEVICE)[: case["batch"] * per]
    state = {"table": order.to(torch.int32).view(case["batch"], per).contiguous(), "page": page, "tokens": sum(q for _, q in seqs)}
    state["lengths"] = torch.tensor([length for length, _ in seqs], dtype=torch.int32, device=DEVICE)
    state["offsets"] = None
    if case["ragged"]:
        state["offsets"] = torch.tensor([0] + [q for _, q in seqs], device=DEVICE).cumsum(0).to(torch.int32)
    counts = torch.tensor([q for _, q in seqs], device=DEVICE)
    # for every token of this step: its sequence and its position, as the plain form needs them
    seq = torch.repeat_interleave(torch.arange(case["batch"], device=DEVICE), counts)
    first = counts.cumsum(0) - counts
    state["seq"], state["pos"] = seq, state["lengths"].long()[seq] - counts[seq] + torch.arange(state["tokens"], device=DEVICE) - first[seq]
    large = 1 + 2 * (torch.rand(h, d, generator=gen, device=DEVICE) < 0.1)
    for name in ("k", "v"):
        if case["op"] == "append":
            state[name] = (torch.randn(state["tokens"], h, d, generator=gen, device=DEVICE) * large).to(dtype)
        codes, scale = torch.zeros(pages, h, page, d // 2, dtype=torch.uint8, device=DEVICE), torch.zeros(pages, h, page, dtype=torch.float16, device=DEVICE)
        if case["op"] == "attend":
            values, scales = _round_rows(torch.randn(pages, h, page, d, generator=gen, device=DEVICE) * large[:, None])
            codes, scale = _pack(values), scales.squeeze(-1).contiguous()
        state[name + "_codes"], state[name + "_scale"] = codes, scale
    return state


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    state = _linear_inputs(case, gen) if case["op"] == "linear" else _cache_inputs(case, gen)
    state["case"] = case
    if case["op"] == "attend":
        state["q"] = torch.randn(state["tokens"], case["heads"], case["head_dim"], generator=gen, device=DEVICE).to(DTYPES[case["dtype"]])
        state["slopes"] = torch.exp2(-8 * torch.arange(1, case["heads"] + 1, device=DEVICE) / case["heads"]) if case["slopes"] else None
        state["prefix"] = torch.full((case["batch"],), case["prefix"], dtype=torch.int32, device=DEVICE) if case["prefix"] else None
    if own:
        package = os.path.join(os.getcwd(), "gptq-2d_b200")
        if package not in sys.path:
            sys.path.insert(0, package)
        import packed_cache
        import packed_linear

        state["L"], state["C"] = packed_linear, packed_cache
        if case["op"] != "linear":
            state["cache"] = packed_cache.PackedCache(state["k_codes"], state["k_scale"], state["v_codes"], state["v_scale"])
        elif case["adapters"]:
            state["adapters"] = packed_linear.LowRankAdapters(state["down"], state["up"], state["scaling"])
    return state


# ---- one pass --------------------------------------------------------------------------------------------------------------------

def _plain_linear(s):
    m, n = s["codes"].shape[0], s["x"].shape[1]
    groups = s["scale"].shape[1]
    w = (_fields(s["codes"]).float().view(m, groups, n // groups) + s["qmin"] - s["zero"][..., None]) * s["scale"][..., None]
    x = s["x"].float()
    y = x @ w.view(m, n).t()
    if s["case"]["adapters"]:
        a, r = s["down"].shape[:2]
        takes = (s["index"][:, None] == torch.arange(a, device=DEVICE)).float() * s["scaling"]
        inner = (x @ s["down"].float().view(a * r, n).t()).view(-1, a, r) * takes[..., None]
        y = y + inner.view(-1, a * r) @ s["up"].float().permute(1, 0, 2).reshape(m, a * r).t()
    return y.to(s["x"].dtype)


def _plain_append(s):
    pages = s["table"].long()[s["seq"], s["pos"] // s["page"]]
    offset = s["pos"] % s["page"]
    k, v = _round_rows(s["k"]), _round_rows(s["v"])
    s["k_codes"][pages, :, offset], s["k_scale"][pages, :, offset] = _pack(k[0]), k[1].squeeze(-1)
    s["v_codes"][pages, :, offset], s["v_scale"][pages, :, offset] = _pack(v[0]), v[1].squeeze(-1)
    read = lambda c, scale: ((_fields(c[pages, :, offset]).float() - 8) * scale[pages, :, offset].float()[..., None]).to(s["k"].dtype)  # noqa: E731
    return read(s["k_codes"], s["k_scale"]), read(s["v_codes"], s["v_scale"])


def _plain_attend(s):
    case = s["case"]
    b, h, d, group = case["batch"], case["kv_heads"], case["head_dim"], case["heads"] // case["kv_heads"]
    per = s["table"].shape[1]
    most, keys = case["queries"], per * case["page"]
    whole = lambda c, scale: ((_fields(c[s["table"].long()]).float() - 8) * scale[s["table"].long()].float()[..., None]).transpose(1, 2).reshape(b, h, 1, keys, d)  # noqa: E731
    # this step's tokens of a sequence behind one another, from row `most` - count on
    row = s["pos"] - s["lengths"].long()[s["seq"]] + most
    q = torch.zeros(b, most, h, group, d, device=DEVICE)
    q[s["seq"], row] = s["q"].float().view(-1, h, group, d)
    u = q.permute(0, 2, 3, 1, 4).reshape(b, h, group * most, d) @ whole(s["k_codes"], s["k_scale"]).squeeze(2).transpose(-1, -2)
    u = (u / math.sqrt(d)).view(b, h, group, most, keys)
    if case["softcap"]:
        u = case["softcap"] * torch.tanh(u / case["softcap"])
    j = torch.arange(keys, device=DEVICE)
    length = s["lengths"].long()[:, None]
    p = length - most + torch.arange(most, device=DEVICE)
    if case["slopes"]:
        u = u + s["slopes"].view(1, h, group, 1, 1) * (j - p[..., None])[:, None, None].float()
    limit = length.expand(b, most)
    if case["causal"]:
        limit = torch.minimum(length, torch.clamp(p + 1, min=0 if s["prefix"] is None else case["prefix"]))
    seen = (j < limit[..., None])[:, None, None]
    u = torch.where(seen, u, torch.full((), -torch.inf, device=DEVICE))
    largest = u.amax(-1, keepdim=True)
    e = torch.exp(u - torch.where(largest == -torch.inf, torch.zeros_like(largest), largest))
    del u
    total = e.sum(-1, keepdim=True)
    o = e.view(b, h, group * most, keys) @ whole(s["v_codes"], s["v_scale"]).squeeze(2)
    o = o.view(b, h, group, most, d) / torch.where(total == 0, torch.ones_like(total), total)
    return o.permute(0, 3, 1, 2, 4)[s["seq"], row].reshape(-1, case["heads"], d).to(s["q"].dtype)


def run(state):
    s, case = state, state["case"]
    if own:
        if case["op"] == "linear":
            return s["L"].packed_linear(s["x"], s["codes"], s["scale"], s["zero"], qmin=s["qmin"], bits=4, adapters=s.get("adapters"), adapter_index=s.get("index"))
        if case["op"] == "append":
            s["C"].append_packed(s["cache"], s["k"], s["v"], s["table"], s["lengths"], s["offsets"])
            return s["C"].read_packed(s["cache"], s["table"], s["lengths"], s["offsets"], tokens=s["tokens"], dtype=s["k"].dtype)
        return s["C"].attend_packed(s["q"], s["cache"], s["table"], s["lengths"], s["offsets"], causal=case["causal"], softcap=case["softcap"], slopes=s["slopes"], prefix=s["prefix"])
    return {"linear": _plain_linear, "append": _plain_append, "attend": _plain_attend}[case["op"]](s)


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    low, high = (lambda c: (c % 16).double()), (lambda c: torch.div(c, 16, rounding_mode="floor").double())
    if case["op"] == "linear":
        if 2.0 * case["m"] * case["n"] * case["tokens"] > 2e12:
            return None
        x, codes = s["x"].double(), s["codes"]
        groups = s["scale"].shape[1]
        width = case["n"] // groups
        y = torch.zeros(case["tokens"], case["m"], dtype=torch.float64, device=DEVICE)
        for first in range(0, case["m"], 2048):  # even columns sit in the lower halves of the bytes
            rows = slice(first, min(case["m"], first + 2048))
            scale = s["scale"].double()[rows].repeat_interleave(width // 2, 1)
            shift = s["qmin"] - s["zero"].double().expand(case["m"], groups)[rows].repeat_interleave(width // 2, 1)
            y[:, rows] = x[:, 0::2] @ (scale * (low(codes[rows]) + shift)).t() + x[:, 1::2] @ (scale * (high(codes[rows]) + shift)).t()
        if case["adapters"]:
            for a in range(case["adapters"]):
                mine = torch.nonzero(s["index"] == a).flatten()
                y[mine] += s["scaling"][a].double() * (x[mine] @ s["down"][a].double().t() @ s["up"][a].double().t())
        return y
    if case["op"] == "append":
        out = []
        for v in (s["k"].double(), s["v"].double()):
            scale = (v.abs().amax(-1, keepdim=True) / 7.5).float().half().double()
            scale[scale == 0] = 1.0
            out.append(torch.clamp(torch.round(v / scale), -8, 7) * scale)
        return tuple(out)
    d, group = case["head_dim"], case["heads"] // case["kv_heads"]
    out, at = torch.zeros(s["tokens"], case["heads"], d, dtype=torch.float64, device=DEVICE), 0
    for b, (length, queries) in enumerate(_sequences(case)):
        pages = s["table"][b].long()
        k, v = (torch.stack((low(s[n + "_codes"][pages]) - 8, high(s[n + "_codes"][pages]) - 8), -1).flatten(-2) * s[n + "_scale"][pages].double()[..., None] for n in ("k", "v"))
        for head in range(case["heads"] if queries and length else 0):
            keys, values = (t[:, head // group].reshape(-1, d)[:length] for t in (k, v))
            u = s["q"][at:at + queries, head].double() @ keys.t() * d ** -0.5
            if case["softcap"]:
                u = case["softcap"] * torch.tanh(u / case["softcap"])
            place, j = torch.arange(length - queries, length, device=DEVICE)[:, None], torch.arange(length, device=DEVICE)[None]
            if case["slopes"]:
                u = u + float(s["slopes"][head]) * (j - place)
            if case["causal"]:
                u = u.masked_fill((j > place) & (j >= case["prefix"]), -math.inf)
            out[at:at + queries, head] = torch.softmax(u, -1) @ values
        at += queries
    return out
