"""Measured cases of the operators that run a quantized language model with what its encodings say:
the product with packed 4-bit weights, the key/value cache held in 8 bits, and attention over it.

* ``linear``: ``y = x . w^T + bias`` with ``w = (code + offset) * scale``, 4-bit codes, one scale per
  output channel and block of input channels (symmetric, asymmetric, or the blockwise grid whose scales
  are integer multiples of a per-channel scale).
* ``append``: keys and values of new tokens written into a paged cache of 8-bit codes with one scale per
  block of tokens and head, followed by reading the touched blocks back as values.
* ``attention``: softmax attention of the newest tokens over such a cache, grouped heads, ragged lengths.

``run`` computes them in plain tensor operations in 32 bits, or, where ``own`` is true, through
``aimet_b200``.
"""

import math

import numpy as np
import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
LEVELS = 127.0  # codes of the cache lie in [-127, 127]
GROWTH = 1.25   # a block's scale that has to grow while the block fills grows by this at least


# ------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------
def _linear(name, tokens, n, k, block, grid, dtype, bias=False):
    return {"name": name, "op": "linear", "tokens": tokens, "n": n, "k": k, "block": block, "grid": grid, "dtype": dtype,
            "bias": bias}


def _append(name, seqs, new, context, heads, dim, page, dtype):
    return {"name": name, "op": "append", "seqs": seqs, "new": new, "context": context, "heads": heads, "dim": dim,
            "page": page, "dtype": dtype}


def _attention(name, seqs, context, heads, group, dim, page, query, dtype, window=0):
    return {"name": name, "op": "attention", "seqs": seqs, "context": context, "heads": heads, "group": group, "dim": dim,
            "page": page, "query": query, "dtype": dtype, "window": window}


def listed():
    return [
        # one token through a square projection: the smallest call of a decode step, latency counts
        _linear("linear one token 4096x4096", 1, 4096, 4096, 128, "sym", "bfloat16"),
        # one token through the wide projection of a feed-forward layer, the blockwise grid that
        # GroupedBlockQuantizeDequantize calibrates
        _linear("linear one token 14336x4096 lpbq", 1, 14336, 4096, 64, "lpbq", "bfloat16"),
        # a few sequences decoded together, a layer whose sizes fit no tile, asymmetric grid, bias
        _linear("linear ragged few tokens", 5, 1000, 2080, 32, "asym", "float16", True),
        # a float32 model, per-channel scales
        _linear("linear float32 per channel", 3, 2048, 4096, 0, "sym", "float32"),
        # a prompt through the wide projection
        _linear("linear prompt 14336x4096", 1500, 14336, 4096, 128, "asym", "bfloat16", True),
        # one decode step of a batch: one new token for every sequence
        _append("append one token each", 64, 1, 2000, 8, 128, 64, "bfloat16"),
        # prompts of ragged lengths enter the cache
        _append("append prompts", 4, 2000, 500, 8, 128, 32, "float16"),
        # a single conversation, short context: latency
        _attention("attention one short sequence", 1, 500, 8, 4, 128, 16, 1, "bfloat16"),
        # a decode step of a batch with ragged contexts
        _attention("attention batch", 64, 4000, 8, 4, 128, 64, 1, "bfloat16"),
        # two very long contexts: few rows, the work lies along the cache
        _attention("attention long contexts", 2, 131072, 8, 8, 128, 128, 1, "bfloat16"),
        # several proposed tokens checked at once, sliding window, odd group
        _attention("attention proposed tokens", 16, 8000, 4, 7, 64, 32, 5, "float16", 1500),
        # float32 queries, head size that is no power of two
        _attention("attention float32", 3, 3001, 2, 3, 80, 16, 2, "float32"),
    ]


def _spread(rng, low, high):
    """An integer of [low, high], spread over the logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["linear", "linear", "append", "attention", "attention"])
    if op == "linear":
        dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
        grid = rng.choice(["sym", "asym", "lpbq"])
        block = rng.choice([16, 32, 64, 128, 256] if grid == "lpbq" else [0, 16, 32, 64, 128, 256])
        tokens = rng.choice([1, _spread(rng, 1, 16), _spread(rng, 1, 64 if dtype == "float32" else 2048)])
        n, k = _spread(rng, 200, 14336), _spread(rng, 128, 14336)
        if block:
            k = max(block, k // block * block)
        while tokens * n * k > 1500 * 14336 * 4096:
            n = n // 2 + 1
        return _linear("drawn", tokens, n, k, block, grid, dtype, rng.random() < 0.5)
    heads, dim = rng.choice([1, 2, 4, 8]), rng.choice([64, 80, 96, 128, 256])
    page = rng.choice([16, 32, 64, 128])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    if op == "append":
        seqs, new = _spread(rng, 1, 128), rng.choice([1, _spread(rng, 1, 4096)])
        while seqs * new * heads * dim > 4 * 2000 * 8 * 128:
            new = new // 2 + 1 if new > 1 else new
            seqs = seqs // 2 + 1 if new == 1 or new * heads * dim > 4 * 2000 * 8 * 128 // 2 else seqs
        return _append("drawn", seqs, new, _spread(rng, 1, 4000), heads, dim, page, dtype)
    seqs, context, query = _spread(rng, 1, 64), _spread(rng, 1, 131072), rng.choice([1, 1, rng.randint(2, 16)])
    group = rng.choice([1, 2, 3, 4, 5, 6, 7, 8, 16])
    most = 2 * 131072 * 8 * 128
    while seqs * context * heads * dim * max(1.0, query * group / 8) > most:
        if seqs > 4 and rng.random() < 0.5:
            seqs = seqs // 2
        else:
            context = context // 2 + 1
    window = rng.choice([0, 0, _spread(rng, 16, 4096)])
    return _attention("drawn", seqs, context, heads, group, dim, page, query, dtype, window)


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def _lengths(case, seed):
    """(new tokens, tokens in the cache) of every sequence, on the host.  append: tokens in the cache
    before the call; attention: including the newest ones.  Of four sequences or more one is idle."""
    r = np.random.RandomState(seed % (2**31 - 1) + 17)
    seqs = case["seqs"]
    most = case["new"] if case["op"] == "append" else case["query"]
    new = r.randint(max(1, most // 3), most + 1, seqs)
    new[0] = most
    context = r.randint(case["context"] // 4, case["context"] + 1, seqs)
    context[-1] = case["context"]
    if seqs >= 4:
        new[seqs // 2] = 0
        context[seqs // 2] = 0
    return new, context


def _touched(case):
    """The most blocks that the new tokens of a sequence can lie in."""
    return (case["new"] + case["page"] - 2) // case["page"] + 1


def _tables(blocks, width, rng):
    """A block table with the pages in no order, -1 behind a sequence's last block, and the number of
    pages: room for `width` blocks of every sequence and a few more (the last one is never in the table)."""
    pages = len(blocks) * width + 3
    order = rng.permutation(pages - 1)
    table = np.full((len(blocks), width), -1, np.int32)
    at = 0
    for s, b in enumerate(blocks):
        table[s, :b] = order[at:at + b]
        at += b
    return table, pages


def _cache(pages, heads, page, dim, g):
    """Codes and scales of a cache in use: every block's largest code is the largest level, channels
    differ in size."""
    dev = "cuda"
    codes, scales = [], []
    for _ in range(2):
        channel = torch.empty(heads, 1, dim, device=dev).uniform_(0.3, 1.7, generator=g)
        c = torch.empty(pages, heads, page, dim, dtype=torch.int8, device=dev)
        s = torch.empty(pages, heads, device=dev)
        step = max(1, (1 << 26) // (heads * page * dim))
        starts = range(0, pages, step)
        for lo in starts:
            x = torch.randn(min(step, pages - lo), heads, page, dim, device=dev, generator=g) * channel
            top = x.abs().amax((2, 3))
            s[lo:lo + step] = top / LEVELS
            c[lo:lo + step] = torch.round(x / (top / LEVELS)[..., None, None]).clamp(-LEVELS, LEVELS).to(torch.int8)
        codes.append(c)
        scales.append(s)
    return codes[0], codes[1], scales[0], scales[1]


def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(int(seed))
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "linear":
        return _prepare_linear(case, g, dtype)
    new, context = _lengths(case, int(seed))
    rng = np.random.RandomState(int(seed) % (2**31 - 1) + 5)
    page, heads, dim = case["page"], case["heads"], case["dim"]
    appends = case["op"] == "append"
    held, most = (context + new, case["context"] + case["new"]) if appends else (context, case["context"])
    table, pages = _tables(-(-held // page), -(-most // page), rng)
    key, value, key_scale, value_scale = _cache(pages, heads, page, dim, g)
    state = {"op": case["op"], "key": key, "value": value, "key_scale": key_scale, "value_scale": value_scale,
             "table": torch.from_numpy(table).to(dev), "context": torch.from_numpy(context.astype(np.int32)).to(dev),
             "new": torch.from_numpy(new.astype(np.int32)).to(dev), "dtype": dtype, "page": page}
    if case["op"] == "append":
        first = context // page
        touched = np.where(new > 0, (context + new - 1) // page - first + 1, 0)
        tail = np.full((case["seqs"], _touched(case)), -1, np.int32)
        for s, b in enumerate(touched):
            tail[s, :b] = table[s, first[s]:first[s] + b]
        state["tail"] = torch.from_numpy(tail).to(dev)
        state["tail_len"] = torch.from_numpy(np.where(new > 0, context % page + new, 0).astype(np.int32)).to(dev)
        # keys and values as a fused projection leaves them: one row per token, keys and values side by side
        both = torch.randn(case["seqs"], case["new"], 2, heads, dim, device=dev, generator=g) * 1.1
        both = both.to(dtype)
        state["new_key"], state["new_value"] = both[:, :, 0], both[:, :, 1]
    else:
        q = torch.randn(case["seqs"], case["query"], heads * case["group"], dim, device=dev, generator=g) * 1.3
        state |= {"query": q.to(dtype), "window": case["window"], "scale": dim ** -0.5}
    if own:  # the handle that a program keeps beside its buffers
        from aimet_b200.kv_cache import Int8KVCache

        state["cache"] = Int8KVCache.from_buffers(key, value, key_scale, value_scale)
    return state


def _prepare_linear(case, g, dtype):
    dev, n, k = "cuda", case["n"], case["k"]
    block = case["block"] or k
    groups = k // block
    qmin = 0 if case["grid"] == "asym" else -8
    codes = torch.round(torch.randn(n, k, device=dev, generator=g) * 2.7 - 0.5)
    offset = None
    if case["grid"] == "asym":
        offset = -torch.round(torch.empty(n, groups, device=dev).uniform_(5.0, 10.0, generator=g))
        codes = codes - torch.repeat_interleave(offset, block, 1)
    codes = codes.clamp(qmin, qmin + 15).to(torch.int8)
    scale = torch.empty(n, groups, device=dev).uniform_(0.4, 1.6, generator=g) * (0.37 / math.sqrt(k))
    state = {"op": "linear", "codes": codes, "block": block, "qmin": qmin, "offset": offset, "int_scale": None, "dtype": dtype}
    if case["grid"] == "lpbq":
        state["int_scale"] = torch.randint(1, 17, (n, groups), device=dev, generator=g).to(torch.uint8)
        scale = scale[:, :1].contiguous() / 16
    state["scale"] = scale
    x = torch.randn(case["tokens"], k, device=dev, generator=g)
    x = x * torch.where(torch.rand(k, device=dev, generator=g) < 0.01, 8.0, 1.0)  # a few large channels
    state["x"] = x.to(dtype)
    state["bias"] = torch.randn(n, device=dev, generator=g).mul(0.5).to(dtype) if case["bias"] else None
    if own:  # the weights as a program lays them out once
        from aimet_b200.int4 import PackedInt4Weight

        state["packed"] = PackedInt4Weight.from_codes(codes, scale, offset, qmin=qmin, int_scale=state["int_scale"])
    return state


# ------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------
def run(state):
    if state["op"] == "linear":
        if own:
            from aimet_b200.int4 import linear_int4

            return linear_int4(state["x"], state["packed"], state["bias"])
        return _plain_linear(state)
    if state["op"] == "append":
        if own:
            cache = state["cache"]
            cache.append(state["new_key"], state["new_value"], state["table"], state["context"], state["new"])
            key, value = cache.gather(state["tail"], state["tail_len"], dtype=state["dtype"])
        else:
            key, value = _plain_append(state)
        return {"key": key, "value": value, "key_scale": state["key_scale"], "value_scale": state["value_scale"]}
    if own:
        return state["cache"].attention(state["query"], state["table"], state["context"], state["new"],
                                        window=state["window"] or None, scale=state["scale"])
    return _plain_attention(state)


def _plain_linear(state):
    scale = state["scale"]
    if state["int_scale"] is not None:
        scale = scale * state["int_scale"].float()
    w = state["codes"].float()
    if state["offset"] is not None:
        w = w + torch.repeat_interleave(state["offset"], state["block"], 1)
    w = w * torch.repeat_interleave(scale, state["block"], 1)
    y = torch.matmul(state["x"].float(), w.t())
    if state["bias"] is not None:
        y = y + state["bias"].float()
    return y.to(state["dtype"])


def _plain_append(state):
    page, context, new = state["page"], state["context"].long(), state["new"].long()
    tail = state["tail"].long()
    seqs, blocks = tail.shape
    kept = context % page  # rows of the first touched block that hold tokens already
    source = torch.arange(blocks * page, device=tail.device)[None] - kept[:, None]
    fresh = (source >= 0) & (source < new[:, None])  # rows that a new token goes to
    source = source.clamp(0, state["new_key"].shape[1] - 1)
    spare = state["key"].shape[0] - 1
    pages = torch.where(tail < 0, spare, tail)
    seq = torch.arange(seqs, device=tail.device)[:, None]
    partly = torch.zeros_like(tail, dtype=torch.bool)
    partly[:, 0] = kept > 0
    out = []
    for x, codes, scales in ((state["new_key"], state["key"], state["key_scale"]),
                             (state["new_value"], state["value"], state["value_scale"])):
        heads, dim = x.shape[2], x.shape[3]
        x = x[seq, source].float().view(seqs, blocks, page, heads, dim).transpose(2, 3)  # [seq, block, head, row, dim]
        put = fresh.view(seqs, blocks, 1, page, 1)
        before, old = codes[pages], scales[pages]
        held = torch.where(partly[..., None], old, torch.zeros_like(old))
        need = (x.abs() * put).amax((3, 4)) / LEVELS
        grown = torch.where(partly[..., None], torch.maximum(need, held * GROWTH), need)
        scale = torch.where(partly[..., None] & (need <= held), held, grown)
        ratio = torch.where(scale > 0, held / scale, torch.ones_like(scale))[..., None, None]
        shrunk = torch.where(partly[..., None, None, None], torch.round(before.float() * ratio), before.float())
        wide = scale[..., None, None]
        quantized = torch.where(wide > 0, torch.round(x / wide).clamp(-LEVELS, LEVELS), torch.zeros_like(x))
        after = torch.where(put, quantized, shrunk)
        there = tail >= 0
        codes[pages] = torch.where(there[..., None, None, None], after, before.float()).to(torch.int8)
        scales[pages] = torch.where(there[..., None], scale, old)
        rows = torch.arange(blocks * page, device=tail.device)[None] < state["tail_len"].long()[:, None]
        values = (after * wide).transpose(2, 3).reshape(seqs, blocks * page, heads, dim)
        out.append(torch.where(rows[..., None, None], values, torch.zeros_like(values)).to(state["dtype"]))
    return out


def _plain_attention(state):
    query, page = state["query"], state["page"]
    seqs, most, all_heads, dim = query.shape
    heads = state["key"].shape[1]
    group = all_heads // heads
    pages = state["table"].long().clamp(min=0)
    length = pages.shape[1] * page

    def values(codes, scales):
        x = codes[pages].float() * scales[pages][..., None, None]
        return x.permute(0, 2, 1, 3, 4).reshape(seqs, heads, length, dim)

    context, new = state["context"].long(), state["new"].long()
    q = query.float().view(seqs, most, heads, group, dim).permute(0, 2, 3, 1, 4).reshape(seqs, heads, group * most, dim)
    score = torch.matmul(q, values(state["key"], state["key_scale"]).transpose(2, 3)) * state["scale"]
    token = torch.arange(most, device=query.device)[None]
    position = context[:, None] - new[:, None] + token  # of every query in its sequence
    at = torch.arange(length, device=query.device)
    sees = (at[None, None] <= position[..., None]) & (token < new[:, None])[..., None]
    if state["window"]:
        sees = sees & (at[None, None] > position[..., None] - state["window"])
    score = score.view(seqs, heads, group, most, length).masked_fill(~sees[:, None, None], float("-inf"))
    top = score.amax(-1, keepdim=True)
    weight = torch.exp(score - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = weight.sum(-1, keepdim=True)
    out = torch.matmul(weight.view(seqs, heads, group * most, length), values(state["value"], state["value_scale"]))
    out = out.view(seqs, heads, group, most, dim) / torch.where(total > 0, total, torch.ones_like(total))
    return out.permute(0, 3, 1, 2, 4).reshape(seqs, most, all_heads, dim).to(state["dtype"])


# ------------------------------------------------------------------------------------------------
# bytes and operations; results in 64 bits
# ------------------------------------------------------------------------------------------------
def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "linear":
        tokens, n, k = case["tokens"], case["n"], case["k"]
        groups = k // (case["block"] or k)
        scales = n * groups * 4 if case["grid"] != "lpbq" else n * groups + n * 4
        zeros = n * groups if case["grid"] == "asym" else 0
        return {"bytes": n * -(-k // 2) + scales + zeros + size * (tokens * k + tokens * n + (n if case["bias"] else 0)),
                "flops": 2 * tokens * n * k}
    heads, dim, page = case["heads"], case["dim"], case["page"]
    new, context = _lengths(case, 1)
    if case["op"] == "append":
        tokens = int(new.sum())
        old = int((context % page)[new > 0].sum())
        blocks = int(np.where(new > 0, (context + new - 1) // page - context // page + 1, 0).sum())
        padded = case["seqs"] * page * _touched(case)
        # new tokens read, their codes written; the touched blocks read and written as values
        return {"bytes": 2 * heads * (dim * (tokens * (size + 1) + tokens + old + padded * size) + 8 * blocks),
                "flops": 2 * heads * dim * 6 * (tokens + old)}
    rows = case["group"]
    seen, pairs = 0, 0
    for n, c in zip(new.tolist(), context.tolist()):
        window = case["window"] or c
        first = max(0, c - n - window + 1) if n else c
        seen += c - first
        for i in range(n):
            position = c - n + i
            pairs += max(0, min(position + 1, window))
    tokens = int(new.sum())
    return {"bytes": 2 * heads * (seen * dim + 4 * -(-seen // page)) + 2 * size * heads * rows * dim * tokens,
            "flops": 4 * heads * rows * dim * pairs}


def exact(case, seed):
    with torch.no_grad():
        state = prepare(case, seed)
        return {"linear": _exact_linear, "append": _exact_append, "attention": _exact_attention}[case["op"]](state)


def _exact_linear(state):
    codes, block = state["codes"].double(), state["block"]
    n, k = codes.shape
    w = codes.view(n, k // block, block)
    if state["offset"] is not None:
        w = w + state["offset"].double()[:, :, None]
    w = w * state["scale"].double()[:, :, None]
    if state["int_scale"] is not None:
        w = w * state["int_scale"].double()[:, :, None]
    y = state["x"].double() @ w.reshape(n, k).T
    return y if state["bias"] is None else y + state["bias"].double()


def _exact_append(state):
    """Sequence by sequence and block by block; a scale is held in 32 bits, everything else in 64."""
    page = state["page"]
    new, context = state["new"].tolist(), state["context"].tolist()
    table = state["table"].tolist()
    seqs, blocks = state["tail"].shape
    found = {}
    for name in ("key", "value"):
        codes, scales, x = state[name], state[name + "_scale"].clone(), state["new_" + name]
        out = torch.zeros(seqs, blocks * page, *x.shape[2:], dtype=torch.float64, device=x.device)
        for s in range(seqs):
            start, stop = context[s], context[s] + new[s]
            first = start // page
            if new[s] == 0:
                continue
            for b in range(first, (stop - 1) // page + 1):
                p, lo, hi = table[s][b], max(start, b * page), min(stop, (b + 1) * page)
                tokens = x[s, lo - start:hi - start].double().transpose(0, 1)  # [head, row, dim]
                scale = (tokens.abs().amax((1, 2)) / LEVELS).float()
                kept = lo - b * page
                base = b * page - first * page
                if kept:
                    old = scales[p].clone()
                    scale = torch.where(scale <= old, old, torch.maximum(scale, (old.double() * GROWTH).float()))
                    ratio = torch.where(scale > 0, old.double() / scale.double(), 1.0)
                    rows = torch.round(codes[p, :, :kept].double() * ratio[:, None, None]) * scale.double()[:, None, None]
                    out[s, base:base + kept] = rows.transpose(0, 1)
                step = scale.double()[:, None, None]
                rows = torch.where(step > 0, torch.round(tokens / step).clamp(-LEVELS, LEVELS), 0.0) * step
                out[s, base + kept:base + kept + hi - lo] = rows.transpose(0, 1)
                scales[p] = scale
        found[name], found[name + "_scale"] = out, scales.double()
    return found


def _exact_attention(state):
    query, page, window = state["query"], state["page"], state["window"]
    heads = state["key"].shape[1]
    seqs, most, all_heads, dim = query.shape
    group = all_heads // heads
    out = torch.zeros(seqs, most, all_heads, dim, dtype=torch.float64, device=query.device)
    for s, (n, c) in enumerate(zip(state["new"].tolist(), state["context"].tolist())):
        if n == 0 or c == 0:
            continue
        pages = state["table"][s, :-(-c // page)].long()
        for h in range(heads):
            k = (state["key"][pages, h].double() * state["key_scale"][pages, h].double()[:, None, None]).reshape(-1, dim)[:c]
            v = (state["value"][pages, h].double() * state["value_scale"][pages, h].double()[:, None, None]).reshape(-1, dim)[:c]
            for i in range(n):
                stop = c - n + i + 1
                start = max(0, stop - window) if window else 0
                if stop <= start:
                    continue
                q = query[s, i, h * group:(h + 1) * group].double()
                weight = torch.softmax(q @ k[start:stop].T * state["scale"], -1)
                out[s, i, h * group:(h + 1) * group] = weight @ v[start:stop]
    return out
