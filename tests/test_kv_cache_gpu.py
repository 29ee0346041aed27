"""The 8-bit key / value cache: what append writes, what gather reads, attention over it.

append: the scale is max * float32(1 / 127) in float32, a code the nearest whole number to x / scale; the quotient is rounded
to float32 before that, which moves it by at most 127 * 2^-24, so |code - x / scale| <= 1/2 + 127 * 2^-24
(and 127 * 2^-22 where a held code is multiplied by a rounded ratio).

attention: with p the exact softmax, an output is off by at most the sum of
* its rounding to the output type, eps / 2 of it;
* sum p |v| times twice the largest error of a score (float32 products and sums over dim: (dim / 16 + 8) * 2^-23
  of sum |q| |k| * scale), the rounding of the weights (2^-11, or 2^-21 for float32 queries, which take two
  float16 terms) and 2^-17 for exponentials, logarithms of the scales and float32 sums;
* what weights below float16's normal range lose: 2^-25 of the largest p |v scale| * 127, per token.
"""

import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu

LEVELS = 127


@pytest.fixture(params=["native calls", "python calls"])
def calls(request, monkeypatch):
    """The extension module's calls, and the same calls made from Python."""
    from aimet_b200 import _lib, int4, kv_cache

    assert _lib.calls is not None
    if request.param == "python calls":
        monkeypatch.setattr(int4, "_calls", None)
        monkeypatch.setattr(kv_cache, "_calls", None)


def make_cache(pages, heads, page, dim, seed=0, spread=0.0):
    from aimet_b200.kv_cache import Int8KVCache

    g = torch.Generator().manual_seed(seed)
    shape = (pages, heads, page, dim)
    key = torch.randint(-LEVELS, LEVELS + 1, shape, generator=g).to(torch.int8)
    value = torch.randint(-LEVELS, LEVELS + 1, shape, generator=g).to(torch.int8)
    ks = (torch.rand(pages, heads, generator=g) + 0.5) / LEVELS * 1.7
    vs = (torch.rand(pages, heads, generator=g) + 0.5) / LEVELS * torch.exp(spread * torch.randn(pages, heads, generator=g))
    return Int8KVCache.from_buffers(key.cuda(), value.cuda(), ks.cuda(), vs.cuda())


def make_table(lens, page, pages, seed=0, width=None):
    """A block table with pages in random order; -7 behind each sequence's last block."""
    g = torch.Generator().manual_seed(seed)
    blocks = [-(-n // page) for n in lens]
    order = torch.randperm(pages, generator=g)
    assert sum(blocks) <= pages
    table = torch.full((len(lens), max([1, *blocks, width or 0])), -7, dtype=torch.int32)
    at = 0
    for s, b in enumerate(blocks):
        table[s, :b] = order[at:at + b].to(torch.int32)
        at += b
    return table.cuda()


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def values_of(cache, which, table, s, n):
    """[heads, n, dim] in 64 bits; rows without a page are NaN-free zeros, flagged in the second result."""
    codes, scales = getattr(cache, which), getattr(cache, which + "_scale")
    page = cache.page_size
    out = torch.zeros(cache.num_heads, n, cache.head_dim, dtype=torch.float64, device="cuda")
    there = torch.zeros(n, dtype=torch.bool, device="cuda")
    step = torch.zeros(cache.num_heads, n, dtype=torch.float64, device="cuda")
    for b in range(-(-n // page)):
        p = int(table[s, b])
        if 0 <= p < cache.num_pages:
            m = min(page, n - b * page)
            out[:, b * page:b * page + m] = codes[p, :, :m].double() * scales[p].double()[:, None, None]
            there[b * page:b * page + m] = True
            step[:, b * page:b * page + m] = scales[p].double()[:, None]
    return out, there, step


def check_attention(cache, query, table, context, new, *, causal=True, window=None, scale=None, seqs=None):
    got, lse = cache.attention(query, table, ints(context), None if new is None else ints(new), causal=causal, window=window,
                               scale=scale, return_lse=True)
    plain = cache.attention(query, table, ints(context), None if new is None else ints(new), causal=causal, window=window, scale=scale)
    assert torch.equal(got, plain)
    assert got.shape == query.shape and got.dtype == query.dtype and lse.dtype == torch.float32
    n_seqs, tokens, heads, dim = query.shape
    group = heads // cache.num_heads
    factor = dim ** -0.5 if scale is None else scale
    half = torch.finfo(query.dtype).eps / 2
    small = 2.0**-21 if query.dtype == torch.float32 else 2.0**-11
    for s in range(n_seqs) if seqs is None else seqs:
        live = tokens if new is None else new[s]
        n = min(context[s], table.shape[1] * cache.page_size)
        k, there, _ = values_of(cache, "key", table, s, n)
        v, _, step = values_of(cache, "value", table, s, n)
        at = torch.arange(n, device="cuda")
        for i in range(tokens):
            pos = context[s] - live + i
            sees = there.clone()
            if causal:
                sees &= at <= pos
            if window:
                sees &= at > pos - window
            if i >= live or not bool(sees.any()):
                assert bool((got[s, i] == 0).all()) and bool((lse[s, i] == float("-inf")).all()), (s, i)
                continue
            q = query[s, i].double().view(cache.num_heads, group, dim)
            score = (q @ k.transpose(1, 2)) * factor
            off = (q.abs() @ k.abs().transpose(1, 2) * abs(factor)).masked_fill(~sees, 0).amax(-1, keepdim=True) * (dim / 16 + 8) * 2.0**-23
            score = score.masked_fill(~sees, float("-inf"))
            p = torch.softmax(score, -1)
            want = p @ v
            bound = half * want.abs() + (p @ v.abs()) * (2 * off + small + 2.0**-17)
            bound = bound + n * 2.0**-25 * (p * step[:, None]).amax(-1, keepdim=True) * LEVELS
            if query.dtype == torch.float16:
                bound = bound + 2.0**-25
            err = (got[s, i].double().view_as(want) - want).abs()
            assert bool((err <= bound).all()), (s, i, float((err / bound).max()))
            lerr = (lse[s, i].double().view(cache.num_heads, group) - torch.logsumexp(score, -1)).abs()
            assert bool((lerr <= 2 * off[..., 0] + 2.0**-17 * (1 + torch.logsumexp(score, -1).abs())).all()), (s, i)
    return got


# ---------------------------------------------------------------------------------------------- attention
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("heads,group,dim,page", [
    (1, 1, 16, 16), (2, 4, 64, 16), (2, 3, 80, 32), (1, 7, 96, 64), (2, 8, 128, 64), (1, 16, 128, 16), (1, 5, 112, 48),
    (3, 2, 256, 32), (1, 4, 160, 128), (1, 17, 64, 16), (1, 33, 48, 16),
])
def test_single_tokens_over_ragged_contexts(dtype, heads, group, dim, page):
    context = [0, 1, 15, 16, 17, page, page + 1, 333]
    cache = make_cache(80, heads, page, dim, seed=dim)
    table = make_table(context, page, 80)
    q = torch.randn(len(context), 1, heads * group, dim, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    check_attention(cache, q, table, context, None)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("heads,group,dim,page,tokens,window,causal", [
    (2, 3, 64, 16, 5, None, True), (1, 4, 128, 32, 8, 33, True), (1, 7, 64, 16, 5, 1, True), (2, 1, 96, 16, 20, 16, True),
    (1, 6, 128, 64, 11, None, False), (1, 2, 256, 16, 9, 100, True), (1, 16, 64, 16, 16, None, True), (1, 3, 80, 16, 3, 40, False),
])
def test_several_tokens_windows_and_padding(calls, dtype, heads, group, dim, page, tokens, window, causal):
    context = [0, 2, tokens, 40, 257, 500]
    new = [0, tokens, tokens, tokens - 2, tokens, 1]  # the second has more tokens than its context
    cache = make_cache(70, heads, page, dim, seed=tokens)
    table = make_table(context, page, 70, width=50)
    q = torch.randn(6, tokens, heads * group, dim, generator=torch.Generator().manual_seed(2)).to(dtype).cuda()
    got = check_attention(cache, q, table, context, new, window=window, causal=causal)
    # what stands behind a sequence's last query is not read
    dirty = q.clone()
    for s, n in enumerate(new):
        dirty[s, n:] = float("nan")
    assert torch.equal(got, cache.attention(dirty, table, ints(context), ints(new), window=window, causal=causal))


@pytest.mark.parametrize("dtype,heads,group,dim,page,context,tokens,window", [
    (torch.bfloat16, 1, 8, 128, 64, [9000], 1, None), (torch.float32, 1, 2, 64, 16, [20011, 70], 2, None),
    (torch.float16, 2, 4, 128, 128, [5000, 3, 0, 12345], 1, None), (torch.bfloat16, 1, 20, 128, 16, [6001], 2, 2500),
    (torch.bfloat16, 1, 1, 256, 32, [8191, 8192, 8193], 1, None), (torch.float16, 1, 4, 64, 16, [16 * 129, 4097], 3, 2048),
])
def test_long_contexts_cut_into_pieces(dtype, heads, group, dim, page, context, tokens, window):
    pages = sum(-(-n // page) for n in context) + 3
    cache = make_cache(pages, heads, page, dim, seed=7)
    table = make_table(context, page, pages)
    q = torch.randn(len(context), tokens, heads * group, dim, generator=torch.Generator().manual_seed(3)).to(dtype).cuda()
    check_attention(cache, q, table, context, [min(tokens, n) for n in context], window=window)
    # a table much wider than the contexts (as a captured step has it) cuts differently
    wide = torch.full((len(context), table.shape[1] * 3), -1, dtype=torch.int32, device="cuda")
    wide[:, : table.shape[1]] = table
    check_attention(cache, q, wide, context, [min(tokens, n) for n in context], window=window)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_what_lies_in_masked_places_does_not_matter(dtype):
    """Rows behind the context, pages of nobody, and pages the table does not name: NaN and infinite scales,
    any codes."""
    context, page = [37, 5, 64], 16
    cache = make_cache(12, 2, page, 64)
    table = make_table(context, page, 12)
    q = torch.randn(3, 1, 4, 64, device="cuda").to(dtype)
    used = set(table[table >= 0].tolist())
    want = check_attention(cache, q, table, context, None)
    for p in set(range(12)) - used:
        cache.key_scale[p] = float("nan")
        cache.value_scale[p] = float("inf")
    cache.key[int(table[0, 2]), :, 5:] = -128  # tokens 37 .. 47 of the first sequence do not exist
    cache.value[int(table[0, 2]), :, 5:] = -128
    assert torch.equal(want, cache.attention(q, table, ints(context)))
    # a hole in a table: its tokens are masked, whatever page 0 holds
    holes = table.clone()
    holes[0, 1], holes[2, 0], holes[1, 0] = -1, 12, 2**31 - 1
    cache.key_scale[0], cache.value_scale[0] = float("nan"), float("inf")
    if 0 in used:
        holes[table == 0] = -5
    got = check_attention(cache, q, holes, context, None)
    assert bool((got[1] == 0).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_scales_of_very_different_size(dtype):
    """Pages whose values are large, tiny or all zero beside each other."""
    context, page = [128, 48], 16
    cache = make_cache(16, 2, page, 64, seed=4)
    table = make_table(context, page, 16)
    for i, f in enumerate((1e-20, 1e20, 1.0, 0.0, 1e-6, 1e6, 0.0, 30.0)):
        cache.value_scale[int(table[0, i])] = f / LEVELS
        cache.key_scale[int(table[0, i])] *= (1.0, 1e-3, 4.0, 0.0, 8.0, 1.0, 3.0, 2.0)[i]
    cache.value_scale[int(table[1, 0])] = 0.0
    cache.value_scale[int(table[1, 1])] = 0.0
    cache.value_scale[int(table[1, 2])] = 0.0
    q = torch.randn(2, 1, 4, 64, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    check_attention(cache, q, table, context, None)


@pytest.mark.parametrize("size", [1e-30, 1e-5, 1e4, 1e30])
def test_queries_of_any_size(size):
    cache = make_cache(4, 1, 16, 64)
    table = make_table([50], 16, 4)
    q = (torch.randn(1, 1, 4, 64, generator=torch.Generator().manual_seed(1)) * size).cuda()
    q[0, 0, 3] = 0
    for dtype in (torch.bfloat16, torch.float32):
        check_attention(cache, q.to(dtype), table, [50], None, scale=0.1 / size)


def test_query_strides_and_alignment(calls):
    cache = make_cache(8, 2, 16, 64)
    table = make_table([70, 40], 16, 8)
    for dtype in (torch.bfloat16, torch.float32):
        base = torch.randn(2, 3, 8, 200, device="cuda").to(dtype)
        heads_first = torch.randn(2, 8, 3, 64, device="cuda").to(dtype).transpose(1, 2)
        for q in (base[..., :64], base[..., 1:65], base[..., 8:72], heads_first, base[:, :1, :1, :64].expand(2, 3, 8, 64),
                  torch.randn(2, 3, 64, 8, device="cuda").to(dtype).transpose(2, 3)):
            check_attention(cache, q, table, [70, 40], None)
    wide = torch.full((2, 20), -1, dtype=torch.int32, device="cuda")
    wide[:, :10:2] = table
    q = torch.randn(2, 1, 4, 64, device="cuda")
    check_attention(cache, q, wide[:, ::2], [70, 40], None)
    check_attention(cache, q, wide.t().contiguous().t()[:, ::2], [70, 40], None)


def test_offsets_beyond_32_bits():
    """A cache of more than 2^31 bytes each for keys and values; the pages used are its last ones."""
    from aimet_b200.kv_cache import Int8KVCache

    pages, heads, page, dim = 8300, 8, 128, 256
    shape = (pages, heads, page, dim)
    cache = Int8KVCache.from_buffers(torch.empty(shape, dtype=torch.int8, device="cuda"), torch.empty(shape, dtype=torch.int8, device="cuda"),
                                     torch.zeros(shape[:2], device="cuda"), torch.zeros(shape[:2], device="cuda"))
    assert cache.key.numel() > 2**31
    table = ints([[pages - 1, pages - 3, 2]])
    x = torch.randn(1, 300, 2, heads, dim, device="cuda").bfloat16()
    cache.append(x[:, :, 0], x[:, :, 1], table, ints([0]))
    key, value = cache.gather(table, ints([300]), 300, torch.float32)
    top = torch.stack([x[0, lo:lo + 128].float().abs().amax((0, 3)) for lo in (0, 128, 256)])  # [block, kv, head]
    step = top.repeat_interleave(128, 0)[:300] / LEVELS
    assert bool(((key[0] - x[0, :, 0].float()).abs() <= step[:, 0, :, None] * 0.5001).all())
    assert bool(((value[0] - x[0, :, 1].float()).abs() <= step[:, 1, :, None] * 0.5001).all())
    q = torch.randn(1, 1, 8, dim, device="cuda").bfloat16()
    check_attention(cache, q, table, [300], None)


def test_results_do_not_depend_on_the_run_or_on_other_sequences():
    context = [3000, 17, 900]
    cache = make_cache(260, 2, 16, 128)
    table = make_table(context, 16, 260)
    q = torch.randn(3, 2, 8, 128, device="cuda").bfloat16()
    first = cache.attention(q, table, ints(context))
    for _ in range(3):
        assert torch.equal(first, cache.attention(q, table, ints(context)))


# ------------------------------------------------------------------------------------------ append, gather
def expected_append(cache, key, value, table, context, new):
    """Checks a cache in place against what append must have made of `before`: returns that check."""
    before = {n: getattr(cache, n).clone() for n in ("key", "value", "key_scale", "value_scale")}
    page = cache.page_size

    def check():
        touched = torch.zeros(cache.num_pages, page, dtype=torch.bool, device="cuda")
        scaled = torch.zeros(cache.num_pages, dtype=torch.bool, device="cuda")
        for s in range(len(context)):
            start, stop = context[s], context[s] + new[s]
            for b in range(start // page, -(-stop // page) if new[s] else 0):
                p = int(table[s, b]) if b < table.shape[1] else -1
                if not 0 <= p < cache.num_pages:
                    continue
                lo, hi = max(start, b * page), min(stop, (b + 1) * page)
                kept = lo - b * page
                touched[p, : hi - b * page] = True
                scaled[p] = True
                for name, x in (("key", key), ("value", value)):
                    t = x[s, lo - start:hi - start].double().transpose(0, 1)
                    finite = torch.where(torch.isfinite(t), t, 0.0)
                    want = finite.abs().amax((1, 2)).float() * torch.tensor(1 / LEVELS, device="cuda")
                    old = before[name + "_scale"][p]
                    if kept:
                        want = torch.where(want <= old, old, torch.maximum(want, (old.double() * 1.25).float()))
                    scale = getattr(cache, name + "_scale")[p]
                    assert torch.equal(scale, want), (name, s, b)
                    code = getattr(cache, name)[p].double()
                    step = scale.double()[:, None, None]
                    ratio = torch.where(step > 0, finite / step, 0.0).clamp(-LEVELS, LEVELS)
                    ratio = torch.where(torch.isinf(t) & (step > 0), torch.sign(t) * LEVELS, ratio)
                    got = code[:, kept:kept + hi - lo]
                    assert bool(((got - ratio).abs() <= 0.5 + 127 * 2.0**-24).all()), (name, s, b)
                    assert bool((got.abs() <= LEVELS).all())
                    if kept:
                        moved = before[name][p, :, :kept].double() * torch.where(step > 0, old.double()[:, None, None] / step, 1.0)
                        assert bool(((code[:, :kept] - moved).abs() <= 0.5 + 127 * 2.0**-22).all()), (name, s, b)
                        same = scale == old
                        assert torch.equal(getattr(cache, name)[p, same, :kept], before[name][p, same, :kept])
        for name in ("key", "value"):  # everything else is as it was
            now, was = getattr(cache, name), before[name]
            keep = ~touched[:, None, :, None].expand_as(now)
            assert torch.equal(now[keep], was[keep])
            sn, sw = getattr(cache, name + "_scale"), before[name + "_scale"]
            assert torch.equal(sn[~scaled].nan_to_num(7.0), sw[~scaled].nan_to_num(7.0))

    return check


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("heads,dim,page,context,new", [
    (1, 16, 16, [0], [1]), (2, 64, 16, [0, 5, 15, 16, 31], [1, 1, 1, 1, 1]), (2, 128, 64, [0, 63, 64, 10], [70, 2, 130, 0]),
    (1, 80, 32, [7, 0, 33], [100, 32, 31]), (3, 256, 16, [1, 14], [40, 3]), (2, 96, 128, [100, 0], [300, 128]), (1, 48, 48, [47, 48], [2, 49]),
])
def test_append(calls, dtype, heads, dim, page, context, new):
    pages = 40
    cache = make_cache(pages, heads, page, dim, seed=page)
    table = make_table([c + n for c, n in zip(context, new)], page, pages)
    g = torch.Generator().manual_seed(len(context))
    most = max(new)
    # a sequence's new tokens are larger, equal or smaller than what its block holds
    size = torch.tensor([0.3, 1.0, 2.5, 40.0, 1e-4])[: len(context)].view(-1, 1, 1, 1, 1)
    x = (torch.randn(len(context), most, 2, heads, dim, generator=g) * size).to(dtype).cuda()
    key, value = x[:, :, 0], x[:, :, 1]
    for s, n in enumerate(new):
        x[s, n:] = float("nan")  # padding
    check = expected_append(cache, key, value, table, context, new)
    cache.append(key, value, table, ints(context), ints(new))
    check()
    # gather gives code * scale, zeros behind the sequence
    held = [c + n for c, n in zip(context, new)]
    for out in (torch.float32, dtype):
        k, v = cache.gather(table, ints(held), max(held) + 3, out)
        assert k.shape == (len(held), max(held) + 3, heads, dim) and k.dtype == out
        for s, n in enumerate(held):
            for got, which in ((k, "key"), (v, "value")):
                codes, scales = getattr(cache, which), getattr(cache, which + "_scale")
                pages_of = table[s, : -(-n // page)].long()
                want = (codes[pages_of].float() * scales[pages_of][..., None, None]).transpose(1, 2).reshape(-1, heads, dim)[:n].to(out)
                assert torch.equal(got[s, :n], want) and bool((got[s, n:] == 0).all())


@pytest.mark.parametrize("vec", [True, False])
def test_append_strides_and_special_values(vec):
    """Keys and values that are slices of wider rows; NaN, infinities, zeros and denormal numbers."""
    for dtype in (torch.bfloat16, torch.float32):
        cache = make_cache(10, 2, 16, 64)
        table = make_table([40, 20], 16, 10)
        wide = torch.randn(2, 20, 2, 300, device="cuda").to(dtype)
        at = 0 if vec else 3
        key, value = wide[..., at:at + 64], torch.randn(2, 2, 20, 64, device="cuda").to(dtype).transpose(1, 2)
        key[0, 3, 0, 5], key[0, 4, 1, 6], key[1, 2, 0, 0] = float("nan"), float("inf"), float("-inf")
        value[0, 12:20, 0] = 0
        value[1, :, 1] = 1e-41
        value[1, 2, 0, :] = float("inf")
        context = [12, 0]
        check = expected_append(cache, key, value, table, context, [20, 20])
        cache.append(key, value, table, ints(context))
        if dtype == torch.float32:  # 1e-41 / 127 is no float32 number: such a block may hold zeros only
            assert bool((cache.value_scale[int(table[1, 0]), 1] * 127 <= 2e-41).all())
        else:
            check()


def test_append_token_by_token_stays_within_its_bound():
    """A block filled one token at a time: every token ends within 2.5 steps of the block's scale, and within
    half a step where the scale did not grow after it; a block written at once is within half a step."""
    for seed in range(3):
        cache = make_cache(3, 2, 64, 64, seed=seed)
        table = ints([[2]])
        x = torch.randn(1, 64, 2, 2, 64, generator=torch.Generator().manual_seed(seed)).cuda()
        x *= torch.linspace(0.05, 3.0, 64, device="cuda").view(1, 64, 1, 1, 1)  # keeps growing
        for i in range(64):
            cache.append(x[:, i:i + 1, 0], x[:, i:i + 1, 1], table, ints([i]))
        key, value = cache.gather(table, ints([64]), 64, torch.float32)
        for got, want, scale in ((key, x[:, :, 0], cache.key_scale[2]), (value, x[:, :, 1], cache.value_scale[2])):
            off = ((got - want).abs() / scale[:, None]).double()
            assert float(off.max()) <= 2.5 + 1e-4
        cache.append(x[:, :, 0], x[:, :, 1], table, ints([0]))
        key, _ = cache.gather(table, ints([64]), 64, torch.float32)
        assert float(((key - x[:, :, 0]).abs() / cache.key_scale[2][:, None]).max()) <= 0.5 + 1e-4


def test_append_drops_what_has_no_page(calls):
    cache = make_cache(6, 1, 16, 32)
    table = ints([[0, -1, 2], [6, 3, 2**31 - 1]])
    x = torch.randn(2, 60, 1, 32, device="cuda")
    check = expected_append(cache, x, x, table, [0, 0], [60, 60])  # 60 tokens: behind the table's end too
    cache.append(x, x, table, ints([0, 0]))
    check()
    key, _ = cache.gather(table, ints([48, 48]), 60, torch.float32)
    assert bool((key[0, 16:32] == 0).all()) and bool((key[1, :16] == 0).all()) and bool((key[:, 48:] == 0).all())


# ---------------------------------------------------------------------------------------------- together
def test_decode_steps_of_a_layer_with_packed_weights_and_the_cache(calls):
    """Prompt, then tokens one by one: projections with packed weights, append, attention, output projection,
    against the same steps in 64 bits on what the cache holds."""
    from test_int4_gpu import assert_close, dequantized, make, packed_of

    from aimet_b200.int4 import linear_int4
    from aimet_b200.kv_cache import Int8KVCache

    heads, group, dim, hidden, page = 2, 3, 64, 256, 16
    wqkv, wout = make((group + 2) * heads * dim, hidden, 64, "lpbq", seed=1), make(hidden, heads * group * dim, 64, "asym", seed=2)
    pq, po = packed_of(*wqkv), packed_of(*wout)
    wo = dequantized(*[wout[i] for i in (0, 1, 2, 4)])
    cache = Int8KVCache(20, heads, page, dim)
    table = make_table([60, 40], page, 20)
    context = torch.zeros(2, dtype=torch.int32, device="cuda")
    dtype = torch.bfloat16
    g = torch.Generator().manual_seed(0)
    for lens in ([37, 20], [1, 1], [1, 1], [1, 1], [0, 4]):
        x = torch.randn(2, max(lens), hidden, generator=g).to(dtype).cuda() * 0.05
        new = ints(lens)
        qkv = linear_int4(x, pq).view(2, max(lens), (group + 2) * heads, dim)
        q, k, v = qkv[:, :, : group * heads], qkv[:, :, group * heads:(group + 1) * heads], qkv[:, :, (group + 1) * heads:]
        check = expected_append(cache, k, v, table, context.tolist(), lens)
        cache.append(k, v, table, context, new)
        check()
        context += new
        y = check_attention(cache, q, table, context.tolist(), lens)
        y = y.reshape(2, max(lens), -1)
        assert_close(linear_int4(y, po), y, wo, weight_in_16=y.shape[0] * y.shape[1] > 8)


def test_steps_captured_into_graphs_and_replayed_side_by_side(calls):
    """Append and attention in one graph each for two caches; both replayed at once, lengths and tokens updated
    between replays; a third cache runs eagerly meanwhile."""
    caches, states = [], []
    for i in range(3):
        cache = make_cache(300, 2, 16, 64, seed=i)
        context = [2000 + i, 31 * i]
        table = make_table([4000, 400], 16, 300, seed=i)
        x = torch.randn(2, 1, 3, 8, 64, device="cuda").bfloat16()
        caches.append(cache)
        states.append([table, ints(context), x])

    def step(cache, table, context, x):
        cache.append(x[:, :, 0, :2], x[:, :, 1, :2], table, context)
        return cache.attention(x[:, :, 2], table, context + 1)

    graphs, streams = [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for i in range(2):
        with torch.cuda.stream(streams[i]):
            graph = torch.cuda.CUDAGraph()
            torch.cuda.synchronize()
            with torch.cuda.graph(graph, stream=streams[i]):
                y = step(caches[i], *states[i])
        graphs.append((graph, y))
    for turn in range(3):
        for table, context, x in states:
            x.normal_()
            context += 1
        befores = [expected_append(c, s[2][:, :, 0, :2], s[2][:, :, 1, :2], s[0], s[1].tolist(), [1, 1]) for c, s in zip(caches, states)]
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i][0].replay()
        eager = step(caches[2], *states[2])
        torch.cuda.synchronize()
        for i, check in enumerate(befores):
            check()
            want = check_attention(caches[i], states[i][2][:, :, 2], states[i][0], (states[i][1] + 1).tolist(), None)
            assert torch.equal(want, graphs[i][1] if i < 2 else eager)


def test_refusals(calls):
    from aimet_b200.kv_cache import Int8KVCache

    cache = make_cache(4, 2, 16, 32)
    table, lens = ints([[0, 1]]), ints([3])
    x = torch.randn(1, 1, 2, 32, device="cuda")
    for sizes, error in (((4, 2, 8, 32), NotImplementedError), ((4, 2, 24, 32), NotImplementedError), ((4, 2, 16, 20), NotImplementedError),
                         ((4, 2, 16, 272), NotImplementedError), ((0, 2, 16, 32), RuntimeError), ((4, 0, 16, 32), RuntimeError),
                         ((4, 2, 2048, 32), NotImplementedError), ((4, 2000, 16, 32), NotImplementedError)):
        with pytest.raises(error):
            Int8KVCache(*sizes)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        Int8KVCache(4, 2, 16, 32, device="cpu")
    with pytest.raises(RuntimeError, match="contiguous"):
        Int8KVCache.from_buffers(cache.key.transpose(2, 3).contiguous().transpose(2, 3), cache.value, cache.key_scale, cache.value_scale)
    with pytest.raises(RuntimeError, match="key_scale"):
        Int8KVCache.from_buffers(cache.key, cache.value, cache.key_scale.half(), cache.value_scale)
    with pytest.raises(RuntimeError, match="no backward pass"):
        cache.append(x.clone().requires_grad_(True), x, table, lens)
    with pytest.raises(RuntimeError, match="no backward pass"):
        cache.attention(x.clone().requires_grad_(True), table, lens)
    with pytest.raises(RuntimeError, match="heads"):
        cache.append(x[:, :, :1], x[:, :, :1], table, lens)
    with pytest.raises(RuntimeError, match="value must be"):
        cache.append(x, x.half(), table, lens)
    with pytest.raises(RuntimeError, match="block_table"):
        cache.append(x, x, table.long(), lens)
    with pytest.raises(RuntimeError, match="block_table"):
        cache.attention(x, table.repeat(2, 1), lens)
    with pytest.raises(RuntimeError, match="context_lens"):
        cache.attention(x, table, lens.long())
    with pytest.raises(RuntimeError, match="context_lens"):
        cache.attention(x, table, lens.cpu())
    with pytest.raises(RuntimeError, match="multiple"):
        cache.attention(torch.randn(1, 1, 3, 32, device="cuda"), table, lens)
    with pytest.raises(RuntimeError, match="window"):
        cache.attention(x, table, lens, window=0)
    with pytest.raises(NotImplementedError, match="float64"):
        cache.attention(x.double(), table, lens)
    with pytest.raises(RuntimeError, match="shape"):
        cache.attention(x[..., :16], table, lens)
    with pytest.raises(NotImplementedError, match="int8"):
        cache.gather(table, lens, dtype=torch.int8)
    for bad in (5.0, "5"):
        with pytest.raises((TypeError, RuntimeError)):
            cache.gather(table, lens, bad)
    with pytest.raises((TypeError, RuntimeError, ctypes.ArgumentError)):
        cache.attention(x, table, lens, window=2.5)
    with pytest.raises((TypeError, ValueError)):
        cache.attention(x, table, lens, scale="big")
    # nothing to do
    empty = torch.randn(0, 1, 2, 32, device="cuda")
    cache.append(empty, empty, table[:0], lens[:0])
    assert cache.attention(empty, table[:0], lens[:0]).shape == (0, 1, 2, 32)
    assert cache.gather(table[:0], lens[:0])[0].shape == (0, 32, 2, 32)
    no_blocks = torch.empty(1, 0, dtype=torch.int32, device="cuda")
    assert bool((cache.attention(x, no_blocks, lens) == 0).all())
    assert bool((cache.gather(no_blocks, lens, 5)[0] == 0).all())
    cache.append(x, x, no_blocks, lens)


# ------------------------------------------------------------------------------------ small weights, limits
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bits", [14, 20, 24, 27])
@pytest.mark.parametrize("n", [4000, 40000])
def test_light_tails_beside_dominating_tokens(dtype, bits, n):
    """Tokens whose weights are 2^-bits of the largest ones', where the largest belong to values of zero: what is
    left is the tail's weighted sum.

    Tolerance: as for attention above, but what a weight loses below float16's normal range is 2^-40 of the
    largest p * step at most: weights are scaled by 2^15 before they are rounded, an absolute step there is 2^-24, half of it
    the rounding."""
    page, dim, group = 16, 64, 2
    pages = n // page + 3
    cache = make_cache(pages, 1, page, dim, seed=bits)
    table = make_table([n], page, pages)
    cache.value.abs_().clamp_(min=64)
    cache.value_scale.mul_(100.0)
    cache.key.zero_()
    # a dominating token at the start of four tiles of every sixteen, so that every warp meets some
    at = torch.arange(n, device="cuda")
    first = at[(at % 16 == 0) & ((at // 16) % 16 < 4)]
    where, row = table[0, first // page].long(), first % page
    cache.key[where, 0, row, 0] = LEVELS
    cache.value[where, 0, row] = 0
    cache.key_scale.fill_(1 / LEVELS)
    q = torch.zeros(1, 1, group, dim, device="cuda")
    q[..., 0] = torch.tensor([bits, bits + 0.5], device="cuda") * 0.6931471805599453
    q[..., 1] = 1.0
    q = q.to(dtype)
    got = cache.attention(q, table, ints([n]), scale=1.0)[0, 0].double()
    k, _, _ = values_of(cache, "key", table, 0, n)
    v, _, step = values_of(cache, "value", table, 0, n)
    score = q[0, 0].double() @ k[0].T
    off = (q[0, 0].double().abs() @ k[0].abs().T).amax(-1, keepdim=True) * (dim / 16 + 8) * 2.0**-23
    p = torch.softmax(score, -1)
    want = p @ v[0]
    half = torch.finfo(dtype).eps / 2
    small = 2.0**-21 if dtype == torch.float32 else 2.0**-11
    bound = half * want.abs() + (p @ v[0].abs()) * (2 * off + small + 2.0**-17) + n * 2.0**-40 * (p * step).amax(-1, keepdim=True) * LEVELS
    if dtype == torch.float16:
        bound = bound + 2.0**-25
    err = (got - want).abs()
    assert bool((err <= bound).all()), float((err / bound).max())


@pytest.mark.parametrize("scale", [0.0, -0.5, 2.0**22])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_scores_of_any_size_stay_finite(dtype, scale):
    """A softmax scale of zero or below, and scores so large that float32 steps are whole powers of two between
    them: a weighted mean of values whatever the scores."""
    cache = make_cache(30, 1, 16, 64, seed=2)
    table = make_table([400], 16, 30)
    q = torch.randn(1, 1, 4, 64, generator=torch.Generator().manual_seed(5)).to(dtype).cuda() * 3
    got, lse = cache.attention(q, table, ints([400]), scale=scale, return_lse=True)
    assert bool(torch.isfinite(got).all()) and bool(torch.isfinite(lse).all())
    if abs(scale) < 1:
        check_attention(cache, q, table, [400], None, scale=scale)
    else:  # one token is all there is
        k, _, _ = values_of(cache, "key", table, 0, 400)
        v, _, _ = values_of(cache, "value", table, 0, 400)
        assert bool((got[0, 0].double() <= v.amax() * 1.01).all())
    # all but one page of values that are zero: what is left is far below the largest score, or not
    cache.value_scale[table[0, 1:].long()] = 0.0
    assert bool(torch.isfinite(cache.attention(q, table, ints([400]), scale=scale)).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("page,width,context,tokens,window,causal", [
    (16, 6, [98, 96, 200], 5, None, True), (16, 6, [98, 110, 400], 5, 40, True), (32, 3, [97, 100, 99], 4, 7, False),
    (16, 700, [11210, 11200, 30000], 20, 300, True), (16, 700, [11205], 8, None, True),
])
def test_contexts_that_reach_behind_the_table(dtype, page, width, context, tokens, window, causal):
    """Tokens behind the table's last block have no page: masked, and positions count them all the same."""
    pages = len(context) * width + 2
    cache = make_cache(pages, 1, page, 64, seed=width)
    table = make_table([width * page] * len(context), page, pages)
    q = torch.randn(len(context), tokens, 3, 64, generator=torch.Generator().manual_seed(6)).to(dtype).cuda()
    check_attention(cache, q, table, context, None, window=window, causal=causal)
    check_attention(cache, q, table, context, [tokens - 2] * len(context), window=window, causal=causal)


@pytest.mark.parametrize("off", [False, True])
def test_forward_mode_derivatives_are_refused(calls, off):
    import torch.autograd.forward_ad as fwad

    cache = make_cache(4, 2, 16, 32)
    table, lens = ints([[0, 1]]), ints([3])
    x = torch.randn(1, 1, 2, 32, device="cuda")
    with torch.set_grad_enabled(not off), fwad.dual_level():
        dual = fwad.make_dual(x, torch.ones_like(x))
        for key, value in ((dual, x), (x, dual)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                cache.append(key, value, table, lens)
        with pytest.raises(RuntimeError, match="forward-mode"):
            cache.attention(dual, table, lens)
        cache.append(x, x, table, lens)
        assert cache.attention(x, table, lens).shape == x.shape


def test_prompts_of_many_heads():
    """More blocks of query rows times heads than one dimension of a grid holds."""
    heads, tokens, dim, page = 256, 4200, 16, 64
    cache = make_cache(70, heads, page, dim, seed=9)
    table = make_table([tokens + 7], page, 70)
    q = torch.randn(1, tokens, heads, dim, generator=torch.Generator().manual_seed(9)).cuda().bfloat16()
    got = cache.attention(q, table, ints([tokens + 7]))
    n = tokens + 7
    k, _, _ = values_of(cache, "key", table, 0, n)
    v, _, step = values_of(cache, "value", table, 0, n)
    sees = torch.arange(n, device="cuda")[None, :] <= torch.arange(7, n, device="cuda")[:, None]
    for h in (0, 1, 100, 254, 255):
        qh = q[0, :, h].double()
        score = (qh @ k[h].T) * dim**-0.5
        off = (qh.abs() @ k[h].abs().T * dim**-0.5).masked_fill(~sees, 0).amax(-1, keepdim=True) * (dim / 16 + 8) * 2.0**-23
        p = torch.softmax(score.masked_fill(~sees, float("-inf")), -1)
        want = p @ v[h]
        bound = 2.0**-8 * want.abs() + (p @ v[h].abs()) * (2 * off + 2.0**-11 + 2.0**-17)
        bound = bound + n * 2.0**-25 * (p * step[h]).amax(-1, keepdim=True) * LEVELS
        assert bool(((got[0, :, h].double() - want).abs() <= bound).all()), h


@pytest.mark.parametrize("vec", [True, False])
def test_append_special_values_of_float32(vec):
    """As above for the smaller types: NaN, infinities, blocks of zeros, slices that start off 16 bytes."""
    cache = make_cache(10, 2, 16, 64)
    table = make_table([40, 20], 16, 10)
    at = 0 if vec else 3
    key = torch.randn(2, 20, 2, 300, device="cuda")[..., at:at + 64]
    value = torch.randn(2, 2, 20, 64, device="cuda").transpose(1, 2)
    key[0, 3, 0, 5], key[0, 4, 1, 6], key[1, 2, 0, 0] = float("nan"), float("inf"), float("-inf")
    value[0, 12:20, 0] = 0
    value[1, :, 1] = 1e-30
    value[1, 2, 0, :] = float("inf")
    check = expected_append(cache, key, value, table, [12, 0], [20, 20])
    cache.append(key, value, table, ints([12, 0]))
    check()
