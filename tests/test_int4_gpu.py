"""Products with packed 4-bit weights against the same product in 64 bits.

Tolerance, element by element, with S = sum |x| |w|: the result is rounded once to the output type (at most
eps / 2 of it); float32 sums take at most k / 16 + 32 additions in a row, each off by at most 2^-23 of S (a
tensor core may truncate); the scale's and the multiplier's own roundings are inside that count.  A weight that
is rounded to 16 bits before the product (many tokens) adds eps / 2 of S.
"""

import pytest
import torch
from torch import nn

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["native calls", "python calls"])
def calls(request, monkeypatch):
    """The extension module's calls, and the same calls made from Python."""
    from aimet_b200 import _lib, int4

    assert _lib.calls is not None
    if request.param == "python calls":
        monkeypatch.setattr(int4, "_calls", None)


def make(n, k, block, grid, seed=0, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    blocks = k // (block or k)
    qmin = 0 if grid == "asym" else -8
    codes = torch.randint(qmin, qmin + 16, (n, k), generator=g).to(torch.int8)
    scale = torch.rand(n, blocks, generator=g) * 0.1 + 0.01
    offset = -torch.randint(0, 16, (n, blocks), generator=g).float() if grid == "asym" else None
    int_scale = None
    if grid == "lpbq":
        int_scale = torch.randint(1, 17, (n, blocks), generator=g).to(torch.uint8)
        scale = scale[:, :1].contiguous()
    dev = lambda t: None if t is None else t.to(device)  # noqa: E731
    return dev(codes), dev(scale), dev(offset), qmin, dev(int_scale)


def dequantized(codes, scale, offset, int_scale):
    n, k = codes.shape
    s = scale.double() if int_scale is None else scale.double() * int_scale.double()
    block = k // s.shape[1]
    w = codes.double()
    if offset is not None:
        w = w + offset.double().repeat_interleave(block, 1)
    return w * s.repeat_interleave(block, 1)


def packed_of(codes, scale, offset, qmin, int_scale):
    from aimet_b200.int4 import PackedInt4Weight

    return PackedInt4Weight.from_codes(codes, scale, offset, qmin=qmin, int_scale=int_scale)


def assert_close(got, x, w, bias=None, weight_in_16=False):
    xd = x.double().reshape(-1, x.shape[-1])
    want = xd @ w.T
    size = xd.abs() @ w.abs().T
    if bias is not None:
        want, size = want + bias.double(), size + bias.double().abs()
    half = torch.finfo(got.dtype).eps / 2
    steps = w.shape[1] / 16 + 32
    bound = half * want.abs() + steps * 2.0**-23 * size * (1 + half)
    if weight_in_16:
        bound = bound + half * size * (1 + half)
    if got.dtype == torch.float16:
        bound = bound + 2.0**-25  # below float16's smallest normal number the step no longer shrinks
    err = (got.double().reshape(want.shape) - want).abs()
    assert bool((err <= bound).all()), f"off by {float((err / bound).max()):.3g} bounds at {int((err / bound).argmax())}"


# tokens from one to several tiles, channels and columns that fit no tile, blocks from 16 to the row
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("grid", ["sym", "asym", "lpbq"])
@pytest.mark.parametrize("tokens,n,k,block", [
    (1, 16, 64, 64), (1, 1, 16, 16), (1, 33, 128, 16), (3, 40, 96, 32), (8, 17, 320, 64), (9, 64, 640, 128), (16, 200, 1024, 256),
    (2, 100, 1040, 16), (5, 48, 144, 48), (7, 31, 480, 96), (4, 24, 1, 0), (1, 50, 77, 0), (3, 65, 1001, 0), (17, 130, 2080, 32),
])
def test_matches_the_product_in_64_bits(dtype, grid, tokens, n, k, block):
    from aimet_b200.int4 import linear_int4

    parts = make(n, k, block, grid, seed=n + k)
    codes, scale, offset, _, int_scale = parts
    g = torch.Generator().manual_seed(tokens)
    x = torch.randn(tokens, k, generator=g).to(dtype).cuda()
    bias = torch.randn(n, generator=g).to(dtype).cuda() if tokens % 2 else None
    got = linear_int4(x, packed_of(*parts), bias)
    assert got.shape == (tokens, n) and got.dtype == dtype
    assert_close(got, x, dequantized(codes, scale, offset, int_scale), bias, weight_in_16=tokens > 8 and dtype != torch.float32)


# many tokens: whole tiles and ragged ones, odd columns, every block class
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("grid,tokens,n,k,block", [
    ("sym", 64, 256, 512, 128), ("asym", 129, 300, 1024, 64), ("lpbq", 257, 130, 768, 32), ("asym", 40, 513, 272, 16),
    ("sym", 100, 128, 333, 0), ("asym", 515, 640, 4096, 128), ("lpbq", 33, 1000, 2048, 256), ("sym", 300, 72, 64, 64),
])
def test_many_tokens(calls, dtype, grid, tokens, n, k, block):
    from aimet_b200.int4 import linear_int4

    parts = make(n, k, block, grid, seed=tokens)
    codes, scale, offset, _, int_scale = parts
    x = torch.randn(tokens, k, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    bias = torch.randn(n, generator=torch.Generator().manual_seed(2)).to(dtype).cuda()
    got = linear_int4(x, packed_of(*parts), bias)
    assert_close(got, x, dequantized(codes, scale, offset, int_scale), bias, weight_in_16=dtype != torch.float32)


# more tiles than SMs, so that a CTA walks several: odd and even numbers of token tiles, a last chunk with one
# column tile and with all four, every block class
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("grid,tokens,n,k,block", [
    ("asym", 513, 6400, 576, 64), ("lpbq", 700, 6300, 320, 32), ("sym", 300, 9500, 272, 16), ("asym", 1024, 5000, 256, 128),
    ("sym", 2000, 2500, 1040, 0), ("asym", 257, 9600, 1024, 32),
])
def test_many_tiles(dtype, grid, tokens, n, k, block):
    from aimet_b200.int4 import linear_int4

    parts = make(n, k, block, grid, seed=tokens)
    codes, scale, offset, _, int_scale = parts
    x = torch.randn(tokens, k, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    bias = torch.randn(n, generator=torch.Generator().manual_seed(2)).to(dtype).cuda()
    p, w = packed_of(*parts), dequantized(codes, scale, offset, int_scale)
    one = linear_int4(x, p, bias)
    assert_close(one, x, w, bias, weight_in_16=True)
    for _ in range(10):
        assert torch.equal(one, linear_int4(x, p, bias))


@pytest.mark.parametrize("tokens", [3, 70])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides_alignment_and_leading_dims(calls, dtype, tokens):
    from aimet_b200.int4 import linear_int4

    parts = make(48, 256, 64, "asym")
    w, p = dequantized(*[parts[i] for i in (0, 1, 2, 4)]), packed_of(*parts)
    base = torch.randn(tokens, 600, device="cuda").to(dtype)
    for x in (base[:, :256], base[:, 1:257], base[:, 3:259], base.t()[:256].t().contiguous().t().contiguous().t(),
              base[:1, :256].expand(tokens, 256), base[::2, 8:264]):
        assert_close(linear_int4(x, p), x, w, weight_in_16=x.shape[0] > 8 and dtype != torch.float32)
    x = base[:2, :512].reshape(2, 2, 256)
    assert linear_int4(x, p).shape == (2, 2, 48)
    assert_close(linear_int4(x, p), x, w)
    assert linear_int4(base[0, :256], p).shape == (48,)
    assert linear_int4(base[:0, :256], p).shape == (0, 48)


def test_float32_values_over_the_whole_range():
    """A float32 activation is cut into terms; large, small and infinite values and NaN survive that."""
    from aimet_b200.int4 import linear_int4

    codes, scale, offset, qmin, _ = make(32, 64, 64, "sym")
    scale = torch.full_like(scale, 2.0**-10)
    w, p = dequantized(codes, scale, None, None), packed_of(codes, scale, None, qmin, None)
    g = torch.Generator().manual_seed(5)
    x = (torch.randn(6, 64, generator=g) * torch.tensor([1e36, 1e-30, 1.0, 1e30, 3e-20, 1e10])[:, None]).cuda()
    x[0] = x[0].clamp(-1e36, 1e36)
    assert_close(linear_int4(x, p), x, w)
    big = torch.zeros(1, 64, device="cuda")
    big[0, 3] = torch.finfo(torch.float32).max  # rounds up past bfloat16's largest value
    assert_close(linear_int4(big, p), big, w)
    for bad in (float("inf"), float("-inf"), float("nan")):
        y = x.clone()
        y[2, 5] = bad
        got, want = linear_int4(y, p), y.float() @ w.float().T
        assert torch.equal(torch.isnan(got[2]), torch.isnan(want[2])) and torch.equal(torch.isinf(got[2]), torch.isinf(want[2]))
        assert_close(got[3:], y[3:], w)


@pytest.mark.parametrize("tokens", [1, 40])
def test_rows_keep_to_themselves(tokens):
    """A row's result does not depend on what else is in the call, and two calls agree to the bit."""
    from aimet_b200.int4 import linear_int4

    parts = make(100, 512, 64, "asym")
    p = packed_of(*parts)
    x = torch.randn(tokens, 512, device="cuda").bfloat16()
    one = linear_int4(x, p)
    assert torch.equal(one, linear_int4(x, p))
    y = x.clone()
    y[-1] = float("nan")
    assert torch.equal(linear_int4(y, p)[:-1], one[:-1])


def test_calls_captured_into_graphs_and_on_other_streams(calls):
    from aimet_b200.int4 import linear_int4

    parts = make(256, 512, 64, "lpbq")
    w, p = dequantized(*[parts[i] for i in (0, 1, 2, 4)]), packed_of(*parts)
    graphs, streams = [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for i, tokens in enumerate((2, 50)):
        x = torch.randn(tokens, 512, device="cuda").half()
        linear_int4(x, p)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=streams[i]):
            y = linear_int4(x, p)
        graphs.append((graph, x, y))
    for _ in range(3):
        for _, x, _ in graphs:
            x.normal_()
        torch.cuda.synchronize()
        for i, (graph, _, _) in enumerate(graphs):
            with torch.cuda.stream(streams[i]):
                graph.replay()
        torch.cuda.synchronize()
        for _, x, y in graphs:
            assert_close(y, x, w, weight_in_16=True)


@pytest.mark.parametrize("kind", ["per_tensor", "per_channel", "blockwise", "asymmetric", "lpbq", "int3"])
def test_packs_what_the_quantizers_calibrate(kind):
    from aimet_b200.int4 import PackedInt4Weight, linear_int4
    from aimet_b200.quantizer import GroupedBlockQuantizeDequantize, QuantizeDequantize

    torch.manual_seed(0)
    weight = (torch.randn(96, 256) * torch.rand(96, 1)).cuda()
    if kind == "lpbq":
        q = GroupedBlockQuantizeDequantize((96, 4), 4, True, 8, block_size=(1, 64), block_grouping=(1, 4))
    else:
        shape, block = {"per_tensor": ((), None), "per_channel": ((96, 1), None)}.get(kind, ((96, 8), (1, 32)))
        q = QuantizeDequantize(shape, 3 if kind == "int3" else 4, kind != "asymmetric", block_size=block)
    q = q.cuda()
    with q.compute_encodings():
        q(weight)
    p = PackedInt4Weight.from_quantizer(weight, q)
    # float32 simulation rounds (code + offset) * scale once more: half a step of each weight
    x = torch.randn(4, 256, device="cuda")
    with torch.no_grad():
        w = q(weight).double()
        got = linear_int4(x, p).double()
    size = x.double().abs() @ w.abs().T
    assert bool(((got - x.double() @ w.T).abs() <= (256 / 16 + 32 + 4) * 2.0**-23 * size).all())
    assert p.nbytes < weight.numel() * 4 / 4
    if kind == "lpbq":
        assert p._desc.scale_kind == 1  # the integer factors are kept as bytes


def test_model_with_packed_weights(calls):
    """nn.precomputed(model, packed=True): same results as the simulated weights up to the sums' rounding."""
    from aimet_b200 import nn as qnn

    torch.manual_seed(0)
    model = nn.Sequential(nn.Linear(64, 96), nn.ReLU(), nn.Linear(96, 40, bias=False)).cuda().eval()
    qnn.quantize_model(model, param_bw=4, act_bw=16)
    x = torch.randn(7, 64, device="cuda")
    with torch.no_grad(), qnn.compute_encodings(model):
        model(x)
    layers = list(qnn.quantized_layers(model))
    with torch.no_grad():
        with qnn.precomputed(model):
            want = model(x)
        with qnn.precomputed(model, packed=True):
            assert all("_packed_weight" in layer.__dict__ and "_held_weight" not in layer.__dict__ for layer in layers)
            got = model(x)
        # 16-bit activation grids: a sum off by its rounding may land one step further (2^-16 of the range),
        # and the second layer multiplies such steps of its 96 inputs
        out_range = float(want.max() - want.min())
        hidden = layers[1].input_quantizers[0]
        step_in = float((hidden.get_max() - hidden.get_min()) / 65535)
        w = layers[1].param_quantizers["weight"](layers[1].layer.weight)
        bound = float(w.abs().sum(1).max()) * step_in * 2 + 2 * out_range / 65535
        assert float((got - want).abs().max()) <= bound
        assert all("_packed_weight" not in layer.__dict__ for layer in layers)
        assert torch.equal(model(x), want)
    with qnn.precomputed(model, packed=True), torch.enable_grad():  # gradients: the simulated weight is used
        y = model(x.requires_grad_(True))
        y.sum().backward()
        assert x.grad is not None and layers[0].layer.weight.grad is not None
    # an 8-bit weight is held as before
    model8 = qnn.quantize_model(nn.Sequential(nn.Linear(64, 8)).cuda(), param_bw=8)
    with torch.no_grad(), qnn.compute_encodings(model8):
        model8(x)
    with torch.no_grad(), qnn.precomputed(model8, packed=True):
        assert "_held_weight" in model8[0].__dict__ and "_packed_weight" not in model8[0].__dict__


def test_refusals(calls):
    from aimet_b200.int4 import PackedInt4Weight, linear_int4

    codes, scale, offset, qmin, _ = make(16, 64, 32, "asym")
    p = packed_of(codes, scale, offset, qmin, None)
    x = torch.randn(2, 64, device="cuda")
    with pytest.raises(RuntimeError, match="no backward pass"):
        linear_int4(x.clone().requires_grad_(True), p)
    with pytest.raises(RuntimeError, match="input features"):
        linear_int4(x[:, :32], p)
    with pytest.raises(RuntimeError, match="bias must be"):
        linear_int4(x, p, torch.zeros(17, device="cuda"))
    with pytest.raises(RuntimeError, match="bias must be"):
        linear_int4(x, p, torch.zeros(16, device="cuda", dtype=torch.half))
    with pytest.raises(NotImplementedError, match="float64"):
        linear_int4(x.double(), p)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        linear_int4(x.cpu(), p)
    with pytest.raises(RuntimeError, match="whole numbers"):
        PackedInt4Weight.from_codes(codes.float() + 0.5, scale, offset, qmin=0)
    with pytest.raises(RuntimeError, match="whole numbers"):
        PackedInt4Weight.from_codes(codes, scale, offset, qmin=1)
    with pytest.raises(RuntimeError, match="do not divide"):
        PackedInt4Weight.from_codes(codes, scale[:8], None, qmin=0)
    with pytest.raises(RuntimeError, match="do not divide"):
        PackedInt4Weight.from_codes(codes[:, :63], scale, None, qmin=0)
    with pytest.raises(NotImplementedError, match="multiple of 16"):
        PackedInt4Weight.from_codes(codes, torch.ones(16, 8, device="cuda"), None, qmin=0)
    with pytest.raises(NotImplementedError, match="whole numbers"):
        PackedInt4Weight.from_codes(codes, scale, offset + 0.5, qmin=0)
    with pytest.raises(NotImplementedError, match="112"):
        PackedInt4Weight.from_codes(codes, scale, offset - 200, qmin=0)
    with pytest.raises(RuntimeError, match="int_scale"):
        PackedInt4Weight.from_codes(codes, scale[:, :1].contiguous(), None, qmin=0, int_scale=torch.full((16, 2), 300, device="cuda"))
    with pytest.raises(RuntimeError, match="non-empty"):
        PackedInt4Weight.from_codes(codes[:0], scale[:0], None, qmin=0)


def test_a_wait_that_gave_up_is_reported_by_the_next_call(calls):
    """The status word is written here by hand: nothing makes a kernel wait."""
    from aimet_b200 import int4

    parts = make(48, 64, 64, "sym")
    p = packed_of(*parts)
    x = torch.randn(64, 64, device="cuda").half()
    want = int4.linear_int4(x, p)
    int4._status._words[torch.cuda.current_device()][1].value = 2
    with pytest.raises(RuntimeError, match="gave up waiting"):
        int4.linear_int4(x, p)
    assert torch.equal(int4.linear_int4(x, p), want)


def test_longest_rows(calls):
    """The most input features of float32, and 16-bit rows of which one token at a time fits shared memory; longer
    ones are refused."""
    from aimet_b200.int4 import MOST_FEATURES, PackedInt4Weight, linear_int4

    for dtype, k in ((torch.float32, MOST_FEATURES[torch.float32]), (torch.bfloat16, 60000), (torch.float16, MOST_FEATURES[torch.float16])):
        codes = torch.randint(-8, 8, (20, k), device="cuda", dtype=torch.int8)
        scale = torch.rand(20, 1, device="cuda") + 0.1
        p = PackedInt4Weight.from_codes(codes, scale)
        for tokens in (1, 2, 3, 40):
            x = torch.randn(tokens, k, device="cuda").to(dtype) * 0.01
            assert_close(linear_int4(x, p), x, dequantized(codes, scale, None, None), weight_in_16=tokens > 2 and dtype != torch.float32)
    p = PackedInt4Weight.from_codes(torch.zeros(16, MOST_FEATURES[torch.float16] + 1, device="cuda"), torch.ones(16, 1, device="cuda"))
    with pytest.raises(NotImplementedError, match="shared memory"):
        linear_int4(torch.zeros(1, p.in_features, device="cuda", dtype=torch.half), p)


def test_zero_points_beyond_the_grid():
    """Offsets need not lie on the grid: every whole zero point up to 112 is subtracted exactly."""
    from aimet_b200.int4 import linear_int4

    codes, scale, _, _, _ = make(32, 128, 32, "asym")
    offset = torch.randint(-112, 113, scale.shape, device="cuda").float()
    offset[0, 0], offset[1, 1] = 112.0, -112.0
    w, p = dequantized(codes, scale, offset, None), packed_of(codes, scale, offset, 0, None)
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        x = torch.randn(3, 128, device="cuda").to(dtype)
        assert_close(linear_int4(x, p), x, w)


def test_a_slow_predecessor_is_not_a_wait_that_gave_up():
    """The tensor-core kernel may become resident while its predecessor in the stream still runs; the limit of its
    waits (two seconds) counts from the predecessor's end.  The predecessor here is attention of one query over
    one page that a table names again and again, by one CTA (the other sequences hold nothing but leave no
    more than one CTA for each), for three seconds or so."""
    from aimet_b200 import _lib, int4
    from aimet_b200.kv_cache import Int8KVCache

    cache = Int8KVCache(1, 1, 1024, 16)
    seqs = 4096
    q = torch.randn(seqs, 1, 1, 16, device="cuda").half()
    blocks = (1 << 30) // 1024
    table = torch.zeros(1, blocks, dtype=torch.int32, device="cuda").expand(seqs, blocks)
    context = torch.zeros(seqs, dtype=torch.int32, device="cuda")

    def timed(tokens):
        context[0] = tokens
        torch.cuda.synchronize()
        start, stop = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        cache.attention(q, table, context)
        stop.record()
        torch.cuda.synchronize()
        return start.elapsed_time(stop)

    timed(1 << 20)
    per_token = timed(1 << 23) / (1 << 23)
    parts = make(512, 256, 64, "sym")
    p = packed_of(*parts)
    x = torch.randn(64, 256, device="cuda").half()
    want = int4.linear_int4(x, p)
    context[0] = min((1 << 30) - 1, int(3000 / per_token))
    torch.cuda.synchronize()
    assert _lib.lib.aimet_b200_kv_attention_scratch_bytes(cache._ref, seqs, 1, 1, blocks, _lib.AB_F16) == 0  # one kernel, nothing behind it
    start, stop = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    cache.attention(q, table, context)
    got = int4.linear_int4(x, p)
    stop.record()
    torch.cuda.synchronize()
    assert start.elapsed_time(stop) > 2200, "the predecessor has to take longer than the limit"
    assert torch.equal(got, want)
    assert torch.equal(int4.linear_int4(x, p), want)  # and nothing is reported


def linear_bound(x, w, bias, out_dtype, weights_in_16):
    """How far two results y = x . w^T + bias may be apart: each is rounded to its type once, sums float32 (as
    in assert_close); `weights_in_16` of the two multiply weights that are rounded to 16 bits."""
    xd = x.double()
    y, size = xd @ w.T, xd.abs() @ w.abs().T
    if bias is not None:
        y, size = y + bias.double(), size + bias.double().abs()
    half = torch.finfo(out_dtype).eps / 2
    sums = (w.shape[1] / 16 + 32) * 2.0**-23 * size
    return 2 * half * y.abs() + (2 * sums + weights_in_16 * half * size) * (1 + half) + 2.0**-24


def layers_of(dtype, seed=0, sizes=((64, 96, True), (96, 40, False)), grid="per_channel"):
    """Linear layers with calibrated 4-bit weight quantizers and no activation quantizers."""
    from aimet_b200 import nn as qnn
    from aimet_b200.quantizer import GroupedBlockQuantizeDequantize, QuantizeDequantize

    def quantizer(n, k):
        if grid == "lpbq":
            return GroupedBlockQuantizeDequantize((n, k // 32), 4, True, 8, block_size=(1, 32), block_grouping=(1, k // 32))
        shape, block = {"per_channel": ((n, 1), None), "asymmetric": ((n, 1), None), "per_tensor": ((), None)}.get(grid, ((n, k // 16), (1, 16)))
        return QuantizeDequantize(shape, 4, grid != "asymmetric", block_size=block)

    torch.manual_seed(seed)
    model = nn.Sequential(*[qnn.QuantizedLayer(nn.Linear(k, n, bias=b), None, None, quantizer(n, k)) for k, n, b in sizes])
    model = model.to("cuda", dtype).eval()
    for layer in model:
        with layer.param_quantizers["weight"].compute_encodings():
            layer.param_quantizers["weight"](layer.layer.weight)
    return model


@pytest.mark.parametrize("grid", ["per_channel", "per_tensor", "asymmetric", "blockwise", "lpbq"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_packed_codes_are_the_simulated_ones(dtype, grid):
    """What a packed weight stands for, read through a product with the unit matrix, against the simulated weight:
    apart by roundings (of the scale, the product and the read-back, half a step each), never by a code."""
    from aimet_b200.int4 import PackedInt4Weight, linear_int4

    for layer in layers_of(dtype, grid=grid, sizes=((256, 384, False), (96, 40, False))):
        quantizer, weight = layer.param_quantizers["weight"], layer.layer.weight
        with torch.no_grad():
            simulated = quantizer(weight).double()
            eye = torch.eye(weight.shape[1], device="cuda")
            packed = linear_int4(eye, PackedInt4Weight.from_quantizer(weight, quantizer)).double().T
        half = torch.finfo(dtype).eps / 2
        assert bool(((packed - simulated).abs() <= (2 * half * (1 + half) + 2.0**-22) * packed.abs()).all())
        scale = quantizer.get_encodings().scale.detach().double()
        assert float(simulated.abs().max()) > 3 * float(scale.min())  # (steps are far wider than that)


@pytest.mark.parametrize("grid", ["per_channel", "per_tensor", "asymmetric", "blockwise", "lpbq"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens", [1, 7, 40, 300])
def test_packed_weights_against_the_weights_held_otherwise(dtype, tokens, grid):
    """precomputed(packed=True) and precomputed() on the same layer, from one token to a prompt."""
    from aimet_b200 import nn as qnn

    model = layers_of(dtype, grid=grid)
    x = torch.randn(tokens, 64, device="cuda").to(dtype)
    with torch.no_grad():
        for layer in model:
            with qnn.precomputed(model):
                want, w = layer(x), layer._held_weight.double()
            with qnn.precomputed(model, packed=True):
                assert "_packed_weight" in layer.__dict__
                got = layer(x)
            assert got.dtype == want.dtype == dtype
            # the held weight is rounded to the type, its scale too where blocks have one, and many tokens round the packed one
            bound = linear_bound(x, w, layer.layer.bias, dtype, 0 if dtype == torch.float32 else 3)
            if dtype == torch.float32:  # (code + offset) * scale rounded to float32: half a step of each weight
                bound = bound + 2.0**-23 * (x.double().abs() @ w.abs().T)
            assert bool(((got.double() - want.double()).abs() <= bound).all())
            x = want


def test_a_context_that_fails_on_entry_leaves_no_frozen_weight(monkeypatch):
    """Packing, or quantizing, the second layer's weight raises: the first layer keeps nothing, and a weight that is
    edited afterwards counts."""
    from aimet_b200 import int4
    from aimet_b200 import nn as qnn
    from aimet_b200.quantizer import QuantizeDequantize

    model = layers_of(torch.float32)
    x = torch.randn(4, 64, device="cuda")
    made = int4.PackedInt4Weight.from_quantizer.__func__

    def breaks(cls, weight, quantizer):
        if weight is model[1].layer.weight:
            raise MemoryError("no room")
        return made(cls, weight, quantizer)

    with monkeypatch.context() as patch:
        patch.setattr(int4.PackedInt4Weight, "from_quantizer", classmethod(breaks))
        with pytest.raises(MemoryError), qnn.precomputed(model, packed=True):
            pass

    def quantizing(self, t):
        if t.shape == model[1].layer.weight.shape:
            raise MemoryError("no room")
        return plain(self, t)

    plain = QuantizeDequantize.forward
    for context in (qnn.precomputed, qnn.compute_encodings):
        with monkeypatch.context() as patch:
            patch.setattr(QuantizeDequantize, "forward", quantizing)
            for layer in model:
                layer.param_quantizers["weight"].allow_overwrite(False)
            with pytest.raises(MemoryError), context(model):
                pass
    for layer in model:
        assert "_packed_weight" not in layer.__dict__ and "_held_weight" not in layer.__dict__
    with torch.no_grad():
        before = model(x)
        model[0].layer.weight.data.mul_(-1)
        assert not torch.equal(before, model(x))


def test_weights_without_codes_are_held_as_they_are():
    """A weight that holds NaN, or an infinity, runs packed as it runs held."""
    from aimet_b200 import nn as qnn

    for grid in ("per_channel", "blockwise"):
        for bad in (float("nan"), float("inf")):
            model = layers_of(torch.float32, grid=grid)
            model[1].layer.weight.data[3, 5] = bad
            x = torch.randn(4, 64, device="cuda")
            with torch.no_grad():
                with qnn.precomputed(model):
                    want = model[1](model[0](x))
                with qnn.precomputed(model, packed=True):
                    assert "_packed_weight" in model[0].__dict__
                    got = model[1](model[0](x))
            assert torch.equal(torch.isnan(got), torch.isnan(want))
            assert bool(((got - want).abs().nan_to_num() <= 1e-4 * want.abs().nan_to_num().amax()).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens", [1, 7, 40])
def test_packed_weights_under_autocast(dtype, tokens):
    """Autocast decides the types of a packed layer's product as it does of the plain one: activations of any type
    it casts, a float32 bias among them."""
    from aimet_b200 import nn as qnn

    model = layers_of(torch.float32)
    layer = model[0]
    for given in (torch.float32, dtype):
        x = torch.randn(tokens, 64, device="cuda").to(given)
        with torch.no_grad(), torch.autocast("cuda", dtype=dtype):
            with qnn.precomputed(model):
                want, w = layer(x), layer._held_weight.double()
                deep = model(x)
            with qnn.precomputed(model, packed=True):
                got = layer(x)
                assert model(x).dtype == deep.dtype == dtype
        assert got.dtype == want.dtype == dtype
        bound = linear_bound(x.to(dtype), w, layer.layer.bias.to(dtype), dtype, 2)
        assert bool(((got.double() - want.double()).abs() <= bound).all())


@pytest.mark.parametrize("off", [False, True])
def test_forward_mode_derivatives_are_refused(calls, off):
    """A tangent would be lost: refused, with gradients off too; a packed layer multiplies with the simulated weight."""
    import torch.autograd.forward_ad as fwad

    from aimet_b200 import nn as qnn
    from aimet_b200.int4 import linear_int4

    parts = make(48, 64, 64, "sym")
    p = packed_of(*parts)
    x, bias = torch.randn(3, 64, device="cuda"), torch.randn(48, device="cuda")
    model = layers_of(torch.float32)
    with torch.set_grad_enabled(not off), fwad.dual_level():
        dual = fwad.make_dual(x, torch.ones_like(x))
        with pytest.raises(RuntimeError, match="forward-mode"):
            linear_int4(dual, p)
        with pytest.raises(RuntimeError, match="forward-mode"):
            linear_int4(x, p, fwad.make_dual(bias, torch.ones_like(bias)))
        assert linear_int4(x, p, bias).shape == (3, 48)
        with fwad._set_fwd_grad_enabled(False):
            assert torch.equal(linear_int4(dual, p), linear_int4(x, p))
        with torch.no_grad():
            with qnn.precomputed(model):
                want = fwad.unpack_dual(model(dual)).tangent
            with qnn.precomputed(model, packed=True):
                got = fwad.unpack_dual(model(dual)).tangent
        assert want is not None and torch.equal(got, want)


@pytest.mark.parametrize("grid", ["sym", "lpbq"])
@pytest.mark.parametrize("tokens", [1, 40])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_scales_near_the_end_of_the_range(dtype, tokens, grid):
    """Scales of 2^120 and more beside small activations: the product is a number of the type."""
    from aimet_b200.int4 import linear_int4

    codes, scale, offset, qmin, int_scale = make(40, 128, 64, grid)
    scale = scale * 2.0**126
    x = (torch.randn(tokens, 128, generator=torch.Generator().manual_seed(3)) * 2.0**-60).to(dtype).cuda()
    w = dequantized(codes, scale, offset, int_scale)
    got = linear_int4(x, packed_of(codes, scale, offset, qmin, int_scale))
    assert_close(got, x, w, weight_in_16=tokens > 8 and dtype != torch.float32)


def test_packed_codes_are_the_simulated_ones_while_gradients_are_spiked():
    """With pivot gradient spiking on, a trainable weight is simulated by division in its own type, a frozen one by
    the fake-quantize arithmetic."""
    from aimet_b200 import nn as qnn
    from aimet_b200 import pgs

    model = layers_of(torch.bfloat16, sizes=((256, 384, False),))
    x = torch.eye(256, device="cuda").bfloat16()
    pgs.enable_pgs()
    try:
        for trainable in (True, False):
            model[0].layer.weight.requires_grad_(trainable)
            with torch.no_grad():
                with qnn.precomputed(model):
                    want = model(x).double()
                with qnn.precomputed(model, packed=True):
                    got = model(x).double()
            assert bool(((got - want).abs() <= 3 * 2.0**-8 * want.abs()).all()), trainable
    finally:
        pgs.disable_pgs()


def test_packed_layers_under_vmap():
    """Tensors that torch.func wraps have no data of their own: the simulated weight is used."""
    from aimet_b200 import nn as qnn

    model = layers_of(torch.float32)
    x = torch.randn(5, 3, 64, device="cuda")
    with torch.no_grad():
        with qnn.precomputed(model):
            want = torch.func.vmap(model)(x)
        with qnn.precomputed(model, packed=True):
            got = torch.func.vmap(model)(x)
    assert torch.equal(got, want)
