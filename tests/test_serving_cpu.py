"""Host-side checks of the packed 4-bit product and the 8-bit cache that need no GPU: what the entry points
refuse before anything touches a device, and how scales are laid out."""

import ctypes

import pytest
import torch


def test_storage_blocks_and_tiled_scales():
    from aimet_b200 import int4

    assert [int4._storage_block(b, 2048) for b in (16, 32, 48, 64, 96, 128, 192, 256, 512, 2048)] == [16, 32, 16, 64, 32, 128, 64, 256, 256, 256]
    assert int4._storage_block(77, 77) == 256 and int4._storage_block(1, 1) == 256
    for bad in (8, 20, 40 + 2):
        with pytest.raises(NotImplementedError, match="multiple of 16"):
            int4._storage_block(bad, bad * 4)
    # channel i, column j finds its scale at [i // 16][j // 256][j % 256 // max(64, block)][i % 16][j % 64 // block]
    for n, k, block in ((5, 96, 32), (20, 64, 16), (17, 384, 128), (16, 96, 48), (3, 77, 77), (33, 640, 320), (2, 1024, 512), (3, 600, 600)):
        blocks = k // block
        param = torch.arange(n * blocks, dtype=torch.float32).view(n, blocks) + 1
        storage = int4._storage_block(block, k)
        tiled = int4._tiled(param, block, storage, k)
        assert tiled.is_contiguous() and tiled.shape[3] == 16
        for row in (0, n - 1):
            for j in (0, 15, 16, 63, k // 2, k - 1):
                if j < k:
                    at = (row // 16, j // 256, j % 256 // max(64, storage), row % 16, j % 64 // storage)
                    assert tiled[at] == param[row, j // block]
        if n % 16:
            assert bool((tiled[-1, :, :, n % 16:] == 0).all())


def test_entry_points_refuse_before_touching_the_device():
    from aimet_b200 import _lib

    lib, one = _lib.lib, 1 << 20  # any aligned non-NULL value: the calls below return before a pointer is used
    assert lib.aimet_b200_int4_codes_bytes(16, 256) == 2048 and lib.aimet_b200_int4_codes_bytes(17, 257) == 4 * 2048
    assert lib.aimet_b200_int4_codes_bytes(0, 64) == _lib.AB_ERR_INVALID
    assert lib.aimet_b200_int4_pack(one, 16, 64, -200, 64, one, None) == _lib.AB_ERR_INVALID and "signed bytes" in _lib.last_error()
    assert lib.aimet_b200_int4_pack(one, 16, 64, 0, 64, one + 4, None) == _lib.AB_ERR_INVALID and "aligned" in _lib.last_error()
    assert lib.aimet_b200_int4_pack(one, 16, 64, 0, 48, one, None) == _lib.AB_ERR_UNSUPPORTED
    assert lib.aimet_b200_int4_pack(None, 16, 64, 0, 64, one, None) == _lib.AB_ERR_INVALID

    def weight(**kw):
        w = _lib.Int4Weight(32, 128, 64, 0, 8, 0, one, one, None, one)
        for name, v in kw.items():
            setattr(w, name, v)
        return w

    def linear(w, x=one, y=one, ldx=128, ldy=32, tokens=2, code=_lib.AB_BF16):
        return lib.aimet_b200_int4_linear(w, x, ldx, None, y, ldy, tokens, code, None, None)

    for kw, code, text in (({"block": 48}, _lib.AB_ERR_UNSUPPORTED, "storage block"), ({"block": 96}, _lib.AB_ERR_UNSUPPORTED, "storage block"),
                           ({"scale_kind": 2}, _lib.AB_ERR_INVALID, "scale_kind"), ({"row_scale": None}, _lib.AB_ERR_INVALID, "row_scale"),
                           ({"zero": 113}, _lib.AB_ERR_INVALID, "zero point"), ({"codes": None}, _lib.AB_ERR_INVALID, "NULL"),
                           ({"codes": one + 8}, _lib.AB_ERR_INVALID, "aligned"), ({"n": 0}, _lib.AB_ERR_INVALID, "0 x 128")):
        assert linear(weight(**kw)) == code and text in _lib.last_error(), kw
    assert linear(weight(), tokens=-1) == _lib.AB_ERR_INVALID
    assert linear(weight(), ldx=127) == _lib.AB_ERR_INVALID and "ldx" in _lib.last_error()
    assert linear(weight(), ldy=31) == _lib.AB_ERR_INVALID and "ldy" in _lib.last_error()
    assert linear(weight(), code=_lib.AB_F64) == _lib.AB_ERR_UNSUPPORTED
    assert linear(weight(), x=None) == _lib.AB_ERR_INVALID
    assert linear(weight(), tokens=0, x=None, y=None) == _lib.AB_OK
    assert linear(weight(), tokens=200) == _lib.AB_ERR_INVALID and "status" in _lib.last_error()

    def cache(**kw):
        c = _lib.KVCache(one, one, one, one, 10, 2, 16, 64, 0)
        for name, v in kw.items():
            setattr(c, name, v)
        return c

    strides = (ctypes.c_int64 * 3)(128, 128, 64)

    def append(c, seqs=1, tokens=1, code=_lib.AB_BF16, table=one, width=4):
        return lib.aimet_b200_kv_append(c, one, one, strides, strides, seqs, tokens, table, width, width, one, None, code, None)

    def gather(c, out=one, code=_lib.AB_BF16):
        return lib.aimet_b200_kv_gather(c, out, out, 1, 5, one, 4, 4, one, code, None)

    def attention(c, seqs=1, tokens=1, group=1, width=4, code=_lib.AB_BF16, window=0, scratch=None, n=0):
        return lib.aimet_b200_kv_attention(c, one, strides, one, None, seqs, tokens, group, one, width, width, one, None, 1, window, 0.1,
                                           code, scratch, n, None)

    for kw in ({"page_size": 8}, {"page_size": 24}, {"page_size": 2048}, {"head_dim": 8}, {"head_dim": 72}, {"head_dim": 512}):
        for call in (append, gather, attention):
            assert call(cache(**kw)) == _lib.AB_ERR_UNSUPPORTED, (kw, call)
    for kw in ({"num_pages": 0}, {"num_pages": 2**31}, {"num_heads": 0}, {"key": None}, {"value_scale": None}, {"value": one + 8}):
        for call in (append, gather, attention):
            assert call(cache(**kw)) == _lib.AB_ERR_INVALID, (kw, call)
    for call in (append, gather, attention):
        assert call(cache(), code=_lib.AB_F64) == _lib.AB_ERR_UNSUPPORTED
    assert append(cache(), table=None) == _lib.AB_ERR_INVALID
    assert append(cache(), seqs=1 << 24, tokens=1 << 20, width=1 << 20) == _lib.AB_ERR_UNSUPPORTED and "in one call" in _lib.last_error()
    assert append(cache(), seqs=0) == _lib.AB_OK and append(cache(), tokens=0) == _lib.AB_OK
    assert gather(cache(), out=one + 8) == _lib.AB_ERR_INVALID and "aligned" in _lib.last_error()
    assert attention(cache(), window=-1) == _lib.AB_ERR_INVALID
    assert attention(cache(), group=0) == _lib.AB_ERR_INVALID
    assert attention(cache(), seqs=70000) == _lib.AB_ERR_INVALID
    assert attention(cache(), width=1 << 28) == _lib.AB_ERR_INVALID
    assert attention(cache(), tokens=1 << 20, group=8) == _lib.AB_ERR_UNSUPPORTED and "query rows" in _lib.last_error()
    assert attention(cache(), tokens=0) == _lib.AB_OK
    need = lib.aimet_b200_kv_attention_scratch_bytes(cache(), 1, 1, 4, 4096, _lib.AB_BF16)
    assert need > 0 and need % 16 == 0
    assert attention(cache(), group=4, width=4096, scratch=one, n=need - 1) == _lib.AB_ERR_SCRATCH
    assert lib.aimet_b200_kv_attention_scratch_bytes(cache(), 1, 1, 4, 1, _lib.AB_BF16) == 0


def test_extension_module_leaves_what_is_not_plain_to_python():
    """Built with the library; CPU tensors, wrong types and wrong shapes come back as None before anything runs."""
    from aimet_b200 import _lib

    calls = _lib.calls
    assert calls is not None
    w = _lib.Int4Weight(32, 128, 64, 0, 8, 0, None, None, None, None)
    status = ctypes.c_int32(0)
    where = (ctypes.addressof(w), 0, ctypes.addressof(status))
    assert calls.linear(torch.zeros(2, 128), None, *where) is None
    assert calls.linear("no tensor", None, *where) is None
    c = _lib.KVCache(None, None, None, None, 10, 2, 16, 64, 0)
    x, ints = torch.zeros(1, 1, 2, 64), torch.zeros(1, dtype=torch.int32)
    assert calls.append(x, x, ints[None], ints, None, ctypes.addressof(c), 0) is None
    assert calls.gather(ints[None], ints, -1, _lib.AB_BF16, ctypes.addressof(c), 0) is None
    assert calls.attention(x, ints[None], ints, None, True, 0, 0.1, False, ctypes.addressof(c), 0) is None
    with pytest.raises(TypeError):
        calls.linear(x)


def test_cpu_tensors_are_refused():
    from aimet_b200.int4 import PackedInt4Weight
    from aimet_b200.kv_cache import Int8KVCache

    with pytest.raises(RuntimeError, match="no CPU fallback"):
        PackedInt4Weight.from_codes(torch.zeros(4, 16), torch.ones(4, 1))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        Int8KVCache(4, 1, 16, 16, device="cpu")
    codes = torch.zeros(4, 1, 16, 16, dtype=torch.int8)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        Int8KVCache.from_buffers(codes, codes.clone(), torch.zeros(4, 1), torch.zeros(4, 1))
    with pytest.raises(NotImplementedError, match="page_size"):
        Int8KVCache.from_buffers(codes[:, :, :8].contiguous(), codes[:, :, :8].contiguous(), torch.zeros(4, 1), torch.zeros(4, 1))


def test_prompts_that_one_grid_does_not_hold_are_taken():
    """Blocks of sixteen query rows times cache heads: up to 2^20 in one call, with no scratch for so many."""
    from aimet_b200 import _lib

    for heads, group, tokens in ((8, 4, 32768), (32, 1, 32768), (8, 8, 131072), (1024, 1, 16000)):
        c = _lib.KVCache(1 << 20, 1 << 20, 1 << 20, 1 << 20, 4096, heads, 64, 128, 0)
        assert _lib.lib.aimet_b200_kv_attention_scratch_bytes(c, 1, tokens, group, 2048, _lib.AB_BF16) == 0, (heads, group, tokens)
    c = _lib.KVCache(1 << 20, 1 << 20, 1 << 20, 1 << 20, 4096, 1024, 64, 128, 0)
    assert _lib.lib.aimet_b200_kv_attention_scratch_bytes(c, 1, 16384, 1, 2048, _lib.AB_BF16) == _lib.AB_ERR_UNSUPPORTED
