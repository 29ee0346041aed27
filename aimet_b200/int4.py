"""Products with 4-bit weights: inference on what the 4-bit weight quantizers calibrate.

:class:`PackedInt4Weight` holds the codes of a ``[out_features, in_features]`` weight in four bits with
their scales (per channel, blockwise along the input channels, or the blockwise grid of
``GroupedBlockQuantizeDequantize`` whose scales are small integers times a per-channel scale), and
:func:`linear_int4` multiplies with it without ever writing the weight out in 16 bits.  The grids and
their names follow aimet_torch (quantization/affine/quantizer.py:1072-1440, affine/encoding.py:560-620);
the reference itself only simulates them.
"""

from __future__ import annotations

import ctypes
import math
from typing import Optional

import torch

from . import _lib, backend
from ._lib import check, lib

__all__ = ["PackedInt4Weight", "linear_int4"]

_TILE_N, _TILE_K, _CHUNK_K = 16, 64, 256
# input features of the longest row that the kernels take
MOST_FEATURES = {torch.float32: 37120, torch.float16: 111360, torch.bfloat16: 111360}
_MOST_PLANS = 512  # input layouts that a weight remembers
_MAX_ZERO = 112  # 16-bit floats subtract zero points up to here exactly


def _storage_block(block: int, in_features: int) -> int:
    """Input channels per scale as the kernels store them: the largest of 16, 32, 64, 128 and 256 that
    divides ``block`` (a scale for the whole row is stored for every 256)."""
    if block == in_features:
        return _CHUNK_K
    for b in (256, 128, 64, 32, 16):
        if block % b == 0:
            return b
    raise NotImplementedError(f"blocks of {block} input channels: a multiple of 16, or the whole row, is supported")


def _tiled(param: torch.Tensor, block: int, storage: int, in_features: int) -> torch.Tensor:
    """[out, blocks] -> the kernels' order [ceil(out / 16)][chunk of 256 columns][entry][16][sub] (zeros
    behind the matrix)."""
    n = param.shape[0]
    chunks, sub = -(-in_features // _CHUNK_K), max(1, _TILE_K // storage)
    entries = _CHUNK_K // max(_TILE_K, storage)
    if block == in_features:
        param = param.expand(n, chunks)
    elif storage != block:
        param = param.repeat_interleave(block // storage, 1)
    out = param.new_zeros(-(-n // _TILE_N) * _TILE_N, chunks * entries * sub)
    out[:n, : param.shape[1]] = param
    return out.view(-1, _TILE_N, chunks, entries, sub).permute(0, 2, 3, 1, 4).contiguous()


_calls = _lib.calls
_current_device = torch._C._cuda_getDevice  # pylint: disable=protected-access
_current_stream = torch._C._cuda_getCurrentRawStream  # pylint: disable=protected-access


class _Status:
    """The word that a kernel's bounded waits write when they give up, per device, in pinned host memory:
    looked at by the next call without waiting for the device."""

    def __init__(self):
        self._words: dict[int, tuple[torch.Tensor, ctypes.c_int32]] = {}

    def address(self, index: int) -> int:
        if index not in self._words:
            word = torch.zeros(1, dtype=torch.int32, pin_memory=True)
            self._words[index] = (word, ctypes.c_int32.from_address(word.data_ptr()))
        return self._words[index][0].data_ptr()

    def checked(self, index: int) -> int:
        word, value = self._words[index]
        if value.value:
            code, value.value = value.value, 0
            raise RuntimeError(f"aimet_b200: an earlier linear_int4 call on cuda:{index} gave up waiting (device status {code}); "
                               "its output is not valid")
        return word.data_ptr()


_status = _Status()


def _simulated_codes(weight: torch.Tensor, encoding) -> torch.Tensor:
    """The codes whose values ``quantize_dequantize`` gives for a weight when no gradient is wanted.  That is what
    ``quantize`` gives, except where the fake-quantize arithmetic runs (per tensor and per channel): there the
    weight is multiplied by 1 / scale in float32 whatever its type, while ``quantize`` divides in the weight's
    type, and quotients near the middle of two codes (in bfloat16 one of sixty) fall differently."""
    scale, offset, qmin, qmax, block = encoding.scale, encoding.offset, encoding.qmin, encoding.qmax, encoding.block_size
    if not backend._takes_fake_quantize_path(weight, scale, offset, block, 0.0, qmin, qmax):  # pylint: disable=protected-access
        return backend.quantize(weight, scale, offset, qmin, qmax, block)
    # (code + offset) * scale in float32, |code + offset| <= 15: the quotient is off by 2^-20 at most
    value = backend.quantize_dequantize(weight.to(torch.float32), scale, offset, qmin, qmax, block)
    return torch.round(value / scale) - offset


class PackedInt4Weight:
    """4-bit codes of a linear layer's weight with their scales, laid out for the CUDA kernels.

    Made by :meth:`from_codes`, :meth:`from_encoding` or :meth:`from_quantizer`; its contents are fixed.
    ``w[n, k] = (code[n, k] + offset[n, b]) * scale[n, b]`` with ``b`` the block of column ``k``.
    """

    def __init__(self, out_features, in_features, block_size, qmin, codes, scales, multiples, zeros, row_scale, zero):
        self.out_features, self.in_features = out_features, in_features
        self.block_size, self.qmin = block_size, qmin
        self._buffers = (codes, scales, zeros, row_scale)  # what the descriptor below points at
        storage = _storage_block(block_size, in_features)
        self._desc = _lib.Int4Weight(out_features, in_features, storage, int(multiples), zero, 0,
                                     codes.data_ptr(), scales.data_ptr(), _lib.ptr(zeros), row_scale.data_ptr())
        self.device = codes.device
        self._ref = ctypes.byref(self._desc)
        self._index = codes.get_device()
        self._address = ctypes.addressof(self._desc)
        self._status = _status.address(self._index)  # made now: a first product may be inside a stream capture, where it could not be
        self._bias_shape = torch.Size((out_features,))
        self._plans: dict = {}  # layout of an input -> what follows from it

    @property
    def nbytes(self) -> int:
        """Bytes on the device."""
        return sum(t.numel() * t.element_size() for t in self._buffers if t is not None)

    def __deepcopy__(self, memo):
        return self  # its contents are fixed

    def __repr__(self):
        return (f"PackedInt4Weight({self.out_features}x{self.in_features}, block_size={self.block_size}, "
                f"device={self.device})")

    @classmethod
    def from_codes(cls, codes: torch.Tensor, scale: torch.Tensor, offset: Optional[torch.Tensor] = None, *,
                   qmin: int = -8, int_scale: Optional[torch.Tensor] = None) -> "PackedInt4Weight":
        """From codes ``[out_features, in_features]`` (whole numbers in ``[qmin, qmin + 15]``, any dtype).

        ``scale``: ``[out_features, blocks]`` (``blocks == 1``: per channel); ``offset``: the same shape,
        whole numbers, or None for zeros.  With ``int_scale`` (``[out_features, blocks]``, whole numbers in
        ``[0, 255]``) the scale of a block is ``int_scale * scale`` and ``scale`` is ``[out_features, 1]``.
        Checks the values, which waits for the device: pack a weight once, not per forward.
        """
        if codes.dim() != 2 or codes.numel() == 0:
            raise RuntimeError(f"codes must be a non-empty matrix, got shape {tuple(codes.shape)}")
        if not codes.is_cuda:
            raise RuntimeError("aimet_b200 operates on CUDA tensors only; there is no CPU fallback")
        n, k = codes.shape
        qmin = int(qmin)
        if not -128 <= qmin <= 112:
            raise RuntimeError(f"codes of [{qmin}, {qmin + 15}] do not fit signed bytes")
        per_block = scale if int_scale is None else int_scale
        if per_block.dim() != 2 or per_block.shape[0] != n or per_block.shape[1] < 1 or k % per_block.shape[1]:
            raise RuntimeError(f"scales of shape {tuple(per_block.shape)} do not divide a weight of shape {(n, k)}")
        if int_scale is not None and tuple(scale.shape) != (n, 1):
            raise RuntimeError(f"with int_scale, scale must have shape {(n, 1)}, got {tuple(scale.shape)}")
        if offset is not None and tuple(offset.shape) != tuple(per_block.shape):
            raise RuntimeError(f"offset must have shape {tuple(per_block.shape)}, got {tuple(offset.shape)}")
        for t in (scale, offset, int_scale):
            if t is not None and t.device != codes.device:
                raise RuntimeError(f"expected all tensors on {codes.device}, got {t.device}")
        with torch.no_grad():
            block = k // per_block.shape[1]
            storage = _storage_block(block, k)
            whole = codes.to(torch.int32)
            if bool(((whole != codes) | (whole < qmin) | (whole > qmin + 15)).any()):
                raise RuntimeError(f"codes must be whole numbers in [{qmin}, {qmin + 15}]")
            if int_scale is None:
                # a power of two per channel is split off, so that what many tokens multiply in 16 bits has a
                # channel's largest scale near 1 whatever the size of the weights
                scale = scale.detach().to(torch.float32)
                top = scale.abs().amax(1)
                top = torch.where(torch.isfinite(top) & (top > 0), top, torch.ones_like(top))
                row_scale = torch.ldexp(torch.ones_like(top), torch.frexp(top).exponent.clamp(-125, 127))
                scales = _tiled(scale / row_scale[:, None], block, storage, k)
            else:
                if bool(((int_scale != int_scale.to(torch.uint8)) | (int_scale < 0) | (int_scale > 255)).any()):
                    raise RuntimeError("int_scale must hold whole numbers in [0, 255]")
                scales = _tiled(int_scale.to(torch.uint8), block, storage, k)
                row_scale = scale.detach().to(torch.float32).reshape(-1).contiguous().clone()
            zeros, zero = None, -qmin
            if offset is not None:
                z = -(offset.detach().double() + qmin)
                if bool(((z != z.round()) | (z.abs() > _MAX_ZERO)).any()):
                    raise NotImplementedError(f"offsets must be whole numbers with |offset + qmin| <= {_MAX_ZERO}")
                if bool((z == z[0, 0]).all()):
                    zero = int(z[0, 0].item())
                else:
                    zeros = _tiled(z.to(torch.int8), block, storage, k)
            elif abs(zero) > _MAX_ZERO:
                raise NotImplementedError(f"qmin={qmin} without an offset: |qmin| <= {_MAX_ZERO} is supported")
            codes8 = whole.to(torch.int8).contiguous()
            packed = torch.empty(lib.aimet_b200_int4_codes_bytes(n, k), dtype=torch.uint8, device=codes.device)
            with _lib.on_device(codes.device):
                check(lib.aimet_b200_int4_pack(codes8.data_ptr(), n, k, qmin, storage, packed.data_ptr(),
                                               _lib.stream_ptr(codes.device)))
                # products request weights before they wait for what precedes them in their stream
                torch.cuda.current_stream(codes.device).synchronize()
        return cls(n, k, block, qmin, packed, scales, int_scale is not None, zeros, row_scale, zero)

    @classmethod
    def from_encoding(cls, weight: torch.Tensor, encoding) -> "PackedInt4Weight":
        """Quantize ``weight`` ``[out_features, in_features]`` with a 4-bit ``AffineEncoding`` (per tensor, per
        output channel, or blockwise along the input channels) and pack the codes: the ones that
        ``quantize_dequantize`` simulates when no gradient is wanted.  What 4 bits cannot hold (a wider grid, a
        scale per input channel, NaN) raises ``NotImplementedError``."""
        if weight.dim() != 2:
            raise NotImplementedError(f"weights of linear layers are packed, got shape {tuple(weight.shape)}")
        if encoding.qmax - encoding.qmin > 15:
            raise NotImplementedError(f"a grid of [{encoding.qmin}, {encoding.qmax}] does not fit 4 bits")
        if not -128 <= encoding.qmin <= 112:
            raise NotImplementedError(f"codes of [{encoding.qmin}, {encoding.qmax}] do not fit signed bytes")
        if encoding.zero_point_shift:
            raise NotImplementedError("a grid with a zero-point shift cannot be packed")
        n, k = weight.shape
        scale, offset = encoding.scale, encoding.offset
        with torch.no_grad():
            if scale.dim() > 2:
                raise NotImplementedError(f"scales of shape {tuple(scale.shape)} for a linear layer's weight")
            codes = _simulated_codes(weight, encoding)
            if not bool(torch.isfinite(codes).all()):
                raise NotImplementedError("a weight or scale that is not a number has no codes")

            def per_channel(p):  # [out or 1, blocks] -> [out, blocks]
                p = p.detach().to(torch.float32).reshape((1,) * (2 - p.dim()) + tuple(p.shape))
                if encoding.block_size is None and p.shape[1] != 1:
                    raise NotImplementedError(f"a scale per input channel (shape {tuple(p.shape)}) cannot be packed")
                return p.repeat_interleave(n // p.shape[0], 0)

            int_scale = None
            shared = getattr(encoding, "per_channel_scale", None)
            if shared is not None and tuple(shared.shape) == (n, 1) and 2 ** (encoding.decompressed_bw - encoding.bitwidth) <= 255:
                int_scale = encoding.per_block_int_scale
                if not torch.equal(int_scale * shared, scale):  # keep exactly the scales that are simulated
                    int_scale = None
            if int_scale is not None:
                return cls.from_codes(codes, shared, per_channel(offset), qmin=encoding.qmin, int_scale=int_scale)
            return cls.from_codes(codes, per_channel(scale), per_channel(offset), qmin=encoding.qmin)

    @classmethod
    def from_quantizer(cls, weight: torch.Tensor, quantizer) -> "PackedInt4Weight":
        """Pack ``weight`` on the grid of a calibrated 4-bit weight quantizer."""
        encoding = quantizer.get_encodings()
        if encoding is None:
            raise RuntimeError("the quantizer has no encodings yet: calibrate it before packing its weight")
        return cls.from_encoding(weight, encoding)


def linear_int4(input: torch.Tensor, weight: PackedInt4Weight, bias: Optional[torch.Tensor] = None) -> torch.Tensor:  # pylint: disable=redefined-builtin
    """``input @ w.T + bias`` for a packed weight: ``[..., in_features] -> [..., out_features]``.

    float32, float16 or bfloat16 activations; sums in float32, one rounding to ``input.dtype``.  A few
    tokens, and float32 always, multiply the integer codes exactly; many tokens multiply weights that are
    rounded to the 16-bit type once, as a simulated 16-bit model's are.  Which of the two runs depends on the
    number of tokens and input features (from 17 tokens on the second; with long rows from three on, where
    they start on 16 bytes).  Rows of up to 37120 input features in
    float32 and 111360 in 16 bits.  For inference: an input or bias that needs a gradient, or carries a
    forward-mode derivative, is refused (train through the quantizer instead).
    """
    if _calls is not None:
        out = _calls.linear(input, bias, weight._address, weight._index, weight._status)  # pylint: disable=protected-access
        if out is not None:
            return out
    signature = (input.shape, input.stride(), input.dtype, input.get_device())
    plan = weight._plans.get(signature)  # pylint: disable=protected-access
    if plan is None:
        plan = _plan_linear(signature, input, weight)
    if torch.is_grad_enabled() and (input.requires_grad or (bias is not None and bias.requires_grad)):
        raise RuntimeError("linear_int4 has no backward pass: call it under torch.no_grad(), or train through the weight's quantizer")
    if _lib.has_tangent(input, bias):
        raise RuntimeError("linear_int4 has no forward-mode derivative: train through the weight's quantizer")
    code, tokens, pitch, out_shape, direct, watched = plan
    if bias is not None:
        if bias.dtype != input.dtype or bias.get_device() != input.get_device() or bias.shape != weight._bias_shape:  # pylint: disable=protected-access
            raise RuntimeError(f"bias must be {input.dtype} of shape {(weight.out_features,)} on {input.device}, "
                               f"got {bias.dtype} of shape {tuple(bias.shape)} on {bias.device}")
        if not bias.is_contiguous():
            bias = bias.contiguous()
    out = input.new_empty(out_shape)
    if tokens == 0:
        return out
    if not direct:
        input = input.reshape(tokens, weight.in_features).contiguous()
    if tokens > 16 and watched and (input.data_ptr() % 16 or pitch % 8):  # the tensor-core kernel wants rows that start on 16 bytes
        pitch = -(-weight.in_features // 8) * 8
        rows = input.reshape(tokens, weight.in_features)
        input = rows.new_empty(tokens, pitch)[:, : weight.in_features].copy_(rows)
    index = weight._index  # pylint: disable=protected-access
    if _current_device() != index:
        with torch.cuda.device(index):
            return linear_int4(input.reshape(out_shape[:-1] + (weight.in_features,)), weight, bias)
    rc = lib.aimet_b200_int4_linear(weight._ref, input.data_ptr(), pitch, None if bias is None else bias.data_ptr(), out.data_ptr(),  # pylint: disable=protected-access
                                    weight.out_features, tokens, code, _status.checked(index) if watched else None,
                                    _current_stream(index))
    if rc:
        check(rc)
    return out


def _plan_linear(signature, x: torch.Tensor, weight: PackedInt4Weight):
    """Checks an input and says how it is read: dtype code, tokens, elements between rows, output shape, whether it
    can be read where it is, whether the library may choose its tensor-core kernel."""
    if not x.is_cuda:
        raise RuntimeError("aimet_b200 operates on CUDA tensors only; there is no CPU fallback")
    code = _lib.DTYPE_CODE.get(x.dtype)
    if code is None or code == _lib.AB_F64:
        raise NotImplementedError(f"linear_int4 takes float32, float16 or bfloat16 activations, got {x.dtype}")
    k = weight.in_features
    if x.dim() == 0 or x.shape[-1] != k:
        raise RuntimeError(f"expected {k} input features, got an input of shape {tuple(x.shape)}")
    if x.device != weight.device:
        raise RuntimeError(f"input is on {x.device}, the weight on {weight.device}")
    tokens = math.prod(x.shape[:-1])
    pitch, direct = k, True
    if tokens:
        # rows at one distance from each other, elements side by side, no overlap
        direct = x.stride(-1) == 1 or k == 1
        outer = [(n, st) for n, st in zip(x.shape[:-1], x.stride()[:-1]) if n > 1]
        if outer:
            pitch = outer[-1][1]
            direct = direct and pitch >= k and all(a[1] == b[0] * b[1] for a, b in zip(outer, outer[1:]))
        if not direct:
            pitch = k
    plan = (code, tokens, pitch, x.shape[:-1] + (weight.out_features,), direct, tokens > 2 and code != _lib.AB_F32)
    if len(weight._plans) >= _MOST_PLANS:  # pylint: disable=protected-access
        weight._plans.clear()  # pylint: disable=protected-access
    weight._plans[signature] = plan  # pylint: disable=protected-access
    return plan
