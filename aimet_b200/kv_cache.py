"""A paged key / value cache held in 8 bits, and attention over it.

:class:`Int8KVCache` keeps the keys and values of a decoder layer as signed 8-bit codes on a symmetric
grid, one scale per page (a block of tokens) and head.  :meth:`Int8KVCache.append` quantizes new tokens
into it, :meth:`Int8KVCache.attention` attends over it reading one byte per element, and
:meth:`Int8KVCache.gather` reads tokens back as values.  Token ``j`` of a sequence lies in row
``j % page_size`` of page ``block_table[sequence, j // page_size]``; which pages belong to whom is the
caller's, lengths and tables stay on the device, nothing waits for the host, so a decode step can be
captured into a CUDA graph.  Inference only: inputs that need a gradient, or carry a forward-mode
derivative, are refused.
"""

from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import check, lib

__all__ = ["Int8KVCache"]

_Strides = ctypes.c_int64 * 3
_MOST_PLANS = 512  # checked argument layouts that a cache remembers


_calls = _lib.calls
_current_device = torch._C._cuda_getDevice  # pylint: disable=protected-access
_current_stream = torch._C._cuda_getCurrentRawStream  # pylint: disable=protected-access


class Int8KVCache:
    """``num_pages`` pages of ``page_size`` tokens for ``num_heads`` key / value heads of ``head_dim``.

    ``key``, ``value``: int8 ``[num_pages, num_heads, page_size, head_dim]``, codes in [-127, 127];
    ``key_scale``, ``value_scale``: float32 ``[num_pages, num_heads]``, not negative; a code stands for
    ``code * scale``.
    ``page_size`` is a multiple of 16 up to 1024, ``head_dim`` a multiple of 16 up to 256.
    """

    def __init__(self, num_pages: int, num_heads: int, page_size: int, head_dim: int, device="cuda"):
        device = torch.device(device)
        if device.type != "cuda":
            raise RuntimeError("aimet_b200 operates on CUDA tensors only; there is no CPU fallback")
        self._check_sizes(num_pages, num_heads, page_size, head_dim)
        shape = (num_pages, num_heads, page_size, head_dim)
        self._adopt(torch.zeros(shape, dtype=torch.int8, device=device), torch.zeros(shape, dtype=torch.int8, device=device),
                    torch.zeros(shape[:2], device=device), torch.zeros(shape[:2], device=device))

    @classmethod
    def from_buffers(cls, key: torch.Tensor, value: torch.Tensor, key_scale: torch.Tensor,
                     value_scale: torch.Tensor) -> "Int8KVCache":
        """A cache over four existing buffers that share no memory (used in place; shapes and dtypes as in the class)."""
        if key.dim() != 4:
            raise RuntimeError(f"key must be [num_pages, num_heads, page_size, head_dim], got shape {tuple(key.shape)}")
        for name, t, dtype, shape in (("key", key, torch.int8, key.shape), ("value", value, torch.int8, key.shape),
                                      ("key_scale", key_scale, torch.float32, key.shape[:2]),
                                      ("value_scale", value_scale, torch.float32, key.shape[:2])):
            if t.dtype != dtype or t.shape != shape or t.device != key.device:
                raise RuntimeError(f"{name} must be {dtype} of shape {tuple(shape)} on {key.device}, got {t.dtype} of shape "
                                   f"{tuple(t.shape)} on {t.device}")
            if not t.is_contiguous():
                raise RuntimeError(f"{name} must be contiguous")
        cls._check_sizes(*key.shape)
        if not key.is_cuda:
            raise RuntimeError("aimet_b200 operates on CUDA tensors only; there is no CPU fallback")
        if key.data_ptr() % 16 or value.data_ptr() % 16:
            raise RuntimeError("key and value must be 16-byte aligned")
        cache = cls.__new__(cls)
        cache._adopt(key, value, key_scale, value_scale)
        return cache

    @staticmethod
    def _check_sizes(num_pages, num_heads, page_size, head_dim):
        if num_pages < 1 or num_heads < 1:
            raise RuntimeError(f"a cache needs pages and heads, got num_pages={num_pages}, num_heads={num_heads}")
        if num_heads > 1024:
            raise NotImplementedError(f"num_heads={num_heads}: up to 1024 are supported")
        if page_size < 16 or page_size % 16 or page_size > 1024:
            raise NotImplementedError(f"page_size={page_size}: a multiple of 16 up to 1024 is supported")
        if head_dim < 16 or head_dim % 16 or head_dim > 256:
            raise NotImplementedError(f"head_dim={head_dim}: a multiple of 16 up to 256 is supported")

    def _adopt(self, key, value, key_scale, value_scale):
        self._buffers = (key, value, key_scale, value_scale)  # what the descriptor below points at
        self.num_pages, self.num_heads, self.page_size, self.head_dim = key.shape
        self.device = key.device
        self._desc = _lib.KVCache(key.data_ptr(), value.data_ptr(), key_scale.data_ptr(), value_scale.data_ptr(),
                                  self.num_pages, self.num_heads, self.page_size, self.head_dim, 0)
        self._ref = ctypes.byref(self._desc)
        self._address = ctypes.addressof(self._desc)
        self._scale = self.head_dim ** -0.5
        self._index = self.device.index if self.device.index is not None else torch.cuda.current_device()
        self._plans: dict = {}  # signature of a call's arguments -> what follows from it

    def _remember(self, signature, plan):
        if len(self._plans) >= _MOST_PLANS:
            self._plans.clear()
        self._plans[signature] = plan
        return plan

    key = property(lambda self: self._buffers[0])
    value = property(lambda self: self._buffers[1])
    key_scale = property(lambda self: self._buffers[2])
    value_scale = property(lambda self: self._buffers[3])

    def __repr__(self):
        return (f"Int8KVCache(num_pages={self.num_pages}, num_heads={self.num_heads}, page_size={self.page_size}, "
                f"head_dim={self.head_dim}, device={self.device})")

    # ---- argument checks: once per layout of the arguments -----------------------------------
    def _check_tokens(self, t: torch.Tensor, name: str) -> int:
        """Checks a [sequences, tokens, heads, head_dim] input; returns its dtype code."""
        if not t.is_cuda:
            raise RuntimeError("aimet_b200 operates on CUDA tensors only; there is no CPU fallback")
        code = _lib.DTYPE_CODE.get(t.dtype)
        if code is None or code == _lib.AB_F64:
            raise NotImplementedError(f"{name} must be float32, float16 or bfloat16, got {t.dtype}")
        if t.dim() != 4 or t.shape[3] != self.head_dim:
            raise RuntimeError(f"{name} must be [sequences, tokens, heads, {self.head_dim}], got shape {tuple(t.shape)}")
        if t.device != self.device:
            raise RuntimeError(f"{name} is on {t.device}, the cache on {self.device}")
        return code

    def _check_table(self, table: torch.Tensor, seqs: int) -> None:
        if table.dtype != torch.int32 or table.dim() != 2 or table.shape[0] != seqs or table.device != self.device:
            raise RuntimeError(f"block_table must be int32 of shape ({seqs}, blocks) on {self.device}, got {table.dtype} of shape "
                               f"{tuple(table.shape)} on {table.device}")

    def _check_lens(self, lens: Optional[torch.Tensor], seqs: int, name: str) -> None:
        if lens is not None and (lens.dtype != torch.int32 or lens.dim() != 1 or lens.shape[0] != seqs or lens.device != self.device):
            raise RuntimeError(f"{name} must be int32 of shape ({seqs},) on {self.device}, got {lens.dtype} of shape "
                               f"{tuple(lens.shape)} on {lens.device}")

    @staticmethod
    def _dense(table, *lens):
        """Block table and lengths as the kernels read them: table entries side by side, lengths contiguous."""
        if table.shape[1] > 1 and table.stride(1) != 1:
            table = table.contiguous()
        return table, *(t if t is None or t.is_contiguous() else t.contiguous() for t in lens)

    # ---- operators -------------------------------------------------------------------------
    def append(self, key: torch.Tensor, value: torch.Tensor, block_table: torch.Tensor, context_lens: torch.Tensor,
               new_lens: Optional[torch.Tensor] = None) -> None:
        """Quantize new tokens into the cache.

        ``key``, ``value``: ``[sequences, tokens, num_heads, head_dim]`` of one dtype, any strides;
        ``context_lens``: int32 tokens that every sequence holds already; ``new_lens``: int32 tokens of
        ``key`` / ``value`` that are real (default: all).  Token ``i`` becomes position ``context_lens + i``.

        A block's scale is the largest magnitude of its tokens over 127.  While a partly filled block
        takes in larger tokens its scale grows, by a quarter at least, and the codes it holds are rounded to
        the new grid: a token ends within 2.5 steps of its value, within half a step if its block was
        written at once.  NaN is stored as zero; infinities as the block's largest level, scales being taken
        from finite values.  Tokens whose table entry is outside ``[0, num_pages)``, or lies behind the
        table's end, are dropped.  Within a call no page may receive tokens of two sequences, or of two blocks
        of one.
        """
        if _calls is not None and _calls.append(key, value, block_table, context_lens, new_lens, self._address, self._index):
            return
        # what the checks of the arguments depend on (nothing of their values or addresses)
        signature = (key.shape, key.stride(), key.dtype, key.get_device(), value.shape, value.stride(), value.dtype, value.get_device(),
                     block_table.shape, block_table.stride(), block_table.dtype, block_table.get_device(), context_lens.shape,
                     context_lens.stride(), context_lens.dtype, context_lens.get_device(),
                     new_lens if new_lens is None else (new_lens.shape, new_lens.stride(), new_lens.dtype, new_lens.get_device()))
        plan = self._plans.get(signature) or self._plan_append(signature, key, value, block_table, context_lens, new_lens)
        if torch.is_grad_enabled() and (key.requires_grad or value.requires_grad):
            raise RuntimeError("append has no backward pass: call it under torch.no_grad()")
        if _lib.has_tangent(key, value):
            raise RuntimeError("append has no forward-mode derivative")
        code, key_strides, value_strides, dense = plan
        if not dense:
            block_table, context_lens, new_lens = self._dense(block_table, context_lens, new_lens)
            if key_strides is None:
                key, value = key.contiguous(), value.contiguous()
                key_strides = value_strides = _Strides(*key.stride()[:3])
        if _current_device() != self._index:
            with torch.cuda.device(self._index):
                return self.append(key, value, block_table, context_lens, new_lens)
        seqs, tokens = key.shape[:2]
        rc = lib.aimet_b200_kv_append(
            self._ref, key.data_ptr(), value.data_ptr(), key_strides, value_strides, seqs, tokens, block_table.data_ptr(),
            block_table.stride(0), block_table.shape[1], context_lens.data_ptr(), None if new_lens is None else new_lens.data_ptr(), code,
            _current_stream(self._index))
        if rc:
            check(rc)

    def _plan_append(self, signature, key, value, table, context, new):
        code = self._check_tokens(key, "key")
        if value.dtype != key.dtype or value.shape != key.shape or value.device != key.device:
            raise RuntimeError(f"value must be {key.dtype} of shape {tuple(key.shape)} on {key.device}, got {value.dtype} of shape "
                               f"{tuple(value.shape)} on {value.device}")
        if key.shape[2] != self.num_heads:
            raise RuntimeError(f"key has {key.shape[2]} heads, the cache {self.num_heads}")
        self._check_table(table, key.shape[0])
        self._check_lens(context, key.shape[0], "context_lens")
        self._check_lens(new, key.shape[0], "new_lens")
        rows = key.stride(3) == 1 and value.stride(3) == 1
        same = self._dense(table, context, new)
        dense = rows and same[0] is table and same[1] is context and same[2] is new
        strides = (_Strides(*key.stride()[:3]), _Strides(*value.stride()[:3])) if rows else (None, None)
        return self._remember(signature, (code, *strides, dense))

    def gather(self, block_table: torch.Tensor, lens: torch.Tensor, length: Optional[int] = None,
               dtype: torch.dtype = torch.bfloat16) -> Tuple[torch.Tensor, torch.Tensor]:
        """Keys and values ``[sequences, length, num_heads, head_dim]`` of the first ``lens`` (int32) tokens
        of every sequence, zeros behind; ``length`` defaults to all that the table can hold."""
        code = _lib.DTYPE_CODE.get(dtype, _lib.AB_F64)
        if _calls is not None and code != _lib.AB_F64 and (length is None or length >= 0):
            out = _calls.gather(block_table, lens, -1 if length is None else length, code, self._address, self._index)
            if out is not None:
                return out
        signature = (block_table.shape, block_table.stride(), block_table.dtype, block_table.get_device(), lens.shape, lens.stride(),
                     lens.dtype, lens.get_device(), length, dtype)
        code, shape = self._plans.get(signature) or self._plan_gather(signature, block_table, lens, length, dtype)
        block_table, lens = self._dense(block_table, lens)
        if _current_device() != self._index:
            with torch.cuda.device(self._index):
                return self.gather(block_table, lens, length, dtype)
        key = lens.new_empty(shape, dtype=dtype)
        value = torch.empty_like(key)
        rc = lib.aimet_b200_kv_gather(self._ref, key.data_ptr(), value.data_ptr(), shape[0], shape[1], block_table.data_ptr(),
                                      block_table.stride(0), block_table.shape[1], lens.data_ptr(), code, _current_stream(self._index))
        if rc:
            check(rc)
        return key, value

    def _plan_gather(self, signature, table, lens, length, dtype):
        code = _lib.DTYPE_CODE.get(dtype)
        if code is None or code == _lib.AB_F64:
            raise NotImplementedError(f"gather gives float32, float16 or bfloat16, not {dtype}")
        seqs = table.shape[0] if table.dim() == 2 else -1
        self._check_table(table, seqs)
        self._check_lens(lens, seqs, "lens")
        if length is None:
            length = table.shape[1] * self.page_size
        if length < 0:
            raise RuntimeError(f"length={length} is negative")
        return self._remember(signature, (code, (seqs, length, self.num_heads, self.head_dim)))

    def attention(self, query: torch.Tensor, block_table: torch.Tensor, context_lens: torch.Tensor,
                  query_lens: Optional[torch.Tensor] = None, *, causal: bool = True, window: Optional[int] = None,
                  scale: Optional[float] = None, return_lse: bool = False):
        """Softmax attention of every sequence's newest tokens over its tokens in the cache.

        ``query``: ``[sequences, tokens, heads, head_dim]``, any strides, ``heads`` a multiple of the
        cache's (consecutive query heads share a cache head); ``context_lens``: int32 tokens in the cache,
        the newest included (append first); ``query_lens``: int32 tokens of ``query`` that are real
        (default: all).  Query ``i`` stands at position ``context_lens - query_lens + i`` and sees positions
        up to its own (``causal``) and after its own minus ``window``, as far as they have a page (positions behind
        the table's end have none); ``scale`` defaults to
        ``head_dim ** -0.5``.  Scores, softmax and sums are float32; float32 queries keep 22 bits.  A token's weight
        is rounded to 11 bits before it multiplies its value (float32 queries: 22), and by at most 2^-40 of the
        largest product of a weight and its value's scale.

        Returns ``[sequences, tokens, heads, head_dim]`` in ``query.dtype``; queries that see nothing, and
        those behind ``query_lens``, give zeros.  With ``return_lse`` also the logarithm of each query's
        softmax sum, float32 ``[sequences, tokens, heads]`` (-inf where it sees nothing), by which results
        over parts of a context can be joined.  In one call up to 65535 sequences, and fewer than 2^20 sixteens of
        query rows (tokens times query heads for each of the cache's) over all of the cache's heads.
        """
        scale = self._scale if scale is None else float(scale)
        if _calls is not None and (window is None or window >= 1):
            out = _calls.attention(query, block_table, context_lens, query_lens, causal, window or 0, scale, return_lse, self._address,
                                   self._index)
            if out is not None:
                return out
        signature = (query.shape, query.stride(), query.dtype, query.get_device(), block_table.shape, block_table.stride(),
                     block_table.dtype, block_table.get_device(), context_lens.shape, context_lens.stride(), context_lens.dtype,
                     context_lens.get_device(), window,
                     query_lens if query_lens is None else (query_lens.shape, query_lens.stride(), query_lens.dtype, query_lens.get_device()))
        plan = self._plans.get(signature) or self._plan_attention(signature, query, block_table, context_lens, query_lens, window)
        if torch.is_grad_enabled() and query.requires_grad:
            raise RuntimeError("attention over the cache has no backward pass: call it under torch.no_grad()")
        if _lib.has_tangent(query):
            raise RuntimeError("attention over the cache has no forward-mode derivative")
        code, strides, group, need, dense = plan
        if not dense:
            block_table, context_lens, query_lens = self._dense(block_table, context_lens, query_lens)
            if strides is None:
                query = query.contiguous()
                strides = _Strides(*query.stride()[:3])
        if _current_device() != self._index:
            with torch.cuda.device(self._index):
                return self.attention(query, block_table, context_lens, query_lens, causal=causal, window=window, scale=scale,
                                      return_lse=return_lse)
        seqs, tokens, heads = query.shape[:3]
        out = query.new_empty(query.shape)
        lse = query.new_empty((seqs, tokens, heads), dtype=torch.float32) if return_lse else None
        if need >= 0:  # there are queries
            # scratch from the caching allocator, call by call: buffers of two streams, or of two captured graphs, are
            # never shared
            part = query.new_empty(need, dtype=torch.uint8) if need else None
            rc = lib.aimet_b200_kv_attention(
                self._ref, query.data_ptr(), strides, out.data_ptr(), None if lse is None else lse.data_ptr(), seqs, tokens, group,
                block_table.data_ptr(), block_table.stride(0), block_table.shape[1], context_lens.data_ptr(),
                None if query_lens is None else query_lens.data_ptr(), causal, window or 0, scale, code,
                None if part is None else part.data_ptr(), need, _current_stream(self._index))
            if rc:
                check(rc)
        return (out, lse) if return_lse else out

    def _plan_attention(self, signature, query, table, context, new, window):
        code = self._check_tokens(query, "query")
        seqs, tokens, heads = query.shape[:3]
        if heads < 1 or heads % self.num_heads:
            raise RuntimeError(f"{heads} query heads are no multiple of the cache's {self.num_heads}")
        if window is not None and window < 1:
            raise RuntimeError(f"window={window}: at least 1, or None for no window")
        self._check_table(table, seqs)
        self._check_lens(context, seqs, "context_lens")
        self._check_lens(new, seqs, "query_lens")
        rows = query.stride(3) == 1
        same = self._dense(table, context, new)
        dense = rows and same[0] is table and same[1] is context and same[2] is new
        group, need = heads // self.num_heads, -1
        if seqs and tokens:
            with _lib.on_device(self.device):
                need = lib.aimet_b200_kv_attention_scratch_bytes(self._ref, seqs, tokens, group, table.shape[1], code)
            check(need)
        return self._remember(signature, (code, _Strides(*query.stride()[:3]) if rows else None, group, need, dense))
