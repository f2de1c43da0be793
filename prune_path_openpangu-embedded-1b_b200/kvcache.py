"""Paged key/value cache: append with the rotary embedding on the way (``ppmoe_kv_append``) and causal
attention of the newest tokens over it (``ppmoe_attend``).

A batch is ragged: ``starts [batch + 1]`` cuts the packed rows of ``q``, ``k`` and ``v`` into each
sequence's newest tokens, ``lengths [batch]`` counts each sequence's positions with these included,
``table [batch, max_pages]`` names its pages (all int32 on the cache's device).  Rows ``starts[b] + i``
stand at position ``lengths[b] - (starts[b + 1] - starts[b]) + i``; position ``p`` lies in row
``p % page_size`` of page ``table[b, p // page_size]``.  The kernels read the three tensors on the
device, so calls captured into a CUDA graph follow what is written into them.  Rows outside every
sequence (padding behind ``starts[batch]``) are not read and their outputs not written.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch
from torch.autograd import forward_ad

from . import _lib
from .rotary import _NONE, RotaryEmbedding, _enter, _has_tangent, _stream, _written

__all__ = ["PagedKVCache"]

_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}
_PAGE_SIZES = (16, 32, 64, 128, 256)


class PagedKVCache:
    """Keys and values of one layer in pages: ``k``, ``v`` ``[num_pages, kv_heads, page_size, head_dim]``.

    ``page_size`` 16, 32, 64, 128 or 256; ``head_dim`` 64 or 128; bf16 or fp16.  Which page belongs to
    which sequence is the caller's table; sequences may share pages that neither appends to.
    """

    def __init__(self, num_pages: int, page_size: int, kv_heads: int, head_dim: int, *,
                 dtype: torch.dtype = torch.bfloat16, device="cuda"):
        if num_pages < 1 or kv_heads < 1:
            raise ValueError(f"num_pages={num_pages} and kv_heads={kv_heads} must be positive")
        self._check(page_size, head_dim, dtype)
        shape = (num_pages, kv_heads, page_size, head_dim)
        self._mount(torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device))

    @classmethod
    def from_tensors(cls, k: torch.Tensor, v: torch.Tensor) -> "PagedKVCache":
        """A cache over given tensors ``[num_pages, kv_heads, page_size, head_dim]``: any strides of whole
        16 bytes with contiguous heads, so ``[num_pages, page_size, kv_heads, head_dim]`` storage goes in as
        its ``transpose(1, 2)``."""
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or k.device != v.device:
            raise ValueError(f"k {list(k.shape)} {k.dtype} on {k.device} and v {list(v.shape)} {v.dtype} on {v.device} "
                             "must be alike, [num_pages, kv_heads, page_size, head_dim]")
        cls._check(k.shape[2], k.shape[3], k.dtype)
        if k.numel() == 0:
            raise ValueError("the cache has no pages")
        if k.requires_grad or v.requires_grad:
            raise ValueError("the cache writes into its tensors: they cannot require gradients")
        if k.data_ptr() == v.data_ptr():
            raise ValueError("keys and values need memory of their own")
        for t in (k, v):
            if t.stride(3) != 1 or any(s % 8 or s == 0 for n, s in zip(t.shape[:3], t.stride()) if n > 1) or t.data_ptr() % 16:
                raise ValueError("cache tensors need contiguous heads, 16-byte alignment and strides of whole 16 bytes")
        self = cls.__new__(cls)
        self._mount(k, v)
        return self

    @staticmethod
    def _check(page_size, head_dim, dtype):
        if page_size not in _PAGE_SIZES:
            raise ValueError(f"page_size={page_size} must be one of {_PAGE_SIZES}")
        if head_dim not in (64, 128):
            raise ValueError(f"head_dim={head_dim} must be 64 or 128")
        if dtype not in _DTYPES:
            raise TypeError(f"the cache holds bf16 or fp16, got {dtype}")

    def _mount(self, k, v):
        if k.device.type != "cuda":
            raise RuntimeError("PagedKVCache runs on CUDA only; got " + str(k.device))
        self._k, self._v = k, v  # (the structure below holds their addresses)
        self.num_pages, self.kv_heads, self.page_size, self.head_dim = k.shape
        self.dtype, self.device = k.dtype, k.device
        self._status = torch.zeros(256, dtype=torch.uint8, device=k.device)

        def strides(t):  # a size of one has any stride: give it a harmless one
            return tuple(s if n > 1 else 8 for n, s in zip(t.shape[:3], t.stride()))

        self._c = _lib.KVCache(k.data_ptr(), v.data_ptr(), *strides(k), *strides(v), *k.shape[:1], self.page_size,
                               self.kv_heads, self.head_dim, _DTYPES[k.dtype], self._status.data_ptr())

    @property
    def k(self) -> torch.Tensor:
        return self._k

    @property
    def v(self) -> torch.Tensor:
        return self._v

    @property
    def _ptr(self) -> int:
        return ctypes.addressof(self._c)

    def __deepcopy__(self, memo):
        return PagedKVCache.from_tensors(self._k.clone(), self._v.clone())

    def __reduce__(self):
        return PagedKVCache.from_tensors, (self._k, self._v)

    # ------------------------------------------------------------------ checks
    def _rows(self, name, x, heads=None):
        """x and its strides, checked."""
        if x.requires_grad and torch.is_grad_enabled():
            raise RuntimeError(f"{name} requires a gradient, and the cache records none: call it under torch.no_grad()")
        if forward_ad._current_level >= 0 and _has_tangent(x):
            raise RuntimeError(f"{name} has a forward-mode tangent, and the cache records none: pass its primal")
        shape = x.shape
        if len(shape) != 3 or shape[2] != self.head_dim or (heads is not None and shape[1] != heads):
            raise ValueError(f"{name} must be [tokens, {heads or 'heads'}, {self.head_dim}], got {list(shape)}")
        if x.dtype is not self.dtype or x.device != self.device:
            raise ValueError(f"{name} must be {self.dtype} on {self.device}, got {x.dtype} on {x.device}")
        s = x.stride()
        if s[2] != 1:
            x = x.contiguous()
            s = x.stride()
        return x, s

    def _batch(self, starts, lengths, table):
        i32, dev, ts = torch.int32, self.device, table.shape
        if (starts.dtype is not i32 or lengths.dtype is not i32 or table.dtype is not i32 or starts.device != dev
                or lengths.device != dev or table.device != dev or len(ts) != 2):
            raise ValueError(f"starts, lengths and table [batch, max_pages] must be int32 on {dev}, got "
                             + ", ".join(f"{t.dtype} {list(t.shape)} on {t.device}" for t in (starts, lengths, table)))
        B, pages = ts
        if starts.shape != (B + 1,) or lengths.shape != (B,) or B < 1 or pages < 1:
            raise ValueError(f"starts {list(starts.shape)}, lengths {list(lengths.shape)} and table {list(ts)} "
                             "must be [batch + 1], [batch] and [batch, max_pages]")
        s = table.stride()
        if not starts.is_contiguous() or not lengths.is_contiguous() or (pages > 1 and s[1] != 1):
            raise ValueError("starts, lengths and the rows of table must be contiguous")
        return starts.data_ptr(), lengths.data_ptr(), table.data_ptr(), s[0], B, pages

    # ------------------------------------------------------------------ calls
    def append(self, q: Optional[torch.Tensor], k: torch.Tensor, v: torch.Tensor, starts: torch.Tensor,
               lengths: torch.Tensor, table: torch.Tensor, *, rotary: Optional[RotaryEmbedding] = None,
               out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
        """Writes the rows of ``k`` (rotated to their positions where ``rotary`` is given) and ``v``
        ``[tokens, kv_heads, head_dim]`` to their places, and returns ``q [tokens, q_heads, head_dim]``
        rotated likewise: a new tensor, or ``out`` (which may be ``q``).  ``q`` None returns None.  Rows
        outside every sequence are not written, in ``out`` neither.  The rows of one call must go to
        different places.  Records no derivatives, and refuses rows that ask for one."""
        k, sk = self._rows("k", k, self.kv_heads)
        v, sv = self._rows("v", v, self.kv_heads)
        T = k.shape[0]
        if v.shape[0] != T or (q is not None and q.shape[0] != T):
            raise ValueError("q, k and v must have the same number of rows")
        if rotary is not None and rotary._head_dim != self.head_dim:
            raise ValueError(f"rotary has head_dim={rotary.head_dim}, the cache {self.head_dim}")
        batch = self._batch(starts, lengths, table)
        Hq, qp, op, sq, so = 0, None, None, _NONE, _NONE
        written = self._k, self._v
        if q is not None:
            q, sq = self._rows("q", q)
            Hq = q.shape[1]
            if out is None:
                out = torch.empty_like(q, memory_format=torch.contiguous_format)
                so = (Hq * self.head_dim, self.head_dim)
            else:
                so = self._out(out, q)
                written += (out,)
            qp, op = q.data_ptr(), out.data_ptr()
        elif out is not None:
            raise ValueError("out without q")
        _written(*written)
        back = _enter(self.device)
        rc = _lib.load().ppmoe_kv_append(
            self._ptr, None if rotary is None else rotary._ptr, qp, sq[0], sq[1], op, so[0], so[1], Hq, k.data_ptr(),
            sk[0], sk[1], v.data_ptr(), sv[0], sv[1], T, *batch, _stream(self.device))
        if back is not None:
            torch.cuda.set_device(back)
        if rc:
            raise _lib.PPMoEError("ppmoe_kv_append", rc, _lib.load().ppmoe_last_error().decode())
        return out

    def attend(self, q: torch.Tensor, starts: torch.Tensor, lengths: torch.Tensor, table: torch.Tensor, *,
               max_new: Optional[int] = None, max_length: Optional[int] = None, scale: Optional[float] = None,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Attention of the rows ``q [tokens, q_heads, head_dim]`` over their sequences' positions up to
        their own (``q_heads`` a multiple of ``kv_heads``; query head ``h`` reads kv head
        ``h // (q_heads / kv_heads)``).  A row at a negative position gives zeros; rows outside every
        sequence are not written.  A row whose every score is -inf is NaN.  ``max_new`` / ``max_length``: the
        most new rows and the greatest length of a sequence as far as the host knows (default: the largest
        possible, all rows in one sequence: a decode step wants ``max_new=1``); they choose how the work is laid
        out, never what is computed.  ``scale`` defaults to ``head_dim ** -0.5``.  ``out`` may be ``q``.
        Records no derivatives, and refuses rows that ask for one."""
        q, sq = self._rows("q", q)
        T, Hq, D = q.shape
        if Hq < 1 or Hq % self.kv_heads:
            raise ValueError(f"q has {Hq} heads: not a multiple of the cache's {self.kv_heads}")
        batch = self._batch(starts, lengths, table)
        cap = batch[5] * self.page_size
        new = T if max_new is None else max(1, min(int(max_new), T))
        length = cap if max_length is None else max(1, min(int(max_length), cap))
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
            so = (Hq * D, D)
        else:
            so = self._out(out, q)
            _written(out)
        scale = D ** -0.5 if scale is None else float(scale)
        lib = _lib.load()
        n = lib.ppmoe_attend_workspace_bytes(T, Hq, self.kv_heads, D, batch[4], new, length)
        ws = torch.empty(n, dtype=torch.uint8, device=self.device) if n else None
        back = _enter(self.device)
        rc = lib.ppmoe_attend(self._ptr, q.data_ptr(), sq[0], sq[1], Hq, T, *batch, scale, new, length, out.data_ptr(),
                              so[0], so[1], None if ws is None else ws.data_ptr(), n, _stream(self.device))
        if back is not None:
            torch.cuda.set_device(back)
        if rc:
            raise _lib.PPMoEError("ppmoe_attend", rc, lib.ppmoe_last_error().decode())
        return out

    def _out(self, out, q):
        s = out.stride()
        if out.shape != q.shape or out.dtype is not q.dtype or out.device != q.device or (out.numel() and s[2] != 1):
            raise ValueError(f"out must be {list(q.shape)} {q.dtype} on {q.device} with contiguous heads")
        if any(n > 1 and x == 0 for n, x in zip(out.shape, s)):
            raise ValueError("out repeats elements")
        return s

    def check_device_status(self) -> None:
        """Wait for the device, all its streams, and raise if a call met a position without a page (its row was
        not stored, or what it gave is not defined); clears the status."""
        torch.cuda.synchronize(self.device)
        back = _enter(self.device)
        try:
            _lib.call("ppmoe_workspace_status", self._status.data_ptr(), _stream(self.device))
        finally:
            if back is not None:
                torch.cuda.set_device(back)
