"""Rotary position embedding on the GPU (``ppmoe_rotary``), forward and backward.

A head's first ``rotary_dim`` values are pairs; pair ``i`` at position ``p`` is turned by the angle
``p * f_i``, ``f_i = base ** (-2 i / rotary_dim)``, optionally scaled for contexts longer than the
trained ones.  The kernel takes the angle from the position itself (reduced in fp64, sine and
cosine in fp32), so there is no table of a largest position and far positions lose nothing.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Tuple

import torch

from . import _lib

__all__ = ["RotaryEmbedding"]

_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16, torch.float32: _lib.DTYPE_F32}


def _stream(device: torch.device) -> int:
    return torch._C._cuda_getCurrentRawStream(device.index)


_NONE = (0, 0, 0, 0)


def _enter(device: torch.device):
    """Makes ``device`` current (a launch goes to the current device); the device to go back to, or None."""
    now = torch.cuda.current_device()
    if now == device.index:
        return None
    torch.cuda.set_device(device)
    return now


class _Rotate(torch.autograd.Function):
    """The rotation by the positions' angles or, inverse, by their negatives; each is the other's gradient."""

    @staticmethod
    def forward(ctx, emb, q, k, positions, inverse):
        ctx.emb, ctx.inverse = emb, inverse
        ctx.save_for_backward(positions)
        ctx.set_materialize_grads(False)
        return emb._launch(q, k, positions, inverse)

    @staticmethod
    def backward(ctx, dq, dk):
        (positions,) = ctx.saved_tensors
        _, need_q, need_k, _, _ = ctx.needs_input_grad
        if not need_q:
            dq = None
        if not need_k:
            dk = None
        first = dk if dq is None else dq
        if first is None:
            return None, None, None, None, None
        rest = None if dq is None else dk
        if torch.is_grad_enabled():  # a gradient of the gradient is wanted
            a, b = _Rotate.apply(ctx.emb, first, rest, positions, not ctx.inverse)
        else:
            a, b = ctx.emb._launch(first, rest, positions, not ctx.inverse)
        return (None, None, a, None, None) if dq is None else (None, a, b, None, None)


class RotaryEmbedding:
    """Rotary embedding of ``[..., tokens, heads, head_dim]`` queries and keys.

    ``rotary_dim`` (default ``head_dim``): the leading values of a head that are rotated; even.
    ``layout``: ``"half"`` pairs value ``i`` with ``i + rotary_dim / 2``, ``"interleaved"`` pairs ``2i``
    with ``2i + 1``.  ``scaling`` for long contexts, a dict:

    * ``{"type": "linear", "factor": s}``: every frequency divided by ``s``;
    * ``{"type": "ntk", "factor": s}``: the base multiplied by ``s ** (rotary_dim / (rotary_dim - 2))``,
      which leaves the fastest pair alone and divides the slowest one by ``s``;
    * ``{"type": "yarn", "factor": s, "original_length": n}`` (and optionally ``beta_fast`` 32,
      ``beta_slow`` 1, ``gain``): pairs that turn more than ``beta_fast`` times within ``n`` positions
      are left alone, those under ``beta_slow`` are divided by ``s``, the ones between are blended by
      their index; rotated values are multiplied by ``gain`` (default ``0.1 ln s + 1``).

    The object holds numbers only (``turns``: turns per position of each pair, fp64 on the host);
    a captured launch keeps its own copy of them.  bf16, fp16 and fp32; values are rounded once.
    To capture a backward pass into a CUDA graph, let no eager graph of the same leaves live: autograd would
    wait for the stream that one was made on, which a capture does not allow.
    """

    def __init__(self, head_dim: int, *, rotary_dim: Optional[int] = None, base: float = 10000.0,
                 layout: str = "half", scaling: Optional[dict] = None):
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        if head_dim < 2 or head_dim > 256 or head_dim % 2:
            raise ValueError(f"head_dim={head_dim} must be even and in [2, 256]")
        if rotary_dim < 2 or rotary_dim > head_dim or rotary_dim % 2:
            raise ValueError(f"rotary_dim={rotary_dim} must be even and in [2, head_dim={head_dim}]")
        if layout not in ("half", "interleaved"):
            raise ValueError(f"layout={layout!r} must be 'half' or 'interleaved'")
        if not (base > 0 and math.isfinite(base)):
            raise ValueError(f"base={base} must be positive and finite")
        self.head_dim, self.rotary_dim, self.layout = head_dim, rotary_dim, layout
        self.gain = 1.0
        pairs = range(rotary_dim // 2)
        sc = dict(scaling or {})
        kind = sc.pop("type", None)
        if scaling is not None and kind not in ("linear", "ntk", "yarn"):
            raise ValueError(f"scaling type {kind!r} must be 'linear', 'ntk' or 'yarn'")
        factor = float(sc.pop("factor", 1.0))
        if not (factor > 0 and math.isfinite(factor)):
            raise ValueError(f"scaling factor {factor} must be positive and finite")
        if kind == "ntk":
            if rotary_dim == 2:
                raise ValueError("ntk scaling needs rotary_dim > 2")
            base = base * factor ** (rotary_dim / (rotary_dim - 2))
        freq = [base ** (-2.0 * i / rotary_dim) for i in pairs]
        if kind == "linear":
            freq = [f / factor for f in freq]
        elif kind == "yarn":
            if "original_length" not in sc or base == 1.0:
                raise ValueError("yarn scaling needs original_length, and a base other than 1")
            n = float(sc.pop("original_length"))
            fast, slow = float(sc.pop("beta_fast", 32.0)), float(sc.pop("beta_slow", 1.0))
            if not (n > 0 and fast > 0 and slow > 0):
                raise ValueError("yarn scaling needs positive original_length, beta_fast and beta_slow")

            def index(turns):  # the pair (a fraction) that turns so often within the trained length
                return rotary_dim * math.log(n / (turns * 2 * math.pi)) / (2 * math.log(base))

            low, high = max(math.floor(index(fast)), 0), min(math.ceil(index(slow)), rotary_dim - 1)
            keep = [1.0 - min(max((i - low) / max(high - low, 1e-3), 0.0), 1.0) for i in pairs]
            freq = [f * k + f / factor * (1.0 - k) for f, k in zip(freq, keep)]
            self.gain = float(sc.pop("gain", 0.1 * math.log(factor) + 1.0))
        if sc:
            raise ValueError(f"unknown scaling entries {sorted(sc)}")
        turns = [f / (2.0 * math.pi) for f in freq]
        self.turns = torch.tensor(turns, dtype=torch.float64)
        self._c = _lib.Rotation(rotary_dim, layout == "interleaved", self.gain)
        self._c.turns[:rotary_dim // 2] = turns

    @property
    def _ptr(self) -> int:  # (of this object's own structure: copies have theirs)
        return ctypes.addressof(self._c)

    # ------------------------------------------------------------------ calls
    def __call__(self, q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor
                 ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
        """Rotated copies of ``q [(batch,) tokens, q_heads, head_dim]`` and ``k`` (same leading sizes, its
        own number of heads; or None).  ``positions [(batch,) tokens]`` or ``[tokens]``, int64 or int32.
        Any strides with contiguous heads; differentiable in ``q`` and ``k``."""
        if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
            return _Rotate.apply(self, q, k, positions, False)
        return self._launch(q, k, positions, False)

    def rotate_(self, q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor) -> None:
        """The same in place (no gradients; ``q`` and ``k`` must not overlap)."""
        for x in (q, k):
            if x is not None and torch.is_grad_enabled() and x.requires_grad:
                raise RuntimeError("rotate_ records no gradients: call the embedding itself, or use torch.no_grad()")
            if x is not None and any(n > 1 and s == 0 for n, s in zip(x.shape, x.stride())):
                raise ValueError("rotate_ needs tensors without repeated elements")
        if k is not None and k.untyped_storage().data_ptr() == q.untyped_storage().data_ptr() and k.data_ptr() == q.data_ptr():
            raise ValueError("rotate_ needs q and k of their own")
        self._launch(q, k, positions, False, (q, k))

    def _launch(self, q, k, positions, inverse, out=None):
        dev, shape, dt = q.device, q.shape, q.dtype
        if dev.type != "cuda":
            raise RuntimeError("RotaryEmbedding runs on CUDA only; got a tensor on " + str(dev))
        n = len(shape)
        if n not in (3, 4) or shape[-1] != self.head_dim:
            raise ValueError(f"q must be [(batch,) tokens, heads, {self.head_dim}], got {list(shape)}")
        code = _DTYPES.get(dt)
        if code is None:
            raise TypeError(f"RotaryEmbedding takes bf16, fp16 or fp32, got {dt}")
        if k is not None:
            ks = k.shape
            if k.dtype is not dt or k.device != dev or ks[:-2] != shape[:-2] or ks[-1] != self.head_dim:
                raise ValueError(f"k {list(ks)} {k.dtype} on {k.device} does not go with q {list(shape)} {dt} on {dev}")
        if positions.device != dev or positions.dtype not in (torch.int64, torch.int32):
            raise ValueError(f"positions must be int64 or int32 on {dev}, got {positions.dtype} on {positions.device}")
        if positions.shape != shape[:-2] and positions.shape != shape[-3:-2]:
            raise ValueError(f"positions {list(positions.shape)} do not go with q {list(shape)}")
        sq = q.stride()
        if sq[-1] != 1:
            q = q.contiguous()
            sq = q.stride()
        B, L, Hq = (shape[0] if n == 4 else 1), shape[-3], shape[-2]
        sk, Hk, k2, sk2 = _NONE, 0, None, _NONE
        if k is not None:
            sk, Hk = k.stride(), ks[-2]
            if sk[-1] != 1:
                k = k.contiguous()
                sk = k.stride()
        if out is None:
            q2 = torch.empty_like(q, memory_format=torch.contiguous_format)
            sq2 = (L * Hq * self.head_dim, Hq * self.head_dim, self.head_dim, 1)
            if k is not None:
                k2 = torch.empty_like(k, memory_format=torch.contiguous_format)
                sk2 = (L * Hk * self.head_dim, Hk * self.head_dim, self.head_dim, 1)
        else:
            q2, k2 = out
            sq2 = sq if n == 4 else (0, *sq)
            if k2 is not None:
                sk2 = sk if n == 4 else (0, *sk)
            if q2.data_ptr() != q.data_ptr() or (k is not None and k2.data_ptr() != k.data_ptr()):
                raise ValueError("rotate_ needs contiguous heads")
        if n == 3:
            sq = (0, *sq)
            if k is not None:
                sk = (0, *sk)
        pb, pt = positions.stride() if positions.dim() == 2 else (0, positions.stride(0))
        back = _enter(dev)
        rc = _lib.load().ppmoe_rotary(
            self._ptr, inverse, q.data_ptr(), sq[0], sq[1], sq[2], q2.data_ptr(), sq2[0], sq2[1], sq2[2], Hq,
            None if k is None else k.data_ptr(), sk[0], sk[1], sk[2], None if k is None else k2.data_ptr(),
            sk2[0], sk2[1], sk2[2], Hk, B, L, self.head_dim, positions.data_ptr(),
            positions.dtype is torch.int64, pb, pt, code, _stream(dev))
        if back is not None:
            torch.cuda.set_device(back)
        if rc:
            raise _lib.PPMoEError("ppmoe_rotary", rc, _lib.load().ppmoe_last_error().decode())
        return q2, k2
