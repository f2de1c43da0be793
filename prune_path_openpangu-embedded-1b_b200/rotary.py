"""Rotary position embedding on the GPU (``ppmoe_rotary``), forward and backward.

A head's first ``rotary_dim`` values are pairs; pair ``i`` at position ``p`` is turned by the angle
``p * f_i``, ``f_i = base ** (-2 i / rotary_dim)``, optionally scaled for contexts longer than the
trained ones.  The kernel takes the angle from the position itself (reduced in fp64, sine and
cosine in fp32), so there is no table of a largest position, and up to 2^31 positions out an angle is
off by less than 2^-19 radians (the fp64 roundings of ``f_i`` and of ``p * f_i``; they grow with ``p``).
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import _lib

__all__ = ["RotaryEmbedding"]

_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16, torch.float32: _lib.DTYPE_F32}


def _stream(device: torch.device) -> int:
    return torch._C._cuda_getCurrentRawStream(device.index)


_POSITIONS = (torch.int64, torch.int32)
_NONE = (0, 0, 0)


def _has_tangent(*tensors: Optional[torch.Tensor]) -> bool:
    """Whether forward-mode differentiation follows one of these (such a tensor requires no gradient)."""
    return (forward_ad._current_level >= 0  # (asked first where a call's host time counts)
            and any(x is not None and forward_ad.unpack_dual(x).tangent is not None for x in tensors))


def _written(*tensors: torch.Tensor) -> None:
    """Tells autograd that a kernel writes into these, so that a backward pass that saved one complains."""
    if torch.is_grad_enabled():
        for x in tensors:
            if x.requires_grad:
                raise RuntimeError("a tensor that requires a gradient cannot be written to: use torch.no_grad()")
    if forward_ad._current_level >= 0 and _has_tangent(*tensors):
        raise RuntimeError("a tensor with a forward-mode tangent cannot be written to")
    torch._C._increment_version(tensors)  # (leaves inference tensors out; what autograd.graph's function calls)


def _heads(x: torch.Tensor, four: bool):
    """x with contiguous heads, and its (batch, token, head) strides."""
    s = x.stride()
    if s[-1] != 1:
        x = x.contiguous()
        s = x.stride()
    return x, s if four else (0, *s)


def _enter(device: torch.device):
    """Makes ``device`` current (a launch goes to the current device); the device to go back to, or None."""
    now = torch.cuda.current_device()
    if now == device.index:
        return None
    torch.cuda.set_device(device)
    return now


class _Rotate(torch.autograd.Function):
    """The rotation by the positions' angles or, inverse, by their negatives; each is the other's gradient.  It is
    linear: tangents (forward mode) are rotated as the values are."""

    @staticmethod
    def forward(ctx, emb, q, k, positions, inverse):
        ctx.emb, ctx.inverse = emb, inverse
        ctx.save_for_backward(positions)
        if forward_ad._current_level >= 0:
            ctx.save_for_forward(positions)
            ctx.like = q.detach(), None if k is None else k.detach()
        ctx.set_materialize_grads(False)
        return emb._launch(q, k, positions, inverse)

    @staticmethod
    def jvp(ctx, _emb, tq, tk, _positions, _inverse):
        (positions,) = ctx.saved_tensors
        if tq is None:  # an output beside one with a tangent has one too
            tq = torch.zeros_like(ctx.like[0])
        if tk is None and ctx.like[1] is not None:
            tk = torch.zeros_like(ctx.like[1])
        return _Rotate.apply(ctx.emb, tq, tk, positions, ctx.inverse)

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
        if torch.is_grad_enabled() or _has_tangent(first, rest):  # a derivative of the gradient is wanted
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
      their index; rotated values are multiplied by ``gain`` (default ``0.1 ln s + 1``, and 1 for ``s``
      below 1).

    The object holds numbers only, which do not change (``turns``: turns per position of each pair, fp64 on the
    host); a captured launch keeps its own copy of them.  bf16, fp16 and fp32; values are rounded once.
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
        self._head_dim = head_dim
        gain = 1.0
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
            gain = float(sc.pop("gain", 0.1 * math.log(max(factor, 1.0)) + 1.0))
        if sc:
            raise ValueError(f"unknown scaling entries {sorted(sc)}")
        self._c = _lib.Rotation(rotary_dim, layout == "interleaved", gain)  # (what the launches read)
        self._c.turns[:rotary_dim // 2] = [f / (2.0 * math.pi) for f in freq]

    @property
    def head_dim(self) -> int:
        return self._head_dim

    @property
    def rotary_dim(self) -> int:
        return self._c.rotary_dim

    @property
    def layout(self) -> str:
        return "interleaved" if self._c.interleaved else "half"

    @property
    def gain(self) -> float:
        return self._c.gain

    @property
    def turns(self) -> torch.Tensor:
        return torch.tensor(self._c.turns[:self._c.rotary_dim // 2], dtype=torch.float64)

    @property
    def _ptr(self) -> int:  # (of this object's own structure: copies have theirs)
        return ctypes.addressof(self._c)

    # ------------------------------------------------------------------ calls
    def __call__(self, q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor
                 ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
        """Rotated copies of ``q [(batch,) tokens, q_heads, head_dim]`` and ``k`` (same leading sizes, its
        own number of heads; or None).  ``positions [(batch,) tokens]`` or ``[tokens]``, int64 or int32.
        Any strides with contiguous heads; differentiable in ``q`` and ``k``, in reverse and in forward mode."""
        if (torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad))) or _has_tangent(q, k):
            return _Rotate.apply(self, q, k, positions, False)
        return self._launch(q, k, positions, False)

    def rotate_(self, q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor) -> None:
        """The same in place (records no derivatives, and refuses tensors that ask for one; ``q`` and ``k`` must not
        overlap)."""
        for x in (q, k):
            if x is not None and any(n > 1 and s == 0 for n, s in zip(x.shape, x.stride())):
                raise ValueError("rotate_ needs tensors without repeated elements")
        if k is not None and k.untyped_storage().data_ptr() == q.untyped_storage().data_ptr() and k.data_ptr() == q.data_ptr():
            raise ValueError("rotate_ needs q and k of their own")
        _written(*(x for x in (q, k) if x is not None))
        self._launch(q, k, positions, False, (q, k))

    def _launch(self, q, k, positions, inverse, out=None):
        dev, shape, dt, D = q.device, q.shape, q.dtype, self._head_dim
        if dev.type != "cuda":
            raise RuntimeError("RotaryEmbedding runs on CUDA only; got a tensor on " + str(dev))
        four = len(shape) == 4
        if not (four or len(shape) == 3) or shape[-1] != D:
            raise ValueError(f"q must be [(batch,) tokens, heads, {D}], got {list(shape)}")
        B, L, Hq = shape[:3] if four else (1, *shape[:2])
        code = _DTYPES.get(dt)
        if code is None:
            raise TypeError(f"RotaryEmbedding takes bf16, fp16 or fp32, got {dt}")
        at = positions.shape
        if positions.device != dev or positions.dtype not in _POSITIONS:
            raise ValueError(f"positions must be int64 or int32 on {dev}, got {positions.dtype} on {positions.device}")
        if at != (L,) and not (four and at == (B, L)):
            raise ValueError(f"positions {list(at)} do not go with q {list(shape)}")
        pb, pt = positions.stride() if len(at) == 2 else (0, positions.stride(0))
        q, sq = _heads(q, four)
        qo = out[0] if out else torch.empty_like(q, memory_format=torch.contiguous_format)
        so = (L * Hq * D, Hq * D, D)
        kp, sk, ko, sko, Hk, k2 = None, _NONE, None, _NONE, 0, None
        if k is not None:
            ks = k.shape
            Hk = ks[-2] if len(ks) == len(shape) else -1
            if k.dtype is not dt or k.device != dev or ks != ((B, L, Hk, D) if four else (L, Hk, D)):
                raise ValueError(f"k {list(ks)} {k.dtype} on {k.device} does not go with q {list(shape)} {dt} on {dev}")
            k, sk = _heads(k, four)
            k2 = out[1] if out else torch.empty_like(k, memory_format=torch.contiguous_format)
            sko = (L * Hk * D, Hk * D, D)
            kp, ko = k.data_ptr(), k2.data_ptr()
        if out:
            so, sko = sq, sk
            if qo.data_ptr() != q.data_ptr() or kp != ko:
                raise ValueError("rotate_ needs contiguous heads")
        back = _enter(dev)
        rc = _lib.load().ppmoe_rotary(
            self._ptr, inverse, q.data_ptr(), sq[0], sq[1], sq[2], qo.data_ptr(), so[0], so[1], so[2], Hq, kp,
            sk[0], sk[1], sk[2], ko, sko[0], sko[1], sko[2], Hk, B, L, D, positions.data_ptr(),
            positions.dtype is torch.int64, pb, pt, code, _stream(dev))
        if back is not None:
            torch.cuda.set_device(back)
        if rc:
            raise _lib.PPMoEError("ppmoe_rotary", rc, _lib.load().ppmoe_last_error().decode())
        return qo, k2
