"""Rotary position embedding under forward-mode differentiation, and as an object of its own."""
import copy
import math
import pickle

import pytest
import torch
from torch.autograd import forward_ad

from conftest import pkg
from paged_helpers import assert_rotation, exact_rotation


def emb(*a, **k):
    return pkg().rotary.RotaryEmbedding(*a, **k)


def data(shape, dtype, device, seed):
    g = torch.Generator(device=device).manual_seed(seed)
    return torch.randn(*shape, generator=g, device=device).to(dtype)


# ------------------------------------------------------------------ CPU
class OnCpu:
    """Stands in for the launch: the rotation in fp64, rounded once."""

    def __init__(self, monkeypatch, e):
        self.e = e
        monkeypatch.setattr(e, "_launch", self)

    def __call__(self, q, k, positions, inverse, out=None):
        return tuple(None if x is None else exact_rotation(self.e, x.detach(), positions, inverse)[0].to(x.dtype) for x in (q, k))


@pytest.mark.parametrize("mode", [torch.enable_grad, torch.no_grad])
def test_tangents_on_cpu(monkeypatch, mode):
    """Which tensors a tangent reaches, and that it is the rotated tangent (the function is linear)."""
    e = emb(8)
    OnCpu(monkeypatch, e)
    q, k, tq, tk = (data((5, h, 8), torch.float64, "cpu", i) for i, h in enumerate((3, 2, 3, 2)))
    pos = torch.arange(5)
    rotated = lambda x: exact_rotation(e, x, pos)[0]  # noqa: E731
    with mode(), forward_ad.dual_level():
        for with_q, with_k in ((True, True), (True, False), (False, True)):
            a = forward_ad.make_dual(q, tq) if with_q else q
            b = forward_ad.make_dual(k, tk) if with_k else k
            for x, t, has, y in zip((q, k), (tq, tk), (with_q, with_k), e(a, b, pos)):
                got, tangent = forward_ad.unpack_dual(y)
                assert torch.equal(got, rotated(x))
                assert torch.equal(tangent, rotated(t) if has else torch.zeros_like(t))
        y, none = e(forward_ad.make_dual(q, tq), None, pos)
        assert none is None and torch.equal(forward_ad.unpack_dual(y).tangent, rotated(tq))
        assert forward_ad.unpack_dual(e(q, None, pos)[0]).tangent is None
        with pytest.raises(RuntimeError, match="tangent"):
            e.rotate_(forward_ad.make_dual(q.clone(), tq), None, pos)


def test_mixed_modes_on_cpu(monkeypatch):
    """Reverse over forward and forward over reverse, against each other's definition by linearity."""
    e = emb(8)
    OnCpu(monkeypatch, e)
    pos = torch.arange(4) * 7
    q, t, w = (data((4, 2, 8), torch.float64, "cpu", i) for i in range(3))
    back = lambda x: exact_rotation(e, x, pos, inverse=True)[0]  # noqa: E731
    with forward_ad.dual_level():
        t2 = t.clone().requires_grad_()
        y = forward_ad.unpack_dual(e(forward_ad.make_dual(q, t2), None, pos)[0]).tangent
        (dt,) = torch.autograd.grad(y, t2, w)
        assert torch.equal(dt, back(w))
        x = q.clone().requires_grad_()
        (dq,) = torch.autograd.grad(e(x, None, pos)[0], x, forward_ad.make_dual(w, t))
        dq, tangent = forward_ad.unpack_dual(dq)
        assert torch.equal(dq, back(w)) and torch.equal(tangent, back(t))


@pytest.mark.parametrize("factor,gain", [(0.5, 1.0), (1.0, 1.0), (2.0, 0.1 * math.log(2.0) + 1.0)])
def test_yarn_gain(factor, gain):
    """The published rule multiplies values only where the context is made longer."""
    assert emb(64, scaling={"type": "yarn", "factor": factor, "original_length": 4096}).gain == gain


def test_an_embedding_does_not_change():
    """What the launches read is what the attributes say, in copies too; none can be set."""
    e = emb(64, rotary_dim=32, layout="interleaved", scaling={"type": "yarn", "factor": 4.0, "original_length": 4096})
    for x in (e, copy.deepcopy(e), pickle.loads(pickle.dumps(e))):
        assert (x.head_dim, x.rotary_dim, x.layout, x.gain) == (64, 32, "interleaved", 0.1 * math.log(4.0) + 1.0)
        assert torch.equal(x.turns, e.turns) and x.turns.dtype == torch.float64 and x.turns.shape == (16,)
        for name, value in (("head_dim", 32), ("rotary_dim", 16), ("layout", "half"), ("gain", 2.0), ("turns", torch.zeros(16))):
            with pytest.raises(AttributeError):
                setattr(x, name, value)
    before = e.turns
    e.turns.zero_()
    assert torch.equal(e.turns, before)


# ------------------------------------------------------------------ GPU
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_tangents(cuda, dtype):
    e = emb(64, rotary_dim=48, scaling={"type": "yarn", "factor": 4.0, "original_length": 64})
    q, k, tq = (data((9, h, 64), dtype, cuda, i) for i, h in enumerate((3, 1, 3)))
    pos = torch.arange(9, device=cuda) * 31
    with forward_ad.dual_level():
        q2, k2 = e(forward_ad.make_dual(q, tq), k, pos)
        q2, t2 = forward_ad.unpack_dual(q2)
        assert torch.equal(q2, e(q, None, pos)[0]) and torch.equal(forward_ad.unpack_dual(k2).primal, e(k, None, pos)[0])
    assert_rotation(t2, *exact_rotation(e, tq, pos))
