"""Rotary position embedding: values and gradients against fp64, refusals."""
import math

import pytest
import torch

from conftest import pkg
from paged_helpers import assert_rotation, exact_rotation

SCALINGS = [None, {"type": "linear", "factor": 4.0}, {"type": "ntk", "factor": 8.0},
            {"type": "yarn", "factor": 8.0, "original_length": 4096}]


def emb(*a, **k):
    return pkg().rotary.RotaryEmbedding(*a, **k)


# ------------------------------------------------------------------ CPU
def test_frequencies():
    e = emb(64)
    assert torch.allclose(e.turns * 2 * math.pi, 10000.0 ** (-torch.arange(32, dtype=torch.float64) / 32), rtol=1e-14, atol=0)
    lin = emb(64, scaling={"type": "linear", "factor": 4.0})
    assert torch.equal(lin.turns, e.turns / 4)
    ntk = emb(64, scaling={"type": "ntk", "factor": 8.0})
    assert ntk.turns[0] == e.turns[0] and math.isclose(ntk.turns[-1] * 8, e.turns[-1], rel_tol=1e-12)
    y = emb(128, scaling={"type": "yarn", "factor": 8.0, "original_length": 4096})
    e = emb(128)
    n = e.turns * 4096  # turns within the trained length
    assert torch.equal(y.turns[n > 40], e.turns[n > 40])
    assert torch.allclose(y.turns[n < 0.8] * 8, e.turns[n < 0.8], rtol=1e-14, atol=0)
    mid = (n < 30) & (n > 1.2)
    assert (y.turns[mid] < e.turns[mid]).all() and (y.turns[mid] * 8 > e.turns[mid]).all()
    assert math.isclose(y.gain, 0.1 * math.log(8.0) + 1)
    assert emb(128, scaling={"type": "yarn", "factor": 8.0, "original_length": 4096, "gain": 1.0}).gain == 1.0


@pytest.mark.parametrize("bad", [
    dict(head_dim=0), dict(head_dim=63), dict(head_dim=258), dict(head_dim=64, rotary_dim=0),
    dict(head_dim=64, rotary_dim=66), dict(head_dim=64, rotary_dim=31), dict(head_dim=64, layout="other"),
    dict(head_dim=64, base=0.0), dict(head_dim=64, base=math.inf), dict(head_dim=64, scaling={"type": "other", "factor": 2.0}),
    dict(head_dim=64, scaling={"factor": 2.0}), dict(head_dim=64, scaling={"type": "linear", "factor": 0.0}),
    dict(head_dim=64, scaling={"type": "linear", "factor": 2.0, "more": 1}), dict(head_dim=64, rotary_dim=2, scaling={"type": "ntk", "factor": 2.0}),
    dict(head_dim=64, scaling={"type": "yarn", "factor": 2.0}), dict(head_dim=64, scaling={"type": "yarn", "factor": 2.0, "original_length": 0}),
])
def test_constructor_refusals(bad):
    with pytest.raises(ValueError):
        emb(bad.pop("head_dim"), **bad)


def test_runs_on_cuda_only():
    with pytest.raises(RuntimeError, match="CUDA only"):
        emb(64)(torch.zeros(2, 1, 64), None, torch.zeros(2, dtype=torch.long))


def test_host_validation_without_gpu():
    lib = pkg()._lib.load()
    e = emb(64)

    def call(heads=1, batch=1, length=2, head_dim=64, rot=64, dtype=0, q=16, pos=16, ptr=None):
        e._c.rotary_dim = rot
        return lib.ppmoe_rotary(e._ptr if ptr is None else ptr, 0, q, 0, 64, 64, q, 0, 64, 64, heads, None, 0, 0, 0, None, 0, 0, 0,
                                0, batch, length, head_dim, pos, 1, 0, 1, dtype, None)

    assert call(length=0) == 0 and call(heads=0) == 0  # nothing to do: no launch
    assert call(head_dim=63) == -2 and call(head_dim=258) == -2 and call(rot=66) == -2 and call(rot=3) == -2
    assert call(ptr=0) == -1 and call(dtype=3) == -2 and call(q=None) == -1 and call(pos=None) == -1
    assert call(batch=-1) == -1 and call(batch=2, length=2**31) == -1 and call(heads=1 << 20) == -2
    assert b"heads" in lib.ppmoe_last_error()


# ------------------------------------------------------------------ GPU
def data(shape, dtype, device, seed):
    g = torch.Generator(device=device).manual_seed(seed)
    return torch.randn(*shape, generator=g, device=device).to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim,rot", [(128, 128), (128, 64), (64, 16), (96, 32), (40, 20), (256, 256), (6, 2), (2, 2), (80, 8)])
def test_rotation(cuda, dtype, layout, dim, rot):
    """Aligned and unaligned head sizes and rotated parts, both layouts and every type."""
    e = emb(dim, rotary_dim=rot, layout=layout)
    q, k = data((2, 9, 5, dim), dtype, cuda, 1), data((2, 9, 3, dim), dtype, cuda, 2)
    pos = torch.tensor([[0, 1, 2, 100, 4095, 65537, 999_999, 7, -3], [5, 5, 5, 6, 7, 8, 9, 10, 11]], device=cuda)
    q2, k2 = e(q, k, pos)
    for x, y in ((q, q2), (k, k2)):
        assert_rotation(y, *exact_rotation(e, x, pos))
        assert torch.equal(y[..., rot:], x[..., rot:])


@pytest.mark.gpu
@pytest.mark.parametrize("scaling", SCALINGS)
def test_scaled_and_far_positions(cuda, scaling):
    e = emb(128, scaling=scaling)
    q = data((1500, 4, 128), torch.float32, cuda, 3)
    pos = (torch.arange(1500, device=cuda) * 701).to(torch.int32)  # up to a million
    q2, none = e(q, None, pos)
    assert none is None
    assert_rotation(q2, *exact_rotation(e, q, pos))


@pytest.mark.gpu
def test_far_positions_keep_relative_angles(cuda):
    """A score depends on the distance alone, a billion positions out."""
    e = emb(64)
    q, k = data((1, 1, 64), torch.float32, cuda, 4), data((1, 1, 64), torch.float32, cuda, 5)
    scores = []
    for p in (0, 1_000_000_000, 2**40):
        q2, k2 = e(q, k, torch.tensor([p + 17], device=cuda))[0], e(k, None, torch.tensor([p], device=cuda))[0]
        scores.append((q2.double() * k2.double()).sum().item())
    bound = 2.0 ** -19 * (q.double().abs() @ k.double().abs().transpose(1, 2)).item() * 2
    # p * turns is rounded in fp64: 2^40 / 2 pi * 2^-53 turns, 2^-15.7 * 2 pi ... radians at the last p
    assert abs(scores[1] - scores[0]) <= bound
    assert abs(scores[2] - scores[0]) <= bound + 4 * 2.0 ** 40 * 2.0 ** -53 * (q.abs().sum() * k.abs().max()).item()


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,heads", [(1, 1), (1, 12), (1023, 2), (1025, 2), (1027, 12), (4096, 24)])
def test_token_counts(cuda, tokens, heads):
    e = emb(128)
    q = data((tokens, heads, 128), torch.bfloat16, cuda, tokens)
    pos = torch.arange(tokens, device=cuda)
    assert_rotation(e(q, None, pos)[0], *exact_rotation(e, q, pos))


@pytest.mark.gpu
def test_empty(cuda):
    e = emb(64)
    q, k = e(torch.empty(0, 4, 64, device=cuda), torch.empty(0, 0, 64, device=cuda), torch.empty(0, dtype=torch.long, device=cuda))
    assert q.shape == (0, 4, 64) and k.shape == (0, 0, 64)


@pytest.mark.gpu
def test_strides(cuda):
    """Parts of a fused projection, head-major tensors, odd offsets, expanded inputs and positions."""
    e = emb(64)
    pos = torch.arange(10, device=cuda)
    fused = data((2, 10, 7, 64), torch.bfloat16, cuda, 1)
    q, k = fused[:, :, :4], fused[:, :, 4:6]
    q2, k2 = e(q, k, pos)
    assert_rotation(q2, *exact_rotation(e, q, pos.expand(2, 10)))
    assert_rotation(k2, *exact_rotation(e, k, pos.expand(2, 10)))
    hm = data((2, 3, 10, 64), torch.bfloat16, cuda, 2).transpose(1, 2)  # [batch, heads, tokens, dim] storage
    assert_rotation(e(hm, None, pos)[0], *exact_rotation(e, hm, pos.expand(2, 10)))
    odd = data((10 * 2 * 64 + 1,), torch.bfloat16, cuda, 3)[1:].view(10, 2, 64)  # 2-byte aligned
    assert_rotation(e(odd, None, pos)[0], *exact_rotation(e, odd, pos))
    wide = data((10, 1, 64), torch.bfloat16, cuda, 4).expand(10, 6, 64)
    assert_rotation(e(wide, None, pos)[0], *exact_rotation(e, wide, pos))
    last = data((10, 64, 2), torch.bfloat16, cuda, 5).transpose(1, 2)  # heads not contiguous
    assert_rotation(e(last, None, pos)[0], *exact_rotation(e, last, pos))


@pytest.mark.gpu
def test_in_place(cuda):
    e = emb(64, rotary_dim=32, layout="interleaved")
    fused = data((10, 7, 64), torch.float16, cuda, 1)
    ref = fused.clone()
    pos = torch.arange(10, device=cuda, dtype=torch.int32)
    e.rotate_(fused[:, :4], fused[:, 4:6], pos)
    q2, k2 = e(ref[:, :4], ref[:, 4:6], pos)
    assert torch.equal(fused[:, :4], q2) and torch.equal(fused[:, 4:6], k2) and torch.equal(fused[:, 6], ref[:, 6])
    with pytest.raises(ValueError):
        e.rotate_(ref[:, :1].expand(10, 4, 64), None, pos)
    with pytest.raises(ValueError):
        e.rotate_(ref, ref, pos)
    with pytest.raises(RuntimeError):
        e.rotate_(ref.clone().requires_grad_(), None, pos)
    w = torch.ones(10, 7, 64, dtype=torch.float16, device=cuda, requires_grad=True)
    x = ref.clone()
    y = (w * x).sum()  # saves x
    e.rotate_(x, None, pos)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():
        z = ref * 1
        e.rotate_(z, None, pos)
    assert torch.equal(z, x)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradients(cuda, dtype, layout):
    """Against the transposed rotation in fp64, and (fp32) against differences of the function."""
    e = emb(64, rotary_dim=48, layout=layout, scaling={"type": "yarn", "factor": 4.0, "original_length": 64})
    q = data((2, 6, 3, 64), dtype, cuda, 1).requires_grad_()
    k = data((2, 6, 1, 64), dtype, cuda, 2).requires_grad_()
    pos = torch.arange(6, device=cuda) * 31
    wq, wk = data((2, 6, 3, 64), dtype, cuda, 3), data((2, 6, 1, 64), dtype, cuda, 4)
    q2, k2 = e(q, k, pos)
    dq, dk = torch.autograd.grad((q2, k2), (q, k), (wq, wk))
    p = pos.expand(2, 6)
    assert_rotation(dq, *exact_rotation(e, wq, p, inverse=True))
    assert_rotation(dk, *exact_rotation(e, wk, p, inverse=True))
    if dtype is torch.float32:
        g = torch.Generator(device=cuda).manual_seed(9)
        step = torch.randn(q.shape, generator=g, device=cuda)
        with torch.no_grad():
            # linear in q: the difference over any step is the derivative; fp32 sums of 1152 terms
            diff = ((e(q + step, k, pos)[0] - e(q - step, k, pos)[0]).double() * wq.double()).sum() / 2
        want = (dq.double() * step.double()).sum()
        assert abs(diff - want) <= 2.0 ** -19 * ((q.abs() + step.abs()).double() * 2).sum() * wq.abs().max()


@pytest.mark.gpu
def test_gradients_of_broadcast_and_partial_use(cuda):
    e = emb(64)
    pos = torch.arange(5, device=cuda)
    base = data((5, 1, 64), torch.float32, cuda, 1).requires_grad_()
    k = data((5, 2, 64), torch.float32, cuda, 2).requires_grad_()
    q2, k2 = e(base.expand(5, 4, 64), k, pos)
    q2.sum().backward()  # the gradient comes as an expanded scalar; k2 is unused
    y, size = exact_rotation(e, torch.ones(5, 4, 64, device=cuda), pos, inverse=True)
    assert ((base.grad.double() - y.sum(1, keepdim=True)).abs() <= 2.0 ** -18 * size.sum(1, keepdim=True)).all()
    assert k.grad is None
    q2, k2 = e(base.expand(5, 4, 64), k, pos)
    (dk,) = torch.autograd.grad(k2, k, torch.ones_like(k2))
    assert_rotation(dk, *exact_rotation(e, torch.ones(5, 2, 64, device=cuda), pos, inverse=True))
    q2, k2 = e(base.detach(), k, pos)  # only k needs a gradient
    (dk2,) = torch.autograd.grad(k2, k, torch.ones_like(k2))
    assert torch.equal(dk2, dk)


@pytest.mark.gpu
def test_second_gradients(cuda):
    """The gradient is linear in the incoming one, and its own gradient the rotation again."""
    e = emb(64, scaling={"type": "yarn", "factor": 4.0, "original_length": 64})
    pos = torch.arange(7, device=cuda) * 13
    q = data((7, 2, 64), torch.float32, cuda, 1).requires_grad_()
    k = data((7, 1, 64), torch.float32, cuda, 2).requires_grad_()
    wq, wk = (data(s, torch.float32, cuda, i).requires_grad_() for i, s in ((3, (7, 2, 64)), (4, (7, 1, 64))))
    dq, dk = torch.autograd.grad(e(q, k, pos), (q, k), (wq, wk), create_graph=True)
    vq, vk = data((7, 2, 64), torch.float32, cuda, 5), data((7, 1, 64), torch.float32, cuda, 6)
    gq, gk = torch.autograd.grad((dq, dk), (wq, wk), (vq, vk))
    assert_rotation(gq, *exact_rotation(e, vq, pos))
    assert_rotation(gk, *exact_rotation(e, vk, pos))


@pytest.mark.gpu
def test_captured_training_step(cuda):
    """Forward and backward in a captured graph (no eager graph of the same leaves lives meanwhile), and the
    check that saved positions have not been written to."""
    e = emb(64)
    pos = torch.arange(9, device=cuda)
    q = data((9, 2, 64), torch.bfloat16, cuda, 1).requires_grad_()
    k = data((9, 1, 64), torch.bfloat16, cuda, 2).requires_grad_()
    wq, wk = data((9, 2, 64), torch.bfloat16, cuda, 3), data((9, 1, 64), torch.bfloat16, cuda, 4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # warm-up, as a capture of autograd wants it
        torch.autograd.grad(e(q, k, pos), (q, k), (wq, wk))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(e(q, k, pos), (q, k), (wq, wk))
    pos += 5
    graph.replay()
    for g, w in zip(got, (wq, wk)):
        assert_rotation(g, *exact_rotation(e, w, pos, inverse=True))
    out = e(q, k, pos)
    pos -= 5
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out, (q, k), (wq, wk))


@pytest.mark.gpu
def test_streams_and_capture(cuda):
    e = emb(128)
    q, k = data((64, 12, 128), torch.bfloat16, cuda, 1), data((64, 12, 128), torch.bfloat16, cuda, 2)
    pos = torch.arange(64, device=cuda)
    want = e(q, k, pos + 1000)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = e(q, k, pos + 1000)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = e(q, k, pos)
    del e  # the graph keeps the frequencies
    pos += 1000
    graph.replay()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.gpu
def test_refusals(cuda):
    e = emb(64)
    q, pos = torch.zeros(4, 2, 64, device=cuda), torch.zeros(4, dtype=torch.long, device=cuda)
    for args in [(q[..., :32], None, pos), (q[0], None, pos), (q, q[:3], pos), (q, q.half(), pos), (q, None, pos[:3]),
                 (q, None, pos.float()), (q, None, pos.cpu())]:
        with pytest.raises(ValueError):
            e(*args)
    with pytest.raises(TypeError):
        e(q.double(), None, pos)
