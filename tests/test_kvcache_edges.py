"""Paged cache and attention where they meet the rest of a program: launches behind them on the stream, autograd,
values and sizes at the borders of what they take."""
import ctypes
import math

import pytest
import torch
from torch.autograd import forward_ad

from conftest import pkg
from gpu_helpers import make_module
from paged_helpers import GARBAGE, Batch, assert_attention, exact_attention


# ------------------------------------------------------------------ CPU
def test_a_table_of_too_many_positions():
    """Counting keys in 32 bits would run over: refused before anything is launched."""
    lib = pkg()._lib.load()
    for page, pages in ((256, (1 << 23) - 31), (16, 1 << 27)):
        cache = pkg()._lib.KVCache(1024, 1024, 2 * page * 64, page * 64, 64, 2 * page * 64, page * 64, 64, 4, page, 2, 64, 0, 256)
        rc = lib.ppmoe_attend(ctypes.byref(cache), 16, 256, 64, 4, 1, 16, 16, 16, pages, 1, pages, 0.125, 1, 64, 16, 256, 64, None, 0, None)
        assert rc == -2 and b"positions" in lib.ppmoe_last_error()


def test_keys_and_values_of_one_memory():
    """An append would write both to the same places."""
    x = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    for v in (x, x.view_as(x)):
        with pytest.raises(ValueError, match="memory of their own"):
            pkg().kvcache.PagedKVCache.from_tensors(x, v)


# ------------------------------------------------------------------ GPU: what follows on the stream
@pytest.mark.gpu
@pytest.mark.parametrize("shared", ["out", "q"])
@pytest.mark.parametrize("seqs,new,length,hk,hints", [
    (16, 1, 8000, 12, dict(max_new=1)),                 # few rows, parts that meet in clusters
    (1, 16, 8000, 1, dict(max_new=1, max_length=1)),    # few rows, one CTA going through all of them
    (1, 16, 8000, 1, dict(max_new=16, max_length=1)),   # tiles in one part
    (1, 16, 8000, 1, dict(max_new=16, max_length=8000)),  # tiles whose parts are joined
])
def test_a_decode_from_host_memory_follows(cuda, shared, seqs, new, length, hk, hints):
    """ppmoe_decode_host's staging copy starts before its wait; where its staging buffer is the attention's output
    or queries, it has to come after the attention all the same."""
    P = pkg()
    b = Batch([new] * seqs, [length] * seqs, hk, 128, 64, torch.bfloat16, cuda, seed=21)
    q = b.normal(12, 2.0)
    want = exact_attention(b, q)
    tokens = q.shape[0]
    layer = P.synth.make_layer(8, 1536, 64, 96)
    m = make_module(layer, 0.95, cuda)
    x = P.synth.make_tokens(8, tokens, 1536)
    ref = m.forward_decode(x.to(cuda)).cpu()
    xh, oh = x.pin_memory(), torch.empty(tokens, 1536, dtype=torch.bfloat16).pin_memory()
    out, od, ws = torch.empty_like(q), torch.empty(tokens, 1536, dtype=torch.bfloat16, device=cuda), m.workspace(tokens)
    staging = out if shared == "out" else q
    cache, s = b.cache(), torch.cuda.current_stream()
    cache.attend(q, b.starts, b.lens, b.table, out=out, **hints)
    P._lib.call("ppmoe_decode_host", xh.data_ptr(), tokens, m.packed().data_ptr(), 1536, 64, 96, 0.95, None, oh.data_ptr(),
                staging.data_ptr(), od.data_ptr(), ws.data_ptr(), ws.numel(), s.cuda_stream)
    s.synchronize()
    m.check_device_status()
    assert torch.equal(staging.view(tokens, 1536).cpu(), x)
    assert torch.equal(oh, ref)
    if shared == "q":
        assert_attention(out, *want)


# ------------------------------------------------------------------ GPU: autograd
@pytest.mark.gpu
@pytest.mark.parametrize("which", ["k", "v"])
def test_append_tells_autograd(cuda, which):
    """A backward pass that saved the cache's tensors (its own, or the given ones) must not use what an append wrote."""
    b = Batch([2], [20], 1, 64, 16, torch.bfloat16, cuda, seed=22)
    cache, k, v = b.cache(), b.normal(1), b.normal(1)
    for saved in (getattr(cache, which), getattr(b, which)):
        w = torch.ones_like(saved, requires_grad=True)
        y = (w * saved).sum()
        cache.append(None, k, v, b.starts, b.lens, b.table)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    with torch.inference_mode():
        cache.append(None, k, v, b.starts, b.lens, b.table)
    cache.k.requires_grad_()
    with pytest.raises(RuntimeError, match="no_grad"):
        cache.append(None, k, v, b.starts, b.lens, b.table)


@pytest.mark.gpu
def test_tangents_are_refused(cuda):
    b = Batch([2], [20], 1, 64, 16, torch.bfloat16, cuda, seed=23)
    cache, q, k, v = b.cache(), b.normal(2), b.normal(1), b.normal(1)
    at = b.starts, b.lens, b.table
    with forward_ad.dual_level():
        dual = lambda x: forward_ad.make_dual(x.clone(), torch.ones_like(x))  # noqa: E731
        for call in (lambda: cache.attend(dual(q), *at), lambda: cache.append(dual(q), k, v, *at), lambda: cache.append(q, dual(k), v, *at),
                     lambda: cache.append(q, k, dual(v), *at), lambda: cache.attend(q, *at, out=dual(q)),
                     lambda: cache.append(q, k, v, *at, out=dual(q))):
            with pytest.raises(RuntimeError, match="tangent"):
                call()
        cache.append(q, k, v, *at)
        cache.attend(q, *at)


# ------------------------------------------------------------------ GPU: values
PLANS = [  # new rows, keys, hints: each way a call is laid out
    pytest.param(1, 300, dict(max_new=1, max_length=1), id="few rows in one part"),
    pytest.param(2, 900, dict(max_new=2, max_length=900), id="few rows in a cluster"),
    pytest.param(3, 9000, dict(max_new=3, max_length=9000), id="few rows joined"),
    pytest.param(70, 300, dict(max_new=70, max_length=300), id="one row tile"),
    pytest.param(70, 300, dict(max_new=1, max_length=300), id="few rows, many times"),
    pytest.param(60, 6000, dict(max_new=60, max_length=6000), id="one row tile joined"),
    pytest.param(300, 900, dict(max_new=300, max_length=900), id="two row tiles"),
    pytest.param(300, 900, dict(max_new=40, max_length=900), id="one row tile, groups in turn"),
    pytest.param(300, 900, dict(max_new=70, max_length=900), id="two row tiles, groups in turn"),
    pytest.param(300, 5000, dict(max_new=300, max_length=5000), id="two row tiles joined"),
]


def store(b, s):
    """Sequence s's keys and values to its pages."""
    pos = torch.arange(b.lengths[s], device=b.device)
    at = b.table[s][pos // b.page].long(), slice(None), pos % b.page
    b.k[at], b.v[at] = b.keys[s], b.values[s]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 128), (torch.float16, 64)])
@pytest.mark.parametrize("new,length,hints", PLANS)
def test_scores_of_minus_infinity(cuda, dtype, dim, new, length, hints):
    """Rows that see such scores alone are NaN, as softmax has it; beside others these keys weigh nothing; a row
    without keys stays 0."""
    b = Batch([new, new, new, 2], [length, length, new, 1], 2, dim, 32, dtype, cuda, seed=24)
    q = b.normal(4, 2.0)
    q[..., 1] = q[..., 1].abs() + 0.5
    b.keys[0][..., 1] = -math.inf              # every key
    b.keys[1][:length - new // 2 - 1, 1, 1] = -math.inf  # one kv head; the last rows see others
    b.keys[2][:new // 2, 0, 1] = -math.inf        # from the sequence's start
    for s in range(3):
        store(b, s)
    out, size = exact_attention(b, q)
    assert out[:new].isnan().all() and out[3 * new - 1].isfinite().all() and (out[-2] == 0).all() and out[-1].isfinite().all()
    assert_attention(b.cache().attend(q, b.starts, b.lens, b.table, **hints), out, size)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 128), (torch.float16, 64)])
@pytest.mark.parametrize("new,length,hints", PLANS)
def test_values_that_are_not_finite(cuda, dtype, dim, new, length, hints):
    """inf and NaN in places that rows of one tile, of both, of one part or of all see: they reach the rows that see
    them, in their column, and no others."""
    b = Batch([new, new, 3], [length, new, 40], 2, dim, 32, dtype, cuda, seed=25)
    for s in (0, 1):
        n = b.lengths[s]
        p = n - new  # the first new row's position
        marks = [[(n - 1, math.nan)], [(n - 1, math.inf)], [(p + new // 2, -math.inf)], [(p + min(10, new - 1), math.inf)],
                 [(p, math.inf), (n - 1, -math.inf)], [(n // 3, math.inf)], [(n // 3, math.inf), (n - 1, -math.inf)],
                 [(min(p + 70, n - 1), math.nan)], [(n // 2, math.nan)], [(n // 2, -math.inf), (min(p + 150, n - 1), -math.inf)]]
        for column, places in enumerate(marks):
            for at, value in places:
                b.values[s][at, column % 2, column if column % 3 else dim - 1 - column] = value
        store(b, s)
    q = b.normal(4, 2.0)
    out, size = exact_attention(b, q)
    assert out.isnan().any() and out.isinf().any() and out[-3:].isfinite().all()
    cache = b.cache()
    assert_attention(cache.attend(q, b.starts, b.lens, b.table, **hints), out, size)
    cache.check_device_status()


@pytest.mark.gpu
@pytest.mark.parametrize("new,length,hints", PLANS)
def test_keys_that_are_not_finite(cuda, new, length, hints):
    """A NaN score makes the rows that see it NaN, one of +inf too (inf - inf); rows before them are as ever."""
    b = Batch([new, new, new], [length, length, new], 1, 64, 16, torch.float16, cuda, seed=26)
    q = b.normal(3, 2.0)
    q[..., 9] = q[..., 9].abs() + 0.5
    b.keys[0][length - (new + 1) // 2, 0, 9] = math.nan
    b.keys[1][length // 2, 0, 9] = math.inf
    b.keys[2][0, 0, 9] = math.nan
    for s in range(3):
        store(b, s)
    out = b.cache().attend(q, b.starts, b.lens, b.table, **hints)
    want = exact_attention(b, q)
    for s, first in enumerate((length - (new + 1) // 2, length // 2, 0)):
        first = max(first - (b.lengths[s] - new), 0)  # new rows before the key
        assert out[s * new + first:(s + 1) * new].isnan().all()
        assert_attention(out[s * new:s * new + first], *(x[s * new:s * new + first] for x in want))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("new,length,hints", PLANS)
def test_huge_scores(cuda, dtype, new, length, hints):
    """Whole-number scores times 2^20: exact in fp32, up to 2^36; each row's weight is shared by its largest."""
    b = Batch([new], [length], 1, 64, 64, dtype, cuda, seed=27)
    g = torch.Generator(device=cuda).manual_seed(1)
    b.keys[0] = torch.randint(-32, 33, (length, 1, 64), generator=g, device=cuda).to(dtype)
    store(b, 0)
    q = torch.randint(-32, 33, (new, 2, 64), generator=g, device=cuda).to(dtype)
    got = b.cache().attend(q, b.starts, b.lens, b.table, scale=2.0 ** 20, **hints)
    assert_attention(got, *exact_attention(b, q, 2.0 ** 20))


@pytest.mark.gpu
@pytest.mark.parametrize("new,length,hints", PLANS)
def test_a_missing_page(cuda, new, length, hints):
    """Ids that the cache does not have are reported; the rows before them and the other sequences are as ever."""
    P = pkg()
    b = Batch([new, new], [length, length], 2, 64, 32, torch.bfloat16, cuda, seed=28)
    cache, q = b.cache(), b.normal(4, 2.0)
    want = exact_attention(b, q)
    last = (length - 1) // 32
    before = max(last * 32 - (length - new), 0)  # sequence 0's rows that do not reach its last page
    for spoil in (GARBAGE, -1, b.k.shape[0]):
        table = b.table.clone()
        table[0, last] = spoil
        out = cache.attend(q, b.starts, b.lens, table, **hints)
        with pytest.raises(P._lib.PPMoEError, match="without a page"):
            cache.check_device_status()
        assert_attention(out[:before], *(x[:before] for x in want))
        assert_attention(out[new:], *(x[new:] for x in want))
    cache.check_device_status()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 128), (torch.float16, 64)])
@pytest.mark.parametrize("new,length,hints", PLANS)
def test_infinite_values_of_vanishing_weight(cuda, dtype, dim, new, length, hints):
    """An infinity that a row sees reaches it however small its weight is, and however that came about: its own score
    2^-200 of the row's largest or -inf, a later key that takes all the weight, a part that weighs nothing beside another."""
    b = Batch([new, new, 1], [length, new, 9], 2, dim, 32, dtype, cuda, seed=29)
    q = b.normal(4, 2.0)
    q[..., 2] = 32.0
    for s in (0, 1):
        n = b.lengths[s]
        p = n - new
        k, v = b.keys[s], b.values[s]
        k[..., 2] = 0.0
        low, early, high, late = n // 3, n // 4, p + new // 2, p + min(10, new - 1)
        k[low, :, 2], k[high, :, 2] = -64.0, 64.0
        v[low, 0, 0], v[low, 1, 0] = math.inf, -math.inf
        v[early, :, 1] = math.inf
        v[late, 0, 3] = math.inf
        v[low, 0, 4], v[early, 0, 4] = math.inf, -math.inf
        v[early, 1, 5], v[late, 1, 5] = -math.inf, -math.inf
        if n > 40:
            k[n // 5, :, 2], v[n // 5, 0, 6] = -math.inf, math.inf
        store(b, s)
    out, size = exact_attention(b, q)
    assert out[-2].isinf().any() and out[-1].isfinite().all()
    got = b.cache().attend(q, b.starts, b.lens, b.table, **hints)
    assert_attention(got, out, size)
    assert torch.equal(b.cache().attend(q, b.starts, b.lens, b.table, out=q, **hints).isnan(), out.isnan())  # (q: read again)
    assert_attention(q, out, size)


@pytest.mark.gpu
def test_a_missing_page_on_another_stream(cuda):
    """The status is that of every call before it, on whichever stream."""
    b = Batch([2], [20], 1, 64, 16, torch.bfloat16, cuda, seed=31)
    cache, k, v = b.cache(), b.normal(1), b.normal(1)
    cache.append(None, k, v, b.starts, b.lens, b.table)
    cache.check_device_status()
    nowhere = torch.full_like(b.table, -1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(50_000_000)  # some 25 ms
        cache.append(None, k, v, b.starts, b.lens, nowhere)
    with pytest.raises(pkg()._lib.PPMoEError, match="without a page"):
        cache.check_device_status()
    cache.check_device_status()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("new,length,hints", PLANS)
def test_a_scale_of_zero(cuda, dtype, new, length, hints):
    """The mean of the values; queries that are not finite are no less so for it (0 * inf, 0 * NaN)."""
    b = Batch([new], [length], 1, 64, 32, dtype, cuda, seed=30)
    q = b.normal(4, 2.0)
    q[:, 1, 5], q[:, 2, 60] = math.nan, -math.inf
    q[0, 3, 0] = math.inf
    got = b.cache().attend(q, b.starts, b.lens, b.table, scale=0.0, **hints)
    out, size = exact_attention(b, q.nan_to_num(0.0, 0.0, 0.0), 0.0)
    assert got[:, 1:3].isnan().all() and got[0, 3].isnan().all()
    assert_attention(got[:, 0], out[:, 0], size[:, 0])
    assert_attention(got[1:, 3], out[1:, 3], size[1:, 3])
