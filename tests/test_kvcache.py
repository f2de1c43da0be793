"""Paged key/value cache: append and attention against fp64, alone and as a decoder uses them; refusals."""
import ctypes
import math

import pytest
import torch

from conftest import pkg
from paged_helpers import GARBAGE, Batch, assert_attention, assert_rotation, exact_attention, exact_rotation, half_step

HEADS = [(12, 12), (8, 2), (8, 1), (15, 3)]


def emb(*a, **k):
    return pkg().rotary.RotaryEmbedding(*a, **k)


# ------------------------------------------------------------------ CPU
def test_constructor_refusals():
    C = pkg().kvcache.PagedKVCache
    for bad in [dict(num_pages=0), dict(page_size=8), dict(page_size=48), dict(page_size=512), dict(kv_heads=0), dict(head_dim=96)]:
        with pytest.raises(ValueError):
            C(**{**dict(num_pages=4, page_size=16, kv_heads=2, head_dim=64, device="cpu"), **bad})
    with pytest.raises(TypeError):
        C(4, 16, 2, 64, dtype=torch.float32, device="cpu")
    with pytest.raises(RuntimeError, match="CUDA only"):
        C(4, 16, 2, 64, device="cpu")
    k = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    for bad in [(k, k[:3]), (k, k.half()), (k[0], k[0]), (k[:0], k[:0]), (k[..., :32], k[..., :32]),
                (k[:1].expand(4, 2, 16, 64), k), (k, k.transpose(2, 3).contiguous().transpose(2, 3))]:
        with pytest.raises(ValueError):
            C.from_tensors(*bad)


def test_host_validation_without_gpu():
    lib = pkg()._lib.load()

    def cache(page=16, dim=64, num=4, kvh=2, k=1024, dtype=0, status=256):
        return ctypes.byref(pkg()._lib.KVCache(k, 1024, 2048, 1024, 64, 2048, 1024, 64, num, page, kvh, dim, dtype, status))

    rotation = pkg()._lib.Rotation(64, 0, 1.0)

    def append(tokens=1, batch=1, mp=4, rot=None, k=16, starts=16, null=False, **c):
        rotation.rotary_dim = rot or 0
        return lib.ppmoe_kv_append(None if null else cache(**c), None if rot is None else ctypes.byref(rotation), None, 0, 0, None,
                                   0, 0, 0, k, 128, 64, 16, 128, 64, tokens, starts, 16, 16, mp, batch, mp, None)

    def attend(tokens=1, hq=4, q=16, batch=1, new=1, length=64, scale=0.125, ws=None, n=0, null=False, **c):
        return lib.ppmoe_attend(None if null else cache(**c), q, 256, 64, hq, tokens, 16, 16, 16, 4, batch, 4, scale, new, length,
                                16, 256, 64, ws, n, None)

    for call in (append, attend):
        assert call(tokens=0) == 0  # nothing to do: no launch
        assert call(null=True) == -1 and call(page=8) == -2 and call(page=24) == -2 and call(page=512) == -2
        assert call(dim=96) == -2 and call(dtype=2) == -2 and call(num=0) == -1 and call(kvh=0) == -1
        assert call(k=1032) == -1 or call is append  # (append's k are the new rows)
        assert call(status=None) == -1 and call(batch=0) == -1 and call(tokens=-1) == -1
    assert append(mp=0) == -1 and append(starts=None) == -1 and append(k=None) == -1
    assert append(rot=66) == -2 and append(rot=3) == -2
    assert attend(hq=3) == -1 and attend(hq=0) == -1 and attend(q=None) == -1
    assert attend(scale=math.inf) == -1 and attend(scale=math.nan) == -1 and attend(scale=3e38) == -1
    assert attend(batch=1 << 20) == -2 and attend(tokens=1 << 30) == -2
    n = lib.ppmoe_attend_workspace_bytes(1, 4, 2, 64, 1, 1, 64 * 1024)
    assert n > 0 and attend(length=64 * 1024) == -5 and attend(length=64 * 1024, ws=1024, n=n - 1) == -5
    assert attend(length=64 * 1024, ws=1040, n=n) == -5 and b"workspace" in lib.ppmoe_last_error()
    for odd in [(0, 4, 2, 64, 1, 1, 64), (1, 4, 0, 64, 1, 1, 64), (1, 1, 2, 64, 1, 1, 64), (1, 4, 2, 64, 0, 1, 64)]:
        assert lib.ppmoe_attend_workspace_bytes(*odd) == 0
    assert lib.ppmoe_attend_workspace_bytes(1, 4, 2, 64, 1, -5, -7) == lib.ppmoe_attend_workspace_bytes(1, 4, 2, 64, 1, 1, 1)


# ------------------------------------------------------------------ GPU: append
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("page,dim,rot,layout", [(16, 128, 128, "half"), (64, 64, 32, "interleaved"), (256, 128, 4, "half"), (32, 64, 0, "half")])
@pytest.mark.parametrize("hq,hk", HEADS)
def test_append(cuda, dtype, page, dim, rot, layout, hq, hk):
    """Every row lands rotated in its place and nothing else changes; rows behind the last sequence, and
    their outputs, are left as they were."""
    e = emb(dim, rotary_dim=rot, layout=layout) if rot else None
    b = Batch([3, 0, 40, 1, 257], [3, 9, 100, 640, 1000], hk, dim, page, dtype, cuda, seed=1, pad=5)
    cache = b.cache()
    fused = b.normal(hq + 2 * hk)
    q, k, v = fused[:, :hq], fused[:, hq:hq + hk], fused[:, hq + hk:]
    out = torch.full_like(q.contiguous(), 7.0)
    want_k, want_v = b.k.clone(), b.v.clone()
    got = cache.append(q, k, v, b.starts, b.lens, b.table, rotary=e, out=out)
    assert got is out
    t = 0
    for s, (n, length) in enumerate(zip(b.new, b.lengths)):
        pos = torch.arange(length - n, length, device=cuda)
        pg, row = b.table[s][pos // page].long(), pos % page
        if e is not None:
            assert_rotation(out[t:t + n], *exact_rotation(e, q[t:t + n], pos))
            assert_rotation(b.k[pg, :, row], *exact_rotation(e, k[t:t + n], pos))
        else:
            assert torch.equal(out[t:t + n], q[t:t + n]) and torch.equal(b.k[pg, :, row], k[t:t + n])
        assert torch.equal(b.v[pg, :, row], v[t:t + n])
        want_k[pg, :, row], want_v[pg, :, row] = b.k[pg, :, row], b.v[pg, :, row]
        t += n
    assert torch.equal(b.k.view(torch.int16), want_k.view(torch.int16))
    assert torch.equal(b.v.view(torch.int16), want_v.view(torch.int16))
    assert (out[t:] == 7).all()
    cache.check_device_status()


@pytest.mark.gpu
def test_append_layouts_and_alignment(cuda):
    """[page, row, head] storage, no queries, in-place queries, rows at 2-byte offsets."""
    e = emb(64)
    b = Batch([20, 7], [30, 40], 2, 64, 16, torch.bfloat16, cuda, nhd=True)
    cache = b.cache()
    k, v, q = b.normal(2), b.normal(2), b.normal(4)
    assert cache.append(None, k, v, b.starts, b.lens, b.table, rotary=e) is None
    first = b.k.clone()
    odd = torch.zeros(27 * 2 * 64 + 1, dtype=torch.bfloat16, device=cuda)[1:].view(27, 2, 64).copy_(k)
    want = cache.append(q, odd, v, b.starts, b.lens, b.table, rotary=e)
    assert torch.equal(first.view(torch.int16), b.k.view(torch.int16))
    q2 = q.clone()
    assert cache.append(q2, k, v, b.starts, b.lens, b.table, rotary=e, out=q2) is q2
    assert torch.equal(q2, want)
    pos = torch.arange(10, 30, device=cuda)
    assert_rotation(b.k[b.table[0][pos // 16].long(), :, pos % 16], *exact_rotation(e, k[:20], pos))


@pytest.mark.gpu
@pytest.mark.parametrize("batch", [1, 31, 32, 33, 1000, 1025, 3000])
def test_append_many_sequences(cuda, batch):
    """The search for a row's sequence, empty sequences among them."""
    r = torch.Generator().manual_seed(batch)
    new = torch.randint(0, 3, (batch,), generator=r).tolist()
    new[0] += 1
    b = Batch(new, [n + 5 for n in new], 1, 64, 16, torch.bfloat16, cuda)
    cache = b.cache()
    k, v = b.normal(1), b.normal(1)
    cache.append(None, k, v, b.starts, b.lens, b.table)
    seq = torch.repeat_interleave(torch.arange(batch, device=cuda), torch.tensor(new, device=cuda))
    pos = 5 + torch.arange(b.tokens, device=cuda) - b.starts[seq].long()
    assert torch.equal(b.k[b.table[seq, pos // 16].long(), :, pos % 16], k)
    assert torch.equal(b.v[b.table[seq, pos // 16].long(), :, pos % 16], v)


@pytest.mark.gpu
def test_append_without_a_page(cuda):
    """Negative positions, positions behind the table, ids the cache does not have: not stored, reported."""
    P = pkg()
    cache = P.kvcache.PagedKVCache(4, 16, 1, 64, device=cuda)
    k = torch.ones(3, 1, 64, dtype=torch.bfloat16, device=cuda)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    for lengths, table in [([2], [[0, 1]]), ([34], [[0, 1]]), ([3], [[-1, 1]]), ([3], [[4, 1]]), ([3], [[GARBAGE, 1]])]:
        cache.k.zero_()
        cache.append(None, k, k, i32(0, 3), i32(*lengths), i32(*table))
        with pytest.raises(P._lib.PPMoEError, match="without a page"):
            cache.check_device_status()
        cache.check_device_status()  # cleared
        stored = {2: 2, 34: 1, 3: 0}[lengths[0]]
        assert int((cache.k != 0).any(-1).sum()) == stored


# ------------------------------------------------------------------ GPU: attention
BATCHES = {
    "one": ([1], [1]),
    "one page": ([1], [16]),
    "a key more": ([1], [17]),
    "steps": ([1] * 7, [1, 15, 16, 17, 128, 129, 1000]),
    "steps, some idle": ([1, 0, 1, 0], [500, 7, 3, 0]),
    "proposals": ([5, 1, 3, 4], [300, 1, 129, 4]),
    "prompts": ([130, 17, 64], [130, 17, 64]),
    "a prompt": ([257], [257]),
    "chunks": ([40, 0, 130, 1], [100, 9, 700, 641]),
    "a chunk": ([300], [1500]),
    "positions before the start": ([6, 140, 2], [4, 100, 0]),
}


@pytest.mark.gpu
@pytest.mark.parametrize("name", BATCHES)
@pytest.mark.parametrize("dtype,dim,page", [(torch.bfloat16, 128, 16), (torch.float16, 64, 32), (torch.bfloat16, 64, 256), (torch.float16, 128, 64)])
@pytest.mark.parametrize("hq,hk", HEADS)
def test_attend(cuda, name, dtype, dim, page, hq, hk):
    """Every row against fp64, with NaN in all places of the cache that no position has, and padding
    rows left as they were."""
    new, lengths = BATCHES[name]
    b = Batch(new, lengths, hk, dim, page, dtype, cuda, seed=3, pad=2)
    cache = b.cache()
    q = b.normal(hq, 2.0)
    out = torch.full_like(q, 7.0)
    cache.attend(q, b.starts, b.lens, b.table, max_new=max(new), max_length=max(lengths), out=out)
    n = sum(new)
    assert (out[n:] == 7).all()
    assert_attention(out[:n], *(x[:n] for x in exact_attention(b, q)), what=name)
    cache.check_device_status()


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hk", [(34, 1), (144, 1), (21, 7), (16, 1), (17, 1)])
@pytest.mark.parametrize("new", [1, 9])
def test_attend_group_sizes(cuda, hq, hk, new):
    b = Batch([new, 1], [200, 333], hk, 64, 16, torch.bfloat16, cuda, seed=4)
    q = b.normal(hq, 2.0)
    assert_attention(b.cache().attend(q, b.starts, b.lens, b.table, max_new=new), *exact_attention(b, q))


@pytest.mark.gpu
@pytest.mark.parametrize("page", [16, 128, 256])
@pytest.mark.parametrize("new,length,hq,hk", [(1, 40001, 4, 2), (16, 20003, 4, 2), (64, 9000, 2, 1), (200, 5000, 4, 2), (700, 2777, 3, 1)])
def test_attend_long(cuda, page, new, length, hq, hk):
    """Few rows over a long axis (split work), chunks behind a long context."""
    b = Batch([new, min(new, 2)], [length, 301], hk, 128, page, torch.bfloat16, cuda, seed=5)
    q = b.normal(hq, 1.5)
    assert_attention(b.cache().attend(q, b.starts, b.lens, b.table, max_new=new, max_length=length), *exact_attention(b, q))


@pytest.mark.gpu
def test_hints_never_change_what_is_computed(cuda):
    """max_new and max_length too small, too large and absent."""
    b = Batch([130, 1, 20], [700, 3000, 20], 2, 128, 32, torch.bfloat16, cuda, seed=6)
    cache, q = b.cache(), b.normal(8, 2.0)
    want = exact_attention(b, q)
    for hints in [{}, dict(max_new=1, max_length=1), dict(max_new=1, max_length=3000), dict(max_new=130, max_length=16),
                  dict(max_new=4, max_length=10**9), dict(max_new=10**9, max_length=3000), dict(max_new=40, max_length=100)]:
        out = torch.full_like(q, 7.0)
        assert_attention(cache.attend(q, b.starts, b.lens, b.table, out=out, **hints), *want, what=str(hints))


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 40])
def test_attend_strides_and_scale(cuda, new):
    """Queries inside a fused projection, [page, row, head] storage, an output with gaps, a scale of its own."""
    b = Batch([new, 1], [90, 250], 2, 128, 16, torch.float16, cuda, seed=7, nhd=True)
    fused = b.normal(8, 1.0)
    q = fused[:, 1:5]
    wide = torch.full((b.tokens, 6, 128), 7.0, dtype=torch.float16, device=cuda)
    out = b.cache().attend(q, b.starts, b.lens, b.table, scale=0.21, out=wide[:, 1:5], max_new=new)
    assert_attention(out, *exact_attention(b, q, 0.21))
    assert (wide[:, 0] == 7).all() and (wide[:, 5] == 7).all()
    odd = torch.zeros(q.numel() + 1, dtype=torch.float16, device=cuda)[1:].view(q.shape).copy_(q)
    gap = torch.zeros(q.numel() + 1, dtype=torch.float16, device=cuda)[1:].view(q.shape)
    assert torch.equal(b.cache().attend(odd, b.starts, b.lens, b.table, scale=0.21, out=gap, max_new=new), out)


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 5, 40, 300])
def test_attend_wide_ranges(cuda, new):
    """Scores that grow along the keys (the running maximum moves at every step), large negative ones,
    and one key that takes all the weight."""
    b = Batch([new], [900], 1, 128, 64, torch.bfloat16, cuda, seed=8)
    q = torch.zeros(new, 2, 128, dtype=torch.bfloat16, device=cuda)
    q[:, 0, 0], q[:, 1, 0] = 8.0, -8.0
    k = b.keys[0]
    k.zero_()
    k[:, 0, 0] = torch.arange(900, device=cuda) // 4
    pos = torch.arange(900, device=cuda)
    b.k[b.table[0][pos // 64].long(), :, pos % 64] = k
    assert_attention(b.cache().attend(q, b.starts, b.lens, b.table, scale=1.0, max_new=new), *exact_attention(b, q, 1.0))
    assert_attention(b.cache().attend(q, b.starts, b.lens, b.table, scale=-0.01, max_new=new), *exact_attention(b, q, -0.01))
    assert_attention(b.cache().attend(q, b.starts, b.lens, b.table, scale=0.0, max_new=new), *exact_attention(b, q, 0.0))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dim,page", [(torch.bfloat16, 128, 16), (torch.float16, 64, 128)])
@pytest.mark.parametrize("new,hint", [(5, 5), (40, 40), (40, 1), (150, 150)])
def test_values_that_are_not_finite(cuda, dtype, dim, page, new, hint):
    """inf and NaN among the newest values and keys reach the rows that see them and no others."""
    b = Batch([new, new], [new + 230, new], 2, dim, page, dtype, cuda, seed=13)
    for s in (0, 1):
        n = b.lengths[s]
        k, v = b.keys[s], b.values[s]
        v[n - 1, 0, 3] = math.nan
        v[n - 1, 1, dim - 1] = math.inf
        v[n - 2, 1, 0], v[n - 2, 1, 1] = -math.inf, math.inf
        v[n - new // 2, 0, 5] = math.inf
        v[n - new // 2 + 1, 0, 5] = -math.inf
        k[n - 1, 1, 7] = math.nan  # the last row's scores
        pos = torch.arange(n, device=cuda)
        at = b.table[s][pos // page].long(), slice(None), pos % page
        b.k[at], b.v[at] = k, v
    q = b.normal(4, 2.0)
    out, size = exact_attention(b, q)
    assert out.isfinite().any() and not out.isfinite().all()
    assert_attention(b.cache().attend(q, b.starts, b.lens, b.table, max_new=hint), out, size)


@pytest.mark.gpu
@pytest.mark.parametrize("new,hint", [(1, 1), (5, 5), (40, 40), (150, 150), (150, 1)])
def test_a_key_that_is_not_a_number(cuda, new, hint):
    """NaN in a sequence's first key: every row of it is NaN, also one that sees no other key; the other
    sequence is as ever."""
    b = Batch([new, new], [new, 300], 1, 64, 16, torch.float16, cuda, seed=14)
    b.keys[0][0, 0, 9] = math.nan
    b.k[b.table[0, 0].long(), 0, 0, 9] = math.nan
    q = b.normal(3, 2.0)
    out = b.cache().attend(q, b.starts, b.lens, b.table, max_new=hint)
    assert out[:new].isnan().all()
    want = exact_attention(b, q)
    assert_attention(out[new:], want[0][new:], want[1][new:])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("new", [1, 20, 200])
def test_attend_huge_scores(cuda, dtype, new):
    """Whole-number scores times 2^20: exact in fp32, up to 2^36; each row's weight is shared by its largest."""
    b = Batch([new], [new + 500], 1, 64, 64, dtype, cuda, seed=15)
    g = torch.Generator(device=cuda).manual_seed(1)
    b.keys[0] = torch.randint(-32, 33, (new + 500, 1, 64), generator=g, device=cuda).to(dtype)
    pos = torch.arange(new + 500, device=cuda)
    b.k[b.table[0][pos // 64].long(), :, pos % 64] = b.keys[0]
    q = torch.randint(-32, 33, (new, 2, 64), generator=g, device=cuda).to(dtype)
    assert_attention(b.cache().attend(q, b.starts, b.lens, b.table, scale=2.0 ** 20, max_new=new), *exact_attention(b, q, 2.0 ** 20))


@pytest.mark.gpu
@pytest.mark.parametrize("new,length", [(1, 3000), (1, 40000), (20, 3000), (200, 900)])
def test_attend_in_place_of_q(cuda, new, length):
    b = Batch([new, 1], [length, 50], 2, 128, 32, torch.bfloat16, cuda, seed=16)
    q = b.normal(6, 2.0)
    want = b.cache().attend(q, b.starts, b.lens, b.table, max_new=new)
    assert b.cache().attend(q, b.starts, b.lens, b.table, max_new=new, out=q) is q
    assert torch.equal(q, want)


@pytest.mark.gpu
def test_copies_and_gradients(cuda):
    import copy
    import pickle
    b = Batch([4], [40], 2, 64, 16, torch.bfloat16, cuda, seed=17)
    cache, q, e = b.cache(), b.normal(4), emb(64)
    k, v = b.normal(2), b.normal(2)
    cache2, e2 = copy.deepcopy(cache), copy.deepcopy(e)
    e3 = pickle.loads(pickle.dumps(e))
    want = cache.append(q, k, v, b.starts, b.lens, b.table, rotary=e)
    del e
    for other in (e2, e3):
        assert torch.equal(cache2.append(q, k, v, b.starts, b.lens, b.table, rotary=other), want)
    assert cache2.k.data_ptr() != cache.k.data_ptr() and torch.equal(cache2.k.view(torch.int16), cache.k.view(torch.int16))
    with pytest.raises(AttributeError):
        cache.k = cache2.k
    q.requires_grad_()
    for call in (lambda: cache.attend(q, b.starts, b.lens, b.table), lambda: cache.append(q, k, v, b.starts, b.lens, b.table)):
        with pytest.raises(RuntimeError, match="no_grad"):
            call()
        with torch.no_grad():
            call()


@pytest.mark.gpu
def test_rows_before_the_first_sequence(cuda):
    """starts need not begin at 0: rows before it are nobody's."""
    b = Batch([3, 2], [50, 60], 1, 64, 16, torch.float16, cuda, seed=18, pad=4)
    q = b.normal(2, 2.0)
    shifted = torch.cat([q[-2:], q[:-2]])
    for new in (1, 16, 40):
        out = torch.full_like(q, 7.0)
        b.cache().attend(shifted, b.starts + 2, b.lens, b.table, max_new=new, out=out)
        assert (out[:2] == 7).all() and (out[7:] == 7).all()
        assert_attention(out[2:7], *(x[:5] for x in exact_attention(b, q)))


@pytest.mark.gpu
def test_offsets_beyond_32_bits(cuda):
    """A cache of more than 2^31 values whose used pages lie at its end."""
    pages, page, hk = 140_000, 256, 1
    C = pkg().kvcache.PagedKVCache
    k = torch.empty(pages, hk, page, 64, dtype=torch.bfloat16, device=cuda)
    v = torch.empty_like(k)
    assert k.numel() > 2**31
    g = torch.Generator(device=cuda).manual_seed(1)
    b = Batch([1, 40], [600, 500], hk, 64, page, torch.bfloat16, cuda, seed=9)
    used = b.k.shape[0]
    b.table = torch.where(b.table == GARBAGE, b.table, b.table + (pages - used))
    k[-used:], v[-used:] = b.k, b.v
    cache = C.from_tensors(k, v)
    q = b.normal(4, 2.0)
    for hint in (1, 40):
        assert_attention(cache.attend(q, b.starts, b.lens, b.table, max_new=hint), *exact_attention(b, q))
    nk, nv = b.normal(1), b.normal(1)
    cache.append(None, nk, nv, b.starts, b.lens, b.table)
    assert torch.equal(k[b.table[0, 2].long(), 0, 599 % 256], nk[0, 0]) and torch.equal(v[b.table[1, 1].long(), 0, 499 % 256], nv[40, 0])
    del k, v, cache
    torch.cuda.empty_cache()


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 40])
def test_attend_without_a_page(cuda, new):
    """Lengths beyond the table and ids that the cache does not have are reported; other sequences are
    computed as ever."""
    P = pkg()
    b = Batch([new, new], [100, 90], 1, 64, 16, torch.bfloat16, cuda, seed=10)
    cache, q = b.cache(), b.normal(2, 2.0)
    want = exact_attention(b, q)
    for spoil in ("id", "negative", "length"):
        table, lens = b.table.clone(), b.lens.clone()
        if spoil == "length":
            lens[0] = 10_000
        else:
            table[0, 2] = GARBAGE if spoil == "id" else -1
        out = cache.attend(q, b.starts, lens, table, max_new=new)
        with pytest.raises(P._lib.PPMoEError, match="without a page"):
            cache.check_device_status()
        assert_attention(out[new:], want[0][new:], want[1][new:])
    cache.check_device_status()


@pytest.mark.gpu
def test_same_bits_every_time(cuda):
    b = Batch([1, 1, 5, 300], [9000, 17, 4000, 2000], 2, 128, 32, torch.bfloat16, cuda, seed=11)
    cache, q = b.cache(), b.normal(8, 2.0)
    for new in (1, 16, 300):
        first = cache.attend(q, b.starts, b.lens, b.table, max_new=new)
        for _ in range(5):
            assert torch.equal(first, cache.attend(q, b.starts, b.lens, b.table, max_new=new))


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 20])
def test_graphs_and_streams(cuda, new):
    """Two captured calls on one cache replayed at once on two streams, following the batch's contents."""
    b = Batch([new, new], [3000, 2000], 2, 128, 32, torch.bfloat16, cuda, seed=12)
    cache, q1 = b.cache(), b.normal(8, 2.0)
    q2 = b.normal(8, 1.0)
    lens = b.lens.clone()
    cache.attend(q1, b.starts, lens, b.table, max_new=new)
    graphs, outs = [], []
    for q in (q1, q2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(cache.attend(q, b.starts, lens, b.table, max_new=new, max_length=3000))
        graphs.append(g)
    lens.copy_(torch.tensor([2500, 1900], device=cuda))
    shorter = Batch([new, new], [3000, 2000], 2, 128, 32, torch.bfloat16, cuda, seed=12)
    shorter.lengths = [2500, 1900]
    shorter.keys = [k[:n] for k, n in zip(shorter.keys, shorter.lengths)]
    shorter.values = [v[:n] for v, n in zip(shorter.values, shorter.lengths)]
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for q, out in zip((q1, q2), outs):
        assert_attention(out, *exact_attention(shorter, q))


@pytest.mark.gpu
def test_refusals(cuda):
    b = Batch([3, 1], [30, 20], 2, 64, 16, torch.bfloat16, cuda)
    cache, q = b.cache(), b.normal(4)
    k = b.normal(2)
    ok = (b.starts, b.lens, b.table)
    for bad in [(b.starts.long(), b.lens, b.table), (b.starts, b.lens.cpu(), b.table), (b.starts[:-1], b.lens, b.table),
                (b.starts, b.lens, b.table[:1]), (b.starts, b.lens, b.table[0]), (b.starts, b.lens, b.table[:, :0]),
                (b.starts[:1], b.lens[:0], b.table[:0]), (b.starts, b.lens, b.table.repeat(1, 2)[:, ::2])]:
        with pytest.raises(ValueError):
            cache.attend(q, *bad)
        with pytest.raises(ValueError):
            cache.append(q, k, k, *bad)
    for bad in [q[:, :3], q[..., :32], q.half(), q[0], q.cpu(), q[:, :0]]:
        with pytest.raises(ValueError):
            cache.attend(bad, *ok)
    for out in [q[:3], q.half(), torch.empty(4, 4, 64, device=cuda, dtype=torch.bfloat16).cpu(), k[:, :1].expand(4, 4, 64)]:
        with pytest.raises(ValueError):
            cache.attend(q, *ok, out=out)
    for args in [(q, k, k[:3]), (q[:3], k, k), (q, q, q), (q, k[:, :1], k)]:
        with pytest.raises(ValueError):
            cache.append(*args, *ok)
    with pytest.raises(ValueError):
        cache.append(q, k, k, *ok, rotary=emb(128))
    with pytest.raises(ValueError):
        cache.append(None, k, k, *ok, out=q)
    with pytest.raises(RuntimeError):
        cache.attend(q, *ok, out=torch.empty_like(q).requires_grad_())
    with pytest.raises(ValueError):
        type(cache).from_tensors(b.k.clone().requires_grad_(), b.v)
    version = q._version
    cache.attend(q, *ok, out=q)
    assert q._version > version
    with torch.inference_mode():
        x = q * 1
        cache.attend(x, *ok, out=x)


# ------------------------------------------------------------------ GPU: together
@pytest.mark.gpu
@pytest.mark.parametrize("dtype,hq,hk,dim", [(torch.bfloat16, 12, 12, 128), (torch.float16, 8, 2, 64)])
def test_chunks_and_steps_together(cuda, dtype, hq, hk, dim):
    """Prompts taken in chunks and then token by token, appended and attended in turn, against causal
    attention in fp64 over the same rotated keys."""
    e = emb(dim)
    cache = pkg().kvcache.PagedKVCache(64, 16, hk, dim, dtype=dtype, device=cuda)
    g = torch.Generator(device=cuda).manual_seed(1)
    total = [150, 61]
    q, k, v = ([torch.randn(n, h, dim, generator=g, device=cuda).to(dtype) for n in total] for h in (hq, hk, hk))
    table = torch.randperm(64, generator=g, device=cuda)[:2 * 12].view(2, 12).to(torch.int32)
    done = [0, 0]
    outs = [[], []]
    for new in [(40, 40), (90, 1), (0, 9), (1, 1), (1, 1), (3, 0), (1, 1), (14, 8)]:
        cut = lambda x: torch.cat([x[s][done[s]:done[s] + new[s]] for s in (0, 1)])  # noqa: E731
        starts = torch.tensor([0, new[0], sum(new)], dtype=torch.int32, device=cuda)
        rows = cut(q), cut(k), cut(v)
        done = [done[s] + new[s] for s in (0, 1)]
        lens = torch.tensor(done, dtype=torch.int32, device=cuda)
        q2 = cache.append(*rows, starts, lens, table, rotary=e)
        o = cache.attend(q2, starts, lens, table, max_new=max(new), max_length=max(done))
        outs[0].append(o[:new[0]])
        outs[1].append(o[new[0]:])
    assert done == total
    for s in (0, 1):
        pos = torch.arange(total[s], device=cuda)
        # the rows as stored: rotated, rounded once
        qr, kr = e(q[s], k[s], pos)
        whole = Batch([total[s]], [total[s]], hk, dim, 16, dtype, cuda)
        whole.keys, whole.values = [kr], [v[s]]
        assert_attention(torch.cat(outs[s]), *exact_attention(whole, qr))


@pytest.mark.gpu
@pytest.mark.parametrize("batch", [1, 4])
def test_decoder_on_pages(cuda, batch):
    """SyntheticDecoder(kv="paged"): captured steps give the eager ones' tokens; every attention it ran agrees
    with fp64 over the keys and values that its cache held then."""
    import importlib
    D = importlib.import_module(pkg().__name__ + ".decoder")
    cfg = D.DecoderConfig(layers=2, hidden=256, heads=2, head_dim=128, vocab=1000, experts=16, group=32, max_seq=70, kv="paged")
    d = D.SyntheticDecoder(cfg, cuda, seed=3, max_batch=4)
    ids = torch.randint(0, 1000, (batch, 20), generator=torch.Generator().manual_seed(1)).to(cuda)
    t_graph, _, _ = d.generate(ids, 12, use_graph=True)
    t_again, _, _ = d.generate(ids, 12, use_graph=True)
    seen, attend = [], pkg().kvcache.PagedKVCache.attend

    def record(cache, q, starts, lengths, table, **hints):
        out = attend(cache, q, starts, lengths, table, **hints)
        seen.append((q.clone(), starts, lengths.clone(), table, cache.k.clone(), cache.v.clone(), out.clone()))
        return out

    pkg().kvcache.PagedKVCache.attend = record
    try:
        t_eager, _, _ = d.generate(ids, 12, use_graph=False)
    finally:
        pkg().kvcache.PagedKVCache.attend = attend
    assert torch.equal(t_graph, t_eager) and torch.equal(t_again, t_eager) and t_eager.shape == (batch, 12)
    assert len(seen) == 2 * 12
    for q, starts, lengths, table, k, v, out in seen:
        new = (starts[1:] - starts[:-1]).tolist()
        b = Batch(new, lengths.tolist(), 2, 128, cfg.page, torch.bfloat16, cuda)
        b.keys, b.values = ([x[table[s].long()].transpose(1, 2).reshape(-1, 2, 128)[:n] for s, n in enumerate(lengths.tolist())]
                            for x in (k, v))
        assert_attention(out, *exact_attention(b, q))
    for cache in d.kv:
        cache.check_device_status()
    with pytest.raises(ValueError):
        D.SyntheticDecoder(D.DecoderConfig(layers=1, kv="other"), cuda)


@pytest.mark.gpu
def test_decoder_forms_agree(cuda):
    """Prompt and first step on pages and on the dense cache, in hidden states of one dense-MLP layer.  Both hold
    q, k, v, weights and outputs in bf16 and differ in a handful of roundings (half a step each, of values
    that a layer's sums keep at their size): within 16 half steps of the largest value."""
    import importlib
    D = importlib.import_module(pkg().__name__ + ".decoder")
    outs = []
    for kv in ("dense", "paged"):
        cfg = D.DecoderConfig(layers=1, hidden=256, heads=4, head_dim=64, vocab=500, experts=8, group=32, max_seq=64, mlp="dense", kv=kv)
        d = D.SyntheticDecoder(cfg, cuda, seed=5)
        d._logits_next = lambda x: x
        ids = torch.randint(0, 500, (3, 21), generator=torch.Generator().manual_seed(2)).to(cuda)
        x = d.prefill(ids)
        y = d._step(ids[:, 0], torch.tensor([21], device=cuda))
        outs.append((x.float(), y.float()))
    for a, b in zip(*outs):
        assert (a - b).abs().max() <= 16 * half_step(torch.bfloat16) * a.abs().max()
