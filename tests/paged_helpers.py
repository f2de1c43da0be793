"""Ragged batches over a paged cache and the fp64 definitions they are checked against."""
import math

import torch

from conftest import pkg

GARBAGE = 1_000_000_007  # a page id no cache has: it may stand wherever a sequence does not reach


def half_step(dtype):
    """Largest relative error of one rounding to `dtype`."""
    return torch.finfo(dtype).eps / 2


def rounded(y, dtype):
    """Largest error of rounding y to `dtype`: half a step, eps / 2 of the value; below the smallest normal
    number n the steps no longer shrink but stay eps n (fp16: n = 2^-14, steps of 2^-24), so half of one is
    eps / 2 of n there."""
    return half_step(dtype) * y.abs().clamp_min(torch.finfo(dtype).tiny)


class Batch:
    """`new[b]` newest rows of sequences with `lengths[b]` positions; pages in random order, NaN in every
    place of the cache that no position of a sequence has, garbage in the table behind each sequence."""

    def __init__(self, new, lengths, kv_heads, dim, page, dtype, device, seed=0, nhd=False, spare_pages=3, pad=0):
        g = torch.Generator(device=device).manual_seed(seed)
        self.new, self.lengths, self.page, self.dim, self.kv_heads = new, lengths, page, dim, kv_heads
        need = [-(-max(n, 0) // page) for n in lengths]
        total, widest = sum(need) + spare_pages, max(max(need), 1) + 1
        ids = torch.randperm(total, generator=g, device=device)
        table = torch.full((len(new), widest), GARBAGE, dtype=torch.int64, device=device)
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = ids[at:at + n]
            at += n
        self.table = table.to(torch.int32)
        self.starts = torch.tensor([0] + new, device=device).cumsum(0).to(torch.int32)
        self.lens = torch.tensor(lengths, dtype=torch.int32, device=device)
        self.tokens = sum(new) + pad
        shape = (total, page, kv_heads, dim) if nhd else (total, kv_heads, page, dim)
        self.k, self.v = (torch.full(shape, math.nan, dtype=dtype, device=device) for _ in range(2))
        if nhd:
            self.k, self.v = self.k.transpose(1, 2), self.v.transpose(1, 2)
        self.keys, self.values = [], []  # per sequence [length, kv_heads, dim]
        for b, n in enumerate(lengths):
            n = max(n, 0)
            pos = torch.arange(n, device=device)
            pg = table[b][pos // page]
            kv = torch.randn(2, n, kv_heads, dim, generator=g, device=device).to(dtype)
            self.k[pg, :, pos % page] = kv[0]
            self.v[pg, :, pos % page] = kv[1]
            self.keys.append(kv[0])
            self.values.append(kv[1])
        self.generator = g
        self.device, self.dtype = device, dtype

    def cache(self):
        return pkg().kvcache.PagedKVCache.from_tensors(self.k, self.v)

    def normal(self, heads, std=1.0):
        return (torch.randn(self.tokens, heads, self.dim, generator=self.generator, device=self.device) * std).to(self.dtype)


def exact_attention(batch, q, scale=None):
    """fp64 attention of every row, and sum_j w_j |v_j|, the scale of its rounding errors."""
    scale = batch.dim ** -0.5 if scale is None else scale
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    size = torch.zeros_like(out)
    group = q.shape[1] // batch.kv_heads
    t = 0
    for b, (n, length) in enumerate(zip(batch.new, batch.lengths)):
        k = batch.keys[b].double().repeat_interleave(group, 1)
        v = batch.values[b].double().repeat_interleave(group, 1)
        pos = torch.arange(length - n, length, device=q.device)
        s = torch.einsum("qhd,khd->hqk", q[t:t + n].double(), k) * scale
        seen = torch.arange(k.shape[0], device=q.device) <= pos[:, None]
        w = torch.softmax(s.masked_fill(~seen, -math.inf), -1)
        w = torch.where(seen.any(-1)[:, None], w, torch.zeros_like(w)) if k.shape[0] else w
        fine = v.isfinite()
        out[t:t + n] = torch.einsum("hqk,khd->qhd", w, torch.where(fine, v, 0.0))
        for j in (~fine).any(-1).any(-1).nonzero()[:, 0].tolist():  # a weight above 0 leaves inf and NaN what they are
            out[t:t + n] += torch.where(seen[:, j, None, None] & ~fine[j], v[j], 0.0)
        size[t:t + n] = torch.einsum("hqk,khd->qhd", w, torch.where(fine, v.abs(), 0.0))
        t += n
    return out, size


def assert_attention(got, out, size, what=""):
    """The weights are rounded to the type once (half a step each, relative), scores are fp32 sums: of at
    most 128 products of standard normal values, off by (128 + 3) 2^-24 scale sum |q k| < 2^-13 each, twice
    that in a weight over the sum of weights: 2^-12 with the exponential's own error; the result is
    rounded once."""
    h = half_step(got.dtype)
    tol = rounded(out, got.dtype) + (h + 2.0 ** -12) * size
    odd = ~out.isfinite()
    same = (got.double() == out) | (got.isnan() & out.isnan())
    bad = torch.where(odd, ~same, ~((got.double() - out).abs() <= tol))
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} off, worst "
                           f"{((got.double() - out).abs() / tol.clamp_min(1e-300)).max().item():.3g} of the bound, "
                           f"first at {bad.nonzero()[0].tolist()}")


def exact_rotation(emb, x, positions, inverse=False):
    """fp64 rotation of x [..., tokens, heads, dim] and |x1| + |x2| of each value's pair."""
    rot = emb.rotary_dim
    # exact reduction of p * turns in fp64 needs p * turns < 2^20 or so to keep 2^-30: true of the tests
    turn = torch.remainder(positions.double()[..., None, None] * emb.turns.to(x.device), 1.0)
    c, s = (emb.gain * f(2 * math.pi * turn) for f in (torch.cos, torch.sin))
    if inverse:
        s = -s
    y, size = x.double().clone(), torch.zeros_like(x.double())
    a, b = ((slice(0, rot // 2), slice(rot // 2, rot)) if emb.layout == "half" else (slice(0, rot, 2), slice(1, rot, 2)))
    x1, x2 = y[..., a].clone(), y[..., b].clone()
    y[..., a], y[..., b] = x1 * c - x2 * s, x2 * c + x1 * s
    size[..., a] = size[..., b] = (x1.abs() + x2.abs()) * emb.gain
    return y, size


def assert_rotation(got, y, size, what=""):
    """One rounding to the type; fp32 errors before it: the reduced angle (2^-22.3 radians), sine and
    cosine (2^-22), gain, two products and a sum (2^-24 each) of values up to |x1| + |x2|: under 2^-20."""
    tol = rounded(y, got.dtype) * (1 + 2.0 ** -10) + 2.0 ** -20 * size
    bad = ~((got.double() - y).abs() <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}"
