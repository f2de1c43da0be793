"""SyntheticDecoder: prompts it has no room for; the rotation inside its paged attention."""
import importlib
import math
import types

import pytest
import torch

from conftest import pkg
from paged_helpers import assert_rotation, exact_rotation


def decoder(device, seed=3, **cfg):
    D = importlib.import_module(pkg().__name__ + ".decoder")
    return D.SyntheticDecoder(D.DecoderConfig(**cfg), device, seed=seed, max_batch=4)


# ------------------------------------------------------------------ CPU
@pytest.mark.parametrize("kv", ["dense", "paged"])
def test_a_prompt_that_is_too_long(kv):
    d = decoder("cpu", layers=1, hidden=128, heads=2, head_dim=64, vocab=50, experts=4, group=16, max_seq=32, mlp="dense", kv=kv)
    with pytest.raises(ValueError, match="max_seq"):
        d.prefill(torch.zeros(2, 33, dtype=torch.long))


# ------------------------------------------------------------------ GPU
@pytest.mark.gpu
@pytest.mark.parametrize("kv", ["dense", "paged"])
def test_captured_steps_after_eager_ones(cuda, kv):
    """Eager steps in between leave the captured step's inputs alone, and so does a batch of another size."""
    d = decoder(cuda, layers=2, hidden=256, heads=2, head_dim=128, vocab=1000, experts=16, group=32, max_seq=70, kv=kv)
    g = torch.Generator().manual_seed(1)
    one, two, three = (torch.randint(0, 1000, (b, n), generator=g).to(cuda) for b, n in ((4, 20), (4, 33), (2, 9)))
    want = [d.generate(x, 12, use_graph=False)[0] for x in (one, two, three)]
    for use_graph, i in ((True, 0), (False, 1), (True, 0), (True, 1), (True, 2), (False, 0), (True, 1)):
        assert torch.equal(d.generate((one, two, three)[i], 12, use_graph=use_graph)[0], want[i])


@pytest.mark.gpu
def test_rotation_in_the_decoder(cuda):
    """Every layer's rows are rotated to the positions they stand at, prompts' and steps', into the cache and on the way
    out; positions off by one would be noticed."""
    d = decoder(cuda, layers=2, hidden=256, heads=4, head_dim=64, vocab=500, experts=8, group=32, max_seq=64, mlp="dense", kv="paged")
    e = types.SimpleNamespace(rotary_dim=64, layout="half", gain=1.0,
                              turns=10000.0 ** (-torch.arange(32, dtype=torch.float64) / 32) / (2 * math.pi))
    seen, append = [], pkg().kvcache.PagedKVCache.append

    def record(cache, q, k, v, starts, lengths, table, **kw):
        given = q.clone(), k.clone(), v.clone()
        out = append(cache, q, k, v, starts, lengths, table, **kw)
        seen.append((*given, starts.tolist(), lengths.tolist(), table.clone(), cache.k.clone(), cache.v.clone(), out.clone()))
        return out

    pkg().kvcache.PagedKVCache.append = record
    try:
        ids = torch.randint(0, 500, (3, 21), generator=torch.Generator().manual_seed(2)).to(cuda)
        d.generate(ids, 4, use_graph=False)
    finally:
        pkg().kvcache.PagedKVCache.append = append
    assert len(seen) == 2 * 4
    for call, (q, k, v, starts, lengths, table, kc, vc, out) in enumerate(seen):
        first = 0 if call < 2 else 21 + call // 2 - 1
        for s in range(3):
            rows = slice(starts[s], starts[s + 1])
            pos = first + torch.arange(starts[s + 1] - starts[s], device=cuda)
            assert int(pos[-1]) + 1 == lengths[s]
            at = table[s].long()[pos // d.cfg.page], slice(None), pos % d.cfg.page
            assert_rotation(out[rows], *exact_rotation(e, q[rows], pos))
            assert_rotation(kc[at], *exact_rotation(e, k[rows], pos))
            assert torch.equal(vc[at], v[rows])
            for x, given in ((out[rows], q), (kc[at], k)):
                with pytest.raises(AssertionError):
                    assert_rotation(x, *exact_rotation(e, given[rows], pos + 1))
