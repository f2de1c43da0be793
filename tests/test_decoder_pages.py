"""SyntheticDecoder: prompts it has no room for; the rotation inside its paged attention."""
import importlib

import pytest
import torch

from conftest import pkg


def decoder(device, seed=3, **cfg):
    D = importlib.import_module(pkg().__name__ + ".decoder")
    return D.SyntheticDecoder(D.DecoderConfig(**cfg), device, seed=seed, max_batch=4)


# ------------------------------------------------------------------ CPU
@pytest.mark.parametrize("kv", ["dense", "paged"])
def test_a_prompt_that_is_too_long(kv):
    d = decoder("cpu", layers=1, hidden=128, heads=2, head_dim=64, vocab=50, experts=4, group=16, max_seq=32, mlp="dense", kv=kv)
    with pytest.raises(ValueError, match="max_seq"):
        d.prefill(torch.zeros(2, 33, dtype=torch.long))
