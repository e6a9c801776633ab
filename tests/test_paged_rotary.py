"""A paged pass refuses layers of another rotary base than its cache's (CPU)."""
from types import SimpleNamespace

import pytest
import torch

from fitllm_b200.layer import rotary_tables
from fitllm_b200.verify import PagedKVCache, paged_layer_forward, paged_verify_pass, verify_pass


def _cache(**kw):
    a = dict(num_layers=2, batch=2, kv_heads=2, head_dim=64, capacity=100, device="cpu", page_size=64)
    a.update(kw)
    return PagedKVCache(**a)


def _layer(theta):
    return SimpleNamespace(cfg=SimpleNamespace(rope_theta=theta, head_dim=64, heads=4, kv_heads=2))


@pytest.mark.parametrize("own,bases", [(1e6, [1e4, 1e4]), (1e4, [1e4, 1e6]), (5e5, [1e6, 1e6])])
def test_layers_of_another_rotary_base_are_refused(own, bases):
    c = _cache(rope_theta=own)
    layers = [_layer(b) for b in bases]
    h = torch.zeros(2, 3, 256, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="rope_theta"):
        verify_pass(layers, h, c)
    with pytest.raises(ValueError, match="rope_theta"):
        paged_verify_pass(layers, h.view(1, 6, 256), c, [3, 3])
    other = next(x for x in layers if x.cfg.rope_theta != own)
    with pytest.raises(ValueError, match="rope_theta"):
        paged_layer_forward(other, h, c.pools[0], c, 3)
    # nothing was reserved
    assert (c.page_table == -1).all()


def test_the_tables_follow_the_base():
    c = _cache(rope_theta=1e4)
    for got, want in zip(c.tables, rotary_tables(128, 64, 1e4, "cpu")):
        assert torch.equal(got, want)
