"""Inputs that carry a forward-mode tangent, and caches that require a gradient, are refused by the calls
that would lose them (no GPU needed: before any device call)."""
import pytest
import torch
from torch.autograd import forward_ad

from fitllm_b200 import ops

BF = torch.bfloat16


def _calls():
    q, k = torch.zeros(2, 3, 4, 64, dtype=BF), torch.zeros(2, 3, 1, 64, dtype=BF)
    cache, prefix = torch.zeros(2, 1, 16, 64, dtype=BF), torch.zeros(2, dtype=torch.int32)
    up, cos = torch.zeros(3, dtype=torch.int32), torch.zeros(16, 32)
    path, acc = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int64)
    x, a, b, y = torch.zeros(6, 256, dtype=BF), torch.zeros(1, 16, 256, dtype=BF), torch.zeros(1, 64, 16, dtype=BF), torch.zeros(6, 64, dtype=BF)
    return {
        "tree_append": ([q, k, k.clone(), cache, cache.clone()], lambda t: ops.tree_append(*t, prefix, up, cos, cos)),
        "tree_attention": ([q, cache, cache.clone()], lambda t: ops.tree_attention(*t, prefix, up)),
        "tree_keep": ([cache, cache.clone()], lambda t: ops.tree_keep(t[:1], t[1:], prefix, path, acc)),
        "multi_lora": ([x, a, b, y, torch.zeros(1)], lambda t: ops.multi_lora(t[0], t[1], t[2], t[4], prefix, t[3])),
    }


@pytest.mark.parametrize("name", ["tree_append", "tree_attention", "tree_keep", "multi_lora"])
def test_tangents_and_gradients(name):
    inputs, call = _calls()[name]
    with pytest.raises(ValueError, match="CUDA|same|must"):  # as ever
        call(inputs)
    for i, x in enumerate(inputs):
        some = list(inputs)
        with forward_ad.dual_level():
            with pytest.raises(ValueError, match="CUDA|same|must"):  # a level alone is nothing
                call(some)
            some[i] = forward_ad.make_dual(x, torch.ones_like(x))
            with torch.no_grad(), pytest.raises(NotImplementedError, match="tangent"):
                call(some)
        some[i] = x.clone().requires_grad_()
        with pytest.raises(NotImplementedError, match="gradient"):
            call(some)
        with torch.no_grad(), pytest.raises(ValueError, match="CUDA|same|must"):
            call(some)


def test_wrapped_projections(monkeypatch):
    from fitllm_b200.lora import AdapterRoute, MultiLoRALinear
    from fitllm_b200.qlora import Linear4bit, grouped_forward
    mod, x = MultiLoRALinear(Linear4bit(64, 64), 2, 16, AdapterRoute()), torch.zeros(3, 1, 64, dtype=BF)
    with forward_ad.dual_level(), torch.no_grad():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: mod(dual), lambda: mod(x, residual=dual), lambda: grouped_forward([mod], dual)):
            with pytest.raises(NotImplementedError, match="tangent"):
                call()
