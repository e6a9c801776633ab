"""Log probabilities have no forward-mode derivative: logits that carry a tangent are refused, with
gradients recorded or not, instead of losing it."""
import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("top", [0, 3])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("grad", [True, False])
def test_a_tangent_is_refused(cuda_dev, top, dtype, grad):
    from fitllm_b200.lm_head import token_logprobs
    z = torch.randn(3, 500, device=cuda_dev).to(dtype)
    ids = torch.arange(3, device=cuda_dev)
    want = token_logprobs(z, ids, top=top)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(z, torch.ones_like(z))
        for logits, at in ((dual, ids), (dual[:, :400], ids), (dual.view(3, 1, 500), ids.view(3, 1)), (dual.t().contiguous().t(), ids)):
            with torch.set_grad_enabled(grad), pytest.raises((RuntimeError, NotImplementedError), match="jvp|forward"):
                token_logprobs(logits, at, top=top)
        # plain tensors inside a level, and a dual's primal, are as ever
        for logits in (z, forward_ad.unpack_dual(dual).primal):
            for a, b in zip(token_logprobs(logits, ids, top=top), want):
                assert torch.equal(a, b)


def test_hidden_states_with_a_tangent_are_refused(cuda_dev):
    from fitllm_b200.lm_head import random_lm_head
    head = random_lm_head(256, 1024, cuda_dev, seed=3)
    h = torch.randn(2, 256, device=cuda_dev).bfloat16()
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(h, torch.ones_like(h))
        with pytest.raises((RuntimeError, NotImplementedError), match="jvp|forward"):
            head.token_logprobs(dual, torch.zeros(2, dtype=torch.int64, device=cuda_dev))
