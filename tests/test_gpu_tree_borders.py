"""Verification behind many refusals without a drafting distribution: what is left of the weight is
a difference, and parts of the vocabulary that refusals have emptied name no token."""
import pytest
import torch

from tests import tree_ref as ref

pytestmark = pytest.mark.gpu

NEVER = 1 - 2.0 ** -24  # a child's number that only a probability of one exceeds


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("b", [1, 5])
def test_emptied_parts_name_no_token(cuda_dev, b, dtype):
    """62 children refused in turn leave a thousandth of the weight, all of it on the last token: the next
    one whatever u_0 is, also where u_0 is a few 1e-9."""
    from fitllm_b200.verify import verify_tree
    v, t, last = 152064, 63, 100_000
    z = torch.full((1, t, v), float("-inf"))
    for shift in range(8):  # other logits, other last digits
        heavy = [5] + [20_000 + 3 * i for i in range(61)]
        z[0, 0, heavy[0]] = 6.09375 + shift / 4
        z[0, 0, heavy[1]] = 6.0 + shift / 4
        z[0, 0, heavy[2:]] = 5.90625 + shift / 4
        z[0, 0, last] = 3.125 + shift / 4
        p = torch.softmax(z[0, 0].double(), 0)
        assert 2.0 ** -10 < p[last] < 1.1e-3
        draft = torch.tensor([[0] + heavy], device=cuda_dev).expand(b, t)
        up = torch.tensor([-1] + [0] * (t - 1), dtype=torch.int32, device=cuda_dev)
        rows = z[:, :1].to(cuda_dev, dtype).expand(b, t, v)
        for first in (0.0, 1e-10, 1e-9, 3e-9, 5e-9, 1e-8, 2e-8, 1e-7, 0.5, NEVER):
            u = torch.full((b, t), NEVER, device=cuda_dev)
            u[:, 0] = first
            r = verify_tree(rows, draft, up, u)
            assert r.accepted.tolist() == [0] * b and r.next_token.tolist() == [last] * b, (shift, first)


@pytest.mark.parametrize("v,dtype", [(9_000, torch.float32), (152_064, torch.bfloat16)])
def test_refused_weight_is_gone(cuda_dev, v, dtype):
    """Chances behind many refusals: a child is accepted below its share of what is left and refused above it,
    to 1e-7 of the share (u is fp32: 6e-8 of it), with the weight spread over parts of other largest logits."""
    from fitllm_b200.verify import verify_tree
    g = torch.Generator().manual_seed(v)
    n, t = 40, 42
    at = torch.randperm(v, generator=g)[:n + 2].tolist()
    z = torch.full((v,), float("-inf"))
    z[at[:n]] = (torch.rand(n, generator=g) * 2 + 6).to(dtype).float()
    z[at[n]], z[at[n + 1]] = 3.0, 3.25
    rows = z.to(cuda_dev, dtype).expand(4, t, v)
    draft = torch.tensor([[0] + at[:n + 1]], device=cuda_dev).expand(4, t)
    up = torch.tensor([-1] + [0] * (t - 1), dtype=torch.int32, device=cuda_dev)
    share = 1 / (1 + 2.718281828459045 ** 0.25)
    u = torch.full((4, t), NEVER, device=cuda_dev)
    u[:, -1] = torch.tensor([share * (1 - 1e-7) - 3e-8, share * (1 + 1e-7) + 3e-8, 0.3, 0.6])
    u[:, 0] = torch.tensor([0.0, 5e-9, 0.5, NEVER])
    r = verify_tree(rows, draft, up, u)
    assert r.accepted.tolist() == [1, 0, 1, 0]
    assert r.path[0, :2].tolist() == [0, t - 1] and r.next_token[[1, 3]].tolist() == [at[n + 1]] * 2
    path, acc, nxt = ref.verify(rows[3], draft[3].tolist(), up.tolist(), u[3], None, 1.0)
    assert (acc, nxt) == (0, at[n + 1])
