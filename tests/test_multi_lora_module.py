"""Wrapped projections with adapters of many requests: what they refuse, with stand-ins for
the kernels (no GPU needed)."""
import pytest
import torch

from fitllm_b200 import ops, qlora
from fitllm_b200.lora import AdapterRoute, MultiLoRALinear
from fitllm_b200.qlora import Linear4bit, grouped_forward


@pytest.fixture
def calls(monkeypatch):
    """Kernels that return zeros and note the adapters' calls."""
    seen = []

    def multi_lora(x, a, b, scale, adapter, y, q_start=None, out=None):
        seen.append((tuple(x.shape), adapter, q_start))
        return y if out is None else out

    def base(self, x, residual=None):
        y = x.new_zeros(*x.shape[:-1], self.out_features)
        return y if residual is None else y + residual

    monkeypatch.setattr(ops, "multi_lora", multi_lora)
    monkeypatch.setattr(Linear4bit, "forward", base)
    monkeypatch.setattr(Linear4bit, "wref", lambda self: None)
    monkeypatch.setattr(ops, "nf4_gemv_grouped", lambda x2, jobs: [x2.new_zeros(x2.shape[0], 64) for _ in jobs])
    return seen


def _wrapped(batch):
    route = AdapterRoute()
    route.adapter = None if batch is None else torch.zeros(batch, dtype=torch.int32)
    return MultiLoRALinear(Linear4bit(64, 64), 2, 16, route)


@pytest.mark.parametrize("batch", [None, 3])
def test_inputs_that_require_a_gradient_are_refused(calls, batch):
    mod = _wrapped(batch)
    x, h = torch.zeros(3, 5, 64, dtype=torch.bfloat16), torch.zeros(3, 5, 64, dtype=torch.bfloat16)
    plain = mod(x, residual=h)
    assert plain.shape == (3, 5, 64) and len(calls) == (batch is not None)
    for args in ((x.clone().requires_grad_(), None), (x, h.clone().requires_grad_())):
        with pytest.raises(NotImplementedError, match="gradient"):
            mod(args[0], residual=args[1])
        with torch.no_grad():
            assert mod(args[0], residual=args[1]).shape == plain.shape
    live = x.clone().requires_grad_()
    with pytest.raises(NotImplementedError, match="gradient"):
        grouped_forward([mod, Linear4bit(64, 64)], live)
    with torch.no_grad():
        assert [y.shape for y in grouped_forward([mod, Linear4bit(64, 64)], live)] == [plain.shape] * 2
    # projections without adapters keep their own rule
    assert not grouped_forward([Linear4bit(64, 64)], live)[0].requires_grad


def test_no_call_takes_the_base_for_the_whole(calls, monkeypatch):
    """A call that does not add the adapters refuses a wrapped projection."""
    monkeypatch.setattr(ops, "nf4_gemv_swiglu", lambda x2, gate, up: x2.new_zeros(x2.shape[0], 64))
    mod, plain, x = _wrapped(3), Linear4bit(64, 64), torch.zeros(3, 1, 64, dtype=torch.bfloat16)
    for pair in ((mod, plain), (plain, mod)):
        with pytest.raises(TypeError, match="MultiLoRALinear"):
            qlora.swiglu_forward(*pair, x)
    with pytest.raises(TypeError, match="MultiLoRALinear"):
        qlora.projection_job(mod)
    assert qlora.swiglu_forward(plain, plain, x).shape == (3, 1, 64)
    grouped_forward([mod, plain, mod], x)
    assert len(calls) == 2  # the adapters of both wrapped ones


def test_a_pass_of_another_batch_is_refused(calls, monkeypatch):
    """A route stays until the next one; a pass that is not of its sequences is no call."""
    from fitllm_b200.lora import MultiLoRAManager
    model = torch.nn.Module()
    model.q_proj = Linear4bit(64, 64)
    m = MultiLoRAManager(4, 16, ("q_proj",))
    m.apply(model)
    mod = model.q_proj

    def run(*lead):
        x = torch.zeros(*lead, 64, dtype=torch.bfloat16)
        assert mod(x).shape == (*lead, 64)
        assert grouped_forward([mod, Linear4bit(64, 64)], x)[0].shape == (*lead, 64)

    def refused(*lead):
        n, x = len(calls), torch.zeros(*lead, 64, dtype=torch.bfloat16)
        for call in (lambda: mod(x), lambda: grouped_forward([mod, Linear4bit(64, 64)], x)):
            with pytest.raises(ValueError, match="route"):
                call()
        assert len(calls) == n

    run(1, 8)  # no route: any batch
    m.route(torch.zeros(4, dtype=torch.int32))
    run(4, 2), run(4, 1), run(4)
    for lead in ((1, 8), (2, 4), (8, 1), (8,), (1, 4)):
        refused(*lead)
    # packed tokens: as many rows as the route's, told or read from its starts
    starts = torch.tensor([0, 3, 3, 7], dtype=torch.int32)
    m.route(torch.zeros(3, dtype=torch.int32), q_start=starts)
    run(1, 7), run(7)
    refused(1, 8), refused(3, 7), refused(1, 6)
    m.route(torch.zeros(3, dtype=torch.int32), q_start=starts, tokens=9)  # two rows of padding
    run(1, 9)
    refused(1, 7)
    m.route(None)
    run(2, 4)
    for bad in (dict(q_start=starts[:3]), dict(q_start=starts.long()), dict(q_start=starts, tokens=-1), dict(tokens=7)):
        with pytest.raises(ValueError, match="route"):
            m.route(torch.zeros(3, dtype=torch.int32), **bad)
    run(2, 4)  # and changes nothing
