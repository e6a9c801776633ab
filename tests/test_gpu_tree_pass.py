"""Passes over trees of drafted tokens on NF4 layers, with adapters of many requests:
projections, append, attention, verification and keep as a serving loop runs them.

Hidden states are held to 1e-2 relative (norm), the bar the projections are held to."""
import threading

import pytest
import torch

from tests import tree_ref as ref

pytestmark = pytest.mark.gpu


def _layers(dev, heads=8, kv_heads=2, head_dim=128, n=2, lora=()):
    from fitllm_b200.layer import DecoderLayer, LayerConfig, add_lora_, quantize_layer_
    cfg = LayerConfig(hidden=heads * head_dim, heads=heads, kv_heads=kv_heads, head_dim=head_dim, intermediate=512)
    layers = []
    for i in range(n):
        layer = DecoderLayer(cfg, device=dev)
        quantize_layer_(layer, seed=70 + i)
        if lora:
            add_lora_(layer, 16, 32.0, lora, seed=i, b_std=0.01)
        layer.eval()
        layers.append(layer)
    return cfg, layers


def _rel(a, b):
    return ((a.float() - b.float()).norm() / b.float().norm()).item()


def test_a_tree_is_its_paths(cuda_dev):
    """Each token's state is the last one of its path run as a chain; the kept path's cache is the
    chain's."""
    from fitllm_b200 import ops
    from fitllm_b200.verify import KVCache, TreeKVCache, TreeVerdict, tree_pass, verify_pass
    cfg, layers = _layers(cuda_dev)
    g = torch.Generator(device=cuda_dev).manual_seed(3)
    b, t, cap, prompt = 2, 9, 96, 37
    parents = [[-1, 0, 0, 1, 1, 2, 5, 3, 6], [-1, 0, 1, 1, -2, 0, 3, -2, 6]]
    up = torch.tensor(parents, dtype=torch.int32, device=cuda_dev)
    h_prompt = torch.randn(b, prompt, cfg.hidden, device=cuda_dev, generator=g).bfloat16()
    h = torch.randn(b, t, cfg.hidden, device=cuda_dev, generator=g).bfloat16()
    cache = TreeKVCache(2, b, cfg.kv_heads, cfg.head_dim, cap, cuda_dev)
    verify_pass(layers, h_prompt, cache, 0)
    cache.set_lengths([prompt, prompt])
    out = tree_pass(layers, h, cache, up)
    assert cache.prefix.tolist() == [prompt, prompt] and ops.device_status() == 0
    for s in range(b):
        for i, (line, _) in ref.lineage(parents[s]).items():
            plain = KVCache(2, b, cfg.kv_heads, cfg.head_dim, cap, cuda_dev)
            verify_pass(layers, h_prompt, plain, 0)
            want = verify_pass(layers, h[:, line], plain, prompt)[s, -1]
            assert _rel(out[s, i], want) < 1e-2, (s, i)
    # ---- paths of different lengths stay; the next tree stands behind them
    path = torch.tensor([[0, 2, 5, 6, 8, -1, -1, -1, -1], [0, 1, -1, -1, -1, -1, -1, -1, -1]], dtype=torch.int32, device=cuda_dev)
    cache.keep(TreeVerdict(path, torch.tensor([4, 1], device=cuda_dev), torch.zeros(2, dtype=torch.int64, device=cuda_dev)))
    assert cache.prefix.tolist() == [prompt + 5, prompt + 2]
    h2 = torch.randn(b, 3, cfg.hidden, device=cuda_dev, generator=g).bfloat16()
    out2 = tree_pass(layers, h2, cache, torch.tensor([-1, 0, 0], dtype=torch.int32, device=cuda_dev))
    for s, line in ((0, [0, 2, 5, 6, 8]), (1, [0, 1])):
        plain = KVCache(2, b, cfg.kv_heads, cfg.head_dim, cap, cuda_dev)
        verify_pass(layers, h_prompt, plain, 0)
        verify_pass(layers, h[:, line], plain, prompt)
        want = verify_pass(layers, h2[:, :2], plain, prompt + len(line))[s]
        assert _rel(out2[s, :2], want) < 1e-2


@pytest.mark.parametrize("t", [3, 40])  # the skinny kernels of up to 64 rows, the GEMM
def test_every_sequence_takes_its_adapter(cuda_dev, t):
    from fitllm_b200.lora import MultiLoRAManager
    from fitllm_b200.verify import TreeKVCache, chain_parents, tree_pass
    targets = ("q_proj", "v_proj", "o_proj", "gate_proj", "down_proj")
    b = 3
    g = torch.Generator(device=cuda_dev).manual_seed(5)
    cfg, layers = _layers(cuda_dev)
    h = torch.randn(b, t, cfg.hidden, device=cuda_dev, generator=g).bfloat16()
    up = chain_parents(t, cuda_dev)

    def run(layers):
        cache = TreeKVCache(2, b, cfg.kv_heads, cfg.head_dim, 64, cuda_dev)
        return tree_pass(layers, h, cache, up)

    base = run(layers)
    # two trained adapters, as PEFT modules around the same weights
    want, states = [], []
    for seed in (1, 2):
        _, own = _layers(cuda_dev, lora=targets)
        state = {}
        for i, layer in enumerate(own):
            for name, mod in layer.lora_modules():
                torch.manual_seed(100 * seed + i)
                with torch.no_grad():
                    mod.lora_A["default"].weight.normal_(0, 0.05)
                    mod.lora_B["default"].weight.normal_(0, 0.05)
                for part in ("lora_A", "lora_B"):
                    state[f"base_model.model.model.layers.{i}.{name}.{part}.weight"] = getattr(mod, part)["default"].weight.detach().cpu()
        want.append(run(own))
        states.append(state)
    model = torch.nn.Module()
    model.layers = torch.nn.ModuleList(layers)
    m = MultiLoRAManager(4, 32, targets)  # rank 16 in slots of 32
    m.apply(model)
    assert len(m.layers) == 10
    assert torch.equal(run(layers), base)  # no route: the model as it is
    for slot, state in ((1, states[0]), (3, states[1])):
        assert m.load(slot, state, alpha=32.0) == 10
    m.route(torch.tensor([3, -1, 1], dtype=torch.int32, device=cuda_dev))
    got = run(layers)
    assert _rel(got[0], want[1][0]) < 1e-2 and _rel(got[2], want[0][2]) < 1e-2 and torch.equal(got[1], base[1])
    assert _rel(got[0], base[0]) > 2e-2  # the adapters are felt
    m.route(None)
    assert torch.equal(run(layers), base)


def test_a_step_is_captured_and_replayed(cuda_dev):
    """tree_pass, logits, verify_tree and keep in one graph: lengths move on the device, and replays
    with new inputs give what eager steps give.  Another graph with a workspace of its own runs between."""
    from fitllm_b200 import ops
    from fitllm_b200.lm_head import random_lm_head
    from fitllm_b200.verify import TreeKVCache, tree_pass, verify_tree
    cfg, layers = _layers(cuda_dev)
    head = random_lm_head(cfg.hidden, 4992, cuda_dev, std=0.1)
    b, t, cap = 2, 6, 200
    up = torch.tensor([[-1, 0, 0, 1, 1, 2], [-1, 0, 1, 2, 3, -2]], dtype=torch.int32, device=cuda_dev)

    def inputs(seed):
        g = torch.Generator(device=cuda_dev).manual_seed(seed)
        return (torch.randn(b, t, cfg.hidden, device=cuda_dev, generator=g).bfloat16(),
                torch.randint(0, 4992, (b, t), device=cuda_dev, generator=g), torch.rand(b, t, device=cuda_dev, generator=g))

    def step(cache, h, tokens, u):
        z = head.logits(tree_pass(layers, h, cache, up))
        # drafts that are often right: the best token of the parent's row for odd tokens
        best = z.argmax(-1).gather(1, up.clamp(min=0).long())
        tokens = torch.where(torch.arange(t, device=cuda_dev) % 2 == 1, best, tokens)
        r = verify_tree(z, tokens, up, u, temperature=0.2)
        cache.keep(r)
        return r

    eager = TreeKVCache(2, b, cfg.kv_heads, cfg.head_dim, cap, cuda_dev)
    want = [step(eager, *inputs(i)) for i in range(4)]
    cache = TreeKVCache(2, b, cfg.kv_heads, cfg.head_dim, cap, cuda_dev)
    static = [x.clone() for x in inputs(0)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(cache, *static)
    side.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(step(cache, *static))
    for x in (*cache.k, *cache.v, cache.prefix):
        x.zero_()
    for i in range(4):
        for x, y in zip(static, inputs(i)):
            x.copy_(y)
        graphs[i % 2].replay()
        assert all(torch.equal(x, y) for x, y in zip(outs[i % 2], want[i])), i
    assert torch.equal(cache.prefix, eager.prefix) and int(cache.prefix.sum()) > 8
    for x, y in zip(cache.k + cache.v, eager.k + eager.v):
        for s in range(b):
            n = int(eager.prefix[s])
            assert torch.equal(x[s, :, :n], y[s, :, :n])
    assert ops.device_status() == 0


def test_a_chain_behind_the_paged_cache(cuda_dev):
    """Drafts of a 4-bit paged cache's pass are verified by random numbers and accepted."""
    from fitllm_b200.lm_head import random_lm_head
    from fitllm_b200.verify import PagedKVCache, chain_parents, verify_pass, verify_tree
    cfg, layers = _layers(cuda_dev)
    head = random_lm_head(cfg.hidden, 3008, cuda_dev, std=0.1)
    cache = PagedKVCache(2, 3, cfg.kv_heads, cfg.head_dim, 128, cuda_dev, page_size=16)
    g = torch.Generator(device=cuda_dev).manual_seed(4)
    h = torch.randn(3, 5, cfg.hidden, device=cuda_dev, generator=g).bfloat16()
    z = head.logits(verify_pass(layers, h, cache))
    up = chain_parents(5, cuda_dev)
    tokens = z.argmax(-1).roll(1, 1)
    r = verify_tree(z, tokens, up, torch.rand(3, 5, device=cuda_dev, generator=g), temperature=0.0)
    assert r.accepted.tolist() == [4, 4, 4] and torch.equal(r.next_token, z[:, -1].argmax(-1))
    cache.advance((r.accepted + 1).tolist())
    assert cache.lengths == [5, 5, 5]


def test_two_threads_on_streams_of_their_own(cuda_dev):
    from fitllm_b200 import ops
    from fitllm_b200.verify import verify_tree
    g = torch.Generator(device=cuda_dev).manual_seed(6)
    sets = []
    for i in range(2):
        q, k, v = (torch.randn(*s, device=cuda_dev, generator=g).bfloat16() for s in ((4, 12, 8, 128), (4, 2, 900, 128), (4, 2, 900, 128)))
        up = (torch.rand(4, 12, device=cuda_dev, generator=g) * torch.arange(12, device=cuda_dev)).int() - 1
        z = torch.randn(4, 12, 9000, device=cuda_dev, generator=g) * 2
        sets.append((q, k, v, torch.tensor([800, 3, 450, 0], dtype=torch.int32, device=cuda_dev), up.contiguous(), z,
                     z.argmax(-1), torch.rand(4, 12, device=cuda_dev, generator=g)))
    x, a, bb = (torch.randn(*s, device=cuda_dev, generator=g).bfloat16() for s in ((48, 512), (3, 16, 512), (3, 1024, 16)))
    y, sc = torch.randn(48, 1024, device=cuda_dev, generator=g).bfloat16(), torch.ones(3, device=cuda_dev)
    ad = torch.tensor([0, 2, -1, 1], dtype=torch.int32, device=cuda_dev)

    def calls(s):
        q, k, v, prefix, up, z, tokens, u = s
        return [ops.tree_attention(q, k, v, prefix, up), *verify_tree(z, tokens, up, u), ops.multi_lora(x, a, bb, sc, ad, y)]

    want = [calls(s) for s in sets]
    torch.cuda.synchronize()
    errors = []

    def work(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(30):
                    got = calls(sets[i])
                    stream.synchronize()
                    assert all(torch.equal(p, w) for p, w in zip(got, want[i]))
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not errors and ops.device_status() == 0
