"""A sequence enters a running batch: its prompt in chains through tree_pass, the others without tokens."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_prompt_enters_one_slot(cuda_dev):
    from fitllm_b200 import ops
    from fitllm_b200.layer import DecoderLayer, LayerConfig, quantize_layer_
    from fitllm_b200.verify import KVCache, TreeKVCache, TreeVerdict, chain_parents, tree_pass, verify_pass
    cfg = LayerConfig(hidden=1024, heads=8, kv_heads=2, head_dim=128, intermediate=512)
    layers = []
    for i in range(2):
        layers.append(DecoderLayer(cfg, device=cuda_dev))
        quantize_layer_(layers[-1], seed=30 + i)
        layers[-1].eval()
    g = torch.Generator(device=cuda_dev).manual_seed(12)
    batch, cap, b, n = 3, 256, 1, 150
    cache = TreeKVCache(2, batch, cfg.kv_heads, cfg.head_dim, cap, cuda_dev)
    verify_pass(layers, torch.randn(batch, 40, cfg.hidden, device=cuda_dev, generator=g).bfloat16(), cache, 0)
    cache.set_lengths([40, 25, 31])
    before = [x.clone() for x in cache.k + cache.v]
    cache.release(b)
    prompt = torch.randn(n, cfg.hidden, device=cuda_dev, generator=g).bfloat16()
    outs = []
    for part in prompt.split(64):
        t = part.shape[0]
        parents = torch.full((batch, t), -2, dtype=torch.int32, device=cuda_dev)
        parents[b] = chain_parents(t, cuda_dev)
        h = torch.zeros(batch, t, cfg.hidden, dtype=torch.bfloat16, device=cuda_dev)
        h[b] = part
        outs.append(tree_pass(layers, h, cache, parents)[b])
        path = torch.arange(t, dtype=torch.int32, device=cuda_dev).repeat(batch, 1)
        accepted = torch.full((batch,), -1, device=cuda_dev)
        accepted[b] = t - 1
        cache.keep(TreeVerdict(path, accepted, accepted))
    assert cache.prefix.tolist() == [40, n, 31] and ops.device_status() == 0
    plain = KVCache(2, 1, cfg.kv_heads, cfg.head_dim, cap, cuda_dev)
    want = verify_pass(layers, prompt[None], plain, 0)[0]
    got = torch.cat(outs)
    assert ((got.float() - want.float()).norm() / want.float().norm()).item() < 1e-2  # the bar of tests/test_gpu_tree_pass.py
    for x, y, z in zip(before, cache.k + cache.v, plain.k + plain.v):
        assert torch.equal(x[0], y[0]) and torch.equal(x[2], y[2])
        assert ((y[b, :, :n].float() - z[0, :, :n].float()).norm() / z[0, :, :n].float().norm()).item() < 1e-2
