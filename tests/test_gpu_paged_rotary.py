"""The paged pass rotates as its layers do, whatever their rotary base: its keys are the coded
rotation of the layer's own, and its output is the contiguous pass's over the same positions."""
import pytest
import torch

from tests import kv4_ref as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("theta", [1e4, 1e6])
@pytest.mark.parametrize("head_dim,heads,kv_heads", [(64, 12, 2), (128, 8, 2)])
def test_a_paged_pass_is_the_contiguous_one(cuda_dev, theta, head_dim, heads, kv_heads):
    from fitllm_b200 import ops
    from fitllm_b200.layer import DecoderLayer, LayerConfig, quantize_layer_, rotary_tables
    from fitllm_b200.verify import KVCache, PagedKVCache, verify_pass
    cfg = LayerConfig(hidden=heads * head_dim, heads=heads, kv_heads=kv_heads, head_dim=head_dim, intermediate=512,
                      rope_theta=theta)
    layers = []
    for i in range(2):
        layer = DecoderLayer(cfg, device=cuda_dev)
        quantize_layer_(layer, seed=60 + i)
        layer.eval()
        layers.append(layer)
    n, batch = 190, 2
    paged = PagedKVCache(2, batch, kv_heads, head_dim, 256, cuda_dev, page_size=32, rope_theta=theta)
    g = torch.Generator(device=cuda_dev).manual_seed(2)
    with torch.no_grad():
        h = torch.randn(batch, n, cfg.hidden, generator=g, device=cuda_dev).bfloat16()
        verify_pass(layers, h, paged)
        paged.advance([n] * batch)
        k_raw = layers[0].self_attn.k_proj(layers[0].input_layernorm(h)).view(batch, n, kv_heads, head_dim)
        cos, sin = (t[:n] for t in rotary_tables(n, head_dim, theta, cuda_dev))
        plain = KVCache(2, batch, kv_heads, head_dim, 256, cuda_dev)
        for b in range(batch):
            want = ref.coded_values(ref.rotate(k_raw[b], cos, sin)).bfloat16()
            assert torch.equal(paged.read(0, b)[0], want)
            for i in range(2):
                for to, x in zip((plain.k[i], plain.v[i]), paged.read(i, b)):
                    to[b, :, :n] = x.transpose(0, 1)
        # one more token over those positions (its own key and value alone are not coded in the
        # contiguous cache); the bar is the projections'
        h = torch.randn(batch, 1, cfg.hidden, generator=g, device=cuda_dev).bfloat16()
        a, b = verify_pass(layers, h, paged).float(), verify_pass(layers, h, plain, n).float()
    assert ops.device_status() == 0
    assert float((a - b).norm() / b.norm()) < 1e-2


def test_a_cache_of_another_base_is_refused(cuda_dev):
    from fitllm_b200.layer import DecoderLayer, LayerConfig, quantize_layer_
    from fitllm_b200.verify import PagedKVCache, verify_pass
    cfg = LayerConfig(hidden=256, heads=4, kv_heads=2, head_dim=64, intermediate=512, rope_theta=1e4)
    layer = DecoderLayer(cfg, device=cuda_dev)
    quantize_layer_(layer, seed=1)
    cache = PagedKVCache(1, 1, 2, 64, 64, cuda_dev)
    with pytest.raises(ValueError, match="rope_theta"):
        verify_pass([layer], torch.zeros(1, 3, 256, device=cuda_dev, dtype=torch.bfloat16), cache)
