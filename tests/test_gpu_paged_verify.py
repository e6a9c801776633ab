"""The verify step over a 4-bit paged cache: append, attention and draft scores run
together on NF4 layers.

The reference is the same pass with its attention restated in fp32 torch over what
the cache holds (read back after the pass), and the drafts' log probabilities from
the same logits in 64 bits.  Tolerance of the hidden states: 1e-2 relative (norm),
the bar the projections are held to."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _layers(dev, heads=12, kv_heads=2, head_dim=64, n=2):
    from fitllm_b200.layer import DecoderLayer, LayerConfig, add_lora_, quantize_layer_
    cfg = LayerConfig(hidden=heads * head_dim, heads=heads, kv_heads=kv_heads, head_dim=head_dim, intermediate=512)
    layers = []
    for i in range(n):
        layer = DecoderLayer(cfg, device=dev)
        quantize_layer_(layer, seed=60 + i)
        add_lora_(layer, 16, 32.0, ("q_proj", "v_proj"), seed=i, b_std=0.01)
        layer.eval()
        layers.append(layer)
    return cfg, layers


def _reference(layers, cfg, h, cache, starts, counts, prefix):
    """The packed pass [1, tokens, hidden] with attention over the cache's own values."""
    from fitllm_b200.layer import apply_rotary
    from fitllm_b200.verify import _layer_forward
    cos, sin = cache.tables
    for i, layer in enumerate(layers):
        def attend(q_raw, k_raw, v_raw):
            out = torch.empty_like(q_raw)
            for b, (a, n, p) in enumerate(zip(starts, counts, prefix)):
                if n == 0:
                    continue
                c, s = (torch.cat([x[p:p + n]] * 2, -1) for x in (cos, sin))
                q = q_raw[0, a:a + n].view(n, cfg.heads, -1).transpose(0, 1).float()
                q, _ = apply_rotary(q, q, c, s)
                k, v = (x.float().transpose(0, 1).repeat_interleave(cfg.heads // cfg.kv_heads, 0)
                        for x in cache.read(i, b))
                w = q.bfloat16().float() @ k.transpose(1, 2) / math.sqrt(cfg.head_dim)
                hidden = torch.arange(p + n, device=h.device)[None] > torch.arange(p, p + n, device=h.device)[:, None]
                o = torch.softmax(w.masked_fill(hidden, float("-inf")), -1) @ v
                out[0, a:a + n] = o.transpose(0, 1).reshape(n, -1).bfloat16()
            return out
        h = _layer_forward(layer, h, attend)
    return h


@pytest.mark.parametrize("head_dim,heads,kv_heads", [(64, 12, 2), (128, 8, 2)])
def test_prompts_then_drafts_over_a_paged_cache(cuda_dev, head_dim, heads, kv_heads):
    from fitllm_b200 import ops
    from fitllm_b200.verify import PagedKVCache, paged_verify_pass, verify_pass
    cfg, layers = _layers(cuda_dev, heads, kv_heads, head_dim)
    cache = PagedKVCache(2, 3, kv_heads, head_dim, 256, cuda_dev, page_size=32)
    g = torch.Generator(device=cuda_dev).manual_seed(2)
    counts, starts = [100, 37, 1], [0, 100, 137]
    with torch.no_grad():
        h = torch.randn(1, 138, cfg.hidden, generator=g, device=cuda_dev).bfloat16()
        out = paged_verify_pass(layers, h, cache, counts)
        cache.advance(counts)
        want = _reference(layers, cfg, h, cache, starts, counts, [0, 0, 0])
        assert float((out.float() - want.float()).norm() / want.float().norm()) < 1e-2
        # five new tokens of each, two of them accepted, then one more
        before = list(cache.lengths)
        h = torch.randn(3, 5, cfg.hidden, generator=g, device=cuda_dev).bfloat16()
        out = verify_pass(layers, h, cache)
        cache.advance([5, 5, 5])
        want = _reference(layers, cfg, h.view(1, 15, -1), cache, [0, 5, 10], [5] * 3, before).view_as(out)
        assert float((out.float() - want.float()).norm() / want.float().norm()) < 1e-2
        first = cache.read(1, 0)
    assert ops.device_status() == 0
    # rejected drafts leave nothing behind: the same tokens again give the same cache
    again = PagedKVCache(2, 3, kv_heads, head_dim, 256, cuda_dev, page_size=32)
    g = torch.Generator(device=cuda_dev).manual_seed(2)
    with torch.no_grad():
        paged_verify_pass(layers, torch.randn(1, 138, cfg.hidden, generator=g, device=cuda_dev).bfloat16(), again, counts)
        again.advance(counts)
        verify_pass(layers, torch.randn(3, 7, cfg.hidden, device=cuda_dev).bfloat16(), again)  # all rejected
        assert torch.equal(verify_pass(layers, h, again), out)
        again.advance([5, 5, 5])
        for x, y in zip(first, again.read(1, 0)):
            assert torch.equal(x, y)


def test_captured_verify_pass_follows_the_cache(cuda_dev):
    from fitllm_b200.verify import PagedKVCache, verify_pass
    cfg, layers = _layers(cuda_dev)
    cache = PagedKVCache(2, 2, 2, 64, 128, cuda_dev, page_size=16)
    h = torch.randn(2, 3, cfg.hidden, device=cuda_dev).bfloat16()
    cache.reserve([128, 128])
    with torch.no_grad():
        verify_pass(layers, h, cache)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = verify_pass(layers, h, cache)
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            got = out.clone()
            assert torch.equal(got, verify_pass(layers, h, cache))
            cache.advance([3, 1])
            h.normal_()


def test_score_drafts_and_head_gradients(cuda_dev):
    from fitllm_b200.lm_head import random_lm_head
    from fitllm_b200.verify import score_drafts
    head = random_lm_head(256, 1024, cuda_dev, seed=3, std=0.3)
    g = torch.Generator(device=cuda_dev).manual_seed(4)
    h = torch.randn(4, 5, 256, generator=g, device=cuda_dev).bfloat16()
    logits = head.logits(h).double()
    best = logits.argmax(-1)
    drafts = best[:, :-1].clone()
    drafts[1, 0] = (drafts[1, 0] + 1) % 1024   # none accepted
    drafts[2, 2] = (drafts[2, 2] + 1) % 1024   # two accepted
    r = score_drafts(head, h, drafts, top=3)
    assert r.accepted.tolist() == [4, 0, 2, 4]
    assert r.next_token.tolist() == [int(best[b, a]) for b, a in enumerate([4, 0, 2, 4])]
    lp = torch.log_softmax(logits, -1)
    assert float((r.logp.double() - lp[:, :-1].gather(-1, drafts[..., None])[..., 0]).abs().max()) < 1e-4
    assert r.top_ids.shape == (4, 5, 3) and r.entropy.shape == (4, 5)
    with pytest.raises(ValueError):
        score_drafts(head, h, drafts[:, :-1])
    # a loss on log probabilities reaches the hidden states
    leaf = h.clone().requires_grad_(True)
    ids = torch.randint(0, 1024, (4, 5), generator=g, device=cuda_dev)
    out = head.token_logprobs(leaf, ids)
    (out.logp.sum() + 0.1 * out.entropy.sum()).backward()
    x = h.double().requires_grad_(True)
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)
    lp = torch.log_softmax(y @ head.weight.double().T, -1)
    (lp.gather(-1, ids[..., None]).sum() - 0.1 * (lp.exp() * lp).sum()).backward()
    # bf16 logits (2^-8 of values of a few units) and bf16 gradients: the projections' bar twice over
    assert float((leaf.grad.double() - x.grad).norm() / x.grad.norm()) < 2e-2
