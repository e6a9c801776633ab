"""Bookkeeping of PagedKVCache (CPU): pages handed out, accepted, released."""
import pytest
import torch

from fitllm_b200.verify import PagedKVCache, paged_verify_pass


def _cache(**kw):
    a = dict(num_layers=2, batch=3, kv_heads=2, head_dim=64, capacity=100, device="cpu", page_size=16, num_pages=9)
    a.update(kw)
    return PagedKVCache(**a)


def test_pages_are_distinct_and_follow_the_lengths():
    c = _cache()
    assert c.page_table.shape == (3, 7) and c.pools[0].shape == (9, 2, 1, 18 * 64) and len(c.pools) == 2
    c.reserve([17, 0, 16])
    assert (c.page_table >= 0).sum(dim=1).tolist() == [2, 0, 1]
    c.reserve([17, 0, 16])  # the same positions again: nothing new
    used = c.page_table[c.page_table >= 0].tolist()
    assert len(used) == 3 and len(set(used)) == 3
    c.advance([17, 0, 3])
    assert c.lengths == [17, 0, 3] and c.prefix.tolist() == [17, 0, 3]
    c.reserve([15, 1, 13])
    assert (c.page_table >= 0).sum(dim=1).tolist() == [2, 1, 1]
    c.release(0)
    assert c.lengths == [0, 0, 3] and c.page_table[0].tolist() == [-1] * 7 and c.prefix.tolist() == [0, 0, 3]
    c.reserve([100, 0, 0])
    used = c.page_table[c.page_table >= 0].tolist()
    assert len(used) == len(set(used)) == 9


def test_refusals_change_nothing():
    c = _cache()
    with pytest.raises(ValueError, match="capacity"):
        c.reserve([101, 0, 0])
    with pytest.raises(RuntimeError, match="pages"):
        c.reserve([100, 48, 0])
    with pytest.raises(ValueError, match="counts"):
        c.reserve([1, 1])
    with pytest.raises(ValueError, match="no 1 positions"):
        c.advance([1, 0, 0])
    assert (c.page_table == -1).all() and c.lengths == [0, 0, 0]
    for bad in (dict(head_dim=96), dict(page_size=24)):
        with pytest.raises(ValueError):
            _cache(**bad)


def test_bytes_read_counts_blocks():
    # 4.5 bits an element, keys and values: 18 * 64 bytes per 16 positions of a head
    assert _cache().bytes_read(160) == 2 * 3 * 2 * 10 * 18 * 64


def test_a_pass_without_new_tokens_is_one_without_layers():
    c = _cache()
    h = torch.zeros(1, 0, 128, dtype=torch.bfloat16)
    assert paged_verify_pass([None], h, c, [0, 0, 0]) is h
    with pytest.raises(ValueError, match="counts"):
        paged_verify_pass([None], h, c, [0, 1, 0])
