"""PagedKVCache accepts no positions that were never reserved (CPU)."""
import pytest

from fitllm_b200.verify import PagedKVCache


def _cache(**kw):
    a = dict(num_layers=2, batch=2, kv_heads=2, head_dim=64, capacity=100, device="cpu", page_size=64)
    a.update(kw)
    return PagedKVCache(**a)


def test_advance_stays_within_what_was_reserved():
    c = _cache()
    c.reserve([5, 0])
    for bad in ([60, 0], [6, 0], [0, 1]):
        with pytest.raises(ValueError, match="positions behind"):
            c.advance(bad)
    assert c.lengths == [0, 0] and c.prefix.tolist() == [0, 0]
    c.advance([3, 0])
    c.advance([2, 0])  # a captured pass that was replayed
    with pytest.raises(ValueError, match="positions behind"):
        c.advance([1, 0])
    c.reserve([1, 7])
    c.advance([1, 7])
    assert c.lengths == [6, 7]
    c.release(0)
    with pytest.raises(ValueError, match="positions behind"):
        c.advance([1, 0])
    c.reserve([2, 0])
    c.advance([2, 0])
    assert c.lengths == [2, 7]


def test_advance_stays_within_the_capacity():
    c = _cache(page_size=16)
    c.reserve([100, 0])
    with pytest.raises(ValueError, match="positions behind"):
        c.advance([112, 0])  # the last page has room for them
    c.advance([100, 0])
    c.reserve([0, 0])


def test_a_smaller_reservation_takes_nothing_back():
    c = _cache()
    c.reserve([100, 100])
    c.reserve([3, 3])
    for _ in range(3):
        c.advance([3, 1])
    assert c.lengths == [9, 3]


def test_reservations_that_fail_leave_the_limit():
    c = _cache(num_pages=1)
    c.reserve([5, 0])
    with pytest.raises(RuntimeError):
        c.reserve([50, 50])
    with pytest.raises(ValueError):
        c.advance([6, 0])
