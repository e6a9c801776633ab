"""Sizes that a call over the 4-bit cache refuses through the Python entry point."""
import pytest

from tests.test_gpu_kv4 import BF, _attend, _case

pytestmark = pytest.mark.gpu


def test_a_max_new_beyond_the_tokens_is_refused(cuda_dev):
    c = _case([5, 5], [1, 2], 1, 1, 128, 16, BF, cuda_dev)
    for many in (4, 1 << 31, 1 << 40, 1 << 62):
        c["max_new"] = many
        with pytest.raises(RuntimeError, match="max_new"):
            _attend(c)
