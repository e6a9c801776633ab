"""Limits of a call over the 4-bit cache: more new tokens of a sequence than max_new.

include/fitq.h: such a sequence records FITQ_ERR_ARG and its tokens beyond max_new are not written; its
first max_new tokens, and every other sequence, are computed."""
import pytest
import torch

from tests import kv4_ref as ref
from tests.test_gpu_kv4 import BF, FP, U, _attend, _case

pytestmark = pytest.mark.gpu
FITQ_ERR_ARG = 1

FORMS = {
    "clusters": ([40, 300], 1),
    "clusters of drafts": ([40, 300], 3),
    "whole runs and cut pairs": ([5000, 30, 2000, 64, 7, 900, 3000, 12], 1),
    "cut pairs": ([6000] * 7, 2),
    "tiles of split positions": ([2000, 40], 70),
    "tiles": ([300, 40] * 10, 70),
}


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("h,kvh,dtype", [(8, 8, BF), (32, 8, FP), (40, 8, BF), (20, 4, FP)])
def test_tokens_beyond_max_new_are_not_written(cuda_dev, form, h, kvh, dtype):
    from fitllm_b200 import ops
    prefix, most = FORMS[form]
    for extra in (1, 5):
        counts = [most] * len(prefix)
        counts[0] += extra
        counts[-1] = max(1, most - 1)
        c = _case(prefix, counts, h, kvh, 128, 64, dtype, cuda_dev, seed=h + extra, head=1, tail=2)
        c["max_new"] = most
        out = torch.full_like(c["q"], 7.0)
        _attend(c, out=out)
        assert ops.device_status() == FITQ_ERR_ARG and ops.device_status() == 0
        kept = [min(n, most) for n in counts]
        want = ref.attention(c["q"], c["pool"], c["table"], c["prefix"], c["starts"], kept)
        rows = ~want.isnan().any(-1).any(-1)
        assert int(rows.sum()) == sum(kept)
        assert bool((out[~rows] == 7).all())
        # an element's bound as in test_gpu_kv4.py: scales up to 0.3
        bound = U[dtype] * (8 * 0.3 + want[rows].abs()) + 2.0 ** -10 * 2 * (8 * 0.3 + 1)
        assert bool(((out.double()[rows] - want[rows]).abs() <= bound).all())
