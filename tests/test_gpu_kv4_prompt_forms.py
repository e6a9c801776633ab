"""Bad pages, hidden garbage and groups without numbers in every form of the many-row attention: one number a
value (bf16) and two (fp16), positions split over CTAs and not, rows of one CTA and of several."""
import pytest
import torch

from tests import kv4_ref as ref
from tests.test_gpu_kv4 import BF, FP, U, _attend, _case

pytestmark = pytest.mark.gpu
FITQ_ERR_ARG = 1

# split positions; none (more row tiles than SMs); groups that do not divide a tile
FORMS = [([700, 133], [40, 70], 8, 2), ([300, 21, 77], [70, 66, 90], 160, 160), ([90, 400], [61, 5], 35, 7)]


def _near(o, want, rows, dtype):
    # an element's bound as in test_gpu_kv4.py: scales up to 0.3
    bound = U[dtype] * (8 * 0.3 + want.abs()) + 2.0 ** -10 * 2 * (8 * 0.3 + 1)
    return bool(((o.double() - want).abs() <= bound)[rows].all())


@pytest.mark.parametrize("prefix,counts,h,kvh", FORMS)
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("d", [64, 128])
def test_what_is_hidden_never_matters(cuda_dev, prefix, counts, h, kvh, dtype, d):
    c = _case(prefix, counts, h, kvh, d, 32, dtype, cuda_dev, seed=d)
    a = _attend(c)
    for b, (p, n) in enumerate(zip(prefix, counts)):
        for pos in range(p + n, c["table"].shape[1] * 32):
            page = int(c["table"][b, pos // 32])
            if page < 0:
                break
            block = c["pool"][page, :, (pos % 32) // 16]
            at, per = 16 * d + (pos % 16) * d // 8, d // 8
            block[:, at:at + per] = 255  # NaN scales and lows of keys and values
    assert torch.equal(a, _attend(c))


@pytest.mark.parametrize("prefix,counts,h,kvh", FORMS)
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bits", [0x7c00, 0xfe00])
def test_a_group_without_numbers_reaches_its_own_rows(cuda_dev, prefix, counts, h, kvh, dtype, d, bits):
    c = _case(prefix, counts, h, kvh, d, 32, dtype, cuda_dev, seed=d + 1)
    want = ref.attention(c["q"], c["pool"], c["table"], c["prefix"], c["starts"], c["counts"])
    spoilt = torch.zeros(want.shape, dtype=torch.bool, device=cuda_dev)
    group = h // kvh
    # values inside the cache and of the last new token: a group's elements; a key inside: all of a head's
    for b, pos, kv, gr, side in ((0, 17, 0, 0, 1), (1, prefix[1] + counts[1] - 1, kvh - 1, d // 64 - 1, 1), (0, 40, kvh - 1, 0, 0)):
        at = 16 * d + ((pos % 16) * 2 * (d // 64) + side * (d // 64) + gr) * 4
        block = c["pool"][int(c["table"][b, pos // 32]), kv, pos % 32 // 16]
        block[at], block[at + 1] = bits & 255, bits >> 8
        for i in range(counts[b]):
            if pos <= prefix[b] + i:
                to = slice(64 * gr, 64 * gr + 64) if side else slice(None)
                spoilt[c["starts"][b] + i, kv * group:(kv + 1) * group, to] = True
    o = _attend(c)
    assert not bool(o[spoilt].isfinite().any())
    assert _near(o, want, ~spoilt & ~want.isnan(), dtype)


@pytest.mark.parametrize("prefix,counts,h,kvh", FORMS)
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("what", ["page", "negative page", "table end", "prefix"])
def test_bad_pages_and_prefixes_are_recorded_and_left_out(cuda_dev, prefix, counts, h, kvh, dtype, what):
    from fitllm_b200 import ops
    c = _case(prefix, counts, h, kvh, 128, 32, dtype, cuda_dev, seed=3)
    want = ref.attention(c["q"], c["pool"], c["table"], c["prefix"], c["starts"], c["counts"])
    if what == "page":
        c["table"][0, 1] = c["pool"].shape[0]
    if what == "negative page":
        c["table"][0, 1] = -7
    if what == "table end":
        c["pre"][0] = 32 * c["table"].shape[1] - 3
    if what == "prefix":
        c["pre"][0] = -1
    out = torch.full_like(c["q"], 7.0)
    o = _attend(c, out=out)
    assert ops.device_status() == FITQ_ERR_ARG and ops.device_status() == 0
    first = slice(c["starts"][0], c["starts"][0] + counts[0])
    others = torch.ones(want.shape, dtype=torch.bool, device=cuda_dev)
    others[first] = False
    assert _near(o, want, others & ~want.isnan(), dtype)
    assert bool(o.isfinite().all())
    if what == "prefix":
        assert bool((o[first] == 0).all())
    if what in ("page", "negative page"):  # positions 32..63 are left out
        k, v = ref.read_sequence(c["pool"], c["table"][0], prefix[0] + counts[0])
        keep = torch.ones(prefix[0] + counts[0], dtype=torch.bool, device=cuda_dev)
        keep[32:64] = False
        hidden = torch.arange(len(keep), device=cuda_dev)[None] > torch.arange(prefix[0], len(keep), device=cuda_dev)[:, None]
        for i in (0, h - 1):
            kv = i // (h // kvh)
            s = c["q"][first, i].double() @ k[kv].nan_to_num(0).T / 128 ** 0.5
            p = torch.softmax(s.masked_fill(hidden | ~keep, float("-inf")), -1)
            left = p @ v[kv].nan_to_num(0)
            assert _near(o[first, i], left, torch.ones_like(left, dtype=torch.bool), dtype)
