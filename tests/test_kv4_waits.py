"""Waits of the 4-bit cache's kernels (read from their sources, no GPU): a warp that goes on to
shuffles, votes and MMAs behind a barrier wait goes on, or gives up, as one."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "fitllm_b200" / "csrc"


def _code(name):
    return re.sub(r"//[^\n]*", "", (CSRC / name).read_text())


def test_the_warp_wait_takes_every_lane_along():
    body = re.search(r"bool mbar_wait_warp\([^)]*\) \{(.*?)\n\}", _code("kv4.cuh"), re.S).group(1)
    assert re.fullmatch(r"\s*return __all_sync\(0xffffffffu, mbar_wait\(bar, parity, abort_flag, status\)\);", body)


@pytest.mark.parametrize("name,alone", [
    ("kv4_attn.cu", []),
    # behind its last commit the issuing warp meets at once, with nothing to skip
    ("kv4_prompt.cu", ["mbar_wait(&b_done, 0, &never, p.status);\n    }\n    __syncwarp();"]),
])
def test_no_lane_gives_up_alone(name, alone):
    code = _code(name)
    for text in alone:
        assert code.count(text) == 1
        code = code.replace(text, "")
    assert not re.search(r"\bmbar_wait\(", code)
    assert "mbar_wait_warp(" in code
