"""Waits of the 4-bit cache's kernels (read from their sources, no GPU): a warp that goes on to
shuffles, votes and MMAs behind a barrier wait goes on, or gives up, as one."""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parents[1] / "fitllm_b200" / "csrc"


def _code(name):
    return re.sub(r"\s+", " ", re.sub(r"//[^\n]*", "", (CSRC / name).read_text()))


def test_the_warp_wait_takes_every_lane_along():
    body = re.search(r"bool mbar_wait_warp\([^)]*\) \{(.*?)\}", _code("kv4.cuh")).group(1)
    assert body.strip() == "return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, status));"


def test_no_lane_of_the_prompt_kernel_gives_up_alone():
    # but for the issuing warp behind its last commit, which meets at once with nothing to skip
    last = "mbar_wait(&b_done, 0, &never, p.status); } __syncwarp();"
    code = _code("kv4_prompt.cu")
    assert code.count(last) == 1 and "mbar_wait_warp(" in code
    assert not re.search(r"\bmbar_wait\(", code.replace(last, ""))


def test_no_lane_of_the_decode_kernel_gives_up_alone():
    code = _code("kv4_attn.cu")
    # a lane whose wait ran out notes it and goes on with its warp
    waits = re.findall(r"if \(!mbar_wait\([^;]*\) (\w+ = \w+);", code)
    assert waits == ["cap = kGaveUp"] and len(re.findall(r"\bmbar_wait\(", code)) == 1
    # up to the first vote, which the note makes true (no scale's size is <= kGaveUp), and where all leave
    step = code[code.index("mbar_wait("):]
    assert re.search(r"constexpr float kGaveUp = -\d", code)
    votes = [m.start() for m in re.finditer(r"__(any|all|ballot|shfl\w*|reduce\w*)_sync", step)]
    assert votes[0] == step.index("__any_sync(0xffffffffu, over)")
    assert step[votes[0]:].startswith(
        "__any_sync(0xffffffffu, over)) { if (__any_sync(0xffffffffu, cap == kGaveUp)) return false;")
    assert "return" not in step[:votes[0]]
    assert step[:votes[0]].count("<= cap)") == 2  # one for either way of scaling the weights
