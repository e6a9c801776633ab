"""Limits of the 4-bit cache's sizes, before any device call (no GPU needed)."""
import subprocess
import sys
from pathlib import Path

import pytest

from fitllm_b200 import _lib

P = 0x10000  # an aligned address that nothing reads
SHAPE = 2

BEYOND = [
    # heads, max_new, max_len, the cache's batch and kv_heads
    (8, 1 << 31, 192, 4, 8), (8, 1 << 40, 192, 4, 8), (8, (1 << 62) + 5, 192, 4, 8), (1, 1 << 40, 192, 1, 1),
    (4096, 1 << 28, 192, 1, 8), (65536, 1, 192, 4, 8), (8, 1 << 30, 192, 1 << 27, 1), (8, 2, 1 << 31, 4, 8),
    (8, 2, 1 << 62, 4, 8), (8, 2, 192, 1 << 27, 8),
]


@pytest.fixture(scope="module")
def L():
    from fitllm_b200 import build
    build.build()
    return _lib.load()


def _cache(batch, kv_heads, tokens=8):
    return _lib.Kv4C(P, P, P, P, tokens, 4, batch, kv_heads, 128, 64, 3)


def test_a_workspace_beyond_the_limits_is_none():
    """In a process of its own: a size that overflowed on the way ended it."""
    code = ("from fitllm_b200 import _lib, build; build.build(); L = _lib.load()\n"
            f"for h, n, m, b, kv in {BEYOND!r}:\n"
            f"    c = _lib.Kv4C({P}, {P}, {P}, {P}, 8, 4, b, kv, 128, 64, 3)\n"
            "    print(L.fitq_kv4_attention_workspace(c, h, n, m), end=' ')\n")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=Path(__file__).resolve().parents[1])
    assert r.returncode == 0, r.stderr[-500:]
    assert r.stdout.split() == ["0"] * len(BEYOND)


@pytest.mark.parametrize("heads,max_new,max_len,batch,kv_heads", BEYOND)
def test_a_call_beyond_the_limits_is_refused(L, heads, max_new, max_len, batch, kv_heads):
    c = _cache(batch, kv_heads)
    assert L.fitq_kv4_attention(c, P, heads * 128, P, heads, 0, max_new, max_len, P, 1 << 40, None) == SHAPE


def test_workspaces_can_be_sized_ahead_of_the_tokens(L):
    # the cache's token count belongs to a call, max_new and max_len are the sizes' own
    for tokens in (0, 8, 4096):
        c = _cache(4, 2, tokens)
        for n in (1, 16, 4096, 131072):
            assert L.fitq_kv4_attention_workspace(c, 8, n, 131072) == L.fitq_kv4_attention_workspace(_cache(4, 2), 8, n, 131072) > 0
