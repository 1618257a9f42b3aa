"""Bounded waits of the paged 8-bit KV cache kernels, by their source: a wait
that gives up ends its warp's work as a whole.  Each lane of a warp counts its
own second, so lanes that decide for themselves can part: those that gave up
leave for the block's last barrier, and the others never pass the next warp
barrier.  No GPU: a wait that runs out is not brought about on one."""

import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vortex-rt_b200", "csrc")


def source(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


def statements(text, word):
    return [s.strip() for s in re.split(r"[;{}]", text) if word in s]


def test_prompt_kernel_votes():
    """Every wait whose result steers a warp of the tcgen05 kernel is voted on; the one behind a failed wait steers
    nothing."""
    waits = statements(source("kv8_prefill_tc.cu"), "mbar_wait_bounded(")
    assert len(waits) >= 5
    for s in waits:
        assert "ok = __all_sync(0xffffffffu, ok && mbar_wait_bounded(" in s or s == "mbar_wait_bounded(drained + t, 0)", s
