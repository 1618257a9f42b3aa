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


def test_token_kernel_ends():
    """A wait of the single-token kernel that gives up, in any lane, is the last but for the copies under way: no page
    behind it is waited for, a second each, and no copy is asked for into a slot whose last one may still land."""
    text = source("kv8_decode.cu")
    refill = text[text.index("auto refill"):]
    refill = refill[:refill.index("};")]
    assert "ok = __all_sync(0xffffffffu, ok)" in refill and "if (ok && issued < 2 * mine)" in refill
    assert re.search(r"for \(uint32_t i = 0; i < mine && ok; \+\+i\)", text)
    waits = statements(text, "mbar_wait_bounded(")
    assert len(waits) == 3 and sum(s.startswith("ok &= ") for s in waits) == 2, waits
    drain = text[text.index("if (!ok) {"):]
    assert drain.index("mbar_wait_bounded") < drain.index("atomicOr") < drain.index("__syncthreads")
