"""Steps of the batch with the 8-bit KV cache on one path of tokens with the
fp32 cache: lengths around the borders of pages, rings and slices.

Both batches are given the same ids as a prompt, so the step behind it starts
from the same tokens wherever their first choices agree; it is asserted that
some do.  Logits lie within 5% of their spread (the bound of
test_gpu_batch_kv8.py: twice what the codes' rounding can add up to)."""

import numpy as np
import pytest

import synth_gguf as sg
import vrt

pytestmark = pytest.mark.gpu


def _spread(a, b):
    a, b = np.asarray(a, np.float64), np.asarray(b, np.float64)
    return np.sqrt(np.mean((a - b) ** 2)) / np.std(b)


@pytest.mark.parametrize("window,lens,chunk", [
    (8, [1, 8, 31, 32, 33, 63, 64, 65], 2048),          # pages
    (70, [69, 70, 71, 511, 512, 513, 600, 640], 2048),  # window, slice, ring of 20 pages
    (70, [581, 582, 583, 607, 608, 609, 1100, 1279], 300),
])
def test_steps_on_one_path(ctx, window, lens, chunk):
    shape = sg.SHAPES["tiny-gqa"].with_(sliding_window=window, context_length=4096, name="path")
    model = vrt.Model(ctx, None, config=vrt.Gemma3Config.from_shape(shape), seed=17, max_positions=1536, prefill_chunk=chunk)
    rng = np.random.default_rng(window)
    prompts = [[2] + rng.integers(3, shape.vocab_size, n - 1).tolist() for n in lens]
    n = len(lens)
    batches = [vrt.Batch(model, n, 1536, keep_logits=True, kv8=kv8) for kv8 in (False, True)]
    compared = 0
    for step in range(6):
        for x in batches:
            for i, p in enumerate(prompts):
                x.prefill(i, p)
        ids = [[x.read(i)[0] for i in range(n)] for x in batches]
        for x in batches:
            x.decode_steps(n, 1)
        a, b = batches
        for i in range(n):
            if ids[0][i] == ids[1][i]:
                compared += 1
                assert _spread(b.logits(i), a.logits(i)) < 0.05, f"{len(prompts[i])} tokens"
        prompts = [p + ids[0][i] for i, p in enumerate(prompts)]  # the fp32 batch's path
    assert compared >= n, f"only {compared} of {6 * n} steps started from the same token"
