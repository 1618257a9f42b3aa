"""Batched decode with the 8-bit KV cache (vrt_batch_create_kv8) against the
fp32 cache's.

A code is off by at most half of 1/127 of its page's largest value, evenly
spread: 1/(127 sqrt(12)) of it, some 0.8% of the values' own spread (the
largest of a page's thousands of values is about 3.5 spreads).  Attention
outputs take that over from the values, and about as much again from the keys
through scores of size 1; the residual stream mixes in unrounded embeddings.  So logits
stay within a few percent of their spread, 5% being twice what the layers can
add up to, while a wrong page, mask or position is off by its whole size."""

import numpy as np
import pytest

import synth_gguf as sg
import vrt

pytestmark = pytest.mark.gpu


def _spread(a, b):
    a, b = np.asarray(a, np.float64), np.asarray(b, np.float64)
    return np.sqrt(np.mean((a - b) ** 2)) / np.std(b)


def _compare(ctx, shape, seed, lens, steps, positions, **kw):
    cfg = vrt.Gemma3Config.from_shape(shape)
    model = vrt.Model(ctx, None, config=cfg, seed=seed, max_positions=positions, **kw)
    rng = np.random.default_rng(seed)
    prompts = [[2] + rng.integers(3, shape.vocab_size, n - 1).tolist() for n in lens]
    a = vrt.Batch(model, len(lens), positions, keep_logits=True)
    b = vrt.Batch(model, len(lens), positions, keep_logits=True, kv8=True)
    for i, p in enumerate(prompts):
        a.prefill(i, p)
        b.prefill(i, p)
        assert _spread(b.logits(i), a.logits(i)) < 0.05, f"prompt {i} of {len(p)}"
    same = list(range(len(lens)))  # sequences whose ids have been the same so far
    for step in range(steps):
        same = [i for i in same if a.read(i)[0] == b.read(i)[0]]
        a.decode_steps(len(lens), 1)
        b.decode_steps(len(lens), 1)
        for i in same:
            assert _spread(b.logits(i), a.logits(i)) < 0.05, f"sequence {i}, step {step}"
    for i, n in enumerate(lens):
        assert b.read(i)[1] == n + steps
    # the ids may part at a near tie: the rest of the positions on one path, the fp32 batch's
    paths = [p + a.read(i)[0][:steps] for i, p in enumerate(prompts)]
    for back in (2, steps // 2):
        for i, path in enumerate(paths):
            for x in (a, b):
                x.prefill(i, path[:len(path) - back])
        first = [a.read(i)[0] == b.read(i)[0] for i in range(len(lens))]
        a.decode_steps(len(lens), 1)
        b.decode_steps(len(lens), 1)
        for i in range(len(lens)):
            if first[i]:
                assert _spread(b.logits(i), a.logits(i)) < 0.05, f"sequence {i}, {back} before the end"
    return model, a, b, prompts


@pytest.mark.parametrize("name,graph", [("tiny", True), ("tiny-gqa", False)])
def test_kv8_batch_tiny(ctx, name, graph):
    """Windows of 8 tokens, prompts around page borders."""
    _, _, b, prompts = _compare(ctx, sg.SHAPES[name], 31, [2, 31, 32, 33, 9, 64], 40, 128, use_graph=graph)
    # a sequence started again gives the same as the first time
    b.prefill(0, prompts[0])
    ids = []
    for _ in range(2):
        b.prefill(1, prompts[1])
        b.decode_steps(2, 40)
        ids.append(b.read(1)[0])
    assert ids[0] == ids[1]


def test_kv8_batch_ring(ctx):
    """Sliding layers whose ring of window and slice is passed several times, prompts in chunks."""
    shape = sg.SHAPES["tiny-gqa"].with_(sliding_window=70, context_length=4096, name="ring")
    _compare(ctx, shape, 5, [1500, 40, 2300], 6, 2400, prefill_chunk=900)


def test_kv8_batch_many(ctx):
    """More than 32 sequences: the fp16 projections."""
    _compare(ctx, sg.SHAPES["tiny-gqa"], 8, [3 + i % 37 for i in range(40)], 3, 64)


def test_kv8_batch_270m(ctx):
    _compare(ctx, sg.SHAPES["270m"], 77, [700, 24, 530], 4, 1024)


def test_kv8_batch_27b_slice(ctx):
    shape = sg.SHAPES["27b"].with_(block_count=6, vocab_size=16384, name="27b-slice")
    _compare(ctx, shape, 27, [1200, 33], 3, 1280)


def test_kv8_batch_refusals(ctx):
    model = vrt.Model(ctx, None, config=vrt.Gemma3Config.from_shape(sg.SHAPES["tiny"]), seed=1, max_positions=32)
    with pytest.raises(vrt.VrtError):
        vrt.Batch(model, 2, 64, kv8=True)
    with pytest.raises(vrt.VrtError):
        vrt.Batch(model, 0, 16, kv8=True)
    b = vrt.Batch(model, 2, 16, kv8=True)
    with pytest.raises(vrt.VrtError, match="not been prefilled"):
        b.decode_steps(2, 1)
    b.prefill(0, [2, 5, 6])
    b.prefill(1, [2])
    with pytest.raises(vrt.VrtError, match="capacity"):
        b.decode_steps(2, 20)
    b.decode_steps(2, 13)
    assert b.read(0)[1] == 16 and b.read(1)[1] == 14
