"""Batched decode of a model without a sliding window (its GGUF metadata may
lack one): every layer sees all positions, as in single-sequence decoding."""

import numpy as np
import pytest

import synth_gguf as sg
import vrt

pytestmark = pytest.mark.gpu


def _model(ctx, positions):
    shape = sg.SHAPES["tiny-gqa"].with_(sliding_window=0, context_length=4096, name="no-window")
    return shape, vrt.Model(ctx, None, config=vrt.Gemma3Config.from_shape(shape), seed=9, max_positions=positions)


def test_fp32_cache(ctx):
    """Logits within 1e-3 of the single-sequence path's, as in the other batch tests."""
    shape, model = _model(ctx, 96)
    rng = np.random.default_rng(2)
    prompts = [[2] + rng.integers(3, shape.vocab_size, n - 1).tolist() for n in (5, 33, 60)]
    b = vrt.Batch(model, 3, 80, keep_logits=True)
    for i, p in enumerate(prompts):
        b.prefill(i, p)
    b.decode_steps(3, 6)
    for i, p in enumerate(prompts):
        model.reset()
        for at, t in enumerate(p + b.read(i)[0][:6]):
            model.decode(t, at, 1)
        a, r = b.logits(i).astype(np.float64), model.logits().astype(np.float64)
        assert np.all(np.abs(a - r) <= 1e-3 + 1e-3 * np.abs(r)), f"sequence {i}: {np.abs(a - r).max():.3g}"


def test_8bit_cache(ctx):
    """More tokens than the ring of a window of 0 and one slice would hold.  Logits are those of the fp32 cache within
    5% of their spread, twice what the codes' rounding can add up to (test_gpu_batch_kv8.py)."""
    shape, model = _model(ctx, 1536)
    rng = np.random.default_rng(3)
    prompts = [[2] + rng.integers(3, shape.vocab_size, n - 1).tolist() for n in (1400, 40, 600)]
    a, b = (vrt.Batch(model, 3, 1500, keep_logits=True, kv8=kv8) for kv8 in (False, True))
    for x in (a, b):
        for i, p in enumerate(prompts):
            x.prefill(i, p)
    first = [a.read(i)[0] == b.read(i)[0] for i in range(3)]
    for i in range(3):
        assert _spread(b.logits(i), a.logits(i)) < 0.05, f"prompt {i}"
    for x in (a, b):
        x.decode_steps(3, 1)
    assert any(first)  # the sequences that were given the same token are compared
    for i in range(3):
        if first[i]:
            assert _spread(b.logits(i), a.logits(i)) < 0.05, f"token of sequence {i}"


def _spread(a, b):
    a, b = np.asarray(a, np.float64), np.asarray(b, np.float64)
    return np.sqrt(np.mean((a - b) ** 2)) / np.std(b)
