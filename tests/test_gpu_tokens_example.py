"""The gradient that examples/score_tokens.py returns, entry by entry."""
import sys

import numpy as np
import pytest
import torch

import tokens_ref as R
from conftest import ROOT
from tensorium_b200.layers import TInt8ConnectedLayer, TNNetState

pytestmark = pytest.mark.gpu


def f64(t):
    return t.double().cpu().numpy()


def test_gradient(ctx):
    """Against the 64-bit gradient of the mean of -logprob at the example's own logits (the same head gives the same bits):
    every given token's entry is negative and every other one positive, and a gradient without either part, or of the
    other sign, is outside the bounds."""
    sys.path.insert(0, str(ROOT / "examples"))
    import score_tokens
    rows, vocab = 9, 1501
    hidden, weights, given, r, grad = score_tokens.main(["--rows", str(rows), "--hidden", "200", "--vocab", str(vocab), "--top", "4"])
    logits = TInt8ConnectedLayer(200, vocab, weights=weights).bind(ctx).forward(TNNetState(hidden))
    assert logits.dtype == grad.dtype == torch.bfloat16
    t = given.cpu().numpy()
    a = np.full(rows, np.float32(-1 / rows), np.float64)
    ref, off = R.gradient(f64(logits), t, 1.0, a, None)
    off = off + 1.01 * R.HALF_ULP["bfloat16"] * (np.abs(ref) + off) + R.TINY["bfloat16"]
    got = f64(grad)
    assert np.all(np.abs(got - ref) <= off)
    hit = np.zeros((rows, vocab), bool)
    hit[np.arange(rows), t] = True
    assert (got[hit] < 0).all() and (got[~hit] > 0).all()
    # what the bounds leave no room for
    p = np.exp(R.logprobs(f64(logits), t, 1.0, 0)["lp"])
    for wrong in (-ref, np.zeros_like(ref), p / rows, ref - p / rows):
        assert (np.abs(wrong - ref) > 10 * off).any(axis=1).all()
