"""Draws whose border lies within the exponential's rounding, held to the tokens
that a border there or a token further on allows, and to no others."""
import numpy as np
import pytest
import torch

import test_request_batch as batch
from test_sample import TORCH, check

gpu = pytest.mark.gpu
ONE = 2.0 ** 40  # a weight of 1
# CUDA's expf is within 2 units in the last place, 2^-22 of the value; the weight is then cut to a whole number.
E = 2.0 ** -22


def permissible(z, u, t, k, top_p, min_p):
    """(tokens that the draw may give, their least and largest probability).  Weights in 64 bits from the operator's
    fp32 exponents; where a sum is within its error of top-p's border, or a weight of min-p's, the token there may
    stay or go."""
    z = np.where(np.isnan(z), -np.inf, z).astype(np.float32) + np.float32(0)
    n, top = len(z), z.max()
    with np.errstate(all="ignore"):
        x = (z - top).astype(np.float32) * np.float32(1 / np.float32(t))
        w = np.where(z == top, 1.0, np.where(x <= 0, np.exp(x.astype(np.float64)), 0.0))
    W = np.floor(w * ONE)
    order = np.lexsort((np.arange(n), -z.astype(np.float64)))
    order = order[:k] if k > 0 else order
    surely, maybe = np.zeros(n, bool), np.zeros(n, bool)
    if top_p < 1:
        before = np.cumsum(W[order]) - W[order]
        need = max(1.0, top_p * W[order].sum())
        # j weights are off by E of their sum and 1 each; with top_p <= 0 the border is 1 unit, whatever the sum
        slack = E * before + np.arange(len(order)) + (E * need + len(order) + 1 if top_p > 0 else 0)
        surely[order[before + slack < need]] = True
        maybe[order[before - slack < need]] = True
        surely[order[0]] = True
    else:
        surely[order] = maybe[order] = True
    if min_p > 0:
        edge = min(min_p, 1.0)
        surely &= (w >= edge * (1 + E)) | (w == 1)
        maybe &= (w >= edge * (1 - E)) | (w == 1)
    low, high = np.where(surely, W, 0.0), np.where(maybe | surely, W, 0.0)
    low_end, high_end = np.cumsum(low), np.cumsum(high)
    err = 2 * E * high_end[-1] + n + 2
    may = (high > 0) & (low_end - low <= u * high_end[-1] + err) & (high_end > u * low_end[-1] - err)
    with np.errstate(all="ignore"):
        return np.flatnonzero(may), W[may] / high_end[-1], W[may] / low_end[-1]


def held(z, got, prob, u, settings, dtype=0):
    z = torch.from_numpy(z.astype(np.float32)).to(TORCH[dtype]).float().numpy()
    t, k, top_p, min_p = (off if v is None else v for v, off in zip(settings, (1.0, 0, 1.0, 0.0)))
    for r in range(len(z)):
        tokens, least, most = permissible(z[r], float(np.float32(u[r])), t, k, float(np.float32(top_p)), float(np.float32(min_p)))
        assert len(tokens) <= 2, "the row says too little"
        at = np.flatnonzero(tokens == got[r])
        assert len(at), (r, int(got[r]), tokens)
        # a weight and a sum, each off by E and by its cuts (n units of a sum that is one weight of 2^40 at least)
        slack = 3 * E + 2 * len(z[r]) / ONE
        assert least[at[0]] * (1 - slack) - 1 / ONE <= prob[r] <= most[at[0]] * (1 + slack) + 1 / ONE


SETTINGS = [(1.0, 0, 0.0, 0.0), (1.0, 700, 0.0, None), (0.6, 0, -1.0, 0.3), (1.0, None, 0.97, None), (1.0, None, 0.83, 0.02),
            (1.0, 20001, 0.9, None), (0.7, 50, 0.9, 0.05), (1.0, None, 0.37, None)]


def rows_of(rng, vocab, spread):
    return np.stack([rng.normal(0, spread, vocab), rng.integers(-4, 4, vocab) * 0.5, np.zeros(vocab),
                     np.where(rng.random(vocab) < 0.9, -1.0, rng.normal(0, 1, vocab))])


def test_few_tokens_are_let_through():
    """Of thousands of tokens the check lets one pass, or two next to a border; without top-p's mass only the first maximum."""
    rng = np.random.default_rng(1)
    z = rows_of(rng, 5000, 1.6).astype(np.float32)
    for settings in SETTINGS:
        t, k, top_p, min_p = (off if v is None else v for v, off in zip(settings, (1.0, 0, 1.0, 0.0)))
        for r in range(4):
            for u in rng.random(8):
                tokens, least, most = permissible(z[r], u, t, k, top_p, min_p)
                assert 1 <= len(tokens) <= 2 and (least <= most).all()
                if top_p <= 0:
                    assert tokens.tolist() == [z[r].argmax()] and least[0] == most[0] == 1


@gpu
@pytest.mark.parametrize("dtype", [0, 1, 30])
@pytest.mark.parametrize("spread,vocab", [(1.6, 128256), (2.2, 100003), (0.5, 32000), (1.6, 700), (3.0, 20001)])
@pytest.mark.parametrize("settings", SETTINGS)
def test_sample_at_the_borders(ctx, dtype, spread, vocab, settings):
    rng = np.random.default_rng(vocab + dtype)
    z = rows_of(rng, vocab, spread)
    for u in (rng.random(4), np.zeros(4), np.full(4, 1 - 2.0 ** -24)):
        got, prob = check(ctx, z, u, settings, dtype)
        held(z, got, prob, u, settings, dtype)


@gpu
@pytest.mark.parametrize("top_p", [0.0, -3.0, 1e-30])
def test_no_top_p_takes_the_first_maximum(ctx, top_p):
    """Of equal maxima the first stays alone, whatever u."""
    rng = np.random.default_rng(5)
    z = np.round(rng.normal(0, 1, (6, 40000)) * 4) / 4
    for settings in ((1.0, None, top_p, None), (0.5, 700, top_p, 0.1), (1.0, 30, top_p, None)):
        got, prob = check(ctx, z, rng.random(6), settings)
        assert got.tolist() == z.argmax(1).tolist() and (prob == 1).all()


@gpu
def test_steps_draw_with_their_own_numbers(ctx):
    """Tokens of whole steps are the draws of their rows' own random numbers and logits."""
    rng = np.random.default_rng(3)
    s = batch.Server(ctx, rng, 12, 90, 16, 160)
    for step in range(6):
        s.fill(rng, *batch.plan(rng, 12, step))
        s.step()
        ctx.check()
        z, u = s.logits.cpu().numpy(), s.u.tolist()
        for r, i in enumerate(s.ids.tolist()):
            tokens = permissible(z[r], u[r], float(np.float32(0.8)), 20, float(np.float32(0.9)), 0.0)[0]
            assert len(tokens) <= 2 and i in tokens
