"""Sampling against a sort in 64 bits.  The oracle forms the weights as the
operator defines them (fp32 exponents, whole multiples of 2^-40), so the kept
set and the token have to be equal; CUDA's expf may be 2 units in the last
place from the exact exponential, so a row whose draw lies within that of a
border may take the neighbour: such rows are recognised by arithmetic."""
import math

import numpy as np
import pytest
import torch

from conftest import to_dev
from shukuchi_b200 import cuda as sc

gpu = pytest.mark.gpu
TORCH = {0: torch.float32, 1: torch.float16, 30: torch.bfloat16}
NONE = 0xFFFFFFFF


def test_refused_without_a_context():
    assert sc.lib().shk_cuda_sample(None, None, 0, 1, 1, 0, None, None, None, None, None, None, None, None) == -1


def kept_weights(z, t, k, top_p, min_p):
    """(weights that stay, in index order; slack of the borders) of one row in 64 bits."""
    z = np.where(np.isnan(z), -np.inf, z).astype(np.float32) + np.float32(0)
    top = z.max()
    with np.errstate(all="ignore"):
        x = (z - top).astype(np.float32) * np.float32(1 / np.float32(t))
        w = np.where(z == top, 1.0, np.where(x <= 0, np.exp(x.astype(np.float64)), 0.0))
    w = np.floor(w * 2.0 ** 40)
    order = np.lexsort((np.arange(len(z)), -z.astype(np.float64)))
    stay = np.zeros(len(z), bool)
    order = order[:k] if k > 0 else order
    close = False
    if top_p < 1:
        before = np.cumsum(w[order]) - w[order]
        need = max(1.0, top_p * w[order].sum())
        close |= bool(np.any(np.abs(before - need) < 4e-7 * need + 1))
        order = order[before < need]
    stay[order] = True
    if min_p > 0:
        edge = min(min_p, 1.0) * 2.0 ** 40
        close |= bool(np.any((np.abs(w - edge) < 4e-7 * edge + 1) & (w < 2.0 ** 40)))
        stay &= w >= edge
    return np.where(stay, w, 0.0), close


def check(ctx, z, u, settings, dtype=0, stride=0, **kw):
    """One call; every row against the oracle.  settings: (temperature, top_k, top_p, min_p) per row, or None for off."""
    rows, vocab = z.shape
    zd = torch.zeros(rows, max(stride, vocab), device="cuda", dtype=TORCH[dtype])
    zd[:, :vocab] = to_dev(z.astype(np.float32)).to(TORCH[dtype])
    args, host = {}, {}
    for name, value, off in zip(("temperature", "top_k", "top_p", "min_p"), settings, (1.0, 0, 1.0, 0.0)):
        host[name] = np.full(rows, off) if value is None else np.broadcast_to(np.asarray(value), (rows,)).astype(
            np.int32 if name == "top_k" else np.float32)
        if value is not None:
            args[name] = to_dev(host[name].copy())
    ud, ids = to_dev(u.astype(np.float32)), torch.full((rows,), -9, dtype=torch.int32, device="cuda")
    prob = torch.full((rows,), -9.0, device="cuda")
    torch.cuda.synchronize()
    ctx.sample(zd.data_ptr(), rows, vocab, ud.data_ptr(), ids.data_ptr(), prob=prob.data_ptr(), dtype=dtype,
               row_stride=stride, **{n: a.data_ptr() for n, a in args.items()}, **kw)
    torch.cuda.synchronize()
    ctx.check()
    got, pr = ids.cpu().numpy().view(np.uint32), prob.cpu().numpy()
    z = zd[:, :vocab].float().cpu().numpy()
    for r in range(rows):
        t, k, top_p, min_p = (host[n][r] for n in ("temperature", "top_k", "top_p", "min_p"))
        clean = np.where(np.isnan(z[r]), -np.inf, z[r])
        if clean.max() == -np.inf:
            assert got[r] == NONE and pr[r] == 0
            continue
        if not t > 0:
            assert got[r] == int(clean.argmax()) and pr[r] == 1
            continue
        w, close = kept_weights(z[r], t, int(k), float(top_p), float(min_p))
        i, total = int(got[r]), w.sum()
        assert i < vocab
        if close:  # a border within rounding: the token is one of a set larger or smaller by it
            continue
        assert w[i] > 0, (r, i)
        ends = np.cumsum(w)
        target = min(max(float(u[r]), 0.0), 1.0) * total
        # weights are off by 2 units of 2^-24 each at most: so are the sums
        slack = 4e-7 * total + vocab
        assert ends[i] - w[i] - slack <= target < ends[i] + slack or (i == np.flatnonzero(w)[-1] and target >= total - slack), r
        assert abs(pr[r] - w[i] / total) <= 6e-7 * w[i] / total + 2.0 ** -40
        if slack < target - (ends[i] - w[i]) and target < ends[i] - slack:
            assert i == int(np.searchsorted(ends, target, side="right"))
    return got, pr


@gpu
@pytest.mark.parametrize("dtype", [0, 1, 30])
@pytest.mark.parametrize("rows,vocab,stride", [(1, 1, 0), (3, 2, 5), (5, 31, 0), (2, 1000, 1001), (7, 4097, 0), (3, 32000, 0),
                                               (2, 128256, 128257), (1, 262144, 0), (40, 777, 0), (200, 129, 131)])
def test_sample(ctx, dtype, rows, vocab, stride):
    """Every setting alone and together, on odd sizes and rows that begin anywhere."""
    rng = np.random.default_rng(vocab)
    z = rng.normal(0, 3, (rows, vocab))
    u = rng.random(rows)
    for settings in ((None,) * 4, (0.7, None, None, None), (1.3, 40, None, None), (None, None, 0.9, None),
                     (0.9, None, None, 0.1), (0.8, 50, 0.95, 0.05), (2.0, 1, None, None), (None, 7, 0.5, None),
                     (1.0, vocab + 3, 0.999, 0.0), (0.0, 5, 0.5, 0.5), (1.0, 0, 0.0, 0.0), (1.0, -4, 1.5, 2.0)):
        check(ctx, z, u, settings, dtype, stride)


@gpu
def test_sample_settings_per_row(ctx):
    rng = np.random.default_rng(9)
    n = 300
    z = rng.normal(0, 2.5, (n, 3001))
    z[:, ::301] += 7
    check(ctx, z, rng.random(n), (np.where(rng.random(n) < 0.2, 0, rng.uniform(0.1, 2, n)), rng.integers(0, 100, n),
                                  rng.uniform(0.05, 1.05, n), rng.uniform(0, 0.4, n) * rng.integers(0, 2, n)))


@gpu
@pytest.mark.parametrize("settings", [(None,) * 4, (1.0, 3, None, None), (1.0, None, 0.5005, None), (1.0, 600, 0.7011, 0.01)])
def test_sample_ties(ctx, settings):
    """Equal logits: the lower index stays; all equal, two values, signed zeros."""
    n, rng = 1000, np.random.default_rng(1)
    z = np.zeros((5, n))
    z[1] = rng.integers(0, 2, n)
    z[2] = rng.integers(-3, 3, n) * 0.5
    z[3, ::2] = -0.0
    z[4] = -1e30
    for u in (0.0, 0.123, 0.5, 0.999999):
        check(ctx, z, np.full(5, u), settings)


@gpu
@pytest.mark.parametrize("vocab", [20000, 70001, 200003])
@pytest.mark.parametrize("settings", [(1.0, 5000, None, None), (0.5, None, 0.61, None), (2.0, 9001, 0.377, 0.2), (1.0, 1, None, None),
                                      (1.0, 700, 0.0, None)])
def test_sample_many_ties(ctx, vocab, settings):
    """Thousands of equal logits at the border, spread over every part of the vocabulary."""
    rng = np.random.default_rng(vocab)
    z = np.stack([rng.integers(-4, 4, vocab) * 0.5, np.zeros(vocab), np.where(rng.random(vocab) < 0.9, -1.0, rng.normal(0, 1, vocab)),
                  -20.0 + 1e-6 * rng.integers(0, 3, vocab)])
    for u in (0.0, 0.3337, 0.999):
        check(ctx, z, np.full(len(z), u), settings)


@gpu
@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("spread,vocab", [(1.6, 128256), (2.2, 100003), (0.5, 32000), (1.0, 40000)])
@pytest.mark.parametrize("settings", [(1.0, None, 0.97, None), (1.0, None, 0.83, 0.02), (1.0, 30011, None, None),
                                      (1.0, 20001, 0.9, None)])
def test_sample_crowded_border(ctx, dtype, spread, vocab, settings):
    """Flat rows: some hundred tokens and more share the border's bin, in 16 bits many with the same logit."""
    rng = np.random.default_rng(vocab + dtype)
    z = rng.normal(0, spread, (5, vocab)).astype(np.float32)
    u = rng.random(5)
    first = check(ctx, z, u, settings, dtype)
    again = check(ctx, z, u, settings, dtype)
    assert all((x == y).all() for x, y in zip(first, again))


@gpu
def test_sample_masked(ctx):
    """-inf, the type's lowest value, NaN and +inf among the logits; a row with nothing left; one token left."""
    rng = np.random.default_rng(2)
    z = rng.normal(0, 2, (9, 517))
    z[0, 5:] = -np.inf
    z[1, :] = -np.inf
    z[2, :] = np.nan
    z[3, ::2] = np.nan
    z[4, 100:] = np.finfo(np.float32).min
    z[5, 7], z[5, 300] = np.inf, np.inf
    z[6, :] = -np.inf
    z[6, 516] = -50
    z[7, :] = np.finfo(np.float32).min
    z[8, :] = np.inf
    for settings in ((None,) * 4, (0.5, 10, 0.9, 0.05), (0.0, None, None, None), (math.inf, None, None, None),
                     (1e-40, None, None, None), (1.0, 3, None, None), (1.0, None, 0.3, None)):
        got, _ = check(ctx, z, rng.random(9), settings)
        assert got[1] == got[2] == NONE and got[6] == 516 and got[5] in (7, 300)


@gpu
def test_sample_random_numbers_at_the_ends(ctx):
    """u = 0 takes the first token that stays, u of 1 and more the last, a negative or NaN u counts as 0."""
    z = np.zeros((6, 100))
    z[:, 0] = z[:, 99] = -np.inf
    got, pr = check(ctx, z, np.array([0.0, 1.0, 7.0, 0.5, 1.0 - 2.0 ** -24, 2.0 ** -30]), (None,) * 4)
    assert got.tolist() == [1, 98, 98, 50, 98, 1] and np.all(pr == np.float32(1 / 98))
    zd, ids = to_dev(z.astype(np.float32)), torch.zeros(2, dtype=torch.int32, device="cuda")
    u = to_dev(np.array([-3, np.nan], np.float32))
    torch.cuda.synchronize()
    ctx.sample(zd.data_ptr(), 2, 100, u.data_ptr(), ids.data_ptr())
    ctx.sync()
    assert ids.tolist() == [1, 1]


@gpu
def test_sample_frequencies(ctx):
    """4096 draws at evenly spread u give each of 8 tokens its share to within one draw."""
    z = np.log(np.array([1, 2, 3, 4, 5, 6, 7, 8]) / 36.0)
    n = 4096
    got, _ = check(ctx, np.broadcast_to(z, (n, 8)), (np.arange(n) + 0.5) / n, (None,) * 4)
    count = np.bincount(got, minlength=8)
    assert np.all(np.abs(count - n * np.arange(1, 9) / 36) <= 1)


@gpu
def test_sample_arguments(ctx):
    z, u, ids = torch.zeros(2, 8, device="cuda"), torch.zeros(2, device="cuda"), torch.full((2,), 5, dtype=torch.int32, device="cuda")
    a = (z.data_ptr(), 2, 8, u.data_ptr(), ids.data_ptr())
    for bad in ((None, 2, 8, a[3], a[4]), (a[0], 2, 0, a[3], a[4]), (a[0], 2, 262145, a[3], a[4]), (a[0], 2, 8, None, a[4]),
                (a[0], 2, 8, a[3], None), (a[0] + 2, 2, 8, a[3], a[4]), (a[0], 65536, 8, a[3], a[4])):
        with pytest.raises(sc.ShkError):
            ctx.sample(*bad)
    for kw in (dict(dtype=12), dict(row_stride=7)):
        with pytest.raises(sc.ShkError):
            ctx.sample(*a, **kw)
    ctx.sample(None, 0, 8, None, None)
    ctx.check()
    assert ids.tolist() == [5, 5]
