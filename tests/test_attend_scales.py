"""Attention over blocks whose V scales lie at the ends of fp32 and far apart."""
import numpy as np
import pytest
import torch

from conftest import to_dev
from shukuchi_b200 import cuda as sc
from test_pages import Pool, attend_reference, dev, from_bytes, p

pytestmark = pytest.mark.gpu
H, KV, SCALE = 8, 2, 0.125


def attend(ctx, pool, table, pos, q):
    blocks, n_kv, block, hd = pool.shape
    for i in range(2):
        pool.d[i].copy_(torch.from_numpy(pool.h[i]))
        pool.ds[i].copy_(torch.from_numpy(pool.hs[i]))
    n = len(pos)
    qd, td, pd = to_dev(q.reshape(n, -1)), dev(table), dev(pos)
    out = torch.full((n, H * hd), 7.0, device="cuda")
    ws = torch.empty(sc.pages_attend_ws(n, H, n_kv, hd), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    pool.pages.attend(n, p(qd), p(out), H, p(pd), p(td), table.shape[1], n, SCALE, p(ws), ws.numel())
    ctx.check()
    return out.double().cpu().numpy().reshape(n, H, hd)


def parts_slack(pool, kind, K, q, table, pos):
    """What the weights' two f16 parts may cost.  A weight (of the softmax, times the scale, which counts as 2^-126 at
    least) whose row's largest is held at 2^14 or more is off by 2^-22 of itself, which the general bound has, or by
    half the smallest f16, 2^-25: 2^-39 of that largest one, times the value's byte."""
    n, hd = len(pos), K.shape[3]
    out = np.zeros((n, H, 1))
    for r in range(n):
        t = np.arange(pos[r] + 1)
        b = table[r][t // 16]
        for h in range(H):
            s = (K[b, h % KV, t % 16].astype(np.float64) @ q[r, h]) * SCALE
            w = np.exp(s - s.max())
            largest = (w / w.sum() * np.maximum(pool.hs[1][b, h % KV].astype(np.float64), 2.0 ** -126)).max()
            size = np.abs(from_bytes(pool.h[1], kind)[b, h % KV, t % 16].astype(np.float64)).sum(0).max()
            out[r, h] = 2.0 ** -39 * largest * size
    return out


@pytest.mark.parametrize("kind", [sc.PAGES_I8, sc.PAGES_E4M3])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("blocks", [2, 300])
@pytest.mark.parametrize("exponent", [-149, -141, -127, -126, -120, -113, -100, 100, 119, 127])
def test_ends_of_the_v_scales(ctx, kind, hd, blocks, exponent):
    """Every V scale near 2^exponent: subnormal scales, the smallest normal one, the largest.  The result is one fp32
    number near the exact one, within half a step of a subnormal more where it is one."""
    rng = np.random.default_rng(abs(exponent))
    pool = Pool(ctx, rng, 2 * blocks, KV, 16, hd, kind)
    if exponent > 110:  # bytes 0 and +-1, so that no value overflows
        one = 1 if kind == sc.PAGES_I8 else 0x38
        pool.h[1] = rng.choice([0, one, 0xFF if kind == sc.PAGES_I8 else 0xB8], pool.shape).astype(np.uint8)
    factor = rng.uniform(1, 1.9, pool.hs[1].shape) if exponent > -149 else 1.0
    pool.hs[1] = (np.full(pool.hs[1].shape, 2.0 ** exponent) * factor).astype(np.float32)
    table, pos = rng.permutation(2 * blocks).reshape(2, blocks), [16 * blocks - 1, 16 * blocks - 7]
    q = rng.normal(0, 1, (2, H, hd)).astype(np.float32)
    got = attend(ctx, pool, table, pos, q)
    K = from_bytes(pool.h[0], kind) * pool.hs[0][..., None, None]
    V = from_bytes(pool.h[1], kind).astype(np.float64) * pool.hs[1].astype(np.float64)[..., None, None]
    ref, lim = attend_reference(q, K, V, table, [0, 1], pos, 16, H, SCALE)
    lim += parts_slack(pool, kind, K, q, table, pos)
    assert np.all(np.abs(got - ref) <= lim + 2.0 ** -150)


@pytest.mark.parametrize("kind", [sc.PAGES_I8, sc.PAGES_E4M3])
@pytest.mark.parametrize("first", [0, 1])
@pytest.mark.parametrize("apart", [10, 20, 30, 45])
def test_v_scales_far_apart(ctx, kind, first, apart):
    """A block whose scale is 2^apart of the others', with zeros in half its dimensions: there the others' values are
    the result, as far as the weights' parts hold them."""
    rng = np.random.default_rng(apart)
    n, hd = 8, 64
    pool = Pool(ctx, rng, n, KV, 16, hd, kind)
    pool.hs[1][:] = rng.uniform(1, 2, pool.hs[1].shape).astype(np.float32)
    large = 0 if first else n - 1
    pool.hs[1][large] *= np.float32(2.0 ** apart)
    pool.h[1][large, :, :, : hd // 2] = 0
    table, pos = np.arange(n).reshape(1, n), [16 * n - 1]
    q = 0.1 * rng.normal(0, 1, (1, H, hd)).astype(np.float32)
    got = attend(ctx, pool, table, pos, q)
    K, V = pool.values()
    ref, lim = attend_reference(q, K, V, table, [0], pos, 16, H, SCALE)
    lim += parts_slack(pool, kind, K, q, table, pos)
    assert np.all(np.abs(got - ref) <= lim)
    if apart <= 20:  # within 2^-15 of the smaller blocks' own values
        small = np.abs(ref[0, :, : hd // 2])
        size = np.abs(V[first: n - 1 + first]).mean()
        assert np.all(np.abs(got - ref)[0, :, : hd // 2] <= 2.0 ** -15 * size) and small.max() > 0.01 * size
