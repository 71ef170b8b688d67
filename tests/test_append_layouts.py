"""Appends of prompts: calls large enough that a CTA takes whole blocks of one
head, several runs, more than 256 tokens, or a run too long for its registers.
Bytes and scales as in test_pages, bit for bit."""
import numpy as np
import pytest
import torch

from conftest import to_dev
from shukuchi_b200 import cuda as sc
from test_pages import TORCH, Pool, append_reference, dev, p

pytestmark = pytest.mark.gpu
F32, F16, BF16 = 0, 1, 30


def prompts(rng, block, n, short):
    """Slots of about n tokens of requests that hold some tokens already, padding rows between some of them, and the
    blocks that they take."""
    slots, blocks = [], 0
    while len(slots) < n:
        have, add = int(rng.integers(0, block)), int(rng.integers(1, short if rng.random() < 0.5 else 5 * block))
        at = np.arange(have, have + add)
        slots += [(blocks + t // block) * block + t % block for t in at.tolist()] + [-1] * int(rng.integers(0, 2))
        blocks += -(-(have + add) // block)
    return np.array(slots), blocks


def run(ctx, rng, kind, dtype, n_kv, hd, block, slots, blocks, pad=8, gain=1.0):
    perm = rng.permutation(blocks)
    slots = np.where(slots >= 0, perm[slots // block] * block + slots % block, slots)
    pool, w = Pool(ctx, rng, blocks, n_kv, block, hd, kind), n_kv * hd
    x = [(rng.normal(0, gain, (len(slots), w + pad)) * np.exp(rng.normal(0, 1, (len(slots), 1)))).astype(np.float32) for _ in range(2)]
    xd, sd = [to_dev(a).to(TORCH[dtype]) for a in x], dev(slots)
    torch.cuda.synchronize()
    pool.pages.append(len(slots), p(xd[0]), p(xd[1]), p(sd), dtype=dtype, row_stride=w + pad)
    ctx.sync()
    twice = [append_reference(pool.h[i], pool.hs[i], xd[i].float().cpu().numpy()[:, :w], slots, block, kind) for i in range(2)]
    if twice[0]:
        with pytest.raises(sc.ShkError):
            ctx.check()
    else:
        ctx.check()
    pool.same()
    return twice[0]


@pytest.mark.parametrize("kind", [sc.PAGES_I8, sc.PAGES_E4M3])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n_kv,hd,block,n,pad", [
    (8, 128, 32, 900, 8),    # a block of one head a CTA
    (8, 64, 64, 2500, 1),    # two blocks a CTA; rows that begin anywhere
    (4, 128, 128, 1500, 0),  # runs that a CTA's registers do not hold
    (4, 64, 256, 1500, 8),
    (40, 64, 32, 2600, 0)])  # more than 256 tokens a CTA
def test_append_of_whole_blocks(ctx, kind, dtype, n_kv, hd, block, n, pad):
    rng = np.random.default_rng(n + block + dtype)
    slots, blocks = prompts(rng, block, n, 40)
    assert not run(ctx, rng, kind, dtype, n_kv, hd, block, slots, blocks, pad)


@pytest.mark.parametrize("kind,dtype", [(sc.PAGES_I8, F32), (sc.PAGES_E4M3, BF16)])
@pytest.mark.parametrize("n_kv,n", [(8, 1500), (256, 2700)])
def test_append_of_many_short_runs(ctx, kind, dtype, n_kv, n):
    """Blocks of 16, a warp to a run and head: several runs a CTA, and (256 heads) more than 256 tokens."""
    rng = np.random.default_rng(n)
    slots, blocks = prompts(rng, 16, n, 9)
    assert not run(ctx, rng, kind, dtype, n_kv, 64, 16, slots, blocks)


@pytest.mark.parametrize("n_kv,hd,block,n", [(8, 64, 32, 2000), (40, 64, 32, 2600), (16, 64, 16, 3000)])
@pytest.mark.parametrize("apart", [1, 40, 300, 1500])
def test_append_of_prompts_refuses_second_runs(ctx, n_kv, hd, block, n, apart):
    """Blocks that come again a few tokens, a CTA, a list of tokens and most of the call later: the first run is stored."""
    rng = np.random.default_rng(apart)
    slots, blocks = prompts(rng, block, n, 40)
    live = np.flatnonzero(slots >= 0)
    for t in rng.choice(live[live < n - apart - 2], 6, replace=False):
        slots[t + apart] = slots[t]
    assert run(ctx, rng, sc.PAGES_I8, F32, n_kv, hd, block, slots, blocks)


def test_append_grows_scales_of_a_long_run(ctx):
    """The later part of whole blocks: earlier rows of the block are rounded again by all of a CTA's warps."""
    rng = np.random.default_rng(4)
    for kind, dtype, hd, block in ((sc.PAGES_I8, F32, 128, 128), (sc.PAGES_E4M3, F16, 64, 256), (sc.PAGES_I8, BF16, 64, 32)):
        blocks = 24
        slots = np.concatenate([b * block + np.arange(block // 4 + b % 5, block) for b in range(blocks)])
        assert not run(ctx, rng, kind, dtype, 8, hd, block, slots, blocks, gain=40.0)
