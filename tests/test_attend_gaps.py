"""Attention where thousands of rows that are nobody's lie between two live ones, as a refused prompt leaves them."""
import numpy as np
import pytest

from shukuchi_b200 import cuda as sc
from test_pages import Pool, run_attend

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("gap", [1, 2, 31, 32, 127, 128, 129, 257, 4000])
@pytest.mark.parametrize("H,KV,hd", [(8, 4, 64), (32, 2, 128), (3, 1, 64)])
def test_attend_across_a_gap(ctx, gap, H, KV, hd):
    """Rows of one, two and five at a time, gaps before, between and behind them; requests of every length, so that parts
    of the work begin and end next to a gap."""
    rng = np.random.default_rng(gap + H)
    lens = [300, 5, 40, 1, 16, 900]
    pool = Pool(ctx, rng, sum(-(-n // 16) for n in lens) + 2, KV, 16, hd, sc.PAGES_I8)
    plan = [(-1, 3)] * (gap // 2)
    for z, rows in ((0, 1), (1, 5), (2, 2), (0, 5), (3, 1), (5, 3), (4, 1)):
        plan += [(z, lens[z] - 1 - int(j)) for j in rng.integers(0, lens[z], rows)] + [(-1, 0)] * gap
    run_attend(ctx, pool, rng, lens, 0, H, 0, plan=plan)


@pytest.mark.parametrize("gap", [3, 128, 3000])
def test_attend_across_a_gap_with_idle_slots(ctx, gap):
    """As many request slots as rows, most of them idle, one row a request."""
    rng = np.random.default_rng(gap)
    lens = [500, 3, 70, 1] + [0] * (4 * gap + 8)
    pool = Pool(ctx, rng, sum(-(-n // 16) for n in lens) + 2, 2, 16, 64, sc.PAGES_E4M3)
    plan = [row for z in range(4) for row in [(z, lens[z] - 1)] + [(-1, 2)] * gap]
    run_attend(ctx, pool, rng, lens, 0, 8, 0, plan=plan)
