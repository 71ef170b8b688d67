"""Block ids outside the pool, from the free stack and in the tables: what they
touch is left out of that call and of all later ones, and never becomes
another request's blocks."""
import numpy as np
import pytest
import torch

from shukuchi_b200 import cuda as sc
from test_pages import Pool, Tables, dev, p

pytestmark = pytest.mark.gpu


def refused(ctx):
    with pytest.raises(sc.ShkError) as e:
        ctx.check()
    assert e.value.code == -8


@pytest.mark.parametrize("bad", [-1, -2 ** 31, 8, 2 ** 31 - 1])
@pytest.mark.parametrize("n_rows", [40, 9000])
def test_assign_marks_rows_of_a_bad_block(ctx, bad, n_rows):
    """Request 0's new block is one outside the pool, request 1's held block too; request 2's are good.  Their rows
    are nobody's in every array, the table forgets what stood there, the good request is served."""
    table = np.array([[3, 0, 7], [bad, 0, 7], [2, 0, 7]])  # beyond what is held: ids of other requests
    free = [6, 4, bad, 0, 0, 0, 0, 0]  # request 0 takes `bad` and 4, request 2 takes 6
    t = Tables([16, 4, 15], [18, 2, 2], table, free, 3, n_rows)
    t.assign(ctx, 16, 8, 3)
    refused(ctx)
    slots, pos, seq = (x.cpu().numpy() for x in t.rows)
    want_pos = [-1] * 16 + [32, 33] + [-1, -1] + [15, 16]
    want_slot = [-1] * 16 + [64, 65] + [-1, -1] + [2 * 16 + 15, 6 * 16]
    want_seq = [-1] * 16 + [0, 0] + [-1, -1] + [2, 2]
    for got, want in zip((slots, pos, seq), (want_slot, want_pos, want_seq)):
        assert got.tolist() == want + [-1] * (n_rows - 22)
    assert t.table.tolist() == [[3, -1, 4], [bad, 0, 7], [2, 6, 7]]
    assert t.last.tolist() == [17, -1, 21] and t.lens.tolist() == [34, 6, 17] and t.counts.tolist() == [0, 22, 0]


def test_a_bad_block_stays_out_of_the_steps_behind_it(ctx):
    """A request takes an id outside the pool; its table held another request's block there.  Nothing of that request
    is read or written, in this step or the next ones."""
    rng = np.random.default_rng(3)
    pool = Pool(ctx, rng, 4, 2, 16, 64, sc.PAGES_I8)
    table, free = dev([[0, 1], [2, 1]]), dev([99, 0, 0, 0])  # request 0 owns 0 and 1; request 1 only 2
    lens, counts = dev([32, 16]), dev([1, 0, 0])
    slots, pos, seq, last = (dev([-7] * n) for n in (2, 2, 2, 2))
    add, x = dev([0, 1]), torch.randn(2, 128, device="cuda")
    q, out = torch.randn(2, 256, device="cuda"), torch.full((2, 256), 7.0, device="cuda")
    ws = torch.empty(sc.pages_attend_ws(2, 4, 2, 64), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    for step in range(3):
        ctx.pages_assign(2, 16, 4, 2, 2, p(lens), p(add), p(table), p(free), p(counts), p(lens), p(counts), p(slots), p(pos),
                         p(seq), p(last))
        refused(ctx)
        assert slots.tolist() == pos.tolist() == seq.tolist() == [-1, -1] and last.tolist() == [-1, -1]
        assert table.tolist() == [[0, 1], [2, -1]] and lens.tolist() == [32, 17 + step]
        pool.pages.append(2, p(x), p(x), p(slots))
        pool.pages.attend(2, p(q), p(out), 4, p(pos), p(table), 2, 2, 0.125, p(ws), ws.numel(), row_seq=p(seq))
        ctx.check()
        pool.same()
        assert (out == 7).all()


@pytest.mark.parametrize("n,stride", [(3, 4), (40, 30), (1200, 9)])
def test_release_leaves_out_bad_ids(ctx, n, stride):
    """Every seventh id is outside the pool: the others go back in order, the height counts them alone."""
    rng = np.random.default_rng(n)
    n_blocks = 3 * n * stride
    have, done = rng.integers(0, 16 * stride + 1, n), rng.integers(0, 2, n)
    table = rng.permutation(n_blocks)[: n * stride].reshape(n, stride)
    hurt = np.where(rng.random(table.shape) < 1 / 7, rng.choice([-1, n_blocks, -2 ** 31, 2 ** 31 - 1], table.shape), table)
    hurt[-1, 0], have[-1], done[-1] = n_blocks, max(1, have[-1]), 1
    free = np.full(n_blocks, -9)
    free[:5] = [1, 2, 3, 4, 5]
    h, d, t, f, height = dev(have), dev(done), dev(hurt), dev(free), dev([5])
    lens = dev(np.full(n, -5))
    ctx.pages_release(n, 16, n_blocks, stride, p(t), p(d), p(h), p(lens), p(f), p(height), p(height))
    refused(ctx)
    back = [i for r in range(n) if done[r] for i in hurt[r, : -(-have[r] // 16)] if 0 <= i < n_blocks]
    assert height.item() == 5 + len(back)
    assert f.tolist()[: 5 + len(back)] == free[:5].tolist() + back
    assert np.array_equal(lens.cpu().numpy(), np.where(done != 0, 0, have))


def test_release_leaves_out_bad_lengths(ctx):
    """A negative length and one that its table row cannot hold stay as they are; the other requests' blocks go back."""
    table, have, done = dev([[0, 1], [2, 3], [4, 5], [6, 7]]), dev([32, -3, 33, 16]), dev([1, 1, 1, 5])
    free, height, lens = dev([8, 9] + [-9] * 8), dev([2]), dev([-5] * 4)
    ctx.pages_release(4, 16, 10, 2, p(table), p(done), p(have), p(lens), p(free), p(height), p(height))
    refused(ctx)
    assert lens.tolist() == [0, -3, 33, 0] and height.item() == 5 and free.tolist()[:5] == [8, 9, 0, 1, 6]
