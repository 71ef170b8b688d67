"""Requests cut short: the blocks behind the last kept token go back, and a
server that rejects drafts step after step keeps every block of its pool."""
import numpy as np
import pytest
import torch

import test_request_batch as batch
from shukuchi_b200 import cuda as sc
from test_pages import append_reference, assign_reference, attend_reference, dev, p, tables_case

gpu = pytest.mark.gpu


def test_refused_without_a_context():
    assert sc.lib().shk_cuda_pages_truncate(None, 1, 16, 1, 1, None, None, None, None, None, None, None, None) == -1


@gpu
@pytest.mark.parametrize("in_place", [None, "have", "keep"])
@pytest.mark.parametrize("n,block,longest", [(1, 16, 40), (7, 32, 500), (1500, 16, 90), (16384, 256, 300)])
def test_truncate(ctx, n, block, longest, in_place):
    rng = np.random.default_rng(n)
    have, _, table, free, stride, n_blocks = tables_case(rng, n, block, longest, 0, 9)
    keep = np.where(rng.random(n) < 0.5, rng.integers(0, longest + 9, n), np.maximum(have - rng.integers(-2, 20, n), 0))
    h, k, t, f, height, after = dev(have), dev(keep), dev(table), dev(free), dev([9]), dev([-5])
    lens = {None: dev(np.full(n, -5)), "have": h, "keep": k}[in_place]
    after = height if in_place else after
    ctx.pages_truncate(n, block, n_blocks, stride, p(t), p(k), p(h), p(lens), p(f), p(height), p(after))
    ctx.check()
    kept = np.minimum(keep, have)
    back = [i for r in range(n) for i in table[r, -(-kept[r] // block): -(-have[r] // block)]]
    free[9: 9 + len(back)] = back
    assert np.array_equal(f.cpu().numpy(), free) and after.item() == 9 + len(back)
    assert np.array_equal(lens.cpu().numpy(), kept) and np.array_equal(t.cpu().numpy(), table)


@gpu
def test_rejected_drafts_give_their_blocks_back(ctx):
    """One token and three drafts a step, of which none to all are accepted: after forty steps no block is lost, and
    the tables are those of the lengths alone.  14 blocks would be gone after a few steps otherwise."""
    rng = np.random.default_rng(1)
    n, block, stride, n_blocks, rows = 3, 16, 8, 14, 12
    table, free = np.full((n, stride), -1), rng.permutation(n_blocks)
    t, f, height, counts = dev(table), dev(free), dev([n_blocks]), dev([0] * 3)
    lens, add, last = dev([0] * n), dev([4] * n), dev([0] * n)
    out = [dev([0] * rows) for _ in range(3)]
    have, n_free = np.zeros(n, int), n_blocks
    for step in range(40):
        ctx.pages_assign(n, block, n_blocks, stride, rows, p(lens), p(add), p(t), p(f), p(height), p(lens), p(counts),
                         *[p(x) for x in out], p(last))
        ctx.check()
        table, after, _, want, c = assign_reference(have, np.full(n, 4), table, free, n_free, block, stride, rows)
        assert np.array_equal(t.cpu().numpy(), table) and counts.tolist() == c and c[2] == 0
        for x, y in zip(out, want):
            assert np.array_equal(x.cpu().numpy(), y)
        # one to four of the tokens stay; a request past 60 tokens ends
        keep = np.where(after > 60, 0, have + rng.integers(1, 5, n))
        back = [i for r in range(n) for i in table[r, -(-keep[r] // block): -(-after[r] // block)]]
        n_free = c[0] + len(back)
        free[c[0]: n_free] = back
        k = dev(keep)
        ctx.pages_truncate(n, block, n_blocks, stride, p(t), p(k), p(lens), p(lens), p(f), p(counts), p(height))
        ctx.check()
        have = keep
        assert height.item() == n_free and np.array_equal(lens.cpu().numpy(), have)
        assert n_free + sum(-(-h // block) for h in have) == n_blocks
        held = [i for r in range(n) for i in table[r, : -(-have[r] // block)]]
        assert sorted(held + f.tolist()[:n_free]) == list(range(n_blocks))


@gpu
def test_truncate_leaves_out_bad_lengths(ctx):
    """Negative lengths to keep and lengths that a table row cannot hold: those requests stay as they are.  A request
    that keeps all it has is not looked at, and a stack that would outgrow the pool takes nothing."""
    table, have, keep = dev([[0, 1], [2, 3], [4, 5], [6, 7], [8, 9]]), dev([32, 17, 33, 16, 40]), dev([16, -1, 5, 0, 40])
    free, height, lens = dev([-9] * 10), dev([0]), dev([-5] * 5)
    call = lambda: ctx.pages_truncate(5, 16, 10, 2, p(table), p(keep), p(have), p(lens), p(free), p(height), p(height))
    call()
    with pytest.raises(sc.ShkError):
        ctx.check()
    assert lens.tolist() == [16, 17, 33, 0, 40] and height.item() == 2 and free.tolist()[:2] == [1, 6]
    height.fill_(9)
    call()
    with pytest.raises(sc.ShkError):
        ctx.check()
    assert lens.tolist() == have.tolist() and height.item() == 9


@gpu
def test_truncate_arguments(ctx):
    x = dev([1] * 16)
    for block, n_blocks, stride, n in ((8, 4, 1, 1), (16, 0, 1, 1), (16, 4, 0, 1), (16, 4, 1, 0), (16, 4, 1, 16385)):
        with pytest.raises(sc.ShkError):
            ctx.pages_truncate(n, block, n_blocks, stride, *[p(x)] * 7)
    for at in range(7):
        for bad in (None, p(x) + 2):
            with pytest.raises(sc.ShkError):
                ctx.pages_truncate(1, 16, 4, 1, *[bad if i == at else p(x) for i in range(7)])
    ctx.check()


class Drafts(batch.Server):
    """A step that begins with the lengths to keep (in `done`), as after a check of drafts."""

    def step(self, stream=None):
        c, n = self.ctx, self.n
        c.pages_truncate(n, self.block, self.n_blocks, self.stride, p(self.table), p(self.done), p(self.lens), p(self.lens),
                         p(self.free), p(self.counts), p(self.counts), stream=stream)
        c.pages_assign(n, self.block, self.n_blocks, self.stride, self.rows, p(self.lens), p(self.add), p(self.table),
                       p(self.free), p(self.counts), p(self.lens), p(self.counts), p(self.slot), p(self.pos), p(self.seq),
                       p(self.last), stream=stream)
        self.pool.pages.append(self.rows, p(self.k), p(self.v), p(self.slot), stream=stream)
        self.pool.pages.attend(self.rows, p(self.q), p(self.out), self.H, p(self.pos), p(self.table), self.stride, n, 0.125,
                               p(self.ws), self.ws.numel(), row_seq=p(self.seq), stream=stream)


@gpu
def test_draft_steps(ctx):
    """Steps of drafts whose rejected rows are cut off again: pools and outputs against the references, and a captured
    step replayed against the calls, bit for bit."""
    eager, graph = (Drafts(ctx, np.random.default_rng(5), 12, 60, 16, 96) for _ in range(2))
    g, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=side):
        graph.step(stream=side.cuda_stream)
    rng, lens = np.random.default_rng(9), np.zeros(12, int)
    for step in range(9):
        # of the four or more tokens that the last step added one to all stay; long requests end
        keep = np.where(lens > 90, 0, np.maximum(lens - rng.integers(0, 4, 12), 0))
        add = np.where(rng.random(12) < 0.2, 0, np.where(keep == 0, rng.integers(1, 40, 12) if step % 3 == 0 else 4, 4))
        for s in (eager, graph):
            s.fill(np.random.default_rng(100 + step), add, keep)
        eager.step()
        g.replay()
        torch.cuda.synchronize()
        ctx.check()
        for a, b in zip(eager.state(), graph.state()):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        lens, counts = eager.lens.cpu().numpy(), eager.counts.tolist()
        assert counts[0] + (-(-lens // 16)).sum() == 60
        slot, pos, seq = (x.cpu().numpy() for x in (eager.slot, eager.pos, eager.seq))
        for i, x in enumerate((eager.k, eager.v)):
            assert not append_reference(eager.pool.h[i], eager.pool.hs[i], x.cpu().numpy(), slot, 16, sc.PAGES_I8)
        eager.pool.same()
        ref, lim = attend_reference(eager.q.cpu().numpy().reshape(96, 8, 64), *eager.pool.values(), eager.table.cpu().numpy(),
                                    seq, pos, 16, 8, 0.125)
        out, live = eager.out.double().cpu().numpy().reshape(96, 8, 64), seq >= 0
        assert np.all(np.abs(out - ref)[live] <= lim[live]) and (out[~live] == 7).all() and live.sum() == counts[1] > 0
