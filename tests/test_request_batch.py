"""The request-batch operators together, as a server's decode loop uses them:
finished requests give their blocks back, the others get blocks, slots and
positions, K/V rows enter the pools, every row attends, logits become tokens.
Each step against the operators' own references; then captured and replayed,
on other streams, and twice at once."""
import numpy as np
import pytest
import torch

from conftest import to_dev
from shukuchi_b200 import cuda as sc
from test_pages import Pool, append_reference, assign_reference, attend_reference, dev, p
from test_sample import kept_weights

pytestmark = pytest.mark.gpu


class Server:
    """Fixed-size device arrays of a decode loop over `slots` requests; step() makes the calls of one step on a stream."""

    def __init__(self, ctx, rng, slots, n_blocks, block, rows, H=8, KV=2, hd=64, vocab=300, kind=sc.PAGES_I8):
        self.ctx, self.n, self.block, self.rows, self.H, self.KV, self.hd, self.vocab = ctx, slots, block, rows, H, KV, hd, vocab
        self.stride, self.n_blocks = 12, n_blocks
        self.pool = Pool(ctx, rng, n_blocks, KV, block, hd, kind)
        self.free = dev(rng.permutation(n_blocks))
        self.counts = dev([n_blocks, 0, 0])  # counts[0]: the free stack's height, updated in place
        self.lens, self.done, self.add = dev([0] * slots), dev([0] * slots), dev([0] * slots)
        self.table = dev(np.full((slots, self.stride), -1))
        self.slot, self.pos, self.seq, self.last = (dev([-7] * n) for n in (rows, rows, rows, slots))
        self.k, self.v = (torch.zeros(rows, KV * hd, device="cuda") for _ in range(2))
        self.q = torch.zeros(rows, H * hd, device="cuda")
        self.out = torch.zeros(rows, H * hd, device="cuda")
        self.logits = torch.zeros(slots, vocab, device="cuda")
        self.u = torch.zeros(slots, device="cuda")
        self.temp, self.top_k = torch.full((slots,), 0.8, device="cuda"), dev([20] * slots)
        self.top_p = torch.full((slots,), 0.9, device="cuda")
        self.ids = dev([-7] * slots)
        self.ws = torch.empty(sc.pages_attend_ws(rows, H, KV, hd), dtype=torch.uint8, device="cuda")

    def step(self, stream=None):
        c, n = self.ctx, self.n
        c.pages_release(n, self.block, self.n_blocks, self.stride, p(self.table), p(self.done), p(self.lens), p(self.lens),
                        p(self.free), p(self.counts), p(self.counts), stream=stream)
        c.pages_assign(n, self.block, self.n_blocks, self.stride, self.rows, p(self.lens), p(self.add), p(self.table),
                       p(self.free), p(self.counts), p(self.lens), p(self.counts), p(self.slot), p(self.pos), p(self.seq),
                       p(self.last), stream=stream)
        self.pool.pages.append(self.rows, p(self.k), p(self.v), p(self.slot), stream=stream)
        self.pool.pages.attend(self.rows, p(self.q), p(self.out), self.H, p(self.pos), p(self.table), self.stride, n, 0.125,
                               p(self.ws), self.ws.numel(), row_seq=p(self.seq), stream=stream)
        c.sample(p(self.logits), n, self.vocab, p(self.u), p(self.ids), temperature=p(self.temp), top_k=p(self.top_k),
                 top_p=p(self.top_p), stream=stream)

    def fill(self, rng, add, done):
        self.add.copy_(dev(add))
        self.done.copy_(dev(done))
        for t in (self.k, self.v, self.q):
            t.copy_(to_dev(rng.normal(0, 1, tuple(t.shape)).astype(np.float32)))
        self.logits.copy_(to_dev(rng.normal(0, 3, tuple(self.logits.shape)).astype(np.float32)))
        self.u.copy_(to_dev(rng.random(self.n).astype(np.float32)))
        self.out.fill_(7.0)
        torch.cuda.synchronize()

    def state(self):
        return [t.clone() for t in (self.lens, self.counts, self.table, self.free, self.slot, self.pos, self.seq, self.last,
                                    self.out, self.ids, *self.pool.d, *self.pool.ds)]


def plan(rng, slots, step):
    """What a scheduler would ask for: prompts, single tokens, a few drafts, idle slots."""
    add = np.where(rng.random(slots) < 0.25, rng.integers(2, 30, slots), 1)
    add[rng.random(slots) < 0.15] = 0
    return add, (rng.random(slots) < 0.2).astype(int) if step else np.zeros(slots, int)


@pytest.mark.parametrize("kind,blocks", [(sc.PAGES_I8, 90), (sc.PAGES_E4M3, 14)])
def test_steps_together(ctx, kind, blocks):
    """Eight steps of twelve request slots (with 14 blocks some are refused), every result against its reference."""
    rng = np.random.default_rng(blocks)
    s = Server(ctx, rng, 12, blocks, 16, 160, kind=kind)
    lens, table, free, n_free = np.zeros(12, int), np.full((12, 12), -1), s.free.cpu().numpy().copy(), blocks
    refused = 0
    for step in range(8):
        add, done = plan(rng, 12, step)
        s.fill(rng, add, done)
        s.step()
        ctx.check()
        # tables
        for r in range(12):
            if done[r]:
                back = table[r, : -(-lens[r] // 16)]
                free[n_free: n_free + len(back)] = back
                n_free += len(back)
                lens[r] = 0
        table, lens, last, rows, counts = assign_reference(lens, add, table, free, n_free, 16, 12, 160)
        n_free = counts[0]
        refused += counts[2]
        assert s.counts.tolist() == counts and np.array_equal(s.lens.cpu().numpy(), lens)
        assert np.array_equal(s.table.cpu().numpy(), table) and np.array_equal(s.free.cpu().numpy(), free)
        assert np.array_equal(s.last.cpu().numpy(), last)
        for got, want in zip((s.slot, s.pos, s.seq), rows):
            assert np.array_equal(got.cpu().numpy(), want)
        # pools
        for i, x in enumerate((s.k, s.v)):
            assert not append_reference(s.pool.h[i], s.pool.hs[i], x.cpu().numpy(), rows[0], 16, kind)
        s.pool.same()
        # attention
        K, V = s.pool.values()
        ref, lim = attend_reference(s.q.cpu().numpy().reshape(160, 8, 64), K, V, table, rows[2], rows[1], 16, 8, 0.125)
        out, live = s.out.double().cpu().numpy().reshape(160, 8, 64), rows[2] >= 0
        assert np.all(np.abs(out - ref)[live] <= lim[live]) and (out[~live] == 7).all()
        # tokens
        for r, i in enumerate(s.ids.tolist()):
            w, close = kept_weights(s.logits[r].cpu().numpy(), 0.8, 20, 0.9, 0.0)
            assert close or w[i] > 0
    assert (refused > 0) == (blocks == 14)


def test_captured_steps_equal_eager_ones(ctx):
    """One captured step replayed seven times gives what seven calls give, bit for bit: lengths, the free stack and the
    pools advance on the device."""
    servers = [Server(ctx, np.random.default_rng(5), 12, 90, 16, 160) for _ in range(2)]
    eager, graph = servers
    g = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=side):
        graph.step(stream=side.cuda_stream)
    for step in range(7):
        rngs = [np.random.default_rng(100 + step) for _ in servers]
        add, done = plan(np.random.default_rng(step), 12, step)
        for s, rng in zip(servers, rngs):
            s.fill(rng, add, done)
        eager.step()
        g.replay()
        torch.cuda.synchronize()
        ctx.check()
        for a, b in zip(eager.state(), graph.state()):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_two_captured_steps_at_once(ctx):
    """Two servers' captured steps, each with its own workspace, replayed on two streams at the same time."""
    make = lambda: [Server(ctx, np.random.default_rng(50 + i), 12, 90, 16, 160) for i in range(2)]
    eager, twin = make(), make()
    graphs, streams = [], [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for s, st in zip(twin, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            s.step(stream=st.cuda_stream)
        graphs.append(g)
    for step in range(6):
        for group in (eager, twin):
            for i, s in enumerate(group):
                add, done = plan(np.random.default_rng(10 * step + i), 12, step)
                s.fill(np.random.default_rng(1000 + 10 * step + i), add, done)
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        for s in eager:
            s.step()
        torch.cuda.synchronize()
        ctx.check()
        for a, b in zip(eager, twin):
            for x, y in zip(a.state(), b.state()):
                assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


def test_on_the_callers_stream(ctx):
    """Inputs written on a stream just before the calls on it, results read on it just after: no other synchronisation."""
    rng = np.random.default_rng(2)
    want = Server(ctx, np.random.default_rng(1), 12, 90, 16, 160)
    got = Server(ctx, np.random.default_rng(1), 12, 90, 16, 160)
    add, done = plan(rng, 12, 0)
    want.fill(np.random.default_rng(3), add, done)
    want.step()
    torch.cuda.synchronize()
    staged = [t.clone() for t in (want.q, want.k, want.v, want.logits, want.u, want.add)]
    st = torch.cuda.Stream()
    got.out.fill_(7.0)
    busy = torch.randn(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        for _ in range(10):
            busy = busy @ busy * 1e-3
        for t, x in zip((got.q, got.k, got.v, got.logits, got.u, got.add), staged):
            t.copy_(x)
        got.step(stream=st.cuda_stream)
        seen = got.state()
    torch.cuda.synchronize()
    ctx.check()
    for a, b in zip(want.state(), seen):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
