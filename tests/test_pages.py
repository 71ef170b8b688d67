"""Paged 8-bit K/V pools: block tables and slots against a loop over the
requests, appended bytes and scales against the format's definition in numpy
(equal bit for bit), attention against a 64-bit softmax over the values that
the pools stand for."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from conftest import to_dev
from shukuchi_b200 import cuda as sc

gpu = pytest.mark.gpu
U = 2.0 ** -24  # half a step of fp32
TORCH = {0: torch.float32, 1: torch.float16, 30: torch.bfloat16}


def dev(a, dtype=np.int32):
    return to_dev(np.asarray(a, dtype))


def p(t):
    return t.data_ptr()


# ---- without a GPU ----

def test_refusals_without_a_context():
    L = sc.lib()
    assert L.shk_cuda_pages_assign(None, C.byref(sc.PagesAssign()), None) == -1
    assert L.shk_cuda_pages_release(None, 1, 16, 1, 1, None, None, None, None, None, None, None, None) == -1
    assert L.shk_cuda_pages_append(None, C.byref(sc.PagesDesc()), 1, None, None, 0, 0, None, None) == -1
    assert L.shk_cuda_pages_read(None, C.byref(sc.PagesDesc()), 1, None, None, None, None) == -1
    assert L.shk_cuda_pages_attend(None, C.byref(sc.PagesDesc()), C.byref(sc.PagesRows()), None) == -1


@pytest.mark.parametrize("shape", [(1, 0, 8, 128), (1, 8, 0, 128), (1, 9, 8, 128), (1, 8, 8, 96), (1, 8, 8, 0)])
def test_workspace_of_a_shape_not_taken(shape):
    assert sc.pages_attend_ws(*shape) == 0
    assert sc.pages_attend_ws(1, 32, 8, 128) > 0


# ---- block tables ----

def assign_reference(have, add, table, free, n_free, block, stride, n_rows):
    """The rule, one request after the other."""
    table, lens, last = table.copy(), have.copy(), np.full(len(have), -1)
    rows = [np.full(n_rows, -1) for _ in range(3)]
    row0 = taken = used = live = refused = 0
    for r, (h, n) in enumerate(zip(have.tolist(), add.tolist())):
        end = row0 + max(n, 0)
        ok = h >= 0 and n >= 0 and h + n <= stride * block and (n == 0 or end <= n_rows)
        if ok:
            need = -(-(h + n) // block) - -(-h // block)
            first = taken
            taken += need  # counted whether or not the blocks suffice
            ok = need == 0 or taken <= n_free
        if not ok:
            refused += 1
        else:
            for j in range(need):
                table[r, -(-h // block) + j] = free[n_free - 1 - first - j]
            used += need
            for i in range(n):
                rows[0][row0 + i] = table[r, (h + i) // block] * block + (h + i) % block
                rows[1][row0 + i] = h + i
                rows[2][row0 + i] = r
            live += n
            lens[r] = h + n
            last[r] = end - 1 if n else -1
        row0 = end
    return table, lens, last, rows, [n_free - used, live, refused]


def tables_case(rng, n, block, longest, chunk, spare):
    have = rng.integers(0, longest + 1, n)
    add = np.where(rng.random(n) < 0.2, rng.integers(0, chunk + 1, n), rng.integers(0, 2, n))
    stride = -(-(longest + chunk) // block)
    held = -(-have // block)
    n_blocks = int(held.sum()) + spare
    ids = rng.permutation(n_blocks)
    table = np.full((n, stride), -7)
    table[np.arange(stride)[None] < held[:, None]] = ids[: held.sum()]
    free = np.full(n_blocks, -9)
    free[:spare] = ids[held.sum():]
    return have, add, table, free, stride, n_blocks


class Tables:
    """The arrays of an assign call on the device."""

    def __init__(self, have, add, table, free, n_free, n_rows, in_place=False):
        n = len(have)
        self.have, self.add, self.table, self.free = dev(have), dev(add), dev(table), dev(free)
        self.counts = dev([n_free, 0, 0])
        self.n_free = self.counts if in_place else dev([n_free])
        self.lens = self.have if in_place else dev(np.full(n, -5))
        self.last = dev(np.full(n, -5))
        self.rows = [dev(np.full(max(n_rows, 1), -5)) for _ in range(3)]
        self.n_rows = n_rows

    def assign(self, ctx, block, n_blocks, stride, **kw):
        ctx.pages_assign(len(self.add), block, n_blocks, stride, self.n_rows, p(self.have), p(self.add), p(self.table),
                         p(self.free), p(self.n_free), p(self.lens), p(self.counts), *[p(t) for t in self.rows],
                         p(self.last), **kw)


@gpu
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("n,block,longest,chunk,spare,n_rows", [
    (1, 16, 0, 1, 1, 1), (1, 16, 40, 17, 4, 40), (3, 32, 200, 65, 2, 64), (64, 16, 3000, 1, 64, 64),
    (300, 64, 900, 300, 40, 5000), (1024, 16, 77, 40, 3000, 20000), (1025, 256, 5000, 600, 700, 90000),
    (5000, 16, 60, 3, 300, 1000), (16384, 16, 20, 2, 9000, 17000)])
def test_assign(ctx, n, block, longest, chunk, spare, n_rows, in_place):
    rng = np.random.default_rng(n + block)
    have, add, table, free, stride, n_blocks = tables_case(rng, n, block, longest, chunk, spare)
    t = Tables(have, add, table, free, spare, n_rows, in_place)
    t.assign(ctx, block, n_blocks, stride)
    ctx.check()
    want = assign_reference(have, add, table, free, spare, block, stride, n_rows)
    assert np.array_equal(t.counts.cpu().numpy(), want[4])
    assert np.array_equal(t.lens.cpu().numpy(), want[1])
    assert np.array_equal(t.last.cpu().numpy(), want[2])
    for got, rows in zip(t.rows, want[3]):
        assert np.array_equal(got.cpu().numpy()[:n_rows], rows)
    assert np.array_equal(t.table.cpu().numpy(), want[0])
    assert np.array_equal(t.free.cpu().numpy(), free)


@gpu
def test_assign_refuses_requests_one_by_one(ctx):
    """Negative lengths, a table outgrown, rows outgrown, too few blocks: each
    request alone is refused; those that need nothing still pass."""
    have = np.array([5, -1, 30, 0, 31, 16, 3, 0])
    add = np.array([1, 2, 40, 33, 1, -1, 1, 0])  # request 2: 70 > 4 blocks of 16; 3: needs 3 of the 2 blocks; 4: fits
    table = np.arange(32).reshape(8, 4)
    free = np.array([40, 41] + [0] * 62)
    for n_rows in (0, 1, 40, 100):
        t = Tables(have, add, table, free, 2, n_rows)
        t.assign(ctx, 16, 64, 4)
        ctx.check()
        want = assign_reference(have, add, table, free, 2, 16, 4, n_rows)
        assert np.array_equal(t.counts.cpu().numpy(), want[4])
        assert np.array_equal(t.lens.cpu().numpy(), want[1])
        for got, rows in zip(t.rows, want[3]):
            assert np.array_equal(got.cpu().numpy()[:n_rows], rows)
        assert np.array_equal(t.table.cpu().numpy(), want[0])


@gpu
def test_assign_leaves_out_bad_block_ids(ctx):
    table = np.array([[3, 99], [1, 0], [2, 0]])  # request 0's second block is outside the pool of 8
    for free, bad in (([4, 5], [0]), ([-2, 5], [0, 2])):  # then a free id below 0, given to request 2
        t = Tables([20, 4, 16], [1, 1, 1], table, free + [0] * 6, 1, 3)
        t.assign(ctx, 16, 8, 2)
        with pytest.raises(sc.ShkError) as e:
            ctx.check()
        assert e.value.code == -8
        slots = t.rows[0].cpu().numpy()
        assert [i for i in range(3) if slots[i] < 0] == bad and slots[1] == 20
    ctx.check()


@gpu
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("n,block,longest", [(1, 16, 40), (7, 32, 500), (1500, 16, 90), (16384, 256, 300)])
def test_release(ctx, n, block, longest, in_place):
    rng = np.random.default_rng(n)
    have, _, table, free, stride, n_blocks = tables_case(rng, n, block, longest, 0, 9)
    done = rng.integers(0, 2, n) * rng.integers(1, 9, n)
    h, lens = dev(have), dev(np.full(n, -5))
    f, height, after = dev(free), dev([9]), dev([-5])
    lens, after = (h, height) if in_place else (lens, after)
    d, t = dev(done), dev(table)
    ctx.pages_release(n, block, n_blocks, stride, p(t), p(d), p(h), p(lens), p(f), p(height), p(after))
    ctx.check()
    back = [i for r in range(n) if done[r] for i in table[r, : -(-have[r] // block)]]
    free[9: 9 + len(back)] = back
    assert np.array_equal(f.cpu().numpy(), free)
    assert after.item() == 9 + len(back)
    assert np.array_equal(lens.cpu().numpy(), np.where(done != 0, 0, have))


@gpu
def test_release_of_more_than_the_pool_is_refused(ctx):
    table, have, done = dev([[0, 1], [2, 3]]), dev([32, 32]), dev([1, 1])
    free, height, lens = dev([0, 1, 2, 3]), dev([1]), dev([-5, -5])
    ctx.pages_release(2, 16, 4, 2, p(table), p(done), p(have), p(lens), p(free), p(height), p(height))
    with pytest.raises(sc.ShkError):
        ctx.check()
    assert height.item() == 1 and lens.tolist() == [32, 32] and free.tolist() == [0, 1, 2, 3]


@gpu
def test_table_arguments(ctx):
    t = Tables([1], [1], [[0]], [0] * 4, 1, 1)
    for block, n_blocks, stride in ((8, 4, 1), (24, 4, 1), (512, 4, 1), (0, 4, 1), (16, 0, 1), (16, 4, 0),
                                    (256, 1 << 23, 1)):
        with pytest.raises(sc.ShkError):
            t.assign(ctx, block, n_blocks, stride)
        with pytest.raises(sc.ShkError):
            ctx.pages_release(1, block, n_blocks, stride, *[p(t.have)] * 7)
    t.n_rows = 1 << 30
    with pytest.raises(sc.ShkError):
        t.assign(ctx, 16, 4, 1)
    for n in (0, 16385):
        with pytest.raises(sc.ShkError):
            ctx.pages_assign(n, 16, 4, 1, 1, *[p(t.have)] * 11)
    with pytest.raises(sc.ShkError):
        ctx.pages_assign(1, 16, 4, 1, 1, *[p(t.have)] * 10, None)
    ctx.check()


@gpu
def test_arrays_of_words_are_aligned(ctx):
    """Every int32 and float array two bytes off: refused before any launch."""
    t = Tables([1], [1], [[0]], [0] * 4, 1, 1)
    x = torch.zeros(4096, device="cuda")
    i = p(t.have)
    for at in range(11):
        with pytest.raises(sc.ShkError):
            ctx.pages_assign(1, 16, 4, 1, 1, *[i + 2 * (j == at) for j in range(11)])
    for at in range(7):
        with pytest.raises(sc.ShkError):
            ctx.pages_release(1, 16, 4, 1, *[i + 2 * (j == at) for j in range(7)])
    pool = Pool(ctx, np.random.default_rng(1), 2, 1, 16, 64, sc.PAGES_I8)
    with pytest.raises(sc.ShkError):
        pool.pages.append(1, p(x), p(x), i + 2)
    for at in range(3):
        with pytest.raises(sc.ShkError):
            pool.pages.read(1, *[(i if j == 0 else p(x)) + 2 * (j == at) for j in range(3)])
    ws = torch.zeros(sc.pages_attend_ws(1, 1, 1, 64), dtype=torch.uint8, device="cuda")
    for bad in ("row_pos", "table", "row_seq"):
        arrays = {n: i + 2 * (n == bad) for n in ("row_pos", "table", "row_seq")}
        with pytest.raises(sc.ShkError):
            pool.pages.attend(1, p(x), p(x) + 4096, 1, table_stride=1, n_seq=1, scale=1.0, ws=p(ws), ws_bytes=ws.numel(), **arrays)
    names = ("u", "out", "prob", "temperature", "top_k", "top_p", "min_p")
    for bad in names:
        with pytest.raises(sc.ShkError):
            ctx.sample(p(x), 1, 8, **{n: i + 2 * (n == bad) for n in names})
    ctx.check()
    pool.same()


# ---- append and read ----

E4M3 = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float().numpy()


def to_bytes(y, kind):
    """Rounded to the pool's type, halves to even; NaN -> 0."""
    y = np.where(np.isnan(y), np.float32(0), y).astype(np.float32)
    if kind == sc.PAGES_I8:
        return np.clip(np.rint(y), -127, 127).astype(np.int8).view(np.uint8)
    return torch.from_numpy(np.clip(y, -448, 448)).to(torch.float8_e4m3fn).view(torch.uint8).numpy()


def from_bytes(b, kind):
    return b.view(np.int8).astype(np.float32) if kind == sc.PAGES_I8 else E4M3[b]


def append_reference(pool, scale, x, slots, block, kind):
    """pool [blocks][kv][block][hd] bytes and scale [blocks][kv], changed in
    place, one run of a block's rows after the other; returns whether a block
    came twice."""
    top, n_kv, hd = np.float32(127 if kind == sc.PAGES_I8 else 448), pool.shape[1], pool.shape[3]
    t, seen, twice = 0, set(), False
    while t < len(slots):
        if slots[t] < 0:
            t += 1
            continue
        b, o = divmod(int(slots[t]), block)
        n = 1
        while t + n < len(slots) and slots[t + n] == slots[t] + n and o + n < block:
            n += 1
        if b in seen:
            twice = True
        else:
            for h in range(n_kv):
                new = x[t:t + n].reshape(n, n_kv, hd)[:, h]
                mag = np.abs(new)
                old = scale[b, h] if o else np.float32(0)
                with np.errstate(all="ignore"):
                    s = max(old, np.float32(np.max(mag[~np.isnan(mag)], initial=0)) / top)
                    if o and s > old:
                        pool[b, h, :o] = to_bytes(from_bytes(pool[b, h, :o], kind) * np.float32(old / s), kind)
                    pool[b, h, o:o + n] = to_bytes(new / s, kind) if s > 0 else 0
                scale[b, h] = s
        seen.add(b)
        t += n
    return twice


class Pool:
    """K and V pools on the device and the same on the host."""

    def __init__(self, ctx, rng, blocks, n_kv, block, hd, kind):
        self.block, self.kind, self.shape = block, kind, (blocks, n_kv, block, hd)
        self.h = [to_bytes(rng.normal(0, 30, self.shape).astype(np.float32), kind) for _ in range(2)]
        self.hs = [rng.uniform(0.005, 0.03, (blocks, n_kv)).astype(np.float32) for _ in range(2)]
        self.d, self.ds = [dev(a, np.uint8) for a in self.h], [dev(a, np.float32) for a in self.hs]
        self.pages = sc.Pages(ctx, p(self.d[0]), p(self.d[1]), p(self.ds[0]), p(self.ds[1]), kind, blocks, n_kv, hd, block)

    def same(self):
        for d, h in zip(self.d + self.ds, self.h + self.hs):
            assert np.array_equal(d.cpu().numpy(), h, equal_nan=h.dtype == np.float32)

    def values(self):
        with np.errstate(all="ignore"):
            return [from_bytes(b, self.kind) * s[..., None, None] for b, s in zip(self.h, self.hs)]


@gpu
@pytest.mark.parametrize("kind", [sc.PAGES_I8, sc.PAGES_E4M3])
@pytest.mark.parametrize("n_kv,hd,block,dtype", [(1, 64, 16, 0), (8, 128, 16, 0), (3, 64, 64, 30), (4, 128, 256, 1),
                                                 (9, 128, 32, 0), (40, 64, 16, 30)])
def test_append(ctx, kind, n_kv, hd, block, dtype):
    """Runs that begin and end anywhere in their blocks, single tokens,
    padding rows, rows further apart than they are wide; then more into the
    same blocks, larger (scales grow) and smaller."""
    rng = np.random.default_rng(hd + block + n_kv)
    pool = Pool(ctx, rng, 12, n_kv, block, hd, kind)
    w = n_kv * hd
    for gain, runs in ((1.0, [(3, 0, block), (0, 0, 1), (5, block - 1, 1), (7, 2, block - 2), (8, 0, 3), (9, 1, 7)]),
                       (3.0, [(0, 1, 1), (8, 3, 5), (9, 8, 1), (1, 0, 2), (2, 4, 1)]),
                       (0.5, [(8, 8, 1), (1, 2, block - 2), (0, 0, 4)])):
        slots = [-1]
        for b, o, n in runs:
            slots += list(range(b * block + o, b * block + o + n)) + [-1] * (b % 2)
        x = [(rng.normal(0, 1, (len(slots), w + 8)) * gain).astype(np.float32) for _ in range(2)]
        for a in x:
            a[1, :5] = 0
            a[2 % len(slots), :hd] = 0  # a head of zeros
        xd = [to_dev(a).to(TORCH[dtype]) for a in x]
        sd = dev(slots)
        pool.pages.append(len(slots), p(xd[0]), p(xd[1]), p(sd), dtype=dtype, row_stride=w + 8)
        ctx.check()
        for i in range(2):
            append_reference(pool.h[i], pool.hs[i], xd[i].float().cpu().numpy()[:, :w], slots, block, kind)
        pool.same()
    # read back, with rows left out
    at = np.array([3 * block + 1, -1, 0, 7 * block + block - 1, -3, 8 * block])
    out = [torch.full((len(at), w), 7.0, device="cuda") for _ in range(2)]
    ad = dev(at)
    pool.pages.read(len(at), p(ad), p(out[0]), p(out[1]))
    ctx.check()
    for o, v in zip(out, pool.values()):
        want = np.where((at >= 0)[:, None], v[at // block, :, at % block].reshape(len(at), w), np.float32(7))
        assert np.array_equal(o.cpu().numpy(), want)


@gpu
@pytest.mark.parametrize("kind", [sc.PAGES_I8, sc.PAGES_E4M3])
def test_append_special_values(ctx, kind):
    """NaN counts for nothing, infinities make the scale infinite, zeros give
    scale 0, subnormals and the largest floats keep the rule; a block that
    begins again forgets its scale."""
    rng = np.random.default_rng(4)
    n_kv, hd, block = 2, 64, 16
    pool = Pool(ctx, rng, 10, n_kv, block, hd, kind)
    x = rng.normal(0, 1, (10, n_kv * hd)).astype(np.float32)
    x[0, 3] = np.nan
    x[1, 5], x[1, 70] = np.inf, np.nan
    x[2, :] = 0
    x[3, :hd] = np.nan
    x[4] *= 1e-41
    x[5, :] = 3e38
    x[5, 9] = -np.inf
    x[6] *= 1e38
    x[7, :] = 1e-45
    x[8, :] = -0.0
    pool.hs[0][9, 0] = pool.hs[1][9, 1] = np.inf  # what a block held before its first place is written again
    pool.ds[0][9, 0] = pool.ds[1][9, 1] = math.inf
    offsets = [3, 0, 0, 0, 0, 4, 2, 0, 5, 0]
    slots = [b * block + o for b, o in enumerate(offsets)]
    xd, sd = to_dev(x), dev(slots)
    pool.pages.append(10, p(xd), p(xd), p(sd))
    ctx.check()
    for i in range(2):
        append_reference(pool.h[i], pool.hs[i], x, slots, block, kind)
    pool.same()


@gpu
def test_append_refuses_a_block_that_comes_twice(ctx):
    """The same slot twice, and a block's rows in two runs: the first run is
    stored, the later one is not, and the check says so."""
    for slots in ([16, 33, 16], [16, 17, 40, 18], [20, 19], [5, 5]):
        pool = Pool(ctx, np.random.default_rng(1), 4, 2, 16, 64, sc.PAGES_I8)
        x = np.random.default_rng(2).normal(0, 5, (len(slots), 128)).astype(np.float32)
        xd, sd = to_dev(x), dev(slots)
        pool.pages.append(len(slots), p(xd), p(xd), p(sd))
        with pytest.raises(sc.ShkError) as e:
            ctx.check()
        assert e.value.code == -8
        for i in range(2):
            assert append_reference(pool.h[i], pool.hs[i], x, slots, 16, sc.PAGES_I8)
        pool.same()


@gpu
def test_append_leaves_out_slots_outside_the_pool(ctx):
    pool = Pool(ctx, np.random.default_rng(1), 4, 2, 16, 64, sc.PAGES_I8)
    x = np.random.default_rng(2).normal(0, 5, (3, 128)).astype(np.float32)
    xd, sd = to_dev(x), dev([64, 3, 2 ** 31 - 1])
    pool.pages.append(3, p(xd), p(xd), p(sd))
    with pytest.raises(sc.ShkError):
        ctx.check()
    for i in range(2):
        append_reference(pool.h[i], pool.hs[i], x, [-1, 3, -1], 16, sc.PAGES_I8)
    pool.same()
    out = torch.full((3, 128), 7.0, device="cuda")
    pool.pages.read(3, p(sd), p(out), p(out))
    with pytest.raises(sc.ShkError):
        ctx.check()
    assert (out[0] == 7).all() and (out[2] == 7).all() and not (out[1] == 7).any()


@gpu
def test_pool_arguments(ctx):
    pool = Pool(ctx, np.random.default_rng(1), 4, 2, 16, 64, sc.PAGES_I8)
    x, s = torch.zeros(4, 128, device="cuda"), dev([0, 1, 2, 3])
    good = (p(pool.d[0]), p(pool.d[1]), p(pool.ds[0]), p(pool.ds[1]), sc.PAGES_I8, 4, 2, 64, 16)
    for at, bad in ((0, None), (0, good[0] + 8), (1, good[1] + 4), (2, None), (3, good[3] + 2), (4, 2), (5, 0),
                    (5, 1 << 28), (6, 0), (6, 1025), (7, 96), (8, 48), (8, 8)):
        args = list(good)
        args[at] = bad
        with pytest.raises(sc.ShkError):
            sc.Pages(ctx, *args).append(1, p(x), p(x), p(s))
        with pytest.raises(sc.ShkError):
            sc.Pages(ctx, *args).read(1, p(s), p(x), p(x))
    g = pool.pages
    for kw in (dict(dtype=12), dict(row_stride=127)):
        with pytest.raises(sc.ShkError):
            g.append(1, p(x), p(x), p(s), **kw)
    for a in ((1, None, p(x), p(s)), (1, p(x), p(x), None), (1, p(x) + 2, p(x), p(s))):
        with pytest.raises(sc.ShkError):
            g.append(*a)
    g.append(0, None, None, None)
    g.read(0, None, None, None)
    ctx.check()
    pool.same()


# ---- attention ----

def attend_reference(q, K, V, table, seq, pos, block, n_heads, scale):
    """64-bit softmax(q K) V per row over the values K, V [blocks][kv][block][hd]; rows that see nothing: 0.
    Also the bound of the kernel's error (see test_attend)."""
    n_kv, hd = K.shape[1], K.shape[3]
    out = np.zeros((len(seq), n_heads, hd))
    lim = np.zeros_like(out)
    for r, (z, n) in enumerate(zip(seq, pos)):
        if z < 0 or n < 0:
            continue
        t = np.arange(n + 1)
        b = table[z][t // block]
        t, b = t[b >= 0], b[b >= 0]
        if not len(t):
            continue
        for h in range(n_heads):
            k = K[b, h % n_kv, t % block].astype(np.float64)
            v = V[b, h % n_kv, t % block].astype(np.float64)
            s = k @ q[r, h].astype(np.float64) * scale
            size = np.abs(k) @ np.abs(q[r, h]).astype(np.float64) * scale
            w = np.exp(s - s.max())
            w /= w.sum()
            o = w @ v
            out[r, h] = o
            lim[r, h] = U * ((24 * size + 4 * np.abs(s) + 8)[:, None] * w[:, None] * np.abs(v - o)).sum(0)
            lim[r, h] += U * (len(t) / 8 + 32) * (w @ np.abs(v))
    return out, lim


def run_attend(ctx, pool, rng, lens, rows, n_heads, dtype, pad=0, qgain=1.0, poison=True, stream=None, plan=None):
    """Attention of `rows` rows per request, or of plan's (request, position) rows in their order, against the
    reference; returns the device arrays.  Everything that no row may
    see is poisoned: places behind each request's end, and blocks of nobody."""
    blocks, n_kv, block, hd = pool.shape
    stride = max(1, max(-(-n // block) for n in lens)) + 1
    ids = rng.permutation(blocks)
    table, at = np.full((len(lens), stride), -3), 0
    for z, n in enumerate(lens):
        c = -(-n // block)
        table[z, :c] = ids[at:at + c]
        at += c
    used = np.zeros((blocks, block), bool)
    for z, n in enumerate(lens):
        t = np.arange(n)
        used[table[z][t // block], t % block] = True
    if poison:
        for i in range(2):
            hidden = np.broadcast_to(~used[:, None, :, None], pool.shape)
            pool.h[i][hidden] = 0x80 if pool.kind == sc.PAGES_I8 else 0x7F  # -128; NaN
            pool.hs[i][~used.any(1)] = np.nan
            pool.d[i].copy_(torch.from_numpy(pool.h[i]))
            pool.ds[i].copy_(torch.from_numpy(pool.hs[i]))
    seq = [z for z in range(len(lens)) for _ in range(rows)] + [-1] * pad
    pos = [n - rows + j for n in lens for j in range(rows)] + [5] * pad
    order = rng.permutation(len(seq))
    seq, pos = (np.array(x) for x in zip(*plan)) if plan else (np.array(seq)[order], np.array(pos)[order])
    w = n_heads * hd
    q = to_dev((rng.normal(0, 1, (len(seq), w + 24)) * qgain).astype(np.float32)).to(TORCH[dtype])
    out = torch.full((len(seq), w + 16), 7.0, device="cuda", dtype=TORCH[dtype])
    ws = torch.full((sc.pages_attend_ws(len(seq), n_heads, n_kv, hd),), 0xFF, dtype=torch.uint8, device="cuda")
    seq_d, pos_d, table_d = dev(seq), dev(pos), dev(table)
    scale = float(np.float32(1 / math.sqrt(hd)))
    torch.cuda.synchronize()
    pool.pages.attend(len(seq), p(q), p(out), n_heads, p(pos_d), p(table_d), stride, len(lens), scale, p(ws), ws.numel(),
                      row_seq=p(seq_d), dtype=dtype, q_stride=w + 24, out_stride=w + 16, stream=stream)
    torch.cuda.synchronize()
    ctx.check()
    K, V = pool.values()
    ref, lim = attend_reference(q.float().cpu().numpy()[:, :w].reshape(-1, n_heads, hd), K, V, table, seq, pos, block,
                                n_heads, scale)
    got = out.double().cpu().numpy()
    assert (got[:, w:] == 7).all()
    assert (got[seq < 0] == 7).all()
    live = seq >= 0
    lim = lim + (torch.finfo(TORCH[dtype]).eps / 2 * np.abs(ref) + torch.finfo(TORCH[dtype]).smallest_normal * 2.0 ** -9
                 if dtype else 0)
    err = np.abs(got[:, :w].reshape(ref.shape) - ref)[live]
    assert np.all(err <= lim[live]), (err / np.maximum(lim[live], 1e-300)).max()
    return q, out, table_d, seq_d, pos_d, ws


# The bound: with u = 2^-24, a score is the sum of hd products of 8-bit values with q held in 22 bits or more (4 u of
# each |q k|), added in at most 8 steps of fp32 (cut off, not rounded: 2 u each) and scaled (4 u): 24 u sum |q k|; the
# exponential adds 4 u |s| + 8 u.  Errors of scores move the output by sum w |ds| |v - out|.  The weighted sum of the
# values is cut off once per 16 positions (2 u each) and rounded a few times over in the merges: (n / 8 + 32) u sum w |v|.
@gpu
@pytest.mark.parametrize("kind", [sc.PAGES_I8, sc.PAGES_E4M3])
@pytest.mark.parametrize("H,KV,hd", [(32, 8, 128), (8, 8, 64), (6, 2, 128), (24, 2, 64), (16, 1, 128), (40, 1, 64)])
@pytest.mark.parametrize("block,lens", [(16, [1, 0, 15, 16, 17, 33]), (32, [31, 300, 2]), (256, [255, 257, 1, 900]),
                                        (64, [1500])])
def test_attend(ctx, kind, H, KV, hd, block, lens):
    rng = np.random.default_rng(H * hd + block)
    pool = Pool(ctx, rng, sum(-(-n // block) for n in lens) + 2, KV, block, hd, kind)
    run_attend(ctx, pool, rng, lens, 1, H, 0, pad=1)


@gpu
@pytest.mark.parametrize("dtype", [0, 1, 30])
@pytest.mark.parametrize("rows", [1, 3])
@pytest.mark.parametrize("block,lens", [(16, [9000, 3]), (128, [129, 20000]), (32, list(range(0, 640, 10)))])
def test_attend_long_and_many(ctx, dtype, rows, block, lens):
    """Lengths that many blocks of threads share, batches that one takes several of; rows before the first position."""
    rng = np.random.default_rng(rows + block)
    pool = Pool(ctx, rng, sum(-(-n // block) for n in lens) + 2, 2, block, 128, sc.PAGES_E4M3 if rows == 3 else sc.PAGES_I8)
    run_attend(ctx, pool, rng, lens, rows, 16, dtype, pad=3)


@gpu
@pytest.mark.parametrize("kind", [sc.PAGES_I8, sc.PAGES_E4M3])
@pytest.mark.parametrize("H,KV,hd", [(8, 8, 64), (16, 8, 128), (6, 2, 64), (32, 8, 128), (10, 2, 128), (16, 2, 64),
                                     (24, 2, 128), (16, 1, 128), (40, 1, 64)])
@pytest.mark.parametrize("block,lens,most", [(16, [40, 1, 0, 150], 7), (64, [70, 2500], 20), (16, [33] * 60, 5)])
def test_attend_rows_of_one_request(ctx, kind, H, KV, hd, block, lens, most):
    """Rows of one request side by side, in any number and order: other positions, the same one twice, ones that see
    nothing, padding between them, requests that come again."""
    rng = np.random.default_rng(H * hd + most)
    pool = Pool(ctx, rng, sum(-(-n // block) for n in lens) + 2, KV, block, hd, kind)
    plan = []
    for z in [*range(len(lens)), *rng.permutation(len(lens))[:3]]:
        top = lens[z]
        at = rng.integers(-1, top, rng.integers(0, most + 1)) if top else np.full(rng.integers(0, 3), -1)
        plan += [(z, int(t)) for t in at] + [(-1, 3)] * int(rng.random() < 0.2)
    plan += [(0, lens[0] - 1)] * 3
    run_attend(ctx, pool, rng, lens, 0, H, 30 if kind else 0, plan=plan)


@gpu
@pytest.mark.parametrize("n_rows,live", [(1000, [0, 127, 128, 999]), (20000, [5, 6, 7, 19999]), (65535, [511, 512, 40000, 65534]),
                                         (65535, [])])
def test_attend_rows_far_apart(ctx, n_rows, live):
    """Few rows among many padding rows: the first ones, the last one, none."""
    rng = np.random.default_rng(n_rows)
    lens = [40, 3]
    pool = Pool(ctx, rng, 6, 2, 16, 64, sc.PAGES_I8)
    plan = [(-1, 3)] * n_rows
    for i, r in enumerate(live):
        plan[r] = (i % 2, lens[i % 2] - 1)
    run_attend(ctx, pool, rng, lens, 0, 2, 0, plan=plan)


@gpu
@pytest.mark.parametrize("H,KV,hd", [(8, 4, 64), (16, 2, 64), (32, 8, 128)])
def test_attend_bad_queries_stay_alone(ctx, H, KV, hd):
    """Rows of one request, every other one NaN or infinite: the ones between are what they are alone."""
    rng = np.random.default_rng(7)
    pool = Pool(ctx, rng, 4, KV, 16, hd, sc.PAGES_E4M3)
    table, seq, pos = rng.permutation(4)[:3].reshape(1, 3), np.zeros(6, int), np.array([47, 40, 41, 3, 20, 47])
    q = rng.normal(0, 1, (6, H, hd)).astype(np.float32)
    ref, lim = attend_reference(q, *pool.values(), table, seq, pos, 16, H, 0.125)
    q[1::2, :, 5] = np.array([np.nan, np.inf, -np.inf])[:, None]
    qd, out = to_dev(q), torch.full((6, H * hd), 7.0, device="cuda")
    ws = torch.empty(sc.pages_attend_ws(6, H, KV, hd), dtype=torch.uint8, device="cuda")
    td, sd, pd = dev(table), dev(seq), dev(pos)
    pool.pages.attend(6, p(qd), p(out), H, p(pd), p(td), 3, 1, 0.125, p(ws), ws.numel(), row_seq=p(sd))
    ctx.check()
    got = out.double().cpu().numpy().reshape(ref.shape)
    assert np.all(np.abs(got - ref)[::2] <= lim[::2])
    assert not np.isfinite(got[1]).any()


@gpu
@pytest.mark.parametrize("scale", [np.inf, np.nan])
def test_attend_hidden_scales(ctx, scale):
    """A block that only the longer row of a request sees, with a scale that is no number: nothing to the others."""
    rng = np.random.default_rng(6)
    plan, lens, block = [(0, 10), (0, 39), (0, 31), (0, 7)], [40], 16
    for kind, H, KV, hd in ((sc.PAGES_I8, 8, 4, 64), (sc.PAGES_E4M3, 32, 4, 64), (sc.PAGES_I8, 8, 2, 128)):
        pool = Pool(ctx, rng, 6, KV, block, hd, kind)
        table = rng.permutation(6)[:3].reshape(1, 3)
        K, V = pool.values()
        for i in range(2):
            pool.hs[i][table[0, 2]] = scale
            pool.ds[i].copy_(torch.from_numpy(pool.hs[i]))
        seq, pos = (np.array(x) for x in zip(*plan))
        q = rng.normal(0, 1, (4, H, hd)).astype(np.float32)
        qd, out = to_dev(q), torch.full((4, H * hd), 7.0, device="cuda")
        ws = torch.empty(sc.pages_attend_ws(4, H, KV, hd), dtype=torch.uint8, device="cuda")
        td, sd, pd = dev(table), dev(seq), dev(pos)
        pool.pages.attend(4, p(qd), p(out), H, p(pd), p(td), 3, 1, 0.125, p(ws), ws.numel(), row_seq=p(sd))
        ctx.check()
        ref, lim = attend_reference(q, K, V, table, seq, pos, block, H, 0.125)
        got = out.double().cpu().numpy().reshape(ref.shape)
        see = [0, 2, 3]
        assert np.all(np.abs(got - ref)[see] <= lim[see])
        assert not np.isfinite(got[1]).any()


@gpu
@pytest.mark.parametrize("qgain", [30.0, 1e-6, 1e6])
def test_attend_sharp_and_flat(ctx, qgain):
    """Scores near 100 and beyond (a near one-hot softmax) and near 0; blocks whose scales differ by 2^40."""
    rng = np.random.default_rng(3)
    lens = [700, 33]
    pool = Pool(ctx, rng, 60, 2, 16, 64, sc.PAGES_I8)
    for i in range(2):
        pool.hs[i] *= np.exp2(rng.integers(-20, 20, pool.hs[i].shape)).astype(np.float32) if i else 1
        pool.ds[i].copy_(torch.from_numpy(pool.hs[i]))
    run_attend(ctx, pool, rng, lens, 1, 8, 0, qgain=qgain)


@gpu
def test_attend_spread_of_work(ctx):
    """One long request among many short ones, and 300 requests of one token."""
    rng = np.random.default_rng(8)
    for lens in ([1] * 300, [5000] + [2] * 40, [1] * 63 + [700]):
        pool = Pool(ctx, rng, sum(-(-n // 16) for n in lens) + 2, 4, 16, 64, sc.PAGES_I8)
        run_attend(ctx, pool, rng, lens, 1, 8, 0)


@gpu
@pytest.mark.parametrize("bad", [-1, 50, 2 ** 31 - 1, -2 ** 31])
def test_attend_leaves_out_bad_blocks(ctx, bad):
    """A block id outside the pool: its positions are left out (all of them: zeros), the others count, the check says so."""
    rng = np.random.default_rng(5)
    pool = Pool(ctx, rng, 50, 2, 16, 64, sc.PAGES_I8)
    table = rng.permutation(50)[:40].reshape(4, 10)
    hurt = table.copy()
    hurt[1, 3] = hurt[2, :] = bad
    seq, pos = [0, 1, 2, 3], [159, 100, 70, 0]
    q = rng.normal(0, 1, (4, 8 * 64)).astype(np.float32)
    qd, out = to_dev(q), torch.full((4, 8 * 64), 7.0, device="cuda")
    ws = torch.empty(sc.pages_attend_ws(4, 8, 2, 64), dtype=torch.uint8, device="cuda")
    td, sd, pd = dev(hurt), dev(seq), dev(pos)
    pool.pages.attend(4, p(qd), p(out), 8, p(pd), p(td), 10, 4, 0.125, p(ws), ws.numel(), row_seq=p(sd))
    with pytest.raises(sc.ShkError) as e:
        ctx.check()
    assert e.value.code == -8
    table[1, 3] = table[2, :] = -1
    K, V = pool.values()
    ref, lim = attend_reference(q.reshape(4, 8, 64), K, V, table, seq, pos, 16, 8, 0.125)
    err = np.abs(out.double().cpu().numpy().reshape(4, 8, 64) - ref)
    assert np.all(err <= lim) and (out[2] == 0).all()


@gpu
def test_attend_leaves_out_bad_rows(ctx):
    """A position past the table and a request that is none see nothing: zeros."""
    rng = np.random.default_rng(5)
    pool = Pool(ctx, rng, 8, 2, 16, 64, sc.PAGES_I8)
    q, out = torch.randn(4, 512, device="cuda"), torch.full((4, 512), 7.0, device="cuda")
    ws = torch.empty(sc.pages_attend_ws(4, 8, 2, 64), dtype=torch.uint8, device="cuda")
    table, seq, pos = dev([[0, 1], [2, 3]]), dev([0, 1, 2, 2 ** 31 - 1]), dev([32, 31, 3, 2 ** 31 - 1])
    pool.pages.attend(4, p(q), p(out), 8, p(pos), p(table), 2, 2, 0.125, p(ws), ws.numel(), row_seq=p(seq))
    with pytest.raises(sc.ShkError):
        ctx.check()
    assert (out[[0, 2, 3]] == 0).all() and (out[1] != 0).any()


@gpu
def test_attend_not_a_number(ctx):
    """NaN and infinities that a row sees make its head NaN, and no other's."""
    rng = np.random.default_rng(5)
    pool = Pool(ctx, rng, 40, 2, 16, 64, sc.PAGES_I8)
    pool.ds[0][1, 0] = math.inf      # request 0, KV head 0: the keys of a block
    pool.ds[1][12, 1] = math.nan     # request 1, KV head 1: the values of a block
    q = torch.randn(4, 4, 64, device="cuda")
    q[2, 1, 5] = math.nan
    q[3, 2, 0] = math.inf
    table = torch.arange(40, dtype=torch.int32, device="cuda").view(4, 10)
    pos, out = dev([150, 150, 150, 150]), torch.zeros(4, 4, 64, device="cuda")
    ws = torch.empty(sc.pages_attend_ws(4, 4, 2, 64), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    pool.pages.attend(4, p(q), p(out), 4, p(pos), p(table), 10, 4, 0.125, p(ws), ws.numel())
    ctx.check()
    nan = out.isnan()
    want = torch.zeros(4, 4, dtype=torch.bool, device="cuda")
    want[0, 0::2] = want[1, 1::2] = want[2, 1] = want[3, 2] = True
    assert (nan.all(2) == want).all() and (nan.any(2) == want).all()


@gpu
def test_attend_arguments(ctx):
    pool = Pool(ctx, np.random.default_rng(1), 4, 2, 16, 64, sc.PAGES_I8)
    q, out, i = torch.zeros(2, 512, device="cuda"), torch.zeros(2, 512, device="cuda"), dev([0, 0])
    n = sc.pages_attend_ws(2, 8, 2, 64)
    ws = torch.zeros(n + 16, dtype=torch.uint8, device="cuda")
    good = dict(n_rows=2, q=p(q), out=p(out), n_heads=8, row_pos=p(i), table=p(i), table_stride=1, n_seq=2, scale=1.0,
                ws=p(ws), ws_bytes=n)
    for bad in (dict(q=None), dict(out=None), dict(n_heads=0), dict(n_heads=7), dict(n_heads=8192), dict(row_pos=None),
                dict(table=None), dict(table_stride=0), dict(n_seq=0), dict(n_seq=1), dict(ws=None), dict(ws=p(ws) + 4),
                dict(ws_bytes=n - 1), dict(dtype=2), dict(q_stride=511), dict(out_stride=100), dict(n_rows=65536),
                dict(q=p(q) + 2), dict(table_stride=1 << 28), dict(out=p(q)), dict(out=p(q) + 2048)):
        with pytest.raises(sc.ShkError):
            pool.pages.attend(**{**good, **bad})
    pool.pages.attend(**{**good, "n_rows": 0})
    pool.pages.attend(**good)
    ctx.check()
