"""Attention whose q and out are columns of one buffer: taken where no element is shared, refused where one is."""
import numpy as np
import pytest
import torch

from conftest import to_dev
from shukuchi_b200 import cuda as sc
from test_pages import Pool, attend_reference, dev, p

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [1, 5])
@pytest.mark.parametrize("swap", [False, True])
def test_q_and_out_between_one_another(ctx, rows, swap):
    """[q | out] and [out | q] in one row each, a gap of one element between them or none: as with separate buffers."""
    rng = np.random.default_rng(rows)
    H, KV, hd, block, w = 4, 2, 64, 16, 256
    pool = Pool(ctx, rng, 8, KV, block, hd, sc.PAGES_I8)
    table, seq, pos = rng.permutation(8)[:3].reshape(1, 3), np.zeros(rows, int), np.array([40, 41, 3, 47, 20])[:rows]
    q = rng.normal(0, 1, (rows, w)).astype(np.float32)
    ref, lim = attend_reference(q.reshape(rows, H, hd), *pool.values(), table, seq, pos, block, H, 0.125)
    td, sd, pd = dev(table), dev(seq), dev(pos)
    ws = torch.empty(sc.pages_attend_ws(rows, H, KV, hd), dtype=torch.uint8, device="cuda")
    for stride, gap in ((2 * w, 0), (2 * w + 1, 1), (2 * w + 3, 0)):
        buf = torch.full((rows, stride), 7.0, device="cuda")
        at_q, at_out = (w + gap, 0) if swap else (0, w + gap)
        buf[:, at_q: at_q + w] = to_dev(q)
        torch.cuda.synchronize()
        call = lambda o: pool.pages.attend(rows, p(buf) + 4 * at_q, p(buf) + 4 * o, H, p(pd), p(td), 3, 1, 0.125, p(ws),
                                           ws.numel(), row_seq=p(sd), q_stride=stride, out_stride=stride)
        call(at_out)
        ctx.check()
        got = buf.cpu().numpy()
        assert np.array_equal(got[:, at_q: at_q + w], q)
        assert np.all(np.abs(got[:, at_out: at_out + w].reshape(ref.shape) - ref) <= lim)
        rest = np.delete(got, np.r_[at_q: at_q + w, at_out: at_out + w], 1)
        assert (rest == 7).all()
        # one element shared: at the nearer end of q, and (by a row further on) at the other one
        near = at_q + w - 1 if at_out > at_q else at_q - w + 1
        for o in [near] + ([at_q + stride - w + 1] if rows > 1 and not swap else []):
            if o >= 0:
                with pytest.raises(sc.ShkError):
                    call(o)
    with pytest.raises(sc.ShkError):  # two strides: the ranges count
        pool.pages.attend(5, p(buf), p(buf) + 4 * w, H, p(pd), p(td), 3, 1, 0.125, p(ws), ws.numel(), row_seq=p(sd),
                          q_stride=2 * w, out_stride=2 * w + 1)
    ctx.check()
