"""Attention over long contexts in fp32: sums of tens of thousands of values are not cut short."""
import math

import pytest
import torch

from shukuchi_b200 import cuda as sc
from test_pages import dev, p

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.mark.parametrize("kind", [sc.PAGES_I8, sc.PAGES_E4M3])
@pytest.mark.parametrize("H,hd,rows", [(8, 64, 1), (8, 128, 1), (4, 64, 4)])
def test_long_sums_keep_their_size(ctx, kind, H, hd, rows):
    """96 requests over one context of 65536 positions, so that each CTA adds up thousands of positions of an item.  How
    much the outputs are too small (or large) altogether, sum (out - exact) exact / sum exact^2: what is cut off the sum
    of 16 positions, which begins at 0, is at most 2 u in each of its two products, 4 u; the exponentials (2^-22 at most,
    of either sign) enter by the weights and by the last factor, 4 u each.  Rounded additions have no sign."""
    n, T, block = 96, 65536, 64
    gen = torch.Generator("cuda").manual_seed(hd + kind)
    shape = (T // block, 1, block, hd)
    x = [torch.randn(shape, device="cuda", generator=gen) for _ in range(2)]
    scale = [torch.empty(T // block, 1, device="cuda").uniform_(0.01, 0.02, generator=gen) for _ in range(2)]
    if kind == sc.PAGES_I8:
        data = [(40 * a).round().clamp(-127, 127).to(torch.int8) for a in x]
    else:
        data = [(40 * a).to(torch.float8_e4m3fn) for a in x]
    K, V = ((a.double() * s.double()[..., None, None]).view(T, hd) for a, s in zip(data, scale))
    table = torch.randperm(T // block, device="cuda", generator=gen, dtype=torch.int32).expand(n, -1).contiguous()
    K, V = (a.view(T // block, block, hd)[table[0].long()].reshape(T, hd) for a in (K, V))
    q = torch.randn(n * rows, H, hd, device="cuda", generator=gen)
    seq, pos = dev([r // rows for r in range(n * rows)]), dev([T - 1] * (n * rows))
    out = torch.empty(n * rows, H, hd, device="cuda")
    ws = torch.empty(sc.pages_attend_ws(n * rows, H, 1, hd), dtype=torch.uint8, device="cuda")
    pages = sc.Pages(ctx, p(data[0]), p(data[1]), p(scale[0]), p(scale[1]), kind, T // block, 1, hd, block)
    torch.cuda.synchronize()
    pages.attend(n * rows, p(q), p(out), H, p(pos), p(table), T // block, n, 1 / math.sqrt(hd), p(ws), ws.numel(), row_seq=p(seq))
    ctx.check()
    factor = float(torch.tensor(1 / math.sqrt(hd)))  # as fp32
    exact = torch.cat([torch.softmax(a.double().reshape(-1, hd) @ K.T * factor, 1) @ V for a in q.split(48)]).view_as(out)
    off = ((out.double() - exact) * exact).sum() / (exact * exact).sum()
    assert abs(off.item()) <= 12 * U, off.item() / U
