"""The experts' block where intermediates, experts' outputs and routing weights
lie far from 1 (tolerances: test_gpu_moe.py, whose terms are written out below;
run on an MI355X)."""
import pytest
import torch

import busfill as bf
import oracle as O
from test_gpu_moe import QTS, Experts

pytestmark = pytest.mark.gpu


def terms(x, a, ids, w):
    """64 bits: the block's outputs, its tolerance without the output's rounding, largest |intermediate| and |expert's output|."""
    T, k = ids.shape
    rw, acc = (0.0 if x.qt == O.Q4_K else 2.0 ** -11), 2.0 ** -18
    want, tol, top_h, top_y = torch.zeros(T, x.N).double(), torch.zeros(T, x.N).double(), 0.0, 0.0
    for j in range(k):
        for e in range(x.E):
            t = torch.nonzero(ids[:, j] == e)[:, 0]
            if len(t) == 0:
                continue
            wg, wu, wd = (m[e] for m in x.w64)
            r, ww = a[t].double(), w[t, j].double()[:, None]
            gt, ut = r @ wg.t(), r @ wu.t()
            dg, du = (r.abs() @ m.abs().t() * (rw + acc) for m in (wg, wu))
            silu = gt * torch.sigmoid(gt)
            h = ww * silu * ut
            dh = ww.abs() * (1.1 * dg * (ut.abs() + du) + silu.abs() * du) + (2.0 ** -11 + 2.0 ** -20) * h.abs() + 2.0 ** -25
            y = h @ wd.t()
            want.index_add_(0, t, y)
            tol.index_add_(0, t, dh @ wd.abs().t() * (1 + rw + acc) + h.abs() @ wd.abs().t() * (rw + acc))
            top_h, top_y = max(top_h, float(h.abs().max())), max(top_y, float(y.abs().max()))
    return want, tol, top_h, top_y


@pytest.mark.parametrize("qt", QTS)
@pytest.mark.parametrize("T", [1, 9, 60, 500])
def test_experts_outputs_beyond_fp16_that_cancel(qt, T):
    """Every row's two terms pass 65504, one above and one below zero, their sum is in range: finite, whatever the number
    of rows (one row, several passes, runs of 64, large runs)."""
    x = Experts(qt, 4, 512, 256, 144, seed=9)
    g = torch.Generator().manual_seed(T)
    a = torch.randn(T, 512, generator=g)
    ids = torch.randint(0, 4, (T, 1), generator=g).expand(T, 2).contiguous()
    w = torch.tensor([[1.0, -0.9995]]).repeat(T, 1)
    # activations scaled so that the intermediates come near 2e4 (they grow with the square)
    _, _, h, y = terms(x, a.half(), ids, w)
    a = (a * (2e4 / h) ** 0.5).half()
    want, tol, h, y = terms(x, a, ids, w)
    grow = 1.0
    while y < 2e5:                                 # down weights as large as needed: their scales, exactly doubled
        y, grow = 2 * y, 2 * grow
    dev, aux = x.dev[2]
    if qt == O.Q4_0_PLANES:
        aux.view(torch.float16).mul_(grow)
    else:
        block = dev.view(-1, 18 if qt == O.Q4_0 else 144)
        head = block[:, :2 if qt == O.Q4_0 else 4].contiguous().view(torch.float16) * grow
        block[:, :head.shape[1] * 2] = head.view(torch.uint8).reshape(block.shape[0], -1)
    x.w64[2] = x.w64[2] * grow
    want, tol, h, y = terms(x, a, ids, w)
    assert h < 6e4 and y > 65504 and float(want.abs().max()) < 6e4
    for otype in (bf.OUT_F32, bf.OUT_F16):
        got = x.run(a, ids, w, otype=otype).cpu().double()
        assert torch.isfinite(got).all()
        t = tol + (2.0 ** -11 * want.abs() + 2.0 ** -25 if otype == bf.OUT_F16 else 0.0)
        assert ((got - want).abs() <= t).all(), float(((got - want).abs() / t).max())
