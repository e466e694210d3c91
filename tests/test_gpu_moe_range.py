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


def weighted(x, a, ids, w):
    """terms(), with the intermediate rounded before the part of the weight outside 1/8 .. 1 is multiplied: 2^-11 of it,
    or 2^-25 times the larger of that part and 1."""
    want, _, top_h, top_y = terms(x, a, ids, w)
    tol, (rw, acc) = torch.zeros_like(want), ((0.0 if x.qt == O.Q4_K else 2.0 ** -11), 2.0 ** -18)
    for j in range(ids.shape[1]):
        for t in range(ids.shape[0]):
            wg, wu, wd = (m[int(ids[t, j])] for m in x.w64)
            r, ww = a[t].double(), abs(float(w[t, j]))
            gt, ut = wg @ r, wu @ r
            dg, du = ((rw + acc) * (m.abs() @ r.abs()) for m in (wg, wu))
            silu = gt * torch.sigmoid(gt)
            h = (ww * silu * ut).abs()
            rest = 8 * ww if ww < 0.125 else max(2.0, ww)
            dh = ww * (1.1 * dg * (ut.abs() + du) + silu.abs() * du) + (2.0 ** -11 + 2.0 ** -20) * h + 2.0 ** -25 * rest
            tol[t] += wd.abs() @ dh * (1 + rw + acc) + wd.abs() @ h * (rw + acc)
    return want, tol, top_h, top_y


@pytest.mark.parametrize("qt", QTS)
@pytest.mark.parametrize("T,E,F", [(1, 8, 256), (1, 8, 1024), (6, 8, 256), (40, 3, 256), (70, 3, 512)])
@pytest.mark.parametrize("size", [1e-6, 3e-4, 0.02])
def test_small_weights_keep_the_intermediates_accuracy(qt, T, E, F, size):
    """Weights that nothing has normalised, intermediates about 0.05."""
    x = Experts(qt, E, 256, F, 136, seed=4)
    g = torch.Generator().manual_seed(T + F)
    a = torch.randn(T, 256, generator=g)
    ids = torch.rand(T, E, generator=g).argsort(1)[:, :2]
    w = size * (0.5 + torch.rand(T, 2, generator=g))
    _, _, h, _ = terms(x, a.half(), ids, torch.ones_like(w))
    a = (a * (0.2 / h) ** 0.5).half()
    want, tol, _, _ = weighted(x, a, ids, w)
    got = x.run(a, ids, w).cpu().double()
    assert ((got - want).abs() <= tol).all(), float(((got - want).abs() / tol).max())


@pytest.mark.parametrize("qt", QTS)
@pytest.mark.parametrize("T,E", [(1, 8), (6, 8), (40, 3), (70, 3)])
def test_weights_bring_large_intermediates_into_range(qt, T, E):
    """Intermediates up to 3e5, beyond fp16, whose weights are about 1/8; weights above 1 and below 0 beside them."""
    x = Experts(qt, E, 256, 256, 136, seed=6)
    g = torch.Generator().manual_seed(T)
    a = torch.randn(T, 256, generator=g)
    ids = torch.rand(T, E, generator=g).argsort(1)[:, :2]
    w = 0.126 + 0.02 * torch.rand(T, 2, generator=g)
    _, _, h, _ = terms(x, a.half(), ids, torch.ones_like(w))
    big = (a * (3e5 / h) ** 0.5).half()
    want, tol, _, _ = weighted(x, big, ids, w)
    got = x.run(big, ids, w).cpu().double()
    assert torch.isfinite(got).all() and ((got - want).abs() <= tol).all()
    w = torch.stack([2.5 + torch.rand(T, generator=g), -torch.rand(T, generator=g)], 1)
    a = a.half()
    want, tol, _, _ = weighted(x, a, ids, w)
    assert ((x.run(a, ids, w).cpu().double() - want).abs() <= tol).all()


@pytest.mark.parametrize("qt", [O.Q4_0, O.Q4_0_PLANES])
@pytest.mark.parametrize("K,F,N", [(96, 288, 33), (224, 32, 40), (32, 96, 1)])
@pytest.mark.parametrize("T", [20, 70])
def test_widths_off_256_with_many_rows(qt, K, F, N, T):
    """fp16 outputs of the kernel of one thread an output, on both sides of 24 slots an expert."""
    Experts(qt, 5, K, F, N).check(T, 3, otype=bf.OUT_F16)
