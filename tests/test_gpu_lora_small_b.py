"""Low-rank adapters whose B is far below 1, fp32 outputs alone (C = 0), against 64 bits (run
on an MI355X).

x picks columns of A, so the inner sums are exact.  Tolerance: they enter the second
product to 2^-22 of the row's largest; (rank / 16 + 4) 2^-23 of the products' sum, where
the matrix unit holds a product of a B below 2^-14 as exactly as one of 2^-14; Y's
rounding, 2^-24."""
import pytest
import torch

import busfill as bf
from test_gpu_lora import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [16, 300])
@pytest.mark.parametrize("rank", [16, 64, 136])
@pytest.mark.parametrize("e", [-12, -15, -18, -20, -22, -24])
def test_small_values_of_b(T, rank, e):
    """B from 2^-12 down to the smallest fp16 number."""
    g = torch.Generator().manual_seed(rank - e)
    c = Case(T, 64, [48], 1, rank, scales=False, ids=[0] * T)
    c.x = torch.zeros(T, 64).half()
    c.x[torch.arange(T), torch.arange(T) % 64] = 1.0
    b = (torch.randn(1, 48, rank, generator=g).clamp(-2, 2) * 2.0 ** e).half()
    c.ab = [(c.ab[0][0], b)]
    c.c = torch.zeros_like(c.c)
    kw = c.device()
    y = torch.empty_like(c.dc)
    bf.lora(c.dx, c.dids, c.parts, c.dc, y, **kw)
    torch.cuda.synchronize()
    s, b = c.x.double() @ c.ab[0][0][0].double().t(), b[0].double()
    want, size = s @ b.t(), b.abs().clamp(min=2.0 ** -14)
    tol = (2.0 ** -22 * s.abs().amax(-1, keepdim=True)) * b.abs().sum(-1) + (rank / 16 + 4) * 2.0 ** -23 * (s.abs() @ size.t())
    assert ((y.cpu().double() - want).abs() <= tol + 2.0 ** -24 * want.abs()).all()
