"""Infinities of the low-rank adapters' B against the formula (run on an MI355X).

X and A are small whole numbers, so the inner sums are exact, zeros among them: what is
infinite, of which sign, and what is NaN is the formula's own.  Finite outputs: s is a whole
number below 2^11, exact in fp16; products and their sum in fp32, (rank / 16 + 4) 2^-23
scale |B| |s|, then one addition and rounding of Y (fp32 2^-23)."""
import pytest
import torch

import busfill as bf

pytestmark = pytest.mark.gpu

F16 = torch.float16
INF = float("inf")


def whole(g, most, *shape):
    return torch.randint(-most, most + 1, shape, generator=g).half()


def formula(x, a, b, c, ids, scales):
    """Y and the sum of magnitudes, in 64 bits, term by term (0 times an infinity is NaN)."""
    y, size = c.double(), c.double().abs()
    for t, e in enumerate(ids.tolist()):
        if e >= 0:
            s = (a[e].double() * x[t].double()).sum(-1)
            p = b[e].double() * s
            y[t] += float(scales[e]) * p.sum(-1)
            size[t] += abs(float(scales[e])) * p.abs().sum(-1)
    return y, size


def call(x, a, b, c, ids, scales):
    (T, K), (E, N, rank) = x.shape, b.shape
    d = [v.cuda() for v in (x, ids, a, b, c, scales)]
    y = torch.empty_like(d[4])
    bf.lora(d[0], d[1], bf.lora_parts([(d[2], d[3], N, 0)]), d[4], y, T=T, K=K, adapters=E, rank=rank, scales=d[5],
            otype=bf.OUT_F16 if c.dtype == F16 else bf.OUT_F32)
    torch.cuda.synchronize()
    return y.cpu()


def check(y, want, size, rank):
    assert torch.equal(torch.isnan(y), torch.isnan(want))
    odd = torch.isinf(want)
    assert torch.equal(y.double()[odd], want[odd])
    ok = torch.isfinite(want)
    tol = ((rank / 16 + 6) * 2.0 ** -23 + (2.0 ** -11 if y.dtype == F16 else 0)) * size + 2.0 ** -24
    assert ((y.double() - want).abs() <= tol)[ok].all()


@pytest.mark.parametrize("otype", [torch.float32, F16])
@pytest.mark.parametrize("rank", [8, 16, 32, 64, 72, 136])
@pytest.mark.parametrize("T", [1, 20, 300])
def test_infinities_of_b(T, rank, otype):
    """Columns with one infinity, with two of one sign or of both, with a NaN, and ordinary ones between them."""
    g = torch.Generator().manual_seed(T + rank)
    E, N, K = 3, 150, 64
    x, a = whole(g, 1, T, K), whole(g, 2, E, rank, K)
    b = (torch.randn(E, N, rank, generator=g) * 0.3).half()
    at = torch.randint(0, rank, (E, N, 2), generator=g)
    for e in range(E):
        for n in range(0, N, 3):
            b[e, n, at[e, n, 0]] = INF if n % 2 else -INF
            if n % 4 == 0:
                b[e, n, at[e, n, 1]] = -INF if n % 8 else INF
            if n % 45 == 0:
                b[e, n, 5] = float("nan")
    ids = torch.randint(-1, E, (T,), generator=g).int() if T > 1 else torch.tensor([1], dtype=torch.int32)
    scales = torch.tensor([0.5, -0.75, 1.25])
    c = torch.randn(T, N, generator=g).to(otype)
    y = call(x, a, b, c, ids, scales)
    want, size = formula(x, a, b, c, ids, scales)
    assert torch.isinf(want).any() and torch.isnan(want).any()
    check(y, want, size, rank)


@pytest.mark.parametrize("rank", [16, 72])
@pytest.mark.parametrize("T", [20, 300])
def test_infinities_of_both(T, rank):
    """Rows with an infinity of X beside columns with one of B: by the signs of the inner sums, finite ones beside infinite ones too."""
    g = torch.Generator().manual_seed(rank)
    K, N = 32, 70
    x, a = whole(g, 2, T, K), whole(g, 2, 1, rank, K)
    a[0, ::2, 3] = 0                                                       # (0 times an infinity: those sums are NaN ...
    x[::2, 3], x[1::2, 4] = INF, -INF
    a[0, :, 4] = torch.where(a[0, :, 4] == 0, 1, a[0, :, 4].float()).half()   # ... these are not)
    x[5::6, 4] = 2
    b = (torch.randn(1, N, rank, generator=g) * 0.3).half()
    b[0, ::5, 7], b[0, 3::10, 2] = INF, -INF
    b[0, 4, :] = 0
    c = torch.randn(T, N, generator=g)
    ids, scales = torch.zeros(T, dtype=torch.int32), torch.tensor([-0.5])
    want, size = formula(x, a, b, c, ids, scales)
    assert torch.isinf(want).any() and torch.isnan(want).any() and torch.isfinite(want).any()
    check(call(x, a, b, c, ids, scales), want, size, rank)


@pytest.mark.parametrize("T", [4, 300])
def test_an_infinity_meets_a_sum_far_below_the_largest(T):
    """2^-34 beside 2^32: the small one keeps its sign, and nothing else of it."""
    K, rank, N = 8, 8, 16
    x, a = torch.zeros(T, K), torch.zeros(1, rank, K)
    x[:, 0], x[:, 1] = 2.0 ** -10, 60000.0
    x[1::2, 0] *= -1
    a[0, 0, 0], a[0, 1, 1], a[0, 2, 1] = 2.0 ** -24, 60000.0, -3.0
    b = torch.ones(1, N, rank)
    b[0, 3:, 0], b[0, :, 3:] = INF, 0.0
    c, ids, scales = torch.zeros(T, N), torch.zeros(T, dtype=torch.int32), torch.ones(1)
    want, size = formula(x.half(), a.half(), b.half(), c, ids, scales)
    assert (want[::2, 3:] == INF).all() and (want[1::2, 3:] == -INF).all() and torch.isfinite(want[:, :3]).all()
    check(call(x.half(), a.half(), b.half(), c, ids, scales), want, size, rank)


@pytest.mark.parametrize("rank", [16, 72])
@pytest.mark.parametrize("T", [20, 300])
def test_infinite_sums_and_the_smallest_b(T, rank):
    """An infinity of X times a B of 2^-24 or of 65504, and of 0 (NaN); a scale of 0 (NaN)."""
    x = torch.ones(T, 8)
    x[::2, 0], x[1::4, 0] = INF, -INF
    a, b = torch.ones(2, rank, 8), torch.ones(2, 40, rank)
    b[:, ::4], b[:, 1::4], b[:, 2::4] = 2.0 ** -24, -(2.0 ** -24), 65504.0
    b[:, 3::8, rank - 1] = 0.0
    ids = (torch.arange(T) % 3 == 1).int()
    scales = torch.tensor([2.0, 0.0])
    c = torch.randn(T, 40, generator=torch.Generator().manual_seed(T))
    want, size = formula(x.half(), a.half(), b.half(), c, ids, scales)
    assert torch.isinf(want).any() and torch.isnan(want).any() and torch.isfinite(want).any()
    check(call(x.half(), a.half(), b.half(), c, ids, scales), want, size, rank)
