"""Attention over the 4-bit cache where probabilities and values lie far from 1:
a first token that takes most of the weight and has no value, tails many powers
of two below it, small values, scores of any size (run on an MI355X).

Tolerance, per output element, with A = sum_t p_t |v_t|: every product of a
probability and a scale is rounded to fp16, by 2^-11 of itself or, where it is
more than 2^25 times below the largest probability times the largest scale, by
2^-36 of that; scores, exponentials and sums are fp32 and stay under 2^-13 of A.
So |o - exact| <= (2^-11 + 2^-13) A + tokens (2^-36 max |v| + 2^-48), the
largest |v| among the tokens that the row sees or that its neighbours in a row
tile (up to 32 tokens further) see.  Outputs are fp32.
"""
import math

import numpy as np
import pytest
import torch

import busfill as bf
import kv4_ref as R
from test_gpu_kv4 import Cache

pytestmark = pytest.mark.gpu


def run(k, v, q, scale, group, absent=None, page=64):
    """S equal sequences: k, v [S][n][heads][dim], q [S][nq][heads group][dim] (all fp16): o and lse, fp32.  Unwritten
    bytes of the cache read as scales of 61280; `absent`: a page that the table leaves out."""
    S, n, heads, dim = k.shape
    nq, per = q.shape[1], (n + page - 1) // page
    c = Cache(S * per, page, heads, dim)
    table = torch.randperm(S * per, generator=torch.Generator().manual_seed(1)).int().reshape(S, per)
    c.data.fill_(0x7B)
    t = torch.arange(n)
    slots = (table.long()[:, t // page] * page + t % page).reshape(-1).cuda()
    if absent is not None:
        table[:, absent] = -1
        slots[(torch.arange(S * n) % n // page == absent).cuda()] = -1
    bf.kv4_store(c.c, k.reshape(S * n, -1).cuda(), v.reshape(S * n, -1).cuda(), slots, S * n)
    o = torch.full((S * nq, heads * group * dim), 9.0, device="cuda")
    lse = torch.full((S * nq, heads * group), 9.0, device="cuda")
    dev = lambda x: torch.as_tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    bf.kv4_attention(c.c, q.reshape(S * nq, -1).cuda(), o, dev(torch.arange(S + 1) * nq), dev([n] * S), table.cuda(), S=S,
                     T=S * nq, q_heads=heads * group, max_q=nq, max_kv=n, scale=scale, lse=lse)
    torch.cuda.synchronize()
    return o.cpu().double().reshape(S, nq, heads * group, dim), lse.cpu().double().reshape(S, nq, heads * group)


def quantize(x):
    """R.quantize of finite values, all blocks at once."""
    a = x.numpy().astype(np.float64).reshape(-1, 32)
    m = np.take_along_axis(a, np.abs(a).argmax(1)[:, None], 1)
    d = np.float16(m / -8).astype(np.float64)
    q = np.clip(np.floor(a / np.where(d == 0, 1, d) + 8.5), 0, 15) - 8
    return torch.from_numpy(np.where(d == 0, 0.0, q * d).reshape(x.shape))


def bound(mass, v, see):
    """The tolerance above; see [rows][n], v [n][dim] (64 bits)."""
    n = v.shape[0]
    last = see.float().cumsum(1).argmax(1)         # (rows see tokens up to one, each)
    near = torch.arange(n)[None] <= last[:, None] + 32
    top = torch.where(near, v.abs().amax(1)[None], 0.0).amax(1, keepdim=True)
    return (2.0 ** -11 + 2.0 ** -13) * mass + n * (2.0 ** -36 * top + 2.0 ** -48)


def causal(n, nq):
    return torch.arange(n)[None] <= n - nq + torch.arange(nq)[:, None]


def check(k, v, q, scale, group, lse_tol=1e-4, absent=None):
    """Every form runs whole; the first and last sequence's first and last heads are compared."""
    S, n, H, dim = k.shape
    nq = q.shape[1]
    got, got_lse = run(k, v, q, scale, group, absent)
    assert torch.isfinite(got).all()
    see, worst = causal(n, nq), 0.0
    if absent is not None:
        see[:, 64 * absent:64 * absent + 64] = False
    for s in {0, S - 1}:
        for h in {0, H - 1}:
            kq, vq = quantize(k[s, :, h]), quantize(v[s, :, h])
            for j in {0, group - 1}:
                i = h * group + j
                want, mass, wl = R.attention(q[s, :, i], kq, vq, scale, see)
                worst = max(worst, float(((got[s, :, i] - want).abs() / bound(mass, vq, see)).max()))
                assert ((got_lse[s, :, i] - wl).abs() <= lse_tol).all()
    assert worst <= 1.0, worst


# Of whole sequences, chunks and prompts: sequences, tokens, heads, group, queries.
FORMS = {"whole": (1, 1100, 2, 5, 1), "eight waves": (24, 1500, 8, 1, 1), "chunks": (1, 8192, 1, 8, 1), "four waves": (20, 3000, 8, 1, 1),
         "queries": (2, 1280, 1, 4, 9), "prompt": (1, 1500, 8, 8, 1500)}


def sink(form, dim, down, size, equal):
    """Keys, values, queries: token 0 has no value and `down` powers of two more weight than the others; their values
    are about `size`, of one sign (so that rounding errors cannot cancel), all equal or random."""
    S, n, heads, group, nq = FORMS[form]
    g = torch.Generator().manual_seed(int(down * 8) + dim)
    k = torch.zeros(S, n, heads, dim)
    k[:, 0] = 1.0
    v = size * (0.4 + 0.6 * torch.rand(S, 1 if equal else n, heads, dim, generator=g)).expand(S, n, heads, dim).clone()
    v[:, 0] = 0.0
    q = torch.ones(S, nq, heads * group, dim)
    q[..., 1:2] += torch.rand(S, nq, heads * group, 1, generator=g)        # (the weights differ a little by row)
    return k.half(), v.half(), q.half(), down * math.log(2) / dim, group


@pytest.mark.parametrize("form", [f for f in FORMS if f != "prompt"])
@pytest.mark.parametrize("down,size", [(12, 0.008), (14.5, 0.1), (15.5, 0.008), (20, 0.008), (20, 1.0), (17, 300.0)])
def test_tail_behind_a_token_without_value(form, down, size):
    dim = {"eight waves": 64, "queries": 256, "four waves": 96}.get(form, 128)
    check(*sink(form, dim, down, size, True))
    check(*sink(form, dim, down, size, False))


@pytest.mark.parametrize("dim,down,size", [(64, 12, 0.008), (96, 15.5, 0.008), (128, 15.5, 0.008), (128, 20, 1.0), (256, 20, 0.1)])
@pytest.mark.parametrize("equal", [True, False])
def test_tail_of_a_prompt(dim, down, size, equal):
    check(*sink("prompt", dim, down, size, equal))


@pytest.mark.parametrize("form", ["whole", "chunks", "prompt"])
@pytest.mark.parametrize("rising", [True, False])
def test_scales_that_change_along_the_sequence(form, rising):
    """Values from 2^-20 to 2^10 along the tokens, either way: the range that products are kept in follows them."""
    S, n, heads, group, nq = FORMS[form]
    g = torch.Generator().manual_seed(4)
    e = torch.linspace(-20, 10, n)
    size = 2.0 ** (e if rising else e.flip(0))
    k = torch.randn(S, n, heads, 64, generator=g)
    v = torch.randn(S, n, heads, 64, generator=g) * size[None, :, None, None]
    q = torch.randn(S, nq, heads * group, 64, generator=g)
    check(k.half(), v.half(), q.half(), 0.125, group)


@pytest.mark.parametrize("form", ["whole", "prompt"])
def test_blocks_of_different_size(form):
    """Columns 2^10 smaller than their neighbours keep their accuracy behind a token without value."""
    k, v, q, scale, group = sink(form, 128, 13, 1.0, True)
    v[..., 32:64] = (v[..., 32:64].float() * 2.0 ** -10).half()
    S, n = k.shape[:2]
    nq = q.shape[1]
    check(k, v, q, scale, group)
    got, _ = run(k, v, q, scale, group)
    want, mass, _ = R.attention(q[0, :, 0], quantize(k[0, :, 0]), quantize(v[0, :, 0]), scale, causal(n, nq))
    # (the small columns' products are 2^-24 of the largest or more: no floor)
    assert ((got[0, :, 0] - want).abs() <= (2.0 ** -11 + 2.0 ** -13) * mass)[:, 32:64].all()


@pytest.mark.parametrize("form", ["whole", "chunks", "prompt"])
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_of_any_size(form, sign):
    """Equal scores near 1e9 and, 2^12 units in their last place below, others that must not count: the mean of the first."""
    S, n, heads, group, nq = FORMS[form]
    g = torch.Generator().manual_seed(7)
    k = torch.full((S, n, heads, 64), 60000.0)
    far = torch.arange(n) % 3 == 1
    k[:, far] = 59000.0
    v = torch.rand(S, n, heads, 64, generator=g) + 0.5
    q = torch.full((S, nq, heads * group, 64), sign * 2345.0)
    if sign < 0:
        k = -k
    check(k.half(), v.half(), q.half(), 0.1234, group, lse_tol=1e9 * 2.0 ** -20)


@pytest.mark.parametrize("nan_keys", [True, False])
def test_nan_scales_do_not_move_the_range(nan_keys):
    """A token of NaN behind the others' view leaves small values behind a token without value as accurate."""
    k, v, q, scale, group = sink("queries", 64, 14, 0.008, True)
    S, n, nq = 2, k.shape[1], q.shape[1]
    k[:, n - 3] = float("nan") if nan_keys else 0.0
    v[:, n - 3] = float("nan")
    got, _ = run(k, v, q, scale, group)
    see = causal(n, nq)[:nq - 3]
    for s in range(S):
        vq = R.quantize(v[s, :, 0]).nan_to_num()
        want, mass, _ = R.attention(q[s, :nq - 3, 0], R.quantize(k[s, :, 0]), vq, scale, see)
        assert ((got[s, :nq - 3, 0] - want).abs() <= bound(mass, vq, see)).all()
        assert got[s, nq - 3:, 0].isnan().all()


@pytest.mark.parametrize("form", ["whole", "chunks", "prompt"])
@pytest.mark.parametrize("page", [3, 5])
def test_pages_that_are_not_there_do_not_move_the_range(form, page):
    check(*sink(form, 128, 16, 0.008, True), absent=page)
