"""Attention over the 4-bit cache with a window and first tokens that stay in
sight, against 64 bits (run on an MI355X).  Tolerances as in test_gpu_kv4.py: the
kernels compute the same products of the tokens that are seen."""
import math

import pytest
import torch

import busfill as bf
import kv4_ref as R
from test_gpu_kv4 import Sequences

pytestmark = pytest.mark.gpu


def attend(s, nqs, group, window, sinks, *, otype=bf.OUT_F32, absent=(), seed=5, max_kv=None, workspace=False, stream=None,
           scale=None, hidden_pages=False):
    hq, d = s.heads * group, s.dim
    scale = 1 / math.sqrt(d) if scale is None else scale
    starts = [0]
    for n in nqs:
        starts.append(starts[-1] + n)
    T = max(1, starts[-1])
    q = torch.randn(T, hq * d, generator=torch.Generator().manual_seed(seed)).half()
    table = s.table.clone()
    for i, p in absent:
        table[i, p] = -1 if p % 2 else s.cache.pages
    if hidden_pages:                                               # pages that no query of a sequence sees: not there
        for i, (n, nq) in enumerate(zip(s.lens, nqs)):
            for p in range((n + s.page - 1) // s.page):
                if p * s.page >= sinks and (p + 1) * s.page <= n - nq + 1 - window:
                    table[i, p] = -1
    kw = dict(S=len(nqs), T=T, q_heads=hq, max_q=max(max(nqs), 1), max_kv=max(s.lens) if max_kv is None else max_kv,
              scale=scale, window=window, otype=otype)
    o = torch.full((T, hq * d), 9.0, dtype=torch.float32 if otype == bf.OUT_F32 else torch.float16, device="cuda")
    lse = torch.full((T, hq), 9.0, device="cuda")
    args = [q.cuda(), o, torch.tensor(starts, dtype=torch.int32).cuda(), torch.tensor(s.lens, dtype=torch.int32).cuda(),
            table.cuda()]
    torch.cuda.synchronize()
    if workspace:
        a = bf.kv4_attention_args(s.cache.c, *args, lse=lse, **kw)
        n = bf.kv4_attention_sinks_workspace_bytes(s.cache.c, a, sinks)
        ws = torch.full((n,), 0xFF, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        bf.kv4_attention_sinks_ws(s.cache.c, a, sinks, ws if n else None, n, stream=stream)
    else:
        bf.kv4_attention_sinks(s.cache.c, *args, sinks=sinks, lse=lse, stream=stream, **kw)
    torch.cuda.synchronize()
    got, got_lse = o.cpu().double(), lse.cpu().double()
    for i, nq in enumerate(nqs):
        n = s.lens[i]
        t = torch.arange(n)
        here = torch.ones(n, dtype=torch.bool)
        for (j, p) in absent:
            if j == i:
                here[p * s.page:(p + 1) * s.page] = False
        pos = n - nq + torch.arange(nq)[:, None]
        see = (t[None] <= pos) & ((t[None] > pos - (window or n + nq)) | (t[None] < sinks)) & here
        for h in range(hq):
            r = slice(starts[i], starts[i + 1])
            want, mass, wl = R.attention(q[r, h * d:(h + 1) * d], s.k[i][:, h // group], s.v[i][:, h // group], scale, see)
            tol = (2.0 ** -11 + 2.0 ** -13) * mass + 2.0 ** -24
            if otype == bf.OUT_F16:
                tol = tol + 2.0 ** -11 * want.abs() + 2.0 ** -25
            err = (got[r, h * d:(h + 1) * d] - want).abs()
            assert (err <= tol).all(), (i, h, float((err / tol).max()))
            empty = torch.isinf(wl)
            assert torch.isinf(got_lse[r, h][empty]).all() and (got_lse[r, h][empty] < 0).all()
            assert ((got_lse[r, h] - wl)[~empty].abs() <= 1e-4).all()
    return o


@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("window,sinks", [(40, 4), (1, 1), (32, 32), (33, 70), (64, 33), (200, 3), (16, 500)])
def test_single_tokens(dim, window, sinks):
    """Windows that begin before, inside and behind the first tokens' tiles; sequences shorter than either."""
    s = Sequences([1, 2, 33, 64, 65, 100, 230, 0], 2, dim)
    attend(s, [1] * 8, 5, window, sinks)


@pytest.mark.parametrize("window,sinks", [(40, 4), (1, 1), (32, 64), (100, 35)])
@pytest.mark.parametrize("nqs,lens", [([4, 1, 7], [140, 1, 7]), ([33, 2], [133, 90]), ([17, 0, 5], [200, 50, 3]), ([100, 61], [230, 61])])
@pytest.mark.parametrize("group", [1, 3, 8])
def test_several_queries(window, sinks, nqs, lens, group):
    """Queries of one row tile whose windows begin on both sides of the first tokens' end."""
    attend(Sequences(lens, 2, 64, max_kv=256), nqs, group, window, sinks, max_kv=256)


@pytest.mark.parametrize("page", [32, 96, 256])
def test_pages_that_no_one_sees(page):
    """Their entries in the table may be negative, as where they were given back."""
    s = Sequences([700, 95, 350], 2, 128, page=page)
    attend(s, [1, 1, 1], 4, 90, 5, otype=bf.OUT_F16, hidden_pages=True)
    attend(s, [7, 1, 2], 4, 90, 40, hidden_pages=True)


@pytest.mark.parametrize("lens", [[6000], [9001, 700, 64, 0, 1]])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("workspace", [False, True])
def test_long_windows_in_chunks(lens, dim, workspace):
    """More tiles than a workgroup takes: chunks with the first tokens' tiles and the window's in one walk."""
    s = Sequences(lens, 1, dim)
    attend(s, [1] * len(lens), 8, 5000, 100, workspace=workspace)
    attend(s, [1] * len(lens), 8, 2000, 3000, workspace=workspace)


@pytest.mark.parametrize("dim", [64, 96, 128, 256])
def test_prompts(dim):
    """Enough rows for the kernel of many queries a sequence."""
    s = Sequences([240, 265, 133, 350, 0, 96, 7, 331], 40, dim, page=32)
    attend(s, [140, 133, 133, 150, 5, 0, 7, 131], 4, 50, 4, otype=bf.OUT_F16)


@pytest.mark.parametrize("window,sinks,group,absent", [(40, 33, 4, ()), (1, 1, 5, ()), (64, 200, 3, ((1, 1), (2, 0))), (100, 32, 7, ((0, 0),))])
def test_prompts_masks(window, sinks, group, absent):
    s = Sequences([300, 330, 164, 177], 48, 64)
    attend(s, [170, 122, 164, 140], group, window, sinks, absent=absent)
    attend(s, [170, 122, 164, 140], group, window, sinks, absent=absent, scale=-0.1)


def test_prompt_longer():
    attend(Sequences([900], 16, 128), [900], 8, 200, 36, otype=bf.OUT_F16)


def test_absent_pages():
    s = Sequences([300, 64, 129], 2, 128)
    attend(s, [1, 1, 1], 4, 70, 10, absent=[(0, 0), (0, 4), (1, 0)])
    attend(s, [40, 3, 129], 2, 70, 10, absent=[(0, 0), (0, 3), (1, 0), (2, 1)])


@pytest.mark.parametrize("nqs", [[1, 1, 1], [70, 5, 64]])
def test_same_bits_as_without(nqs):
    """No first tokens, or no window: bf_kv4_attention's bits."""
    s = Sequences([2600, 333, 64], 2, 64)
    assert torch.equal(attend(s, nqs, 4, 2000, 0), s.check(nqs, 4, window=2000))
    assert torch.equal(attend(s, nqs, 4, 0, 7), s.check(nqs, 4))


def test_same_bits_again():
    s = Sequences([7000], 1, 128)
    a = attend(s, [1], 8, 5000, 64).clone()
    for _ in range(3):
        assert torch.equal(a, attend(s, [1], 8, 5000, 64))


@pytest.mark.parametrize("heads,nq", [(1, 64), (128, 200)])
def test_nan_tokens_reach_only_those_who_see_them(heads, nq):
    """Token 3 (a first one) and token 40 are NaN: rows from 3 on see the first, rows 40 .. 49 the other too."""
    s = Sequences([nq], heads, 64)
    q = torch.randn(nq, heads * 4 * 64).half().cuda()
    dev = lambda x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    nan = torch.full((1, heads, 64), float("nan")).half().cuda()

    def rows(sinks):
        o = torch.empty(nq, heads * 4 * 64, device="cuda")
        bf.kv4_attention_sinks(s.cache.c, q, o, dev([0, nq]), dev([nq]), s.table.cuda(), sinks=sinks, S=1, T=nq,
                               q_heads=heads * 4, max_q=nq, max_kv=nq, scale=0.1, window=10)
        return o.isnan().all(-1).cpu(), o.isnan().any(-1).cpu()

    slot = lambda t: (s.table[0, t // 64].long() * 64 + t % 64).reshape(1).cuda()  # noqa: E731
    bf.kv4_store(s.cache.c, nan, nan, slot(40), 1)
    t = torch.arange(nq)
    for x in rows(4):
        assert torch.equal(x, (t >= 40) & (t < 50))
    bf.kv4_store(s.cache.c, nan, nan, slot(3), 1)
    for x in rows(3):
        assert torch.equal(x, ((t >= 3) & (t < 13)) | ((t >= 40) & (t < 50)))
    for x in rows(4):
        assert torch.equal(x, t >= 3)


def test_other_stream():
    attend(Sequences([9000, 17], 2, 128), [1, 1], 4, 3000, 4, otype=bf.OUT_F16, stream=torch.cuda.Stream())


def test_captured_step_as_the_window_moves():
    """A captured call replayed as the sequence grows past its window and over a page's end."""
    s = Sequences([512], 2, 64)
    q = torch.randn(1, 8 * 64).half().cuda()
    lens, tab = torch.tensor([60], dtype=torch.int32).cuda(), s.table.cuda()
    starts, o, want = torch.tensor([0, 1], dtype=torch.int32).cuda(), torch.empty(1, 512, device="cuda"), torch.empty(1, 512, device="cuda")
    step = lambda out: bf.kv4_attention_sinks(s.cache.c, q, out, starts, lens, tab, sinks=4, S=1, T=1, q_heads=8, max_q=1,  # noqa: E731
                                              max_kv=512, scale=0.125, window=64)
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        step(o)
    st.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        step(o)
    for n in (61, 64, 65, 69, 96, 97, 128, 200, 512):
        lens.fill_(n)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        step(want)
        assert torch.equal(o, want) and torch.isfinite(o).all()
