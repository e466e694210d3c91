"""The 4-bit key/value cache and attention over it against 64-bit references
(run on an MI355X).

Tolerance of attention, per output element, with A = sum_t p_t |v_t|: each
product p d is rounded to fp16 (2^-11 of it at most), scores and exponentials
are fp32 (their errors, a few 2^-24 of sums of |q k| under 100 here, stay under
2^-14 of p), so |o - exact| <= (2^-11 + 2^-13) A, plus the output's own rounding
(fp16: 2^-11 |o| + 2^-25).  lse: fp32 scores and log2, 1e-4 absolute.
"""
import math

import pytest
import torch

import busfill as bf
import kv4_ref as R

pytestmark = pytest.mark.gpu


class Cache:
    """A cache whose unwritten bytes are 0xFF: scales that read as NaN, codes of 15."""

    def __init__(self, pages, page, heads, dim):
        self.page, self.heads, self.dim, self.pages = page, heads, dim, pages
        self.data = torch.full((bf.kv4_bytes(pages, page, heads, dim),), 0xFF, dtype=torch.uint8, device="cuda")
        self.c = bf.kv4_cache(self.data, pages, page, heads, dim)


def rows(n, heads, dim, seed):
    g = torch.Generator().manual_seed(seed)
    k = torch.randn(n, heads, dim, generator=g)
    k[..., 5::41] *= 4
    return k.half(), torch.randn(n, heads, dim, generator=g).half()


def same(got, want):
    w = want.to(torch.float16)
    return torch.equal(torch.nan_to_num(got.cpu(), nan=7e3), torch.nan_to_num(w, nan=7e3))


@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("heads,T,page,start", [(1, 1, 32, 0), (2, 1, 64, 63), (3, 40, 32, 5), (2, 97, 64, 31), (8, 130, 256, 0)])
def test_store_and_load(dim, heads, T, page, start):
    pages = (start + T + page - 1) // page + 2
    c = Cache(pages, page, heads, dim)
    k, v = rows(T, heads, dim, T + dim)
    perm = torch.randperm(pages, generator=torch.Generator().manual_seed(3))
    at = torch.arange(start, start + T)
    slots = (perm[at // page] * page + at % page).cuda()
    bf.kv4_store(c.c, k.cuda(), v.cuda(), slots, T)
    k2, v2 = torch.full_like(k, -1).cuda(), torch.full_like(v, -1).cuda()
    bf.kv4_load(c.c, slots, k2, v2, T)
    assert same(k2, R.quantize(k)) and same(v2, R.quantize(v))
    # nothing but the tokens' own bytes changed: their records hold 36 dim bytes for 32 tokens
    assert int((c.data != 0xFF).sum()) <= T * heads * 36 * dim // 32
    untouched = torch.tensor([s for s in range(pages * page) if s not in set(slots.tolist())][:33], dtype=torch.int64)
    if len(untouched):
        a, b = (torch.zeros(len(untouched), heads, dim, dtype=torch.float16, device="cuda") for _ in range(2))
        bf.kv4_load(c.c, untouched.cuda(), a, b, len(untouched))
        assert a.isnan().all() and b.isnan().all()


def test_store_corner_values():
    """Zeros, subnormals, equal magnitudes of both signs, ties between codes, the largest values, infinities, NaN."""
    x = torch.zeros(10, 1, 64, dtype=torch.float16)
    x[1, 0, :32] = 2.0 ** -24 * torch.arange(32)               # scales of subnormals
    x[2, 0, 3], x[2, 0, 9] = 4.0, -4.0                          # +m first
    x[3, 0, 3], x[3, 0, 9] = -4.0, 4.0                          # -m first
    x[4, 0, :32] = torch.arange(32) * 0.25 - 4.0                # exact half steps (d = 0.5)
    x[5, 0] = torch.linspace(-65504, 65504, 64)
    x[6, 0, 40] = float("inf")
    x[7, 0, 2] = float("nan")
    x[8, 0] = -0.0
    x[9, 0, :4] = torch.tensor([3.0, 3.0, -3.0, 1.5])
    c = Cache(1, 32, 1, 64)
    slots = torch.arange(10).cuda() + 11
    bf.kv4_store(c.c, x.cuda(), x.flip(0).cuda(), slots, 10)
    k2, v2 = torch.empty_like(x).cuda(), torch.empty_like(x).cuda()
    bf.kv4_load(c.c, slots, k2, v2, 10)
    assert same(k2, R.quantize(x)) and same(v2, R.quantize(x.flip(0)))


def test_store_strides_and_skipped_slots():
    c = Cache(2, 64, 2, 128)
    T = 50
    k, v = rows(T, 2, 128, 1)
    wide = torch.zeros(T, 7168, dtype=torch.float16)
    wide[:, 512:768], wide[:, 768:1024] = k.reshape(T, -1), v.reshape(T, -1)
    wide = wide.cuda()
    slots = torch.randperm(128)[:T]
    slots[::7] = -1
    slots[3] = 128                                              # past the cache
    slots = slots.cuda()
    bf.kv4_store(c.c, wide[:, 512:], wide[:, 768:], slots, T, ldk=7168, ldv=7168)
    k2, v2 = torch.full((T, 256), 5.0).half().cuda(), torch.full((T, 256), 5.0).half().cuda()
    bf.kv4_load(c.c, slots, k2, v2, T)
    gone = ((slots < 0) | (slots > 127)).cpu()
    wk, wv = R.quantize(k), R.quantize(v)
    wk[gone], wv[gone] = 0, 0
    assert same(k2.reshape(k.shape), wk) and same(v2.reshape(v.shape), wv)
    assert int((c.data != 0xFF).sum()) <= int((~gone).sum()) * 2 * 36 * 4


class Sequences:
    """Sequences with pages in no order, keys and values in a cache and in 64 bits."""

    def __init__(self, lens, heads, dim, page=64, seed=1, max_kv=None):
        self.lens, self.heads, self.dim, self.page = lens, heads, dim, page
        per = [(n + page - 1) // page for n in lens]
        pages = sum(per) + 1
        g = torch.Generator().manual_seed(seed)
        perm = torch.randperm(pages, generator=g)
        self.ldt = max(max(per), ((max_kv or 0) + page - 1) // page, 1)
        table = torch.full((len(lens), self.ldt), -1, dtype=torch.int32)
        self.cache = Cache(pages, page, heads, dim)
        self.k, self.v, at = [], [], 0
        for s, n in enumerate(lens):
            table[s, :per[s]] = perm[at:at + per[s]].int()
            if n:
                k, v = rows(n, heads, dim, seed + 31 * s)
                t = torch.arange(n)
                slots = perm[at + t // page] * page + t % page
                bf.kv4_store(self.cache.c, k.cuda(), v.cuda(), slots.cuda(), n)
                self.k.append(R.quantize(k))
                self.v.append(R.quantize(v))
            else:
                self.k.append(torch.zeros(0, heads, dim).double())
                self.v.append(torch.zeros(0, heads, dim).double())
            at += per[s]
        self.table = table

    def check(self, nqs, group, *, causal=True, window=0, otype=bf.OUT_F32, scale=None, absent=(), seed=5, max_kv=None,
              max_q=None, pad=0, qscale=1.0, workspace=False, stream=None):
        hq, d = self.heads * group, self.dim
        scale = 1 / math.sqrt(d) if scale is None else scale
        starts = [0]
        for n in nqs:
            starts.append(starts[-1] + n)
        T = max(1, starts[-1])
        g = torch.Generator().manual_seed(seed)
        q = (torch.randn(T, hq * d + pad, generator=g) * qscale).half()
        table = self.table.clone()
        for s, p in absent:
            table[s, p] = -1 if p % 2 else self.cache.pages
        kw = dict(S=len(nqs), T=T, q_heads=hq, max_q=max_q or max(max(nqs), 1),
                  max_kv=max(self.lens) if max_kv is None else max_kv, scale=scale, causal=causal, window=window,
                  otype=otype, ldq=hq * d + pad, ldo=hq * d + pad)
        o = torch.full((T, hq * d + pad), 9.0, dtype=torch.float32 if otype == bf.OUT_F32 else torch.float16, device="cuda")
        lse = torch.full((T, hq), 9.0, device="cuda")
        args = [q.cuda(), o, torch.tensor(starts, dtype=torch.int32).cuda(), torch.tensor(self.lens, dtype=torch.int32).cuda(),
                table.cuda()]
        torch.cuda.synchronize()
        if workspace:
            a = bf.kv4_attention_args(self.cache.c, *args, lse=lse, **kw)
            n = bf.kv4_attention_workspace_bytes(self.cache.c, a)
            ws = torch.full((n,), 0xFF, dtype=torch.uint8, device="cuda")
            torch.cuda.synchronize()
            bf.kv4_attention_ws(self.cache.c, a, ws if n else None, n, stream=stream)
        else:
            bf.kv4_attention(self.cache.c, *args, lse=lse, stream=stream, **kw)
        torch.cuda.synchronize()
        got, got_lse = o.cpu().double(), lse.cpu().double()
        assert (got[:, hq * d:] == 9.0).all()
        for s, nq in enumerate(nqs):
            n = self.lens[s]
            t = torch.arange(n)
            here = torch.ones(n, dtype=torch.bool)
            for (ss, p) in absent:
                if ss == s:
                    here[p * self.page:(p + 1) * self.page] = False
            pos = n - nq + torch.arange(nq)[:, None]
            see = (t[None] <= pos if causal else torch.ones(nq, n, dtype=torch.bool)) & here
            if window:
                see = see & (t[None] > pos - window)
            for h in range(hq):
                r = slice(starts[s], starts[s + 1])
                qq = q[r, h * d:(h + 1) * d]
                want, mass, wl = R.attention(qq, self.k[s][:, h // group], self.v[s][:, h // group], scale, see)
                tol = (2.0 ** -11 + 2.0 ** -13) * mass + 2.0 ** -24
                if otype == bf.OUT_F16:
                    tol = tol + 2.0 ** -11 * want.abs() + 2.0 ** -25
                err = (got[r, h * d:(h + 1) * d] - want).abs()
                assert (err <= tol).all(), (s, h, float((err / tol).max()))
                empty = torch.isinf(wl)
                assert torch.isinf(got_lse[r, h][empty]).all() and (got_lse[r, h][empty] < 0).all()
                assert ((got_lse[r, h] - wl)[~empty].abs() <= 1e-4).all()
        return o


@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("heads,group", [(1, 1), (2, 5), (1, 16), (3, 8)])
def test_single_tokens(dim, heads, group):
    """One query a sequence: lengths from one token to several records, a page that ends inside one."""
    Sequences([1, 2, 31, 32, 33, 64, 65, 200, 0], heads, dim).check([1] * 9, group)


@pytest.mark.parametrize("page", [32, 96, 256])
def test_page_sizes(page):
    Sequences([1, 95, 97, 300], 2, 128, page=page).check([1] * 4, 4, otype=bf.OUT_F16)


@pytest.mark.parametrize("lens", [[3000], [5001, 700, 64, 0, 1]])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("workspace", [False, True])
def test_long_sequences_in_chunks(lens, dim, workspace):
    """More records than a workgroup's: the chunks' results joined, beside sequences of one chunk."""
    Sequences(lens, 1, dim).check([1] * len(lens), 8, workspace=workspace)


@pytest.mark.parametrize("nqs,lens", [([4, 1, 7], [40, 1, 7]), ([33, 2], [33, 90]), ([17, 0, 5], [200, 50, 3]),
                                      ([130], [130]), ([100, 61], [230, 61])])
@pytest.mark.parametrize("group", [1, 3, 8])
def test_several_queries(nqs, lens, group):
    """Causal masks inside a record, row tiles that begin inside a query's heads, queries that stand before the first
    cached token (5 queries over 3 tokens) and see nothing."""
    Sequences(lens, 2, 64, max_kv=256).check(nqs, group, max_kv=256)


@pytest.mark.parametrize("dim", [64, 96, 128, 256])
def test_prompts(dim):
    """Enough rows for the kernel of many queries a sequence: whole and partial row tiles, queries behind cached tokens,
    sequences without queries and without tokens, a page that ends inside a record."""
    s = Sequences([40, 65, 33, 150, 0, 96, 7, 31], 40, dim, page=32)
    s.check([40, 33, 33, 50, 5, 0, 9, 31], 4, otype=bf.OUT_F16, pad=8)


@pytest.mark.parametrize("heads,causal,window,group,absent", [
    (40, False, 0, 4, ()), (64, True, 40, 3, ()), (32, True, 0, 16, ((1, 1), (2, 0))), (48, True, 1, 5, ()), (32, True, 0, 7, ())])
def test_prompts_masks(heads, causal, window, group, absent):
    s = Sequences([100, 130, 64, 77], heads, 64)
    s.check([70, 22, 64, 40], group, causal=causal, window=window, absent=absent)
    s.check([70, 22, 64, 40], group, causal=causal, window=window, absent=absent, scale=-0.1)


def test_prompt_longer():
    """Several rounds of units on the chip, rows that see up to 20 records."""
    Sequences([600], 16, 128).check([600], 8, otype=bf.OUT_F16)


def test_prompt_nan_tokens_reach_only_those_who_see_them():
    s = Sequences([120], 128, 64)
    k = torch.full((1, 128, 64), float("nan")).half().cuda()
    slot = (s.table[0, 0].long() * 64 + 40).reshape(1).cuda()
    for nan_keys in (True, False):
        bf.kv4_store(s.cache.c, k if nan_keys else torch.zeros_like(k), k, slot, 1)
        q = torch.randn(120, 512 * 64).half().cuda()
        o = torch.empty(120, 512 * 64, device="cuda")
        dev = lambda x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
        bf.kv4_attention(s.cache.c, q, o, dev([0, 120]), dev([120]), s.table.cuda(), S=1, T=120, q_heads=512, max_q=120,
                         max_kv=120, scale=0.1)
        assert not o[:40].isnan().any() and o[40:].isnan().all()


@pytest.mark.parametrize("nqs,lens", [([1, 1], [70, 333]), ([9], [9]), ([40], [170])])
def test_not_causal(nqs, lens):
    Sequences(lens, 2, 128).check(nqs, 2, causal=False)


@pytest.mark.parametrize("window", [1, 31, 32, 100, 5000])
def test_window(window):
    s = Sequences([260, 33, 64, 2], 2, 64)
    s.check([1, 1, 1, 1], 4, window=window)
    s.check([70, 5, 64, 2], 4, window=window)


def test_absent_pages():
    """Pages that are not there are seen by no one; a sequence with none left gives zeros."""
    s = Sequences([300, 64, 129], 2, 128)
    s.check([1, 1, 1], 4, absent=[(0, 1), (0, 4), (1, 0)])
    s.check([40, 3, 129], 2, absent=[(0, 0), (0, 3), (1, 0), (2, 1)])


def test_rows_are_left_alone_and_bounds_cut():
    """Query rows of no sequence stay as they were; kv_len above max_kv is cut to it."""
    s = Sequences([100], 1, 64)
    o = torch.full((6, 64), 9.0, device="cuda")
    q = torch.randn(6, 64).half().cuda()
    kw = dict(S=1, T=6, q_heads=1, max_q=2, scale=0.1)
    dev = lambda x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    bf.kv4_attention(s.cache.c, q, o, dev([2, 4]), dev([100]), s.table.cuda(), max_kv=100, **kw)
    assert (o[[0, 1, 4, 5]] == 9.0).all() and (o[2:4] != 9.0).all()
    a, b = torch.zeros(6, 64, device="cuda"), torch.zeros(6, 64, device="cuda")
    bf.kv4_attention(s.cache.c, q, a, dev([2, 4]), dev([100]), s.table.cuda(), max_kv=70, **kw)
    bf.kv4_attention(s.cache.c, q, b, dev([2, 4]), dev([70]), s.table.cuda(), max_kv=70, **kw)
    assert torch.equal(a, b)
    # q_start past T and running backwards: cut, nothing written
    bf.kv4_attention(s.cache.c, q, a, dev([4, 2]), dev([100]), s.table.cuda(), max_kv=100, **kw)
    assert torch.equal(a, b)


@pytest.mark.parametrize("qscale", [1e-4, 60.0, 1.2e4])
def test_query_magnitudes(qscale):
    """Queries from subnormal to near fp16's largest (scale chosen so that the scores stay in range)."""
    Sequences([150], 2, 64).check([1], 4, qscale=qscale, scale=0.125 / qscale)


@pytest.mark.parametrize("scale", [0.0, -0.1])
def test_scales_of_zero_and_below(scale):
    Sequences([45, 130], 2, 64).check([3, 1], 2, scale=scale)


def test_sharp_softmax():
    """Scores hundreds apart: the running maximum climbs from record to record.  (The score's fp32 error, 2^-22 of
    sums of |q k| near 3000, is part of p here: up to 2^-10, hence values of one sign and a bound on the whole.)"""
    s = Sequences([400], 1, 64, seed=9)
    order = (s.k[0][:, 0] @ torch.ones(64).double()).argsort()
    slots = torch.arange(400)
    table = s.table[0].long()
    slots = (table[slots // 64] * 64 + slots % 64).cuda()
    k, v = s.k[0][order].half(), s.v[0][order].half()
    bf.kv4_store(s.cache.c, k.cuda(), v.cuda(), slots, 400)
    q = torch.full((1, 64), 8.0).half()
    o = torch.empty(1, 64, device="cuda")
    dev = lambda x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    bf.kv4_attention(s.cache.c, q.cuda(), o, dev([0, 1]), dev([400]), s.table.cuda(), S=1, T=1, q_heads=1, max_q=1,
                     max_kv=400, scale=1.0)
    want, mass, _ = R.attention(q, R.quantize(k)[:, 0], R.quantize(v)[:, 0], 1.0, torch.ones(1, 400, dtype=torch.bool))
    assert ((o.cpu().double() - want).abs() <= 2.0 ** -9 * mass + 2.0 ** -20).all()


def test_nan_tokens_reach_only_those_who_see_them():
    s = Sequences([64], 1, 64)
    k = torch.full((1, 1, 64), float("nan")).half().cuda()
    slot = (s.table[0, 0].long() * 64 + 40).reshape(1).cuda()
    bf.kv4_store(s.cache.c, k, k, slot, 1)
    q = torch.randn(64, 64).half().cuda()
    o = torch.empty(64, 64, device="cuda")
    dev = lambda x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    bf.kv4_attention(s.cache.c, q, o, dev([0, 64]), dev([64]), s.table.cuda(), S=1, T=64, q_heads=1, max_q=64, max_kv=64,
                     scale=0.1)
    assert not o[:40].isnan().any() and o[40:].isnan().all()


def test_other_stream_and_strides():
    st = torch.cuda.Stream()
    Sequences([900, 17], 2, 128).check([1, 1], 4, pad=24, otype=bf.OUT_F16, stream=st)


def test_same_bits_again():
    """No result depends on the order in which workgroups run."""
    s = Sequences([4000], 1, 128)
    a = s.check([1], 8).clone()
    for _ in range(3):
        assert torch.equal(a, s.check([1], 8))


@pytest.mark.parametrize("nq", [1, 300])
def test_cache_of_more_than_4_gb(nq):
    """Pages on both sides of 2^32 bytes: single tokens and, with 300 queries, the kernel of many queries."""
    s = Sequences([330, 300], 8, 256, page=256)
    pages = 8000
    big = Cache.__new__(Cache)
    big.page, big.heads, big.dim, big.pages = 256, 8, 256, pages
    big.data = torch.empty(bf.kv4_bytes(pages, 256, 8, 256), dtype=torch.uint8, device="cuda")
    assert big.data.numel() > 1 << 32
    big.c = bf.kv4_cache(big.data, pages, 256, 8, 256)
    k = torch.empty(630, 8, 256, dtype=torch.float16, device="cuda")
    v, table, at = torch.empty_like(k), torch.tensor([[pages - 1, 3], [0, pages - 2]], dtype=torch.int32), 0
    for i, n in enumerate(s.lens):                             # the same values, at other places
        t = torch.arange(n)
        old, new = (p[i].long()[t // 256] * 256 + t % 256 for p in (s.table, table))
        bf.kv4_load(s.cache.c, old.cuda(), k[at:], v[at:], n)
        bf.kv4_store(big.c, k[at:], v[at:], new.cuda(), n)
        k2, v2 = torch.empty_like(k[:n]), torch.empty_like(v[:n])
        bf.kv4_load(big.c, new.cuda(), k2, v2, n)
        s.k[i], s.v[i] = k2.cpu().double(), v2.cpu().double()
        for got, kept in ((s.k[i], k[at:at + n]), (s.v[i], v[at:at + n])):
            want = R.quantize(kept.cpu())
            assert torch.equal(got, want.half().double())
            got.copy_(want)
        torch.cuda.synchronize()
        at += n
    s.cache, s.table, s.ldt = big, table, 2
    s.check([nq, nq], 16)


def test_captured_decode_step():
    """Store and attention in a graph, replayed as the sequences grow: the lengths live in device memory."""
    heads, dim, page, most = 2, 64, 64, 512
    pages = most // page
    c = Cache(pages, page, heads, dim)
    table = torch.randperm(pages).int().reshape(1, -1)
    k, v = rows(most, heads, dim, 3)
    n0 = 300
    t = torch.arange(most)
    slots = (table[0].long()[t // page] * page + t % page).cuda()
    bf.kv4_store(c.c, k.cuda(), v.cuda(), slots, n0)
    q = torch.randn(1, 8 * dim).half().cuda()
    kin, vin, sin = k[:1].cuda().clone(), v[:1].cuda().clone(), slots[:1].clone()
    lens = torch.tensor([n0], dtype=torch.int32).cuda()
    o, tab, starts = torch.empty(1, 8 * dim, device="cuda"), table.cuda(), torch.tensor([0, 1], dtype=torch.int32).cuda()
    kw = dict(S=1, T=1, q_heads=8, max_q=1, max_kv=most, scale=0.125)

    def step(out):
        bf.kv4_store(c.c, kin, vin, sin, 1)
        bf.kv4_attention(c.c, q, out, starts, lens, tab, **kw)

    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        sin.copy_(slots[n0:n0 + 1])
        lens.fill_(n0 + 1)
        kin.copy_(k[n0:n0 + 1])
        vin.copy_(v[n0:n0 + 1])
        step(o)
    st.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        step(o)
    for n in range(n0, n0 + 5):
        kin.copy_(k[n:n + 1])
        vin.copy_(v[n:n + 1])
        sin.copy_(slots[n:n + 1])
        lens.fill_(n + 1)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = torch.empty_like(o)
        step(want)
        assert torch.equal(o, want)
