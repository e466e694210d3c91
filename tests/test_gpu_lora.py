"""Low-rank adapters of many rows against 64 bits (run on an MI355X).

Tolerance, with s = A x and m = |A| |x|: an inner sum is a chain of at most K / 32 +
40 additions in fp32 (matrix steps, pieces), each off by 2^-23 of what it holds at most: (K / 32 + 40) 2^-23
m; s enters the second product to 2^-21 of the row's largest, whose sum over the ranks is as
exact as the first: scale |B| (ds + 2^-21 max |s|) + (rank / 16 + 4) 2^-23 scale |B| |s|; then one
rounding of Y (fp32 2^-23 with the addition, fp16 2^-11, 2^-25 where subnormal)."""
import pytest
import torch

import busfill as bf

pytestmark = pytest.mark.gpu

F16, F32 = torch.float16, torch.float32


class Case:
    def __init__(self, T, K, widths, adapters, rank, *, ids=None, ranks=None, scales=True, otype=bf.OUT_F32, gap=0, pad=0,
                 seed=1, garbage=True):
        g = torch.Generator().manual_seed(seed + T * 7 + K)
        self.T, self.K, self.widths, self.adapters, self.rank, self.otype = T, K, widths, adapters, rank, otype
        self.x = torch.randn(T, K, generator=g).half()
        self.x[:, ::19] *= 5
        self.ids = torch.randint(0, adapters, (T,), generator=g).int() if ids is None else torch.tensor(ids, dtype=torch.int32)
        self.ranks = None if ranks is None else torch.tensor(ranks, dtype=torch.int32)
        self.scales = torch.rand(adapters, generator=g) + 0.5 if scales else None
        if scales:
            self.scales[0] = -0.7
        self.ab, self.at, at = [], [], gap
        for n in widths:
            a = (torch.randn(adapters, rank, K, generator=g) / K ** 0.5).half()
            b = (torch.randn(adapters, n, rank, generator=g) * 0.3).half()
            if ranks is not None and garbage:                      # what lies past a rank may be anything
                for e, r in enumerate(ranks):
                    a[e, max(r, 0):] = float("nan")
                    b[e, :, max(r, 0):] = float("inf")
            self.ab.append((a, b))
            self.at.append(at)
            at += n + gap
        self.width = at + pad
        self.c = torch.randn(T, self.width, generator=g).to(F32 if otype == bf.OUT_F32 else F16)

    def want(self):
        y = self.c.double()
        tol = torch.zeros_like(y)
        for (a, b), n, at in zip(self.ab, self.widths, self.at):
            for t in range(self.T):
                e = int(self.ids[t])
                if not 0 <= e < self.adapters:
                    continue
                r = self.rank if self.ranks is None else min(max(int(self.ranks[e]), 0), self.rank)
                f = 1.0 if self.scales is None else float(self.scales[e])
                ar, br, x = a[e, :r].double(), b[e, :, :r].double(), self.x[t].double()
                s, m = ar @ x, ar.abs() @ x.abs()
                ds = (self.K / 32 + 40) * 2.0 ** -23 * m + 2.0 ** -21 * (s.abs().max() if r else 0)
                y[t, at:at + n] += f * (br @ s)
                tol[t, at:at + n] = abs(f) * (br.abs() @ (ds + (r / 16 + 4) * 2.0 ** -23 * s.abs()))
        tol = tol * (1 + 2.0 ** -10) + (2.0 ** -23 + (2.0 ** -11 if self.otype == bf.OUT_F16 else 0)) * y.abs() + 2.0 ** -24
        return y, tol

    def device(self):
        d = lambda v: None if v is None else v.cuda()  # noqa: E731
        self.dab = [(a.cuda(), b.cuda()) for a, b in self.ab]
        self.parts = bf.lora_parts([(a, b, n, at) for (a, b), n, at in zip(self.dab, self.widths, self.at)])
        self.dx, self.dids, self.dranks, self.dscales, self.dc = d(self.x), d(self.ids), d(self.ranks), d(self.scales), d(self.c)
        torch.cuda.synchronize()
        return dict(T=self.T, K=self.K, adapters=self.adapters, rank=self.rank, scales=self.dscales, ranks=self.dranks,
                    ldc=self.width, ldy=self.width, otype=self.otype)

    def check(self, y):
        want, tol = self.want()
        y = y.cpu()
        touched = torch.zeros(self.width, dtype=torch.bool)
        for n, at in zip(self.widths, self.at):
            touched[at:at + n] = True
        err = (y.double() - want).abs()[:, touched]
        assert (err <= tol[:, touched]).all(), float((err / tol[:, touched]).max())
        none = (self.ids < 0) | (self.ids >= self.adapters)
        assert torch.equal(y[none][:, touched], self.c[none][:, touched])
        return touched

    def run(self, *, place="out", workspace=False, stream=None):
        kw = self.device()
        y = self.dc if place == "in" else torch.full_like(self.dc, 9.0)
        torch.cuda.synchronize()
        if workspace:
            a = bf.lora_args(self.dx, self.dids, self.parts, self.dc, y, **kw)
            n = bf.lora_workspace_bytes(a)
            ws = torch.full((n,), 0xFF, dtype=torch.uint8, device="cuda")
            torch.cuda.synchronize()
            bf.lora_ws(a, ws, n, stream=stream)
        else:
            bf.lora(self.dx, self.dids, self.parts, self.dc, y, stream=stream, **kw)
        torch.cuda.synchronize()
        touched = self.check(y)
        left = y.cpu()[:, ~touched]
        assert torch.equal(left, self.c[:, ~touched] if place == "in" else torch.full_like(left, 9.0))
        return y


@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 40, 128, 129, 300])
@pytest.mark.parametrize("rank,adapters", [(8, 1), (16, 5), (64, 3), (72, 20)])
def test_rows_and_ranks(T, rank, adapters):
    Case(T, 264, [80], adapters, rank).run()


@pytest.mark.parametrize("K", [8, 24, 32, 40, 256, 1000, 5120])
def test_inputs(K):
    Case(19, K, [33], 4, 16).run()
    Case(1, K, [64], 2, 24, otype=bf.OUT_F16).run()


@pytest.mark.parametrize("widths", [[1], [7], [16], [65], [300], [130, 1, 64], [16, 32, 48, 64]])
@pytest.mark.parametrize("gap,pad", [(0, 0), (3, 2), (8, 16)])
@pytest.mark.parametrize("otype", [bf.OUT_F32, bf.OUT_F16])
def test_parts_and_columns(widths, gap, pad, otype):
    Case(21, 64, widths, 6, 32, gap=gap, pad=pad, otype=otype).run()


@pytest.mark.parametrize("place", ["in", "out"])
@pytest.mark.parametrize("otype", [bf.OUT_F32, bf.OUT_F16])
def test_rows_without_an_adapter(place, otype):
    """Ids below 0 and from `adapters` on: a copy, or nothing where Y is C."""
    ids = [-1, 3, 0, 4, 100, -2 ** 31, 2 ** 31 - 1, 2, 2, -1] * 5
    Case(50, 128, [96, 32], 4, 16, ids=ids, otype=otype).run(place=place)
    Case(4, 128, [96, 32], 4, 16, ids=[-1] * 4, otype=otype).run(place=place)


@pytest.mark.parametrize("T", [9, 200])
@pytest.mark.parametrize("rank", [16, 64, 136])
def test_ranks_of_their_own(T, rank):
    """Ranks from none to all, odd ones, below 0 and above rank; what lies past them is NaN and infinite."""
    Case(T, 128, [70], 9, rank, ranks=[0, 1, 7, 8, 9, 15, rank - 1, rank, -4]).run()
    Case(T, 128, [70], 2, rank, ranks=[rank + 5, 13], garbage=False).run()


@pytest.mark.parametrize("T,ids", [(64, "runs"), (500, "runs"), (500, "mixed"), (2000, "runs")])
def test_prompts(T, ids):
    which = [min(5, t * 6 // T) for t in range(T)] if ids == "runs" else [(t * 7) % 13 - 1 for t in range(T)]
    Case(T, 512, [200, 56], 12, 16 if T == 2000 else 64, ids=which, otype=bf.OUT_F16).run(workspace=True)


@pytest.mark.parametrize("T,widths,rank,otype", [
    (1100, [4200], 16, bf.OUT_F16), (1100, [4200], 64, bf.OUT_F32), (700, [3000, 1030], 32, bf.OUT_F32), (300, [260], 136, bf.OUT_F16),
    (600, [4100, 7], 72, bf.OUT_F32), (257, [64], 8, bf.OUT_F16)])
def test_many_rows_and_columns(T, widths, rank, otype):
    """Workgroups that take several blocks of columns, blocks of ranks and adapters in turn; tiles of one adapter, of several
    and of none."""
    ids = [min(3, t * 4 // T) if t % 230 < 200 else (t % 5) - 1 for t in range(T)]
    c = Case(T, 96, widths, 4, rank, ids=ids, ranks=[rank, rank - 3, max(1, rank // 3), rank], otype=otype, pad=8)
    c.run()


def test_many_rows_in_place():
    ids = [t // 100 - 1 for t in range(900)]
    Case(900, 64, [3500], 7, 16, ids=ids, otype=bf.OUT_F16).run(place="in")


def test_one_row_among_many_of_another():
    """Tiles whose rows are of one adapter but for the last."""
    Case(48, 96, [40], 3, 8, ids=([1] * 15 + [2]) * 3).run()


def test_no_scales_strided_rows_and_alignment():
    c = Case(20, 120, [45], 3, 16, scales=False)
    kw = c.device()
    wide = torch.full((20, 136), float("nan"), dtype=F16, device="cuda")
    wide[:, :120] = c.dx
    base = torch.full((20 * 46 + 1,), 9.0, device="cuda")
    y = base[1:].view(20, 46)                                      # rows off 16 bytes
    kw.update(ldx=136, ldy=46)
    bf.lora(wide, c.dids, c.parts, c.dc, y, **kw)
    torch.cuda.synchronize()
    c.check(y[:, :45])
    assert (y[:, 45] == 9.0).all()


def test_small_and_large_values():
    """Inner sums from 2^-40 to 2^20: s is taken to fp16 times a power of two of its own."""
    for e in (-14, -9, 6):
        c = Case(18, 256, [48], 3, 16)
        c.x = (c.x.float() * 2.0 ** e).half()
        c.ab = [((a.float() * 2.0 ** e).half(), b) for a, b in c.ab]
        c.c = c.c * 2.0 ** (2 * e)
        c.run()


def test_rows_of_infinities_and_nan():
    """A row that is not finite is not finite in its output, and leaves the others alone."""
    c = Case(20, 64, [50], 2, 16)
    c.x[3, 5], c.x[11, 60] = float("inf"), float("nan")
    kw = c.device()
    y = torch.empty_like(c.dc)
    bf.lora(c.dx, c.dids, c.parts, c.dc, y, **kw)
    assert (~torch.isfinite(y[[3, 11]])).all()
    rest = [t for t in range(20) if t not in (3, 11)]
    want, tol = c.want()
    assert ((y.cpu().double() - want).abs() <= tol)[rest].all()


def test_zero_adapter_gives_the_input():
    c = Case(17, 64, [32], 2, 8)
    c.ab = [(a, torch.zeros_like(b)) for a, b in c.ab]
    assert torch.equal(c.run().cpu(), c.c)
    c.ab = [(torch.zeros_like(a), torch.ones_like(b)) for a, b in c.ab]
    assert torch.equal(c.run().cpu(), c.c)


def test_adapters_of_more_than_4_gb():
    """The last adapter of a pool past 2^32 bytes."""
    K, rank, E = 8192, 64, 4500
    pool = torch.zeros(E, rank, K, dtype=F16, device="cuda")
    assert pool.numel() * 2 > 1 << 32
    c = Case(5, K, [40], 3, rank, ids=[0, 1, 2, -1, 2])
    kw = c.device()
    B = torch.zeros(E, 40, rank, dtype=F16, device="cuda")
    where = torch.tensor([0, E // 2 + 1, E - 1])
    pool[where.cuda()], B[where.cuda()] = c.dab[0][0], c.dab[0][1]
    ids = torch.where(c.ids >= 0, where[c.ids.clamp(min=0).long()].int(), c.ids).cuda()
    scales = torch.zeros(E, device="cuda")
    scales[where.cuda()] = c.dscales
    y = torch.empty_like(c.dc)
    kw.update(adapters=E, scales=scales)
    bf.lora(c.dx, ids, bf.lora_parts([(pool, B, 40, 0)]), c.dc, y, **kw)
    c.check(y)


def test_same_bits_in_any_company():
    """A row's result depends neither on its neighbours' adapters nor on the run (same T: the same cuts of K)."""
    a = Case(40, 512, [100], 6, 32)
    first = a.run().clone()
    for _ in range(3):
        assert torch.equal(first, a.run())
    b = Case(40, 512, [100], 6, 32)
    b.ids = b.ids.clone()
    b.ids[:20] = (b.ids[:20] + 1) % 6
    assert torch.equal(first[20:], b.run()[20:])


def test_other_stream_and_graph():
    c = Case(9, 640, [128, 64], 5, 16, otype=bf.OUT_F16)
    kw = c.device()
    y, z = torch.empty_like(c.dc), torch.empty_like(c.dc)
    a = bf.lora_args(c.dx, c.dids, c.parts, c.dc, y, **kw)
    n = bf.lora_workspace_bytes(a)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        bf.lora_ws(a, ws, n)
    for i in range(4):
        c.dids.copy_((c.dids + 1) % 5)
        c.dx.mul_(1.1)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        bf.lora(c.dx, c.dids, c.parts, c.dc, z, **kw)
        assert torch.equal(y, z)
    # the library's workspace is not grown under capture
    fresh, big = torch.cuda.Stream(), Case(400, 640, [128, 64], 5, 512, otype=bf.OUT_F16)
    kw = big.device()
    out = torch.empty_like(big.dc)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=fresh):
        with pytest.raises(bf.BusfillError) as err:
            bf.lora(big.dx, big.dids, big.parts, big.dc, out, **kw)
    assert err.value.status == bf.ERR_UNSUPPORTED


@pytest.mark.parametrize("T,adapters,rank,otype", [
    (300, 64, 16, bf.OUT_F16), (700, 9, 64, bf.OUT_F32), (257, 128, 72, bf.OUT_F16), (4097, 3, 8, bf.OUT_F16),
    (9000, 40, 16, bf.OUT_F32), (4160, 2047, 8, bf.OUT_F32)])
@pytest.mark.parametrize("place", ["in", "out"])
def test_many_rows_in_no_order(T, adapters, rank, otype, place):
    """Rows that are sorted by adapter: more than the sort takes at once, adapters with one row, many, none, rows without one."""
    g = torch.Generator().manual_seed(T)
    ids = torch.randint(-1, adapters + 1, (T,), generator=g)
    ids[torch.rand(T, generator=g) < 0.3] = adapters // 2                  # many of one
    if adapters > 5:
        ids[ids == 3] = 4                                                  # none of another
    Case(T, 40, [70], adapters, rank, ids=ids.tolist(), ranks=[(7 * e) % (rank + 1) for e in range(adapters)], otype=otype,
         pad=2).run(place=place, workspace=True)


@pytest.mark.parametrize("T,adapters", [(300, 151), (300, 2500), (5000, 2048)])
def test_many_rows_of_as_many_adapters(T, adapters):
    """Fewer than two rows an adapter, or more adapters than the sort counts: rows as they come."""
    Case(T, 24, [20], adapters, 8).run()


def test_sorted_rows_give_the_same_bits():
    """The order that rows come in, and the one that the sort gives an adapter's rows, change no bits."""
    c = Case(1500, 640, [260], 7, 32, otype=bf.OUT_F32)
    kw = c.device()

    def call(x, ids, into):
        y = torch.empty_like(into)
        bf.lora(x, ids, c.parts, into, y, **kw)
        torch.cuda.synchronize()
        return y

    first = call(c.dx, c.dids, c.dc)
    for i in range(4):
        p = torch.randperm(1500, generator=torch.Generator().manual_seed(i)).cuda() if i else c.dids.argsort(stable=True)
        assert torch.equal(call(c.dx[p].contiguous(), c.dids[p].contiguous(), c.dc[p].contiguous()), first[p])


@pytest.mark.parametrize("T", [3, 40, 300])
def test_rank_1024(T):
    Case(T, 128, [90], 2, 1024, ranks=[1024, 777]).run()


@pytest.mark.parametrize("T", [20, 300])
def test_infinities_reach_the_output_as_the_formula_has_them(T):
    """An infinity in a row of X: every output infinite with the sign of the sum, or NaN where infinities of both signs meet."""
    c = Case(T, 64, [48], 2, 16, ids=[0] * T)
    c.x[3, 5], c.x[7, 9] = float("inf"), float("-inf")
    kw = c.device()
    y = torch.empty_like(c.dc)
    bf.lora(c.dx, c.dids, c.parts, c.dc, y, **kw)
    torch.cuda.synchronize()
    (a, b), s = c.ab[0], float(c.scales[0])
    for t, r in ((3, 16), (7, 16)):
        want = c.c[t].double() + s * (b[0].double() @ (a[0].double() @ c.x[t].double()))
        assert torch.equal(torch.isnan(y[t].cpu()), torch.isnan(want))
    # one rank: no infinities of both signs
    kw["ranks"] = torch.ones(2, dtype=torch.int32, device="cuda")
    bf.lora(c.dx, c.dids, c.parts, c.dc, y, **kw)
    torch.cuda.synchronize()
    for t in (3, 7):
        want = c.c[t].double() + s * (b[0, :, :1].double() @ (a[0, :1].double() @ c.x[t].double()))
        assert torch.isinf(want).any() and torch.equal(y[t].cpu().double(), want)


@pytest.mark.parametrize("T", [30, 400])
@pytest.mark.parametrize("otype", [bf.OUT_F32, bf.OUT_F16])
def test_rows_apart(T, otype):
    """X, C and Y with strides of their own; what lies between the rows is left alone."""
    c = Case(T, 88, [60, 20], 5, 24, ids=[(3 * t) % 7 - 1 for t in range(T)], otype=otype)
    kw = c.device()
    x = torch.full((T, 104), float("nan"), dtype=F16, device="cuda")
    x[:, :88] = c.dx
    into = torch.full((T, 96), float("nan"), dtype=c.dc.dtype, device="cuda")
    into[:, :80] = c.dc
    y = torch.full((T, 85), 9.0, dtype=c.dc.dtype, device="cuda")
    kw.update(ldx=104, ldc=96, ldy=85)
    torch.cuda.synchronize()
    bf.lora(x, c.dids, c.parts, into, y, **kw)
    torch.cuda.synchronize()
    c.check(y[:, :80])
    assert (y[:, 80:] == 9.0).all()


def test_many_rows_in_a_graph_and_on_two_streams():
    """Replays sort the ids of the moment; calls at once on two streams have workspaces of their own."""
    c = Case(700, 640, [260], 9, 32, otype=bf.OUT_F16)
    kw = c.device()
    y, z, w = (torch.empty_like(c.dc) for _ in range(3))
    a = bf.lora_args(c.dx, c.dids, c.parts, c.dc, y, **kw)
    n = bf.lora_workspace_bytes(a)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=one):
        bf.lora_ws(a, ws, n)
    other = torch.empty_like(c.dids)
    for i in range(4):
        c.dids.copy_((c.dids * 5 + 1 + i) % 11 - 1)                        # (some without an adapter)
        other.copy_(c.dids.flip(0))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        bf.lora(c.dx, c.dids, c.parts, c.dc, z, stream=one.cuda_stream, **kw)
        bf.lora(c.dx, other, c.parts, c.dc, w, stream=two.cuda_stream, **kw)
        torch.cuda.synchronize()
        c.ids = c.dids.cpu()
        c.check(y)
        assert torch.equal(y, z)
        c.ids = other.cpu()
        c.check(w)


@pytest.mark.parametrize("T,adapters", [(128, 8), (129, 7), (129, 8), (129, 64), (129, 65), (256, 7), (257, 7)])
@pytest.mark.parametrize("rank", [16, 96])
def test_where_the_sort_begins(T, adapters, rank):
    Case(T, 72, [90, 6], adapters, rank, otype=bf.OUT_F16).run()
