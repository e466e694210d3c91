"""The example's decoder layer with a window, first tokens in sight and adapters:
its steps between the linears against 64 bits from the step's own inputs, and its
captured decode step against a prompt (run on an MI355X).

Tolerances are those of the operators' own tests: the norm 2^-11 + 2^-18 of itself,
a rotated element 2^-11 of itself and 2^-20 of its pair, attention 2^-11 + 2^-13 of
the values' mass and 2^-11 of itself; adapters from the projection's fp16 output (one
more rounding, 2^-11 of each) with inner sums within 2^-17 of their terms."""
import os
import sys

import pytest
import torch

import busfill as bf
import kv4_ref as R

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
import moe_decoder as M  # noqa: E402

pytestmark = pytest.mark.gpu


def small(**kw):
    return M.Shape(width=512, q_heads=8, kv_heads=2, dim=64, experts=16, chosen=3, ffn=256, **kw)


def adapted(y, x, pairs, widths, ids):
    """y in 64 bits with the adapters of x, and the tolerance of the sums."""
    y, tol, at = y.double(), torch.zeros(y.shape).double(), 0
    for (a, b), n in zip(pairs, widths):
        for t, e in enumerate(ids.tolist()):
            if e >= 0:
                ar, br, xt = a[e].double().cpu(), b[e].double().cpu(), x[t].double()
                s = ar @ xt
                y[t, at:at + n] += br @ s
                tol[t, at:at + n] = br.abs() @ (2.0 ** -17 * (ar.abs() @ xt.abs()) + 2.0 ** -20 * s.abs())
        at += n
    return y, tol


def test_steps_between_the_linears():
    s, streams, n = small(window=20, sinks=3, adapters=4, rank=24), 3, 75
    layer = M.Layer(s, seed=4)
    cache = M.Cache(s, streams, n)
    x = torch.randn(streams, n, s.width, device="cuda")
    who = torch.tensor([2, -1, 0], dtype=torch.int32, device="cuda")
    b = M.prompt(layer, cache, streams, x, who)
    torch.cuda.synchronize()
    rows, ids = streams * n, who.cpu().repeat_interleave(n)
    xd = x.cpu().double().view(rows, -1)
    h1 = xd / (xd.square().mean(-1, keepdim=True) + 1e-6).sqrt()
    assert ((b.h1.cpu().double() - h1).abs() <= (2.0 ** -11 + 2.0 ** -18) * h1.abs() + 2.0 ** -25).all()
    # queries and keys: the projection's fp16 rows, adapters on top, rotated
    base = torch.empty(rows, s.qkv, dtype=torch.float16, device="cuda")
    bf.gemm(bf.Q4_K, layer.wqkv, None, b.h1, base, rows, s.qkv, s.width, otype=bf.OUT_F16)
    q, tol = adapted(base.cpu(), b.h1.cpu(), layer.on_qkv, [512, 128, 128], ids)
    tol = tol + 2.0 ** -11 * q.abs() + 2.0 ** -24
    got = b.qkv.cpu().double()
    assert ((got[:, 640:] - q[:, 640:]).abs() <= tol[:, 640:]).all()             # (values: not rotated)
    t = torch.arange(n).repeat(streams).double()[:, None, None] * layer.freq.cpu().double()
    c, sn = torch.cos(t), torch.sin(t)
    p0, p1 = q[:, :640].view(rows, 10, 64).split(32, -1)
    t0, t1 = tol[:, :640].view(rows, 10, 64).split(32, -1)
    want = torch.cat([p0 * c - p1 * sn, p1 * c + p0 * sn], -1)
    size = torch.cat([p0.abs() + p1.abs()] * 2, -1)
    off = torch.cat([t0 * c.abs() + t1 * sn.abs(), t1 * c.abs() + t0 * sn.abs()], -1)
    assert ((got[:, :640].view(rows, 10, 64) - want).abs() <= off + 2.0 ** -20 * size + 2.0 ** -11 * want.abs() + 2.0 ** -24).all()
    # attention over what the cache holds of the rows
    heads, pos = b.qkv.cpu().view(streams, n, -1, s.dim), torch.arange(n)
    see = (pos[None] <= pos[:, None]) & ((pos[None] > pos[:, None] - 20) | (pos[None] < 3))
    att = b.att.cpu().double().view(streams, n, s.q_heads, s.dim)
    for st in range(streams):
        k, v = R.quantize(heads[st, :, 8:10]), R.quantize(heads[st, :, 10:])
        for h in range(s.q_heads):
            want, mass, _ = R.attention(heads[st, :, h], k[:, h // 4], v[:, h // 4], s.dim ** -0.5, see)
            assert ((att[st, :, h] - want).abs() <= (2.0 ** -11 + 2.0 ** -13) * mass + 2.0 ** -11 * want.abs() + 2.0 ** -24).all()
    # the second norm: of x and the output projection with its adapter
    y = torch.empty(rows, s.width, dtype=torch.float16, device="cuda")
    bf.gemm(bf.Q4_K, layer.wo, None, b.att, y, rows, s.width, 512, otype=bf.OUT_F16)
    y, tol = adapted(y.cpu(), b.att.cpu(), layer.on_out, [512], ids)
    r = xd + y
    tol = tol + 2.0 ** -11 * y.abs() + 2.0 ** -24 + 2.0 ** -23 * r.abs()
    root = (r.square().mean(-1, keepdim=True) + 1e-6).sqrt()
    h2 = r / root
    # r's error moves the root by at most the errors' own root mean square
    tol = (tol + h2.abs() * tol.square().mean(-1, keepdim=True).sqrt()) / root * (1 + 2.0 ** -8)
    assert ((b.h2.cpu().double() - h2).abs() <= tol + (2.0 ** -11 + 2.0 ** -18) * h2.abs() + 2.0 ** -25).all()


@pytest.mark.parametrize("window,sinks,adapters", [(0, 0, 0), (24, 4, 0), (16, 2, 3)])
def test_decode_graph_continues_a_prompt(window, sinks, adapters):
    """Seven tokens decoded one by one by the captured step give the rows that the whole prompt gives, wherever both
    choose the same experts: fp16 rows in between, so within a few of their roundings (4e-3), but for what those
    roundings do to the cache.  A key or value x that is off by one of them, 2^-10 |x|, is off by up to 8 2^-10 = 2^-7 of
    its block's step d (|x| <= 8 d), so it gets another code with a probability of up to 2^-7, d away: 2^-3.5 d in the root
    mean square, with d = max / 8 = 0.41 of the values' deviation (the largest of 32 is near 3.3 of it) 0.036 of it.  Of w
    tokens that a query sees with about equal weights up to seven were decoded: their values move the attention's output by
    0.036 sqrt(7 / w) of itself, their keys (scores of deviation near 1 move by 0.036) as much again, 0.051 sqrt(7 / w)
    together.  That output, an average of w, is at most 1 / sqrt(w) of the values' size, and its projection at most as much
    of x (adapters add less than their projection), the experts' block of the moved rows as much again: 2 / sqrt(w).  Without
    a window, w = 62 to 68, that is 4e-3; with 18 tokens in sight 1.5e-2."""
    s, streams, n, more = small(window=window, sinks=sinks, adapters=adapters), 3, 61, 7
    layer = M.Layer(s, seed=5)
    who = torch.tensor([1, 0, -1], dtype=torch.int32, device="cuda") if adapters else None
    x = torch.randn(streams, n + more, s.width, device="cuda")
    whole = M.prompt(layer, M.Cache(s, streams, n + more), streams, x, who)
    cache = M.Cache(s, streams, n + more + 1)
    M.prompt(layer, cache, streams, x[:, :n], who)
    d = M.Decoder(layer, cache, streams, n, who)
    want, ids = whole.x.view(streams, n + more, -1), whole.ids.view(streams, n + more, -1)
    seen = window + sinks if window else n + 1
    tol = 4e-3 + 0.051 * (7 / seen) ** 0.5 * 2 / seen ** 0.5
    same = 0
    for i in range(more):
        got = d.step(x[:, n + i]).clone()
        torch.cuda.synchronize()
        for st in range(streams):
            if not torch.equal(d.b.ids[st].sort().values, ids[st, n + i].sort().values):
                continue
            same += 1
            a, w = got[st].double(), want[st, n + i].double()
            assert float((a - w).norm()) <= tol * float(w.norm())
    assert same >= streams * more - 3


def test_captured_steps_are_the_eager_ones():
    """The captured step, replayed as the sequences pass the window and pages' ends, gives the bits of the same calls made
    one by one."""
    s, streams, n = small(window=40, sinks=4, adapters=3), 4, 58
    layer = M.Layer(s, seed=6)
    who = torch.tensor([1, 0, -1, 1], dtype=torch.int32, device="cuda")
    x = torch.randn(streams, n + 12, s.width, device="cuda")
    caches = [M.Cache(s, streams, n + 13) for _ in range(2)]
    for c in caches:
        c.data.zero_()
        M.prompt(layer, c, streams, x[:, :n], who)
    d, e = M.Decoder(layer, caches[0], streams, n, who), M.Decoder(layer, caches[1], streams, n, who)
    torch.cuda.synchronize()
    for i in range(12):
        got = d.step(x[:, n + i]).clone()
        e.b.x.copy_(x[:, n + i])
        layer(caches[1], e.b)
        e._at(e.length + 1)
        torch.cuda.synchronize()
        assert torch.equal(got, e.b.x) and torch.equal(caches[0].data, caches[1].data)
