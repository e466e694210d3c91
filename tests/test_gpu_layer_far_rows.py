"""Norm, append and adapters whose rows lie more than 4 GB apart, and calls from several
host threads (run on an MI355X)."""
import threading

import pytest
import torch

import busfill as bf
from test_gpu_kv4_append import frequencies, near, rotated
from test_gpu_lora import Case
from test_gpu_norm import F16, F32, check_h, inputs, reference

pytestmark = pytest.mark.gpu


def far(x, ld):
    """x's rows on the GPU, ld elements apart (what lies between them is never read)."""
    out = torch.empty(x.shape[0] * ld, dtype=x.dtype, device="cuda").view(x.shape[0], ld)
    out[:, :x.shape[1]] = x.cuda()
    return out


@pytest.mark.parametrize("K,ld", [(640, (1 << 30) + 8), (637, (1 << 30) + 7)])
def test_norm(K, ld):
    x, d, w = inputs(4, K, F16, F16, F32, K)
    xs, ds = far(x, ld), far(d, ld)
    assert xs.numel() * 2 > 1 << 32
    bf.rms_norm(xs, 4, K, delta=ds, R=xs, weight=w.cuda(), H=ds, ldx=ld, ldd=ld, ldr=ld, ldh=ld)
    torch.cuda.synchronize()
    assert torch.equal(xs[:, :K].cpu(), (x.float() + d.float()).half())
    check_h(ds[:, :K], reference(x, d, w, 0.0, 1e-6))


@pytest.mark.parametrize("T,ldx,ldy", [(3, (1 << 30) + 8, (1 << 29) + 4), (300, 1 << 23, 1 << 22)])
def test_adapters(T, ldx, ldy):
    """(few rows, and rows sorted by adapter; Y over C)"""
    c = Case(T, 96, [70], 3, 16, ids=[t % 4 - 1 for t in range(T)])
    kw = c.device()
    x, y = far(c.x, ldx), far(c.c, ldy)
    assert x.numel() * 2 > 1 << 32 and y.numel() * 4 > 1 << 32
    kw.update(ldx=ldx, ldc=ldy, ldy=ldy)
    bf.lora(x, c.dids, c.parts, y, y, **kw)
    torch.cuda.synchronize()
    c.check(y[:, :70])


def test_append():
    """Queries, keys and values 4 GB apart, rotated in place."""
    T, hq, h, d, ld = 4, 3, 1, 64, (1 << 30) + 8
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(T, n * d, generator=g).half() for n in (hq, h, h))
    rows = far(torch.cat([q, k, v], -1), ld)
    data = torch.zeros(bf.kv4_bytes(1, 64, h, d), dtype=torch.uint8, device="cuda")
    cache = bf.kv4_cache(data, 1, 64, h, d)
    slots, position, freq = torch.tensor([7, 50, 0, 63]), torch.tensor([5, 900, 0, 131072]), frequencies(d).float()
    bf.kv4_append(cache, rows[:, hq * d:], rows[:, (hq + h) * d:], slots.cuda(), position.cuda(), freq.cuda(), T, Q=rows, Q_out=rows,
                  q_heads=hq, K_out=rows[:, hq * d:], ldq=ld, ldqo=ld, ldk=ld, ldko=ld, ldv=ld)
    torch.cuda.synchronize()
    assert near(rows[:, :hq * d].reshape(T, hq, d), rotated(q.view(T, hq, d), position, freq, d, bf.ROPE_HALVES, 1.0))
    assert near(rows[:, hq * d:(hq + h) * d].reshape(T, h, d), rotated(k.view(T, h, d), position, freq, d, bf.ROPE_HALVES, 1.0))
    want = torch.zeros_like(data)
    other = bf.kv4_cache(want, 1, 64, h, d)
    bf.kv4_store(other, rows[:, hq * d:(hq + h) * d].contiguous(), v.cuda(), slots.cuda(), T)
    torch.cuda.synchronize()
    assert torch.equal(data, want)


def test_calls_from_several_threads():
    """Four threads on one stream, each with calls of its own that share the stream's workspace: the results of calls alone."""
    cases = [Case(T, 640, [130], E, rank, otype=bf.OUT_F16, seed=i) for i, (T, E, rank) in
             enumerate([(5, 4, 16), (300, 9, 64), (90, 3, 72), (700, 20, 136)])]
    kws = [c.device() for c in cases]
    x, d, w = (t.cuda() for t in inputs(40, 640, F32, F16, F32, 2))
    alone, normed = [], torch.empty(40, 640, dtype=F16, device="cuda")
    for c, kw in zip(cases, kws):
        alone.append(torch.empty_like(c.dc))
        bf.lora(c.dx, c.dids, c.parts, c.dc, alone[-1], **kw)
    bf.rms_norm(x, 40, 640, delta=d, weight=w, H=normed)
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    out = [[(torch.empty_like(c.dc), torch.empty_like(normed)) for _ in range(20)] for c in cases]
    errors = []

    def work(i):
        try:
            for y, h in out[i]:
                bf.lora(cases[i].dx, cases[i].dids, cases[i].parts, cases[i].dc, y, stream=st, **kws[i])
                bf.rms_norm(x, 40, 640, delta=d, weight=w, H=h, stream=st)
        except Exception as e:                                             # (a thread's exception would be lost)
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors
    for c, a, ys in zip(cases, alone, out):
        c.check(a)
        assert all(torch.equal(a, y) and torch.equal(normed, h) for y, h in ys)
