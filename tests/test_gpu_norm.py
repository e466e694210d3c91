"""Residual addition and root-mean-square norm against 64 bits (run on an MI355X).

Tolerances: r is one fp32 addition, exactly torch's.  The sum of squares adds at
most 32 squares a thread and 26 partial sums after that, every term positive:
within 58 2^-24 of itself, half of that in its root; then a division, a root and
three products: y is within 2^-18 of itself before its rounding to fp16 (2^-11,
2^-25 where subnormal).  A code's value is within half a step dd of y (and the
2^-18 y, and 127 roundings of the quotient: 2^-16 dd).
"""
import pytest
import torch

import busfill as bf

pytestmark = pytest.mark.gpu

F16, F32 = torch.float16, torch.float32


def q8_views(aq, T, K):
    n, b = T * K, T * K // 32
    return (aq[:n].view(torch.int8).view(T, K // 32, 32), aq[n:n + 4 * b].view(F32).view(T, K // 32),
            aq[n + 4 * b:n + 8 * b].view(torch.int32).view(T, K // 32))


def padded(x, ld):
    """x's rows on the GPU in rows of ld elements that are NaN behind them; a view of x's shape."""
    out = torch.full((x.shape[0], ld), float("nan"), dtype=x.dtype, device="cuda")
    out[:, :x.shape[1]] = x.cuda()
    return out


def inputs(T, K, xt, dt, wt, seed):
    g = torch.Generator().manual_seed(seed)
    x = (2 * torch.randn(T, K, generator=g)).to(xt)
    x[:, ::37] *= 9
    d = None if dt is None else torch.randn(T, K, generator=g).to(dt)
    w = None if wt is None else (1 + 0.3 * torch.randn(K, generator=g)).to(wt)
    return x, d, w


def reference(x, d, w, offset, eps):
    r = x.double() if d is None else x.double() + d.double()
    y = r / (r.square().mean(-1, keepdim=True) + eps).sqrt()
    return y * ((1.0 if w is None else w.double()) + offset)


def check_h(h, y):
    assert ((h.cpu().double() - y).abs() <= (2.0 ** -11 + 2.0 ** -18) * y.abs() + 2.0 ** -25).all()


def check_q8(aq, y, T, K):
    q, d, s = (v.cpu() for v in q8_views(aq, T, K))
    b = y.view(T, K // 32, 32)
    assert ((d.double() - b.abs().amax(-1) / 127).abs() <= 2.0 ** -17 * d.double() + 2.0 ** -149).all()
    err = (q.double() * d.double()[..., None] - b).abs()
    assert (err <= (0.5 + 2.0 ** -10) * d.double()[..., None] + 2.0 ** -149).all()
    assert torch.equal(s, q.sum(-1, dtype=torch.int32))


@pytest.mark.parametrize("K", [1, 7, 8, 31, 32, 100, 256, 520, 5120, 8192, 8200, 8224, 20000, 32768])
@pytest.mark.parametrize("xt,dt,wt", [(F32, F16, F32), (F16, F16, F16), (F32, F32, None), (F16, None, F32)])
def test_norm(K, xt, dt, wt):
    T = 3
    x, d, w = inputs(T, K, xt, dt, wt, K)
    y = reference(x, d, w, 0.0, 1e-6)
    h, r = torch.full((T, K), 7.0, dtype=F16, device="cuda"), torch.empty(T, K, dtype=xt, device="cuda")
    aq = torch.full((bf.q8_bytes(T, K) + 64,), 0x55, dtype=torch.uint8, device="cuda") if K % 32 == 0 else None
    bf.rms_norm(x.cuda(), T, K, delta=None if d is None else d.cuda(), R=r, weight=None if w is None else w.cuda(), H=h, Aq=aq)
    assert torch.equal(r.cpu(), x if d is None else (x.float() + d.float()).to(xt))
    check_h(h, y)
    if aq is not None:
        check_q8(aq, y, T, K)
        assert (aq[bf.q8_bytes(T, K):] == 0x55).all()
        only = torch.empty_like(aq)                                # codes alone: the same bits
        bf.rms_norm(x.cuda(), T, K, delta=None if d is None else d.cuda(), weight=None if w is None else w.cuda(), Aq=only)
        assert torch.equal(only[:bf.q8_bytes(T, K)], aq[:bf.q8_bytes(T, K)])


@pytest.mark.parametrize("K,pad,off", [(256, 8, 0), (256, 3, 0), (320, 0, 1), (96, 5, 2), (1056, 24, 4)])
@pytest.mark.parametrize("T", [1, 70])
def test_strides_and_alignments(K, pad, off, T):
    """Rows longer than K, rows and starts off 16 bytes, in place; what lies between rows stays."""
    x, d, w = inputs(T, K, F32, F16, F32, K + pad)
    y = reference(x, d, w, 1.0, 1e-5)
    ld = K + pad
    base = torch.full((T * ld + 8,), float("nan"), device="cuda")
    xs = base[off:off + T * ld].view(T, ld)
    xs[:, :K] = x.cuda()
    ds = padded(d, ld)
    h = torch.full((T, ld), 7.0, dtype=F16, device="cuda")
    aq = torch.empty(bf.q8_bytes(T, K), dtype=torch.uint8, device="cuda")
    bf.rms_norm(xs, T, K, delta=ds, R=xs, weight=w.cuda(), offset=1.0, eps=1e-5, H=h, Aq=aq, ldx=ld, ldd=ld, ldr=ld, ldh=ld)
    check_h(h[:, :K], y)
    check_q8(aq, y, T, K)
    assert torch.equal(xs[:, :K].cpu(), x + d.float())
    assert (h[:, K:] == 7.0).all() and xs[:, K:].isnan().all()
    # the fp16 rows over delta
    xs[:, :K] = x.cuda()
    bf.rms_norm(xs, T, K, delta=ds, weight=w.cuda(), offset=1.0, eps=1e-5, H=ds, ldx=ld, ldd=ld, ldh=ld)
    assert torch.equal(ds[:, :K], h[:, :K]) and torch.equal(xs[:, :K].cpu(), x)


def test_many_rows():
    x, d, w = inputs(1500, 640, F16, F16, F16, 5)
    h = torch.empty(1500, 640, dtype=F16, device="cuda")
    bf.rms_norm(x.cuda(), 1500, 640, delta=d.cuda(), weight=w.cuda(), H=h)
    check_h(h, reference(x, d, w, 0.0, 1e-6))


@pytest.mark.parametrize("K", [64, 100])
@pytest.mark.parametrize("size,eps", [(1e30, 1e-6), (3e38, 1e-6), (1e-30, 0.0), (1e-41, 0.0), (1e-30, 1e-6), (1e-12, 1e-20)])
def test_rows_beyond_the_squares_range(K, size, eps):
    """Rows whose squares leave fp32's range, beside an ordinary one."""
    g = torch.Generator().manual_seed(3)
    x = (torch.rand(3, K, generator=g) + 0.5) * torch.sign(torch.randn(3, K, generator=g))
    x[0] *= size / 1.5
    x[2] *= size / 1.5
    h = torch.empty(3, K, dtype=F16, device="cuda")
    bf.rms_norm(x.cuda(), 3, K, eps=eps, H=h)
    check_h(h, reference(x, None, None, 0.0, eps))


@pytest.mark.parametrize("K", [64, 96 + 2])
def test_zero_rows_infinities_nan(K):
    """Zero rows give zeros (eps > 0); an infinity or NaN makes its own row NaN there, and no other row."""
    x = torch.randn(5, K, generator=torch.Generator().manual_seed(1))
    x[0] = 0
    x[2, 3] = float("inf")
    x[3, 40] = float("nan")
    h = torch.empty(5, K, dtype=F16, device="cuda")
    aq = torch.empty(bf.q8_bytes(5, 64) if K == 64 else 16, dtype=torch.uint8, device="cuda")
    bf.rms_norm(x.cuda(), 5, K, H=h, Aq=aq if K == 64 else None)
    assert (h[0] == 0).all() and h[2, 3].isnan() and (h[2, 4:] == 0).all() and h[3].isnan().all()
    check_h(h[[1, 4]], reference(x[[1, 4]], None, None, 0.0, 1e-6))
    if K == 64:
        q, d, s = (v.cpu() for v in q8_views(aq, 5, 64))
        assert (q[0] == 0).all() and (d[0] == 0).all() and (s[0] == 0).all()
        assert d[2, 0].isnan() and d[2, 1] == 0 and d[3].isnan().all() and (q[2:4] == 0).all() and (s[2:4] == 0).all()
        assert torch.isfinite(d[[1, 4]]).all()


def test_codes_feed_the_integer_gemm():
    """bf_gemm_q8 takes the codes: within half a step of each of what the GEMM gives of the fp16 rows."""
    import oracle as O
    T, K, N = 5, 512, 96
    x, d, w = inputs(T, K, F32, F16, F32, 9)
    W = O.gen_weights(O.Q4_K, N, K, seed=3)
    Wd = torch.from_numpy(W.W).cuda()
    aq = torch.empty(bf.q8_bytes(T, K), dtype=torch.uint8, device="cuda")
    C = torch.empty(T, N, device="cuda")
    bf.rms_norm(x.cuda(), T, K, delta=d.cuda(), weight=w.cuda(), Aq=aq)
    bf.gemm_q8(O.Q4_K, Wd, None, aq, C, T, N, K)
    y = reference(x, d, w, 0.0, 1e-6)
    wf = torch.from_numpy(O.dequant_f32(W).reshape(N, K)).double()
    step = (y.view(T, -1, 32).abs().amax(-1, keepdim=True) / 127).expand(T, K // 32, 32).reshape(T, K)
    tol = (0.5 + 2.0 ** -10) * (step @ wf.abs().t()) + 2.0 ** -16 * (y.abs() @ wf.abs().t())
    assert ((C.cpu().double() - y @ wf.t()).abs() <= tol).all()


def test_other_stream_and_graph():
    T, K = 9, 2048
    x, d, w = (t.cuda() for t in inputs(T, K, F32, F16, F32, 4))
    a, b = (torch.empty(T, K, dtype=F16, device="cuda") for _ in range(2))
    r = torch.empty_like(x)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    bf.rms_norm(x, T, K, delta=d, R=r, weight=w, H=a, stream=st)
    st.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        bf.rms_norm(x, T, K, delta=d, R=r, weight=w, H=a)
    for i in range(3):
        x.mul_(1.5)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        bf.rms_norm(x, T, K, delta=d, weight=w, H=b)
        assert torch.equal(a, b) and torch.equal(r, x + d.float())
