"""The residual norm's long rows that are not of whole 16-byte pieces (run on an MI355X), up
to 128 KB of LDS a row.

Tolerance: a thread adds 32 squares, at most four such sums, then 6 + 4 across lanes and
waves: the sum within 46 2^-24, the root half of that, then a division, a root, a
reciprocal and two products, 2^-24 each: y within 28 2^-24; dd = amax / 127 within 29."""
import pytest
import torch

import busfill as bf
from test_gpu_norm import F16, F32, check_h, check_q8, inputs, padded, q8_views, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("K", [8191, 8193, 16387, 20001, 32767])
@pytest.mark.parametrize("xt,dt,wt", [(F32, F16, F32), (F16, None, None)])
def test_odd_lengths(K, xt, dt, wt):
    x, d, w = inputs(3, K, xt, dt, wt, K)
    h, r = torch.empty(3, K, dtype=F16, device="cuda"), torch.empty(3, K, dtype=xt, device="cuda")
    on = lambda v: None if v is None else v.cuda()  # noqa: E731
    bf.rms_norm(on(x), 3, K, delta=on(d), R=r, weight=on(w), H=h)
    torch.cuda.synchronize()
    assert torch.equal(r.cpu(), x if d is None else (x.float() + d.float()).to(xt))
    check_h(h, reference(x, d, w, 0.0, 1e-6))


@pytest.mark.parametrize("K", [8224, 20000, 32768])
def test_odd_strides_with_codes(K):
    x, d, w = inputs(2, K, F32, F16, F32, K)
    y = reference(x, d, w, 1.0, 1e-5)
    h = torch.empty(2, K, dtype=F16, device="cuda")
    aq = torch.empty(bf.q8_bytes(2, K), dtype=torch.uint8, device="cuda")
    bf.rms_norm(padded(x, K + 3), 2, K, delta=padded(d, K + 1), weight=w.cuda(), offset=1.0, eps=1e-5, H=h, Aq=aq, ldx=K + 3,
                ldd=K + 1)
    torch.cuda.synchronize()
    check_h(h, y)
    check_q8(aq, y, 2, K)


@pytest.mark.parametrize("K,ld", [(32768, 32769), (32768, 32768)])
def test_sums_that_round_one_way(K, ld):
    """Rows of one value whose partial sums all round the same way: the scales show y's 32 bits."""
    for value in (1.3862042, 1.0001, 1.9173, 0.7):
        x = torch.full((1, K), value)
        aq = torch.empty(bf.q8_bytes(1, K), dtype=torch.uint8, device="cuda")
        bf.rms_norm(padded(x, ld), 1, K, eps=0.0, Aq=aq, ldx=ld)
        torch.cuda.synchronize()
        q, d, _ = q8_views(aq, 1, K)
        assert (q == 127).all() and ((d.cpu().double() * 127 - 1).abs() <= 29 * 2.0 ** -24).all()


@pytest.mark.parametrize("K", [20001, 32767])
@pytest.mark.parametrize("size,eps", [(3e38, 1e-6), (1e-30, 0.0)])
def test_squares_out_of_range(K, size, eps):
    x = (torch.rand(2, K, generator=torch.Generator().manual_seed(3)) + 0.5) * (size / 1.5)
    h = torch.empty(2, K, dtype=F16, device="cuda")
    bf.rms_norm(x.cuda(), 2, K, eps=eps, H=h)
    torch.cuda.synchronize()
    check_h(h, reference(x, None, None, 0.0, eps))
