"""The residual norm's int8 codes where two codes are equally near, bit for bit what
bf_quantize_q8 gives (run on an MI355X): code = round(y / dd), dd = amax / 127, the
quotient rounded to fp32, half away from zero.

Rows of ones with eps = 0: the mean of the squares, its root and its reciprocal are
exactly 1, so y is the weight itself."""
import numpy as np
import pytest
import torch

import busfill as bf

pytestmark = pytest.mark.gpu

f32 = np.float32


def codes(y):
    """(codes, scales) of fp32 y [blocks][32]."""
    dd = (np.abs(y).max(-1, keepdims=True) / f32(127)).astype(f32)
    q = (y / dd).astype(f32).astype(np.float64)
    return np.sign(q) * np.floor(np.abs(q) + 0.5), dd[:, 0]


def half_blocks():
    """fp16 blocks of one largest value and values whose quotient is next to half way between two codes."""
    values = np.arange(0x1000, 0x3FFF, dtype=np.uint16).view(np.float16)
    blocks = []
    for m in range(1024, 2048):
        amax = f32(m / 1024)
        dd = f32(amax / f32(127))
        y = values[values.astype(f32) < amax]
        q = y.astype(np.float64) / np.float64(dd)
        near = y[np.abs(q - np.floor(q) - 0.5) < 2.0 ** -16][:31]
        if len(near):
            blocks.append(np.concatenate([[np.float16(amax)], near, np.zeros(31 - len(near), np.float16)]))
    y = np.stack(blocks)
    y[1::2] *= -1
    return y


def norm_codes(w, T, K, ld):
    x = torch.ones(T, ld, device="cuda")
    h = torch.empty(T, K, dtype=torch.float16, device="cuda")
    aq = torch.empty(bf.q8_bytes(T, K), dtype=torch.uint8, device="cuda")
    bf.rms_norm(x, T, K, weight=w.cuda(), eps=0.0, H=h, Aq=aq, ldx=ld)
    torch.cuda.synchronize()
    return h, aq


@pytest.mark.parametrize("pad", [0, 1])
def test_fp16_values_as_quantize_q8(pad):
    """(rows of 16-byte pieces, and rows that are not)"""
    y = half_blocks()
    per = 200                                                              # blocks a row
    for at in range(0, len(y), per):
        w = torch.from_numpy(y[at:at + per].reshape(-1).copy())
        K = w.numel()
        h, aq = norm_codes(w, 2, K, K + pad)
        assert torch.equal(h.cpu(), w.repeat(2, 1))
        want = torch.empty_like(aq)
        bf.quantize_q8(h, want, 2, K)
        torch.cuda.synchronize()
        assert torch.equal(aq, want)


@pytest.mark.parametrize("pad", [0, 1])
def test_fp32_values_next_to_half_way(pad):
    rng = np.random.default_rng(5)
    y = np.zeros((1000, 32), f32)
    for b in range(1000):
        amax = f32(rng.uniform(1, 2) * 2.0 ** rng.integers(-20, 20))
        half = ((rng.integers(0, 127, 31) + 0.5) * np.float64(f32(amax / f32(127)))).astype(f32)
        y[b, 0], y[b, 1:] = amax, np.nextafter(half, half * f32(rng.choice([0.5, 1, 2])))
    y *= rng.choice([-1, 1], y.shape).astype(f32)
    q, dd = codes(y)
    K = y.size
    _, aq = norm_codes(torch.from_numpy(y.reshape(-1)), 1, K, K + pad)
    aq = aq.cpu().numpy()
    got = aq[:K].view(np.int8).reshape(q.shape)
    assert (got == q).all(), int((got != q).sum())
    assert (aq[K:K + K // 8].view(f32) == dd).all()
    assert (aq[K + K // 8:K + K // 4].view(np.int32) == q.sum(-1)).all()
