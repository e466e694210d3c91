"""Rotation by position with the 4-bit cache's store against 64 bits (run on an
MI355X).

Tolerance of a rotated element of the pair (a, b): the angle's fraction of a turn
is rounded to fp32 (2^-25 of a turn, 2^-22 radians), sine and cosine are within
2^-22, their products with a and b and the sum within 2^-23 of |a| + |b|: 2^-20
(|a| + |b|) |factor| in all, then the rounding to fp16 (2^-11, 2^-25 where
subnormal).  What the cache holds is, bit for bit, what bf_kv4_store makes of the
rotated fp16 keys.
"""
import pytest
import torch

import busfill as bf

pytestmark = pytest.mark.gpu


def frequencies(rot, theta=10000.0):
    return theta ** (-torch.arange(0, rot, 2).double() / rot)


def rotated(x, position, freq, rot, style, factor):
    """x [T][heads][D] in 64 bits, and the pairs' sizes."""
    t = position.double()[:, None, None] * freq.double()
    c, s = torch.cos(t) * factor, torch.sin(t) * factor
    x = x.double()
    r = x[..., :rot]
    a, b = (r[..., :rot // 2], r[..., rot // 2:]) if style == bf.ROPE_HALVES else (r[..., 0::2], r[..., 1::2])
    p, q, size = a * c - b * s, b * c + a * s, (a.abs() + b.abs()) * abs(factor)
    join = (lambda u, v: torch.cat([u, v], -1)) if style == bf.ROPE_HALVES else (lambda u, v: torch.stack([u, v], -1).flatten(-2))
    return torch.cat([join(p, q), x[..., rot:]], -1), torch.cat([join(size, size), torch.zeros_like(x[..., rot:])], -1)


def near(got, want):
    y, size = want
    return ((got.cpu().double() - y).abs() <= 2.0 ** -20 * size + 2.0 ** -11 * y.abs() + 2.0 ** -25).all()


def run(T, hq, h, d, rot, style, *, factor=1.0, start=0, step=1, page=64, place="out", pad=0, seed=0, skip=(), freq=None,
        position=None, stream=None):
    g = torch.Generator().manual_seed(seed + T)
    q, k, v = (torch.randn(T, n, d, generator=g).half() for n in (hq, h, h))
    k[..., 5::41] *= 4
    position = torch.arange(T) * step + start if position is None else position
    freq = frequencies(rot).float() if freq is None else freq
    pages = T // page + 2
    slots = torch.randperm(pages * page, generator=g)[:T]
    for i, s in skip:
        slots[i] = s
    wide = torch.full((T, (hq + 2 * h) * d + pad), 9.0, dtype=torch.float16)
    wide[:, :hq * d], wide[:, hq * d:(hq + h) * d] = q.reshape(T, -1), k.reshape(T, -1)
    wide[:, (hq + h) * d:(hq + 2 * h) * d] = v.reshape(T, -1)
    wide, ld = wide.cuda(), wide.shape[1]
    caches = []
    for _ in range(2):
        data = torch.full((bf.kv4_bytes(pages, page, h, d),), 0xFF, dtype=torch.uint8, device="cuda")
        caches.append((data, bf.kv4_cache(data, pages, page, h, d)))
    qo, ko = (torch.full((T, n * d), 9.0, dtype=torch.float16, device="cuda") for n in (hq, h))
    kw = dict(rot=rot, style=style, factor=factor, ldk=ld, ldv=ld, stream=stream)
    slots, pos, fr = slots.cuda(), position.cuda(), freq.cuda()
    torch.cuda.synchronize()
    qin, kin, vin = wide, wide[:, hq * d:], wide[:, (hq + h) * d:]
    if place == "in":                                              # over the rows themselves
        bf.kv4_append(caches[0][1], kin, vin, slots, pos, fr, T, Q=qin, Q_out=qin, q_heads=hq, K_out=kin, ldq=ld, ldqo=ld, ldko=ld, **kw)
        torch.cuda.synchronize()
        qo, ko = wide[:, :hq * d].contiguous(), wide[:, hq * d:(hq + h) * d].contiguous()
        assert torch.equal(wide[:, (hq + h) * d:(hq + 2 * h) * d].cpu(), v.reshape(T, -1))
    elif place == "out":
        bf.kv4_append(caches[0][1], kin, vin, slots, pos, fr, T, Q=qin, Q_out=qo, q_heads=hq, K_out=ko, ldq=ld, **kw)
    else:                                                          # keys and values alone
        bf.kv4_append(caches[0][1], kin, vin, slots, pos, fr, T, **kw)
        torch.cuda.synchronize()
        bf.kv4_append(caches[1][1], kin, vin, slots, pos, fr, T, K_out=ko, **kw)
        torch.cuda.synchronize()
        caches[1][0].fill_(0xFF)
    torch.cuda.synchronize()
    if place != "none":
        assert near(qo.view(T, hq, d), rotated(q, position, freq, rot, style, factor))
    assert near(ko.view(T, h, d), rotated(k, position, freq, rot, style, factor))
    assert (wide[:, (hq + 2 * h) * d:] == 9.0).all()
    bf.kv4_store(caches[1][1], ko, v.reshape(T, -1).cuda(), slots, T)
    assert torch.equal(caches[0][0], caches[1][0])
    return caches[0][0], qo


@pytest.mark.parametrize("d,rot", [(64, 64), (64, 32), (64, 16), (96, 96), (96, 48), (128, 128), (128, 64), (256, 256), (256, 112)])
@pytest.mark.parametrize("style", [bf.ROPE_HALVES, bf.ROPE_PAIRS])
@pytest.mark.parametrize("T,hq,h", [(1, 1, 1), (5, 6, 3), (70, 40, 8)])
def test_append(d, rot, style, T, hq, h):
    run(T, hq, h, d, rot, style, place="out", start=3)


@pytest.mark.parametrize("place", ["in", "none"])
@pytest.mark.parametrize("style", [bf.ROPE_HALVES, bf.ROPE_PAIRS])
@pytest.mark.parametrize("d,page", [(64, 32), (96, 256), (128, 64), (256, 96)])
def test_in_place_and_keys_alone(place, style, d, page):
    run(33, 10, 2, d, d, style, place=place, pad=16, page=page)


@pytest.mark.parametrize("start,step", [(0, 0), (131000, 7), (-5000, 31), (2 ** 31 - 40, 1), (-2 ** 31, 1), (10 ** 6, 977)])
def test_far_positions(start, step):
    """Positions up to 2^31 either way: the reference's own products round at 2^-22 radians there (64 bits of 2^31 2^-52
    and 24-bit frequencies are exact), within the tolerance."""
    run(30, 4, 2, 128, 128, bf.ROPE_HALVES, start=start, step=step)


def test_many_tokens():
    run(1300, 5, 1, 128, 128, bf.ROPE_HALVES, start=100)
    run(700, 16, 4, 64, 32, bf.ROPE_PAIRS, start=9)


@pytest.mark.parametrize("factor", [0.0, -1.0, 1.3689])
def test_factors(factor):
    run(6, 4, 2, 64, 64, bf.ROPE_HALVES, factor=factor)


def test_frequencies_of_any_kind():
    """A table with zeros, negative and large values."""
    f = torch.tensor([0.0, -0.5, 3.0, 100.0, 1e-6, 2.0, 7.5, 1e4] * 4)
    run(12, 4, 2, 64, 64, bf.ROPE_HALVES, freq=f, start=50)


def test_skipped_slots_are_rotated_all_the_same():
    run(20, 4, 2, 128, 128, bf.ROPE_HALVES, skip=((0, -1), (7, 1 << 40), (19, -2 ** 62)))


def test_corner_values():
    """Keys and values of zeros, subnormals, equal magnitudes, the largest, infinities and NaN at position 0 (which leaves
    them as they are): the cache as kv4_store leaves it."""
    x = torch.zeros(12, 1, 64, dtype=torch.float16)
    x[1, 0, :32] = 2.0 ** -24 * torch.arange(32)
    x[2, 0, 3], x[2, 0, 9] = 4.0, -4.0
    x[3, 0, 3], x[3, 0, 9] = -4.0, 4.0
    x[4, 0, :32] = torch.arange(32) * 0.25 - 4.0
    x[5, 0] = torch.linspace(-65504, 65504, 64)
    x[6, 0, 40] = float("inf")
    x[7, 0, 2] = float("nan")
    x[8, 0] = -0.0
    x[9, 0, :4] = torch.tensor([3.0, 3.0, -3.0, 1.5])
    x[10, 0, 31], x[10, 0, 30] = -2.0, 2.0
    x[11, 0, 8], x[11, 0, 7] = 2.0, -2.0
    data = [torch.zeros(bf.kv4_bytes(1, 32, 1, 64), dtype=torch.uint8, device="cuda") for _ in range(2)]
    a, b = (bf.kv4_cache(d, 1, 32, 1, 64) for d in data)
    ko, zero = torch.empty_like(x).cuda(), torch.zeros(12, dtype=torch.int64, device="cuda")
    slots = torch.arange(12).cuda() + 9
    bf.kv4_append(a, x.cuda(), x.flip(0).cuda(), slots, zero, frequencies(64).float().cuda(), 12, K_out=ko)
    bf.kv4_store(b, ko, x.flip(0).cuda(), slots, 12)
    assert torch.equal(data[0], data[1])
    keep = torch.ones(64, dtype=torch.bool)
    keep[[40, 8, 2, 34]] = False                                   # (inf 0 and NaN reach the pair's other half)
    assert torch.equal(ko.cpu()[..., keep], x[..., keep])
    k2, v2 = torch.empty_like(ko), torch.empty_like(ko)
    bf.kv4_load(a, slots, k2, v2, 12)
    assert k2[6, 0, 32:].isnan().all() and k2[7, 0, :32].isnan().all()


def test_other_stream_and_same_bits():
    st = torch.cuda.Stream()
    a = run(40, 8, 2, 128, 128, bf.ROPE_HALVES, stream=st)
    b = run(40, 8, 2, 128, 128, bf.ROPE_HALVES)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_graph_of_a_growing_sequence():
    """A captured append whose position and slot live in device memory."""
    d, h, hq = 128, 2, 8
    data = [torch.zeros(bf.kv4_bytes(2, 64, h, d), dtype=torch.uint8, device="cuda") for _ in range(2)]
    a, b = (bf.kv4_cache(x, 2, 64, h, d) for x in data)
    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(1, n * d, generator=g).half().cuda() for n in (hq, h, h))
    qo, qo2 = torch.empty_like(q), torch.empty_like(q)
    pos, slot, f = torch.zeros(1, dtype=torch.int64).cuda(), torch.zeros(1, dtype=torch.int64).cuda(), frequencies(d).float().cuda()
    step = lambda c, out: bf.kv4_append(c, k, v, slot, pos, f, 1, Q=q, Q_out=out, q_heads=hq)  # noqa: E731
    st = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=st):
        step(a, qo)
    for i in range(5):
        pos.fill_(1000 + i)
        slot.fill_(60 + i)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        step(b, qo2)
        assert torch.equal(qo, qo2) and torch.equal(data[0], data[1])


def test_cache_of_more_than_4_gb():
    pages = 8000
    data = torch.empty(bf.kv4_bytes(pages, 256, 8, 256), dtype=torch.uint8, device="cuda")
    assert data.numel() > 1 << 32
    c = bf.kv4_cache(data, pages, 256, 8, 256)
    g = torch.Generator().manual_seed(2)
    k, v = (torch.randn(4, 8, 256, generator=g).half().cuda() for _ in range(2))
    slots = torch.tensor([0, pages * 256 - 1, (pages - 3) * 256 + 77, 5 * 256 + 31]).cuda()
    ko, k2, v2, k3, v3 = (torch.empty_like(k) for _ in range(5))
    bf.kv4_append(c, k, v, slots, torch.arange(4).cuda() + 70000, frequencies(256).float().cuda(), 4, K_out=ko)
    bf.kv4_load(c, slots, k2, v2, 4)
    bf.kv4_store(c, ko, v, slots, 4)
    bf.kv4_load(c, slots, k3, v3, 4)
    assert torch.equal(k2, k3) and torch.equal(v2, v3) and (k2 != 0).any()
