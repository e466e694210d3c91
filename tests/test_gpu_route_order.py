"""Routing with logits and biases that are NaN, infinite or the type's lowest
value, against the definition row by row in 64 bits (run on an MI355X).

Order: a NaN is the least of all, then -inf, then the finite values; equal ones
by index.  An expert whose logit is NaN has score NaN and takes no part in the
others' softmax; logits of +inf share the softmax among them.  Weights are fp32
exponentials and one division: 1e-5 of themselves, as in test_gpu_moe.py.
"""
import numpy as np
import pytest
import torch

import busfill as bf
from test_gpu_moe import route

pytestmark = pytest.mark.gpu

NAN, INF, LOW = float("nan"), float("inf"), -3.4028234663852886e38
E = 16


def falling(v):
    """Indices by falling value, NaN last, equal ones by index."""
    nan = np.isnan(v)
    return np.lexsort((np.arange(len(v)), -np.where(nan, 0.0, v), nan))


def scores(x, sigmoid):
    nan, s = np.isnan(x), np.empty(len(x))
    if sigmoid:
        with np.errstate(over="ignore"):
            return 1 / (1 + np.exp(-x))
    m = np.max(x[~nan]) if (~nan).any() else -np.inf
    s[:] = 0.0 if m == -np.inf else (x == m) if m == np.inf else np.exp(np.where(nan, m, x) - m)
    total = s[~nan].sum()
    return np.where(nan, np.nan, s / total if total else s)


def ref(x, bias, k, sigmoid, groups, top, renorm):
    s = scores(x, sigmoid)
    v = s if bias is None else s + bias
    order = x.copy() if bias is None else v.copy()
    out = np.zeros(len(x), bool)
    if groups > 1:
        g = np.where(np.isnan(v), -np.inf, v).reshape(groups, -1)
        two = -np.sort(-g, 1)[:, :2]
        best = two.sum(1) if g.shape[1] > 1 else two[:, 0]
        keep = falling(best)[:top]
        out[:] = ~np.isin(np.arange(len(x)) // g.shape[1], keep)
    ids = [i for i in falling(order) if not out[i]][:k]
    w = s[ids]
    if renorm:
        w = w / w.sum() if w.sum() != 0 else w * 0
    return np.array(ids), w


def decided(x, bias, sigmoid, groups, top):
    """The choice of groups does not hang on fp32 rounding (sums less than 1e-6 apart)."""
    if groups == 1 or top == groups or bias is None:
        return True
    v = scores(x, sigmoid) + bias
    two = -np.sort(-np.where(np.isnan(v), -np.inf, v).reshape(groups, -1), 1)[:, :2]
    best = np.sort(two.sum(1))[::-1]
    a, b = best[top - 1], best[top]
    return not np.isfinite(a) or not np.isfinite(b) or a - b > 1e-6


def rows():
    g = np.random.default_rng(11)
    base = g.permutation(E) * 0.37 - 2.0           # well apart: nothing hangs on rounding
    out = []

    def add(**at):
        r = base.copy()
        for i, val in at.items():
            r[int(i[1:])] = val
        out.append(r)

    add(_3=NAN)
    add(_0=NAN, _15=NAN)
    add(_0=NAN, _1=NAN, _2=NAN, _3=NAN)            # a whole group of four
    add(_4=NAN, _5=NAN, _6=NAN, _8=NAN, _9=NAN, _10=NAN)
    add(_2=NAN, _7=-INF)                           # the NaN stands before, and must come after
    add(_2=-INF, _7=LOW, _9=-INF, _11=NAN)
    add(_2=LOW, _5=LOW, _6=-INF)
    add(_6=INF)
    add(_6=INF, _9=INF, _1=NAN)
    add(_3=0.0, _5=-0.0, _8=0.0)
    out.append(np.full(E, NAN))
    out.append(np.full(E, -INF))
    out.append(np.where(np.arange(E) % 2, NAN, -INF))
    out.append(np.where(np.arange(E) % 3, NAN, base))
    out.append(np.where(np.arange(E) % 3, -INF, LOW))
    return np.stack(out)


@pytest.mark.parametrize("groups,top,k", [(1, 1, 4), (1, 1, E), (4, 2, 5), (4, 4, 9), (8, 3, 6), (2, 1, 8)])
@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("bias", [None, "some", "odd"])
@pytest.mark.parametrize("renorm", [True, False])
def test_order(groups, top, k, sigmoid, bias, renorm):
    x = rows().astype(np.float32).astype(np.float64)
    b = None
    if bias is not None:
        b = np.linspace(3.0, 0.0, E)[np.random.default_rng(2).permutation(E)]
        if bias == "odd":
            b[4], b[9], b[12] = NAN, -INF, LOW
        b = b.astype(np.float32).astype(np.float64)
    ids, w = route(torch.from_numpy(x).float(), k, bias=None if b is None else torch.from_numpy(b).float(),
                   score=bf.SCORE_SIGMOID if sigmoid else bf.SCORE_SOFTMAX, groups=groups, top=top, renorm=renorm)
    sure = [t for t in range(len(x)) if decided(x[t], b, sigmoid, groups, top)]
    assert len(sure) >= len(x) - 2                 # (rows of no weight but the biases', twice)
    for t in sure:
        ri, rw = ref(x[t], b, k, sigmoid, groups, top, renorm)
        assert ids[t].tolist() == ri.tolist(), t
        got = w[t].numpy()
        assert (np.isnan(got) == np.isnan(rw)).all(), t
        ok = ~np.isnan(rw)
        assert (np.abs(got - rw)[ok] <= 1e-5 * rw[ok] + 1e-12).all(), t


@pytest.mark.parametrize("E_", [60, 129, 1000])
def test_order_of_many(E_):
    """Several experts a lane; fp16 logits, NaN and both infinities among them, groups that share lanes."""
    g = torch.Generator().manual_seed(E_)
    x = (torch.randperm(E_, generator=g).float() / 64 - 6).repeat(5, 1)
    for t in range(5):
        at = torch.randperm(E_, generator=g)
        x[t, at[:t]], x[t, at[t:2 * t]] = NAN, -INF
    x[4, 7] = INF
    x = x.half()
    for groups, top in ((1, 1), (E_ // 20, 2)) if E_ % 20 == 0 else ((1, 1), (3, 2) if E_ % 3 == 0 else (1, 1)):
        k = 20
        ids, w = route(x, k, groups=groups, top=top, renorm=False)
        for t in range(5):
            ri, rw = ref(x[t].double().numpy(), None, k, False, groups, top, False)
            assert ids[t].tolist() == ri.tolist(), (groups, t)
            assert (np.abs(w[t].numpy() - rw) <= 1e-5 * rw + 1e-12).all()
