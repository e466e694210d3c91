"""The example's mixture-of-experts decoder layer, every step of it against 64
bits from the step's own inputs, and its captured decode step against a prompt
(run on an MI355X)."""
import os
import sys

import numpy as np
import pytest
import torch

import kv4_ref as R
import oracle as O

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
import moe_decoder as M  # noqa: E402

pytestmark = pytest.mark.gpu


def small():
    return M.Shape(width=512, q_heads=8, kv_heads=2, dim=64, experts=16, chosen=3, ffn=256)


def dequant(w, n, k):
    return torch.from_numpy(O.dequant_f32(O.QWeights(O.Q4_K, n, k, w.cpu().numpy().reshape(-1))).astype(np.float64).reshape(n, k))


def test_layer_from_step_to_step():
    s, streams, n = small(), 3, 45
    layer = M.Layer(s, seed=4)
    cache = M.Cache(s, streams, n)
    x = torch.randn(streams, n, s.width, device="cuda")
    b = M.prompt(layer, cache, streams, x)
    torch.cuda.synchronize()
    rows = streams * n
    # attention over what the cache holds of the rotated rows
    heads = b.qkv.cpu().view(streams, n, -1, s.dim)
    see = torch.ones(n, n, dtype=torch.bool).tril()
    att = b.att.cpu().double().view(streams, n, s.q_heads, s.dim)
    for st in range(streams):
        k, v = R.quantize(heads[st, :, 8:10]), R.quantize(heads[st, :, 10:])
        for h in range(s.q_heads):
            want, mass, _ = R.attention(heads[st, :, h], k[:, h // 4], v[:, h // 4], s.dim ** -0.5, see)
            tol = (2.0 ** -11 + 2.0 ** -13) * mass + 2.0 ** -11 * want.abs() + 2.0 ** -24
            assert ((att[st, :, h] - want).abs() <= tol).all()
    # the routing of the layer's own logits
    lg = b.logits.cpu().double()
    h2, wr = b.h2.cpu().double(), dequant(layer.wr, s.experts, s.width)
    assert ((lg - h2 @ wr.t()).abs() <= (2.0 ** -11 + 2.0 ** -18) * (h2.abs() @ wr.abs().t())).all()
    w, ids = torch.softmax(lg, -1).sort(dim=-1, descending=True, stable=True)
    w, ids = w[:, :3] / w[:, :3].sum(-1, keepdim=True), ids[:, :3]
    assert torch.equal(b.ids.cpu().long(), ids) and ((b.weights.cpu() - w).abs() <= 1e-6).all()
    # the experts' block of the layer's own choice; its terms' rounding as one fp16 rounding of each intermediate
    e, f = s.experts, s.ffn
    wg, wu = (dequant(m, e * f, s.width).view(e, f, -1) for m in (layer.gate, layer.up))
    wd = dequant(layer.down, e * s.width, f).view(e, s.width, f)
    want, tol = torch.zeros(rows, s.width).double(), torch.zeros(rows, s.width).double()
    for j in range(3):
        for t in range(rows):
            i = int(ids[t, j])
            g, u = wg[i] @ h2[t], wu[i] @ h2[t]
            dg, du = (2.0 ** -18 * (m[i].abs() @ h2[t].abs()) for m in (wg, wu))
            silu, wt = g * torch.sigmoid(g), float(b.weights[t, j])
            h = wt * silu * u
            dh = wt * (1.1 * dg * (u.abs() + du) + silu.abs() * du) + (2.0 ** -11 + 2.0 ** -20) * h.abs() + 2.0 ** -25
            want[t] += wd[i] @ h
            # an expert's sum is rounded as the output is, the outputs once more
            tol[t] += wd[i].abs() @ (dh + 2.0 ** -18 * h.abs()) + 2.0 ** -11 * (wd[i] @ h).abs() + 2.0 ** -24
    tol = tol * (1 + 2.0 ** -10) + 2.0 ** -11 * want.abs()
    assert ((b.y.cpu().double() - want).abs() <= tol).all()


def test_decode_graph_continues_a_prompt():
    """Seven tokens decoded one by one by the captured step give the rows that the whole prompt gives, wherever both
    choose the same experts: fp16 rows in between, so within a few of their roundings."""
    s, streams, n, more = small(), 3, 61, 7
    layer = M.Layer(s, seed=5)
    x = torch.randn(streams, n + more, s.width, device="cuda")
    whole = M.prompt(layer, M.Cache(s, streams, n + more), streams, x)
    cache = M.Cache(s, streams, n + more + 1)
    M.prompt(layer, cache, streams, x[:, :n])
    d = M.Decoder(layer, cache, streams, n)
    want, ids = whole.x.view(streams, n + more, -1), whole.ids.view(streams, n + more, -1)
    same = 0
    for i in range(more):
        got = d.step(x[:, n + i]).clone()
        torch.cuda.synchronize()
        for st in range(streams):
            if not torch.equal(d.b.ids[st].sort().values, ids[st, n + i].sort().values):
                continue
            same += 1
            a, w = got[st].double(), want[st, n + i].double()
            assert float((a - w).norm()) <= 4e-3 * float(w.norm())
    assert same >= streams * more - 3
