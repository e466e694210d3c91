"""What the operators around the quantized linears cost: the 4-bit key/value
cache (its store and read-back), attention over it, routing to experts and the
experts' feed-forward blocks in the 4-bit weight formats.

Where ``own`` is false, ``run`` computes each operator in its plain form:
elementary torch operations in 32 bits, rounded once at the end.  Where it is
true, ``run`` makes the calls a program makes of the ``busfill`` package.
``exact`` computes the same outputs from the definitions in 64 bits.

Attention's and the experts' outputs are the fp16 rows that the next linear
takes.  Sizes are the repository's own (5120 wide, 7168 = 5120 + 2 * 1024 for a layer's
query, key and value projections, i.e. 40 query heads over 8 key/value heads of
128; batches of 1, 8, 32; 2000-token prompts) or generic ones.
"""
import math

import torch

own = False

DEV = "cuda"
PAGE = 64
GROUP = 32                                       # values that share a scale, in the cache and in Q4_0 weights
# multiply-adds and cache elements of the largest listed cases: no drawn one is larger
MOST_PAIRS = 2000 * 2001 // 2 * 40 * 128         # attention: (query, key) pairs x head elements
MOST_CACHED = 32 * 8192 * 8 * 128                # cached elements of one attention call
MOST_EXPERT = 2000 * 8 * 4096 * 1792             # experts: rows x weights of one projection
MOST_WEIGHTS = 64 * 4096 * 1792


def listed():
    return [
        # one decode step of 32 streams: each appends its token to a layer's cache (read back as a prefix copy does)
        {"name": "store_decode_32", "kind": "store", "T": 32, "H": 8, "D": 128, "start": 511, "whole": False},
        # a 2000-token prompt appended behind 37 cached tokens, so that it starts and ends inside the cache's tiles
        {"name": "store_prompt_2000", "kind": "store", "T": 2000, "H": 8, "D": 128, "start": 37, "whole": True},
        # one stream early in its answer: the smallest call, where latency counts
        {"name": "attn_decode_1x519", "kind": "attn", "S": 1, "nq": 1, "kv": 519, "spread": False, "Hq": 40, "H": 8,
         "D": 128, "window": 0},
        # 32 concurrent streams of ragged lengths up to 8000 tokens
        {"name": "attn_decode_32x8000", "kind": "attn", "S": 32, "nq": 1, "kv": 8000, "spread": True, "Hq": 40, "H": 8,
         "D": 128, "window": 0},
        # one stream with a long document
        {"name": "attn_decode_1x131072", "kind": "attn", "S": 1, "nq": 1, "kv": 131072, "spread": False, "Hq": 32,
         "H": 4, "D": 128, "window": 0},
        # four drafted tokens a stream checked at once, a model with heads of 64 and a sliding window
        {"name": "attn_draft_8x4_window", "kind": "attn", "S": 8, "nq": 4, "kv": 4099, "spread": True, "Hq": 16, "H": 8,
         "D": 64, "window": 1024},
        # a 2000-token prompt over the cache that holds it
        {"name": "attn_prompt_2000", "kind": "attn", "S": 1, "nq": 2000, "kv": 2000, "spread": False, "Hq": 40, "H": 8,
         "D": 128, "window": 0},
        # a decode step's routing: softmax scores, eight of 64
        {"name": "route_decode_32", "kind": "route", "T": 32, "E": 64, "k": 8, "score": "softmax", "biased": False,
         "groups": 1, "top": 1, "renorm": True, "factor": 1.0, "logits": "f32"},
        # a prompt chunk's routing: sigmoid scores with a balance bias, four of eight groups, eight of 256
        {"name": "route_prompt_4096", "kind": "route", "T": 4096, "E": 256, "k": 8, "score": "sigmoid", "biased": True,
         "groups": 8, "top": 4, "renorm": True, "factor": 2.5, "logits": "f32"},
        # the experts' block for one token
        {"name": "experts_m1", "kind": "experts", "fmt": "q4_k", "T": 1, "E": 64, "k": 8, "K": 2048, "F": 1024},
        # 32 streams, nearly every expert in use
        {"name": "experts_m32", "kind": "experts", "fmt": "q4_k", "T": 32, "E": 64, "k": 8, "K": 5120, "F": 1280},
        # a 2000-token prompt, about 250 rows an expert
        {"name": "experts_prompt_2000", "kind": "experts", "fmt": "q4_0", "T": 2000, "E": 64, "k": 8, "K": 4096,
         "F": 1792},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _not(n, avoid, step):
    return n + step if n == avoid else n


def draw(rng):
    kind = rng.choice(["store", "attn", "attn", "attn", "prompt", "prompt", "route", "route", "experts", "experts",
                       "experts", "experts"])
    d = rng.choice([64, 96, 128, 128, 256])
    h = rng.choice([1, 2, 4, 8])
    if kind == "store":
        whole = rng.random() < 0.5
        return {"kind": kind, "T": _log(rng, 1, 2000 if whole else 256), "H": h, "D": d, "start": rng.randint(0, 700),
                "whole": whole}
    if kind in ("attn", "prompt"):
        group = rng.choice([1, 2, 4, 5, 8, 16])
        window = rng.choice([0, 0, 0, rng.randint(16, 2048)])
        if kind == "prompt":
            h = min(h, max(1, 40 // group))
            nq = _log(rng, 17, min(2000, math.isqrt(2 * MOST_PAIRS // (group * h * d))))
            kv, s = nq + rng.choice([0, 0, rng.randint(1, 500)]), rng.choice([1, 1, 2, 3])
            while s * nq * (2 * kv - nq) * group * h * d > 2 * MOST_PAIRS:
                s, kv = max(1, s - 1), max(nq, kv // 2)
                if s == 1 and kv == nq:
                    break
        else:
            nq, s = rng.choice([1, 1, 1, 1, 2, 4, 7]), _log(rng, 1, 64)
            kv = _log(rng, max(nq, 16), min(131072, MOST_CACHED // (s * h * d)))
        return {"kind": "attn", "S": s, "nq": nq, "kv": kv, "spread": s > 1, "Hq": group * h, "H": h, "D": d,
                "window": window}
    if kind == "route":
        score = rng.choice(["softmax", "sigmoid"])
        groups = rng.choice([1, 1, 4, 8])
        e = groups * _log(rng, max(4, 8 // groups), 512 // groups)
        top = rng.randint(1, groups) if groups > 1 else 1
        return {"kind": kind, "T": _log(rng, 1, 4096), "E": e, "k": rng.randint(1, min(12, top * (e // groups))),
                "score": score, "biased": score == "sigmoid" and rng.random() < 0.7, "groups": groups, "top": top,
                "renorm": rng.random() < 0.7, "factor": rng.choice([1.0, 2.5]), "logits": rng.choice(["f32", "f16"])}
    fmt = rng.choice(["q4_0", "planes", "q4_k", "q4_k"])
    width = _not(256 * max(2, _log(rng, 512, 5120) // 256), 12 * 256, 256)
    f = _not(256 * max(1, _log(rng, 256, 2560) // 256), 12 * 256, 256)
    e, t = rng.choice([8, 16, 60, 64, 128]), _log(rng, 1, 2000)
    k = min(e, rng.choice([1, 2, 4, 6, 8]))
    while e * width * f > MOST_WEIGHTS:
        e //= 2
    k = min(k, e)
    return {"kind": "experts", "fmt": fmt, "T": max(1, min(t, MOST_EXPERT // (k * width * f))), "E": e, "k": k,
            "K": width, "F": f}


# ------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 2654435761 % (1 << 62) + 29)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _keys(g, n, h, d):
    """Keys and values as a projection gives them: unit normal, keys with a few channels of larger magnitude."""
    k = _randn(g, n, h, d)
    k[..., 5::41] *= 4
    return k.to(torch.float16), _randn(g, n, h, d).to(torch.float16)


def _lens(case):
    """Cached tokens of every stream (the queries' own among them): from a quarter of kv to kv where spread."""
    if not case["spread"]:
        return [case["kv"]] * case["S"]
    lo, n = max(case["nq"], case["kv"] // 4), max(1, case["S"] - 1)
    return [case["kv"] - (case["kv"] - lo) * (i * 7 % case["S"]) // n for i in range(case["S"])]


def _seen(case):
    """Visible (query, key) pairs of every stream."""
    out = []
    for n in _lens(case):
        pos = range(n - case["nq"], n)
        out.append(sum(min(p + 1, case["window"]) if case["window"] else p + 1 for p in pos))
    return out


def _reached(case):
    """Cached tokens that some query of the stream sees."""
    w = case["window"] + case["nq"] - 1 if case["window"] else 1 << 40
    return [min(n, w) for n in _lens(case)]


def _scores64(case, logits, bias):
    x = logits.double()
    s = torch.softmax(x, -1) if case["score"] == "softmax" else 1 / (1 + torch.exp(-x))
    return s, s if bias is None else s + bias.double()


def _grouped64(case, sel):
    """The experts of the kept groups, and each group's score."""
    t, e = sel.shape
    n = case["groups"]
    g = sel.reshape(t, n, e // n)
    best = torch.sort(g, -1, descending=True).values[..., :2].sum(-1)
    order = torch.sort(best, dim=-1, descending=True, stable=True).indices[:, :case["top"]]
    keep = torch.zeros(t, n, dtype=torch.bool, device=sel.device)
    keep.scatter_(1, order, True)
    return keep[:, :, None].expand(t, n, e // n).reshape(t, e), best


def _undecided(case, logits, bias):
    """Rows whose choice hangs on differences that 32 bits do not resolve (equal scores are resolved: by index)."""
    s, sel = _scores64(case, logits, bias)
    near = torch.zeros(logits.shape[0], dtype=torch.bool, device=logits.device)

    def close(v, n):
        v = torch.sort(v, -1, descending=True).values[:, :n + 1]
        gap = v[:, :-1] - v[:, 1:]
        return ((gap > 0) & (gap < 4e-6 * v[:, :-1].abs())).any(-1)

    if case["groups"] > 1:
        keep, best = _grouped64(case, sel)
        near |= close(best, case["top"])
        sel = sel.masked_fill(~keep, -1e30)
    return near | close(sel, case["k"])


def _logits(case, g):
    dtype = torch.float16 if case["logits"] == "f16" else torch.float32
    t, e = case["T"], case["E"]
    popular = 0.5 * _randn(g, e)
    x = (1.5 * _randn(g, t, e) + popular).to(dtype)
    bias = 0.05 * _randn(g, e) - 0.1 * popular if case["biased"] else None
    for _ in range(6):
        bad = _undecided(case, x, bias)
        x = torch.where(bad[:, None], (1.5 * _randn(g, t, e) + popular).to(dtype), x)
    return x, bias


def _half_bytes(x):
    return x.to(torch.float16).contiguous().view(torch.uint8).reshape(*x.shape, 2)


def _codes(g, *shape):
    return _randn(g, *shape).mul_(2.7).add_(7.8).round_().clamp_(0, 15).to(torch.uint8)


def _weights(fmt, n, k, g):
    """(W, W_aux) of n x k weights with a standard deviation near 0.02, in one format's bytes."""
    if fmt == "q4_k":
        nb = k // 256
        d = torch.rand(n, nb, generator=g, device=DEV).mul_(1.2e-4).add_(1.1e-4)
        sc = torch.randint(24, 64, (n, nb, 8), generator=g, device=DEV, dtype=torch.uint8)
        m = (sc.int() + torch.randint(-4, 5, (n, nb, 8), generator=g, device=DEV, dtype=torch.int32)).clamp_(0, 63)
        m = m.to(torch.uint8)
        q = _codes(g, n, nb, 4, 2, 32)
        blk = torch.empty(n, nb, 144, dtype=torch.uint8, device=DEV)
        blk[..., 0:2] = _half_bytes(d)
        blk[..., 2:4] = _half_bytes(d * 7.8)
        blk[..., 4:8] = sc[..., :4] | ((sc[..., 4:] >> 4) << 6)
        blk[..., 8:12] = m[..., :4] | ((m[..., 4:] >> 4) << 6)
        blk[..., 12:16] = (sc[..., 4:] & 15) | ((m[..., 4:] & 15) << 4)
        blk[..., 16:] = (q[..., 0, :] | (q[..., 1, :] << 4)).reshape(n, nb, 128)
        return blk.reshape(n, nb * 144), None
    nb = k // 32
    d = torch.rand(n, nb, generator=g, device=DEV).mul_(0.009).add_(0.004)
    if fmt == "q4_0":
        q = _codes(g, n, nb, 2, 16)
        blk = torch.empty(n, nb, 18, dtype=torch.uint8, device=DEV)
        blk[..., 0:2] = _half_bytes(d)
        blk[..., 2:] = q[:, :, 0] | (q[:, :, 1] << 4)
        return blk.reshape(n, nb * 18), None
    q = _codes(g, n, k // 2, 2)
    return q[..., 0] | (q[..., 1] << 4), d.to(torch.float16)


def _expert_inputs(case, g):
    """Every expert's matrices one after the other, normalised rows, and a router's answer (each row's experts differ)."""
    t, e, k, width, f = case["T"], case["E"], case["k"], case["K"], case["F"]
    ws = [_weights(case["fmt"], e * n, m, g) for n, m in ((f, width), (f, width), (width, f))]
    x = _randn(g, t, width)
    x[:, ::509] *= 4
    top = torch.topk(torch.rand(t, e, generator=g, device=DEV), k, -1)
    w = torch.softmax(2 * _randn(g, t, k), -1)
    return ws, x.to(torch.float16), top.indices.to(torch.int32), w.contiguous()


def _pages(case, g):
    """A page table with the pages of all streams in no order, and the slot of every cached token."""
    lens = _lens(case)
    per = [(n + PAGE - 1) // PAGE for n in lens]
    perm = torch.randperm(sum(per), generator=g, device=DEV)
    table = torch.zeros(len(lens), max(per), dtype=torch.int32, device=DEV)
    slots, at = [], 0
    for i, n in enumerate(lens):
        mine = perm[at:at + per[i]]
        table[i, :per[i]] = mine.to(torch.int32)
        t = torch.arange(n, device=DEV)
        slots.append(mine[t // PAGE] * PAGE + t % PAGE)
        at += per[i]
    return table, torch.cat(slots), sum(per)


def _attn_inputs(case, seed):
    g = _gen(seed)
    lens = _lens(case)
    k, v = _keys(g, sum(lens), case["H"], case["D"])
    q = _randn(g, case["S"] * case["nq"], case["Hq"], case["D"]).to(torch.float16)
    return g, lens, q, k, v


def _store_inputs(case, seed):
    g = _gen(seed)
    k, v = _keys(g, case["T"], case["H"], case["D"])
    if case["whole"]:                              # one stream's consecutive tokens
        slots = torch.arange(case["start"], case["start"] + case["T"], device=DEV)
        pages = (case["start"] + case["T"] + PAGE - 1) // PAGE
        perm = torch.randperm(pages, generator=g, device=DEV)
        slots = perm[slots // PAGE] * PAGE + slots % PAGE
    else:                                          # one token of each stream, every stream with pages of its own
        per = (case["start"] + PAGE) // PAGE
        pages = per * case["T"]
        at = (case["start"] + 13 * torch.arange(case["T"], device=DEV)) % (per * PAGE)
        slots = torch.arange(case["T"], device=DEV) * (per * PAGE) + at
    return k, v, slots, pages


# ------------------------------------------------------------------ plain forms
def _quantize(x):
    """Codes and scales of 32 values each: d = the value of largest magnitude / -8 in fp16, code floor(x / d + 8.5)."""
    b = x.float().reshape(*x.shape[:-1], -1, GROUP)
    a = b.abs()
    at = (a == a.amax(-1, keepdim=True)).to(torch.uint8).argmax(-1, keepdim=True)
    d = (b.gather(-1, at) / -8).to(torch.float16)
    q = torch.floor(b / d.float() + 8.5).clamp_(0, 15)
    q = torch.where(d == 0, torch.full_like(q, 8), q)
    return q.to(torch.uint8), d


def _pack(x):
    q, d = _quantize(x)
    q = q.reshape(*x.shape[:-1], x.shape[-1] // 2, 2)
    return q[..., 0] | (q[..., 1] << 4), d.squeeze(-1)


def _unpack(codes, d):
    q = torch.stack([codes & 15, codes >> 4], -1).reshape(*d.shape, GROUP).float()
    return (q.sub_(8).mul_(d.float()[..., None])).reshape(*codes.shape[:-1], codes.shape[-1] * 2)


def _plain_store(s):
    out = []
    for x in (s["k"], s["v"]):
        q, d = _quantize(x)
        out.append(((q.float() - 8) * d.float()).to(torch.float16).reshape(x.shape))
    return out


def _plain_attn(s):
    c = s["case"]
    n, nq, hq, h, d = c["S"], c["nq"], c["Hq"], c["H"], c["D"]
    r, most = hq // h, max(_reached(c))
    lens, first, seen = s["lens"][:, None], s["first"][:, None], torch.arange(most, device=DEV)
    t = torch.clamp(lens - c["nq"] - c["window"] + 1, min=0) + seen if c["window"] else seen.expand(n, most)   # positions
    at = first + torch.minimum(t, lens - 1)
    k = _unpack(s["kq"][at], s["kd"][at]).transpose(1, 2)                        # [S][H][most][D]
    v = _unpack(s["vq"][at], s["vd"][at]).transpose(1, 2)
    q = s["q"].float().reshape(n, nq, h, r, d).permute(0, 2, 3, 1, 4).reshape(n, h, r * nq, d)
    x = torch.matmul(q, k.transpose(2, 3)).mul_(s["scale"]).reshape(n, h, r, nq, most)
    p = (lens - nq + torch.arange(nq, device=DEV))[:, :, None]                   # the queries' positions
    hide = t[:, None, :] > p
    if c["window"]:
        hide = hide | (t[:, None, :] <= p - c["window"])
    x = x.masked_fill_(hide[:, None, None], float("-inf"))
    x = torch.exp(x - x.amax(-1, keepdim=True)).reshape(n, h, r * nq, most)
    o = torch.matmul(x, v) / x.sum(-1, keepdim=True)
    return o.reshape(n, h, r, nq, d).permute(0, 3, 1, 2, 4).reshape(n * nq, hq, d).to(torch.float16)


def _plain_route(s):
    c, x = s["case"], s["x"].float()
    if c["score"] == "softmax":
        score = torch.exp(x - x.amax(-1, keepdim=True))
        score = score / score.sum(-1, keepdim=True)
    else:
        score = 1 / (1 + torch.exp(-x))
    sel = score if s["bias"] is None else score + s["bias"]
    if c["groups"] > 1:
        t, e = x.shape
        g = sel.reshape(t, c["groups"], e // c["groups"])
        best = torch.sort(g, -1, descending=True).values[..., :2].sum(-1)
        order = torch.sort(best, dim=-1, descending=True, stable=True).indices[:, :c["top"]]
        keep = torch.zeros_like(best, dtype=torch.bool).scatter_(1, order, True)
        sel = g.masked_fill(~keep[..., None], float("-inf")).reshape(t, e)
    ids = torch.sort(sel, dim=-1, descending=True, stable=True).indices[:, :c["k"]]
    w = score.gather(1, ids)
    if c["renorm"]:
        w = w / w.sum(-1, keepdim=True)
    return [ids.to(torch.int32), w * c["factor"]]


def _dequant(fmt, w, aux, n, k):
    if fmt == "q4_k":
        b = w.reshape(n, k // 256, 144)
        h = b[..., :4].contiguous().view(torch.float16).float()
        s = b[..., 4:16].int()
        lo, mid, hi = s[..., 0:4], s[..., 4:8], s[..., 8:12]
        sc = torch.cat([lo & 63, (hi & 15) | ((lo >> 6) << 4)], -1).float() * h[..., 0:1]
        mn = torch.cat([mid & 63, (hi >> 4) | ((mid >> 6) << 4)], -1).float() * h[..., 1:2]
        q = b[..., 16:].reshape(n, k // 256, 4, 1, 32)
        q = torch.cat([q & 15, q >> 4], 3).reshape(n, k // 256, 8, 32).float()
        return q.mul_(sc[..., None]).sub_(mn[..., None]).reshape(n, k)
    if fmt == "q4_0":
        b = w.reshape(n, k // 32, 18)
        d = b[..., :2].contiguous().view(torch.float16).float()
        q = torch.cat([b[..., 2:] & 15, b[..., 2:] >> 4], -1).float()
    else:
        d = aux.float()[..., None]
        q = torch.stack([w & 15, w >> 4], -1).reshape(n, k // 32, 32).float()
    return q.sub_(8).mul_(d).reshape(n, k)


def _expert(ws, i, e, n):
    w, aux = ws[i]
    return w[e * n:(e + 1) * n], None if aux is None else aux[e * n:(e + 1) * n]


def _plain_experts(s):
    """All experts in use at once: their weights decoded, their rows side by side, padded to the longest list."""
    c = s["case"]
    t, k, width, f, fmt = c["T"], c["k"], c["K"], c["F"], c["fmt"]
    used, which = torch.unique(s["ids"], return_inverse=True)
    which, n = which.reshape(-1), used.numel()
    order = torch.sort(which, stable=True).indices
    count = torch.bincount(which, minlength=n)
    place = torch.empty_like(which)
    place[order] = torch.arange(t * k, device=DEV) - (torch.cumsum(count, 0) - count)[which[order]]
    a = torch.zeros(n, int(count.max()), width, dtype=torch.float32, device=DEV)
    a[which, place] = s["x"].float().repeat_interleave(k, 0)

    def linear(x, i, rows, cols):
        w, aux = s["ws"][i]
        w = w.reshape(c["E"], rows, -1)[used].reshape(n * rows, -1)
        aux = None if aux is None else aux.reshape(c["E"], rows, -1)[used].reshape(n * rows, -1)
        return torch.matmul(x, _dequant(fmt, w, aux, n * rows, cols).reshape(n, rows, cols).transpose(1, 2))

    g = linear(a, 0, f, width)
    y = linear(g / (1 + torch.exp(-g)) * linear(a, 1, f, width), 2, width, f)
    return (y[which, place].reshape(t, k, width) * s["w"][..., None]).sum(1).to(torch.float16)


# ------------------------------------------------------------------ the four parts that are measured
def _package():
    import os
    import sys
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "bus-fill_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import busfill
    return busfill


def prepare(case, seed):
    s = {"case": case}
    bf = _package() if own else None
    s["bf"] = bf
    if case["kind"] == "store":
        s["k"], s["v"], s["slots"], pages = _store_inputs(case, seed)
        if own:
            s["data"] = torch.zeros(bf.kv4_bytes(pages, PAGE, case["H"], case["D"]), dtype=torch.uint8, device=DEV)
            s["cache"] = bf.kv4_cache(s["data"], pages, PAGE, case["H"], case["D"])
            s["out"] = [torch.empty_like(s["k"]), torch.empty_like(s["v"])]
    elif case["kind"] == "attn":
        g, lens, s["q"], k, v = _attn_inputs(case, seed)
        s["scale"] = 1 / math.sqrt(case["D"])
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
        if own:
            s["table"], slots, pages = _pages(case, g)
            s["data"] = torch.zeros(bf.kv4_bytes(pages, PAGE, case["H"], case["D"]), dtype=torch.uint8, device=DEV)
            s["cache"] = bf.kv4_cache(s["data"], pages, PAGE, case["H"], case["D"])
            bf.kv4_store(s["cache"], k, v, slots, sum(lens))
            s["starts"] = torch.arange(0, (case["S"] + 1) * case["nq"], case["nq"], dtype=torch.int32, device=DEV)
            s["o"] = torch.empty(s["q"].shape, dtype=torch.float16, device=DEV)
        else:
            s["first"] = torch.cumsum(s["lens"], 0) - s["lens"]
            (s["kq"], s["kd"]), (s["vq"], s["vd"]) = _pack(k), _pack(v)
    elif case["kind"] == "route":
        s["x"], s["bias"] = _logits(case, _gen(seed))
        if own:
            s["out"] = [torch.empty(case["T"], case["k"], dtype=torch.int32, device=DEV),
                        torch.empty(case["T"], case["k"], dtype=torch.float32, device=DEV)]
    else:
        s["ws"], s["x"], s["ids"], s["w"] = _expert_inputs(case, _gen(seed))
        if own:
            s["y"] = torch.empty(case["T"], case["K"], dtype=torch.float16, device=DEV)
    return s


def run(s):
    c, bf = s["case"], s["bf"]
    kind = c["kind"]
    if bf is None:
        if kind == "store":
            return _plain_store(s)
        if kind == "attn":
            return [_plain_attn(s)]
        if kind == "route":
            return _plain_route(s)
        return [_plain_experts(s)]
    if kind == "store":
        bf.kv4_store(s["cache"], s["k"], s["v"], s["slots"], c["T"])
        bf.kv4_load(s["cache"], s["slots"], s["out"][0], s["out"][1], c["T"])
        return s["out"]
    if kind == "attn":
        bf.kv4_attention(s["cache"], s["q"], s["o"], s["starts"], s["lens"], s["table"], S=c["S"],
                         T=c["S"] * c["nq"], q_heads=c["Hq"], max_q=c["nq"], max_kv=c["kv"], scale=s["scale"],
                         window=c["window"], otype=bf.OUT_F16)
        return [s["o"]]
    if kind == "route":
        bf.moe_route(s["x"], s["out"][0], s["out"][1], c["T"], c["E"], c["k"], bias=s["bias"],
                     score=bf.SCORE_SOFTMAX if c["score"] == "softmax" else bf.SCORE_SIGMOID, groups=c["groups"],
                     top_groups=c["top"], renorm=c["renorm"], factor=c["factor"])
        return s["out"]
    bf.moe_ffn({"q4_0": bf.Q4_0, "planes": bf.Q4_0_PLANES, "q4_k": bf.Q4_K}[c["fmt"]], s["ws"][0], s["ws"][1],
               s["ws"][2], s["x"], s["ids"], s["w"], s["y"], T=c["T"], K=c["K"], F=c["F"], N=c["K"], E=c["E"],
               k=c["k"], otype=bf.OUT_F16)
    return [s["y"]]


def work(case):
    kind = case["kind"]
    if kind == "store":                            # fp16 rows in, 4.5 bits a value written and read back, fp16 rows out
        n = 2 * case["T"] * case["H"] * case["D"]
        return {"bytes": 2 * n + 9 * n // 16 + 9 * n // 16 + 2 * n, "flops": 4 * n}
    if kind == "attn":
        rows = case["S"] * case["nq"] * case["Hq"] * case["D"]
        return {"bytes": sum(_reached(case)) * case["H"] * case["D"] * 9 // 8
                + rows * 4,
                "flops": 4 * case["D"] * case["Hq"] * sum(_seen(case))}
    if kind == "route":
        t, e = case["T"], case["E"]
        return {"bytes": t * e * (2 if case["logits"] == "f16" else 4) + t * case["k"] * 8, "flops": 4 * t * e}
    t, e, k = case["T"], case["E"], case["k"]
    used = e * (1 - (1 - k / e) ** t)              # experts that some row chose, on average
    weights = 3 * case["K"] * case["F"]
    return {"bytes": int(used * weights * 9 / 16) + t * case["K"] * 4 + 8 * t * k,
            "flops": 2 * t * k * weights}


# ------------------------------------------------------------------ 64-bit results
def _exact_cached(x):
    """What the cache stands for, from the definition in 64 bits."""
    b = x.double().reshape(*x.shape[:-1], -1, GROUP)
    hi, lo = b.amax(-1), b.amin(-1)
    first_hi = (b == hi[..., None]).to(torch.uint8).argmax(-1)
    first_lo = (b == lo[..., None]).to(torch.uint8).argmax(-1)
    m = torch.where(hi > -lo, hi, torch.where(hi < -lo, lo, torch.where(first_hi <= first_lo, hi, lo)))
    d = (m / -8).to(torch.float16).double()[..., None]
    safe = torch.where(d == 0, torch.ones_like(d), d)
    return ((torch.floor(b / safe + 8.5).clamp(0, 15) - 8) * d).reshape(x.shape)


def _exact_weights(fmt, w, aux, n, k):
    """n x k weights from the formats' definitions, weight by weight, in 64 bits."""
    i = torch.arange(k, device=DEV)
    if fmt == "planes":
        q = (w[:, i // 2].int() >> (4 * (i % 2)).int()) & 15
        return (q - 8).double() * aux[:, i // 32].double()
    if fmt == "q4_0":
        at = i // 32 * 18
        q = (w[:, at + 2 + i % 16].int() >> (i % 32 // 16 * 4).int()) & 15
        return (q - 8).double() * w.reshape(n, -1, 18)[..., :2].contiguous().view(torch.float16)[..., 0].double()[:, i // 32]
    at, j = i // 256 * 144, i % 256 // 32            # super-block, sub-block
    h = w.reshape(n, -1, 144)[..., :4].contiguous().view(torch.float16).double()
    q = (w[:, at + 16 + j // 2 * 32 + i % 32].int() >> (j % 2 * 4).int()) & 15
    low, low4 = j < 4, j % 4
    sc = torch.where(low, w[:, at + 4 + low4] & 63, (w[:, at + 12 + low4] & 15) | (w[:, at + 4 + low4] >> 6 << 4))
    mn = torch.where(low, w[:, at + 8 + low4] & 63, (w[:, at + 12 + low4] >> 4) | (w[:, at + 8 + low4] >> 6 << 4))
    return h[:, i // 256, 0] * sc.double() * q.double() - h[:, i // 256, 1] * mn.double()


def exact(case, seed):
    kind = case["kind"]
    if kind == "store":
        k, v, _, _ = _store_inputs(case, seed)
        return [_exact_cached(k), _exact_cached(v)]
    if kind == "attn":
        _, lens, q, k, v = _attn_inputs(case, seed)
        nq, r = case["nq"], case["Hq"] // case["H"]
        out = torch.empty(q.shape, dtype=torch.float64, device=DEV)
        at = 0
        for i, n in enumerate(lens):
            pos = torch.arange(n - nq, n, device=DEV)[:, None]
            t = torch.arange(n, device=DEV)[None, :]
            see = (t <= pos) & (t > pos - (case["window"] or n + 1))
            for h in range(case["H"]):
                kk, vv = _exact_cached(k[at:at + n, h]), _exact_cached(v[at:at + n, h])
                for j in range(h * r, (h + 1) * r):
                    x = (q[i * nq:(i + 1) * nq, j].double() @ kk.t()) / math.sqrt(case["D"])
                    out[i * nq:(i + 1) * nq, j] = torch.softmax(x.masked_fill(~see, float("-inf")), -1) @ vv
            at += n
        return [out]
    if kind == "route":
        x, bias = _logits(case, _gen(seed))
        score, sel = _scores64(case, x, bias)
        if case["groups"] > 1:
            sel = sel.masked_fill(~_grouped64(case, sel)[0], float("-inf"))
        ids = torch.sort(sel, dim=-1, descending=True, stable=True).indices[:, :case["k"]]
        w = score.gather(1, ids)
        if case["renorm"]:
            w = w / w.sum(-1, keepdim=True)
        return [ids.to(torch.int32), w * case["factor"]]
    ws, x, ids, w = _expert_inputs(case, _gen(seed))
    out = torch.zeros(case["T"], case["K"], dtype=torch.float64, device=DEV)
    chosen = torch.zeros(case["T"], case["E"], dtype=torch.float64, device=DEV)
    chosen.scatter_(1, ids.long(), w.double())     # a row's experts differ, so nothing is overwritten
    for e in range(case["E"]):
        rows = torch.nonzero(chosen[:, e])[:, 0]
        if rows.numel() == 0:
            continue
        a = x[rows].double()
        f, width, fmt = case["F"], case["K"], case["fmt"]
        g = a @ _exact_weights(fmt, *_expert(ws, 0, e, f), f, width).t()
        u = a @ _exact_weights(fmt, *_expert(ws, 1, e, f), f, width).t()
        y = (g * torch.sigmoid(g) * u) @ _exact_weights(fmt, *_expert(ws, 2, e, width), width, f).t()
        out.index_add_(0, rows, y * chosen[rows, e][:, None])
    return [out]
