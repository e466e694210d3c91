"""What a decoder layer's steps around its 4-bit projections cost: the residual
norm (fp16 rows, or the int8 rows of the integer-dot path), the rotation of
queries and keys with the 4-bit cache's store, attention with a window and a few
first tokens that stay visible, and low-rank adapters of many requests beside a
shared projection.

Where ``own`` is false, ``run`` computes each operator in its plain form:
elementary torch operations in 32 bits (angles in 64), rounded once at the end.
Where it is true, ``run`` makes the calls a program makes of the ``busfill``
package.  ``exact`` computes the same outputs from the definitions in 64 bits.

Sizes are the repository's own (5120 wide, 7168 = 5120 + 2 * 1024 for a layer's
query, key and value projections, i.e. 40 query heads over 8 key/value heads of
128; batches of 1, 16, 32; 2000-token prompts) or generic ones.
"""
import math

import torch

own = False

DEV = "cuda"
PAGE = 64
GROUP = 32                                       # values that share a scale, in the cache and in int8 rows
# the largest listed cases: no drawn one is larger
MOST_NORM = 2000 * 5120                          # values of one norm
MOST_APPEND = 2000 * 56 * 128                    # query, key and value elements of one append
MOST_PAIRS = 2000 * 512 * 40 * 128               # attention: (query, key) pairs x head elements
MOST_CACHED = 32 * 8000 * 8 * 128                # cached elements of one attention call
MOST_LORA = 2000 * 64 * (5120 + 5120)            # adapters: rows x rank x (inputs + outputs)
MOST_ADAPTERS = 32 * 64 * (5120 + 7168)          # elements of all adapters


def listed():
    return [
        # a decode step of 32 streams: the attention's output joins the fp32 residual, fp16 rows for the next projection
        {"name": "norm_decode_32", "kind": "norm", "T": 32, "K": 5120, "x": "f32", "delta": "f16", "weight": "f32",
         "offset": 0.0, "out": "f16"},
        # a decode step of 16 streams that goes on in the integer-dot path: int8 rows with a scale for 32 values
        {"name": "norm_q8_16", "kind": "norm", "T": 16, "K": 5120, "x": "f16", "delta": "f16", "weight": "f16",
         "offset": 0.0, "out": "q8"},
        # a 2000-token prompt
        {"name": "norm_prompt_2000", "kind": "norm", "T": 2000, "K": 5120, "x": "f32", "delta": "f16", "weight": "f32",
         "offset": 0.0, "out": "f16"},
        # one token of each of 32 streams, far into their texts
        {"name": "append_decode_32", "kind": "append", "T": 32, "Hq": 40, "H": 8, "D": 128, "rot": 128, "style": "halves",
         "theta": 1e6, "start": 7000, "whole": False},
        # a 2000-token prompt behind 37 cached tokens
        {"name": "append_prompt_2000", "kind": "append", "T": 2000, "Hq": 40, "H": 8, "D": 128, "rot": 128,
         "style": "halves", "theta": 10000.0, "start": 37, "whole": True},
        # one stream early on, its window just passed: the smallest call, where latency counts
        {"name": "sinks_decode_1x1200", "kind": "attn", "S": 1, "nq": 1, "kv": 1200, "spread": False, "Hq": 40, "H": 8,
         "D": 128, "window": 1024, "sinks": 4},
        # 32 streams of ragged lengths up to 8000 tokens, a window of 2048
        {"name": "sinks_decode_32x8000", "kind": "attn", "S": 32, "nq": 1, "kv": 8000, "spread": True, "Hq": 40, "H": 8,
         "D": 128, "window": 2048, "sinks": 4},
        # one stream of endless text with a long window, its instructions (100 tokens) kept in sight
        {"name": "sinks_decode_1x131072", "kind": "attn", "S": 1, "nq": 1, "kv": 131072, "spread": False, "Hq": 32, "H": 4,
         "D": 128, "window": 32768, "sinks": 100},
        # a 2000-token prompt of a model with a window of 512
        {"name": "sinks_prompt_2000", "kind": "attn", "S": 1, "nq": 2000, "kv": 2000, "spread": False, "Hq": 40, "H": 8,
         "D": 128, "window": 512, "sinks": 4},
        # one request's adapter beside a layer's query, key and value projections
        {"name": "lora_m1", "kind": "lora", "T": 1, "K": 5120, "parts": "qkv", "E": 8, "rank": 16, "mixed": False,
         "runs": False, "out": "f16"},
        # 32 requests with adapters of their own choice, of ranks from 16 to 64, some with none
        {"name": "lora_m32", "kind": "lora", "T": 32, "K": 5120, "parts": "qkv", "E": 32, "rank": 64, "mixed": True,
         "runs": False, "out": "f16"},
        # prompts of 2000 tokens in all, of a handful of requests, beside the output projection
        {"name": "lora_prompt_2000", "kind": "lora", "T": 2000, "K": 5120, "parts": "5120", "E": 8, "rank": 64,
         "mixed": False, "runs": True, "out": "f16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "append", "append", "attn", "attn", "prompt", "lora", "lora", "lora"])
    if kind == "norm":
        out = rng.choice(["f16", "f16", "q8"])
        k = 32 * _log(rng, 8, 256) if out == "q8" else rng.choice([256 * _log(rng, 1, 32), _log(rng, 64, 8192)])
        return {"kind": kind, "T": _log(rng, 1, min(4000, MOST_NORM // k)), "K": k, "x": rng.choice(["f32", "f16"]),
                "delta": rng.choice(["f16", "f16", "f32", "none"]), "weight": rng.choice(["f32", "f16"]),
                "offset": rng.choice([0.0, 0.0, 1.0]), "out": out}
    d = rng.choice([64, 96, 128, 128, 256])
    h = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 4, 5, 8])
    if kind == "append":
        whole = rng.random() < 0.5
        most = max(1, MOST_APPEND // ((group + 2) * h * d))
        return {"kind": kind, "T": _log(rng, 1, min(2000 if whole else 256, most)), "Hq": group * h, "H": h, "D": d,
                "rot": rng.choice([d, d, d // 2, 32]), "style": rng.choice(["halves", "pairs"]),
                "theta": rng.choice([10000.0, 500000.0, 1e6]), "start": _log(rng, 1, 131072), "whole": whole}
    if kind in ("attn", "prompt"):
        window = _log(rng, 16, 8192)
        sinks = rng.choice([1, 4, 4, rng.randint(1, 200)])
        if kind == "prompt":
            nq = _log(rng, 17, 2000)
            while nq * min(nq, window) * group * h * d > MOST_PAIRS:
                nq = nq * 2 // 3
            return {"kind": "attn", "S": 1, "nq": nq, "kv": nq + rng.choice([0, 0, rng.randint(1, 500)]), "spread": False,
                    "Hq": group * h, "H": h, "D": d, "window": window, "sinks": sinks}
        nq, s = rng.choice([1, 1, 1, 1, 2, 4, 7]), _log(rng, 1, 64)
        return {"kind": "attn", "S": s, "nq": nq, "kv": _log(rng, 16, min(131072, MOST_CACHED // (s * h * d))),
                "spread": s > 1, "Hq": group * h, "H": h, "D": d, "window": window, "sinks": sinks}
    rank = rng.choice([8, 16, 16, 32, 64])
    k, n = 256 * _log(rng, 2, 28), _log(rng, 256, 7168)
    e = rng.randint(1, 64)
    while e * rank * (k + n) > MOST_ADAPTERS:
        e = (e + 1) // 2
    t = _log(rng, 1, min(2000, MOST_LORA // (rank * (k + n))))
    return {"kind": kind, "T": t, "K": k, "parts": rng.choice([str(n), str(n), "%d,%d" % (n - n // 4, n // 4)]), "E": e,
            "rank": rank, "mixed": rng.random() < 0.4, "runs": t > 64 and rng.random() < 0.7, "out": rng.choice(["f16", "f32"])}


# ------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 2654435761 % (1 << 62) + 31)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _type(name):
    return {"f16": torch.float16, "f32": torch.float32}[name]


def _norm_inputs(case, seed):
    """Residual rows with a few large channels, what the last block adds, and weights near 1 (less the offset)."""
    g = _gen(seed)
    t, k = case["T"], case["K"]
    x = 2 * _randn(g, t, k)
    x[:, ::509] *= 16
    x = x.to(_type(case["x"]))
    delta = None if case["delta"] == "none" else _randn(g, t, k).to(_type(case["delta"]))
    w = (1 + 0.3 * _randn(g, k) - case["offset"]).to(_type(case["weight"]))
    if case["out"] == "q8":                        # no value half way between two codes, where 32 bits do not decide
        for _ in range(8):
            v = (x.double() if delta is None else x.double() + delta.double()) * (w.double() + case["offset"])
            b = v.reshape(t, -1, GROUP).abs()
            u = 127 * b / b.amax(-1, keepdim=True)
            near = ((u - torch.floor(u) - 0.5).abs() < 2e-4).reshape(t, k)
            x = torch.where(near, (x.float() * 1.0137).to(x.dtype), x)
    return x, delta, w


def _freq(case):
    i = torch.arange(0, case["rot"], 2, dtype=torch.float64, device=DEV)
    return torch.pow(torch.tensor(case["theta"], dtype=torch.float64, device=DEV), -i / case["rot"]).float()


def _pair(x, case):
    """The two elements of every rotated pair of x [...][D]."""
    r = x[..., :case["rot"]]
    if case["style"] == "halves":
        return r[..., :case["rot"] // 2], r[..., case["rot"] // 2:]
    return r[..., 0::2], r[..., 1::2]


def _paired(a, b, x, case):
    """x with its pairs replaced by a and b."""
    r = torch.cat([a, b], -1) if case["style"] == "halves" else torch.stack([a, b], -1).flatten(-2)
    return torch.cat([r, x[..., case["rot"]:].to(r.dtype)], -1)


def _rotated64(x, position, freq, case):
    """x [T][heads][D] rotated by its positions, and the sums of the products' magnitudes."""
    angle = position.double()[:, None] * freq.double()
    c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    a, b = _pair(x.double(), case)
    return _paired(a * c - b * s, b * c + a * s, x.double(), case), a.abs() + b.abs()


def _append_inputs(case, seed):
    g = _gen(seed)
    t, d, freq = case["T"], case["D"], _freq(case)
    q = _randn(g, t, case["Hq"], d).to(torch.float16)
    v = _randn(g, t, case["H"], d).to(torch.float16)
    if case["whole"]:                              # one stream's consecutive tokens
        position = torch.arange(case["start"], case["start"] + t, device=DEV)
        slots = position % (t + PAGE)
        pages = (t + 2 * PAGE - 1) // PAGE
        perm = torch.randperm(pages, generator=g, device=DEV)
        slots = perm[slots // PAGE] * PAGE + slots % PAGE
    else:                                          # one token of each stream, every stream with pages of its own
        position = case["start"] + 13 * torch.arange(t, device=DEV)
        slots = torch.arange(t, device=DEV) * PAGE + position % PAGE
        pages = t

    def keys():
        k = _randn(g, t, case["H"], d)
        k[..., 5::41] *= 4
        return k.to(torch.float16)

    k = keys()
    for _ in range(10):                            # no rotated key half way between two fp16 numbers, where 32 bits do not decide
        r, size = _rotated64(k, position, freq, case)
        bad = [(x + 1e-6 * size).to(torch.float16) != (x - 1e-6 * size).to(torch.float16) for x in _pair(r, case)]
        bad = bad[0] | bad[1]
        bad = _paired(bad, bad, torch.zeros_like(k, dtype=torch.bool), case)
        k = torch.where(bad, keys(), k)
    return q, k, v, position, slots, freq, pages


def _lens(case):
    """Cached tokens of every stream (the queries' own among them): from a quarter of kv to kv where spread."""
    kv = max(case["kv"], case["nq"])
    if not case["spread"]:
        return [kv] * case["S"]
    lo, n = max(case["nq"], kv // 4), max(1, case["S"] - 1)
    return [kv - (kv - lo) * (i * 7 % case["S"]) // n for i in range(case["S"])]


def _seen(case):
    """Visible (query, key) pairs of every stream."""
    w, k = case["window"], case["sinks"]
    return [sum(min(p + 1, w) + min(k, max(0, p + 1 - w)) for p in range(n - case["nq"], n)) for n in _lens(case)]


def _reached(case):
    """Cached tokens that some query of the stream sees."""
    w = case["window"] + case["nq"] - 1
    return [min(n, w) + min(case["sinks"], max(0, n - w)) for n in _lens(case)]


def _attn_inputs(case, seed):
    g = _gen(seed)
    lens = _lens(case)
    k = _randn(g, sum(lens), case["H"], case["D"])
    k[..., 5::41] *= 4
    v = _randn(g, sum(lens), case["H"], case["D"])
    q = _randn(g, case["S"] * case["nq"], case["Hq"], case["D"])
    first = torch.cumsum(torch.tensor(lens), 0) - torch.tensor(lens)
    for i, n in zip(first.tolist(), lens):         # first tokens that draw attention, as in trained models
        k[i:i + min(case["sinks"], n)] += 0.3 * q.reshape(-1, case["H"], case["Hq"] // case["H"], case["D"]).mean((0, 2))
    return g, lens, q.to(torch.float16), k.to(torch.float16), v.to(torch.float16)


def _pages(case, lens, g):
    """A page table with the pages of all streams in no order, and the slot of every cached token."""
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


def _widths(case):
    return [5120, 1024, 1024] if case["parts"] == "qkv" else [int(n) for n in case["parts"].split(",")]


def _lora_inputs(case, seed):
    """Rows, every row's adapter (-1: none), adapters with their ranks and scales, and the projection's output."""
    g = _gen(seed)
    t, k, e, r = case["T"], case["K"], case["E"], case["rank"]
    x = _randn(g, t, k)
    x[:, ::509] *= 4
    if case["runs"]:                               # requests one after the other
        cuts = torch.sort(torch.randint(0, t, (5,), generator=g, device=DEV)).values
        which = torch.searchsorted(cuts, torch.arange(t, device=DEV), right=True)
        ids = torch.randperm(max(e, 6), generator=g, device=DEV)[which] % e
    else:
        ids = torch.randint(0, e, (t,), generator=g, device=DEV)
        if t > 1:
            ids = torch.where(torch.rand(t, generator=g, device=DEV) < 0.1, torch.full_like(ids, -1), ids)
    ranks = torch.full((e,), r, device=DEV)
    if case["mixed"]:
        ranks = torch.clamp(r >> torch.randint(0, 3, (e,), generator=g, device=DEV), min=4)
    scales = 0.5 + torch.rand(e, generator=g, device=DEV)
    ab = [((_randn(g, e, r, k) / math.sqrt(k)).to(torch.float16), (0.3 * _randn(g, e, n, r) / math.sqrt(r)).to(torch.float16))
          for n in _widths(case)]
    c = _randn(g, t, sum(_widths(case))).to(_type(case["out"]))
    return x.to(torch.float16), ids.to(torch.int32), ranks.to(torch.int32), scales, ab, c


# ------------------------------------------------------------------ plain forms
def _plain_norm(s):
    c = s["case"]
    r = s["x"].float() if s["delta"] is None else s["x"].float() + s["delta"].float()
    y = r / torch.sqrt((r * r).mean(-1, keepdim=True) + s["eps"]) * (s["w"].float() + c["offset"])
    if c["out"] == "f16":
        return [r.to(s["x"].dtype), y.to(torch.float16)]
    b = y.reshape(c["T"], -1, GROUP)
    d = b.abs().amax(-1, keepdim=True) / 127
    q = torch.sign(b) * torch.floor(b.abs() / d + 0.5)
    return [r.to(s["x"].dtype), torch.where(d == 0, torch.zeros_like(q), q) * d]


def _quantize(x):
    """Codes and scales of 32 values each: d = the value of largest magnitude / -8 in fp16, code floor(x / d + 8.5)."""
    b = x.float().reshape(*x.shape[:-1], -1, GROUP)
    a = b.abs()
    at = (a == a.amax(-1, keepdim=True)).to(torch.uint8).argmax(-1, keepdim=True)
    d = (b.gather(-1, at) / -8).to(torch.float16)
    q = torch.floor(b / d.float() + 8.5).clamp_(0, 15)
    q = torch.where(d == 0, torch.full_like(q, 8), q)
    return q, d


def _plain_append(s):
    c = s["case"]
    turns = s["position"].double()[:, None] * (s["freq"].double() / (2 * math.pi))
    angle = 2 * math.pi * (turns - torch.round(turns))
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    out = []
    for x in (s["q"], s["k"]):
        a, b = _pair(x.float(), c)
        out.append(_paired(a * cos - b * sin, b * cos + a * sin, x.float(), c).to(torch.float16))
    for i, x in ((1, out[1]), (2, s["v"])):
        q, d = _quantize(x)
        out[i:] = [((q - 8) * d.float()).to(torch.float16).reshape(x.shape)]
    return out


def _pack(x):
    q, d = _quantize(x)
    q = q.to(torch.uint8).reshape(*x.shape[:-1], x.shape[-1] // 2, 2)
    return q[..., 0] | (q[..., 1] << 4), d.squeeze(-1)


def _unpack(codes, d):
    q = torch.stack([codes & 15, codes >> 4], -1).reshape(*d.shape, GROUP).float()
    return (q.sub_(8).mul_(d.float()[..., None])).reshape(*codes.shape[:-1], codes.shape[-1] * 2)


def _plain_attn(s):
    """The sinks' tokens and those from the first query's window on, gathered; hidden ones masked."""
    c = s["case"]
    n, nq, hq, h, d = c["S"], c["nq"], c["Hq"], c["H"], c["D"]
    r, most = hq // h, max(_reached(c))
    lens, first, seen = s["lens"][:, None], s["first"][:, None], torch.arange(most, device=DEV)
    begin = torch.clamp(lens - nq - c["window"] + 1, min=c["sinks"])
    t = torch.where(seen < c["sinks"], seen, begin - c["sinks"] + seen)          # positions
    at = first + torch.minimum(t, lens - 1)
    k = _unpack(s["kq"][at], s["kd"][at]).transpose(1, 2)                        # [S][H][most][D]
    v = _unpack(s["vq"][at], s["vd"][at]).transpose(1, 2)
    q = s["q"].float().reshape(n, nq, h, r, d).permute(0, 2, 3, 1, 4).reshape(n, h, r * nq, d)
    x = torch.matmul(q, k.transpose(2, 3)).mul_(s["scale"]).reshape(n, h, r, nq, most)
    p = (lens - nq + torch.arange(nq, device=DEV))[:, :, None]                   # the queries' positions
    t = t[:, None, :]
    hide = (t > p) | ((t <= p - c["window"]) & (t >= c["sinks"]))
    x = x.masked_fill_(hide[:, None, None], float("-inf"))
    x = torch.exp(x - x.amax(-1, keepdim=True)).reshape(n, h, r * nq, most)
    o = torch.matmul(x, v) / x.sum(-1, keepdim=True)
    return o.reshape(n, h, r, nq, d).permute(0, 3, 1, 2, 4).reshape(n * nq, hq, d).to(torch.float16)


def _plain_lora(s):
    """All adapters at once: every row's products with all of them, those of other adapters and past the rank as zeros."""
    c = s["case"]
    e, r = c["E"], c["rank"]
    mine = (s["ids"][:, None] == torch.arange(e, device=DEV))[:, :, None] & (torch.arange(r, device=DEV) < s["ranks"][:, None])
    keep = mine * s["scales"][:, None]                                           # [T][E][r]
    x = s["x"].float()
    y = [torch.matmul(torch.matmul(x, a.float().reshape(e * r, -1).t()) * keep.reshape(-1, e * r),
                      b.float().transpose(1, 2).reshape(e * r, -1)) for a, b in s["ab"]]
    return (s["c"].float() + torch.cat(y, -1)).to(s["c"].dtype)


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
    s = {"case": case, "bf": _package() if own else None}
    bf = s["bf"]
    if case["kind"] == "norm":
        s["x"], s["delta"], s["w"] = _norm_inputs(case, seed)
        s["eps"] = 1e-6
        if own:
            s["r"] = torch.empty_like(s["x"])
            if case["out"] == "f16":
                s["h"] = torch.empty(case["T"], case["K"], dtype=torch.float16, device=DEV)
            else:
                n, blocks = case["T"] * case["K"], case["T"] * case["K"] // GROUP
                s["aq"] = torch.empty(bf.q8_bytes(case["T"], case["K"]), dtype=torch.uint8, device=DEV)
                s["q"] = s["aq"][:n].view(torch.int8).reshape(case["T"], -1, GROUP)
                s["d"] = s["aq"][n:n + 4 * blocks].view(torch.float32).reshape(case["T"], -1, 1)
    elif case["kind"] == "append":
        s["q"], s["k"], s["v"], s["position"], s["slots"], s["freq"], pages = _append_inputs(case, seed)
        if own:
            s["data"] = torch.zeros(bf.kv4_bytes(pages, PAGE, case["H"], case["D"]), dtype=torch.uint8, device=DEV)
            s["cache"] = bf.kv4_cache(s["data"], pages, PAGE, case["H"], case["D"])
            s["out"] = [torch.empty_like(s["q"]), torch.empty_like(s["k"]), torch.empty_like(s["v"])]
    elif case["kind"] == "attn":
        g, lens, s["q"], k, v = _attn_inputs(case, seed)
        s["scale"] = 1 / math.sqrt(case["D"])
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
        if own:
            s["table"], slots, pages = _pages(case, lens, g)
            s["data"] = torch.zeros(bf.kv4_bytes(pages, PAGE, case["H"], case["D"]), dtype=torch.uint8, device=DEV)
            s["cache"] = bf.kv4_cache(s["data"], pages, PAGE, case["H"], case["D"])
            bf.kv4_store(s["cache"], k, v, slots, sum(lens))
            s["starts"] = torch.arange(0, (case["S"] + 1) * case["nq"], case["nq"], dtype=torch.int32, device=DEV)
            s["o"] = torch.empty(s["q"].shape, dtype=torch.float16, device=DEV)
            s["most"] = max(lens)
        else:
            s["first"] = torch.cumsum(s["lens"], 0) - s["lens"]
            (s["kq"], s["kd"]), (s["vq"], s["vd"]) = _pack(k), _pack(v)
    else:
        s["x"], s["ids"], s["ranks"], s["scales"], s["ab"], s["c"] = _lora_inputs(case, seed)
        if own:
            at = [sum(_widths(case)[:i]) for i in range(len(_widths(case)))]
            s["parts"] = bf.lora_parts([(a, b, n, i) for (a, b), n, i in zip(s["ab"], _widths(case), at)])
            s["y"] = torch.empty_like(s["c"])
    return s


def run(s):
    c, bf = s["case"], s["bf"]
    kind = c["kind"]
    if bf is None:
        if kind == "norm":
            return _plain_norm(s)
        if kind == "append":
            return _plain_append(s)
        return [_plain_attn(s) if kind == "attn" else _plain_lora(s)]
    if kind == "norm":
        if c["out"] == "f16":
            bf.rms_norm(s["x"], c["T"], c["K"], delta=s["delta"], R=s["r"], weight=s["w"], offset=c["offset"], eps=s["eps"],
                        H=s["h"])
            return [s["r"], s["h"]]
        bf.rms_norm(s["x"], c["T"], c["K"], delta=s["delta"], R=s["r"], weight=s["w"], offset=c["offset"], eps=s["eps"],
                    Aq=s["aq"])
        return [s["r"], torch.mul(s["q"], s["d"])]
    if kind == "append":
        bf.kv4_append(s["cache"], s["k"], s["v"], s["slots"], s["position"], s["freq"], c["T"], Q=s["q"], Q_out=s["out"][0],
                      q_heads=c["Hq"], rot=c["rot"], style=bf.ROPE_HALVES if c["style"] == "halves" else bf.ROPE_PAIRS)
        bf.kv4_load(s["cache"], s["slots"], s["out"][1], s["out"][2], c["T"])
        return s["out"]
    if kind == "attn":
        bf.kv4_attention_sinks(s["cache"], s["q"], s["o"], s["starts"], s["lens"], s["table"], sinks=c["sinks"], S=c["S"],
                               T=c["S"] * c["nq"], q_heads=c["Hq"], max_q=c["nq"], max_kv=s["most"], scale=s["scale"],
                               window=c["window"], otype=bf.OUT_F16)
        return [s["o"]]
    bf.lora(s["x"], s["ids"], s["parts"], s["c"], s["y"], T=c["T"], K=c["K"], adapters=c["E"], rank=c["rank"],
            ranks=s["ranks"], scales=s["scales"], ldc=s["c"].shape[1], ldy=s["c"].shape[1],
            otype=bf.OUT_F16 if c["out"] == "f16" else bf.OUT_F32)
    return [s["y"]]


def work(case):
    kind = case["kind"]
    size = {"f16": 2, "f32": 4, "none": 0}
    if kind == "norm":
        n = case["T"] * case["K"]
        out = 2 if case["out"] == "f16" else 1.25
        return {"bytes": int(n * (2 * size[case["x"]] + size[case["delta"]] + out)) + case["K"] * size[case["weight"]],
                "flops": 6 * n}
    if kind == "append":                           # queries in and out; keys and values in, 4.5 bits written and read, out
        q, kv = case["T"] * case["Hq"] * case["D"], 2 * case["T"] * case["H"] * case["D"]
        return {"bytes": 4 * q + 4 * kv + 2 * (9 * kv // 16) + 16 * case["T"], "flops": 3 * (q + kv // 2) + 4 * kv}
    if kind == "attn":
        rows = case["S"] * case["nq"] * case["Hq"] * case["D"]
        return {"bytes": sum(_reached(case)) * case["H"] * case["D"] * 9 // 8 + rows * 4,
                "flops": 4 * case["D"] * case["Hq"] * sum(_seen(case))}
    t, e, k, n = case["T"], case["E"], case["K"], sum(_widths(case))
    r = case["rank"] * (1.75 / 3 if case["mixed"] else 1)                        # the ranks' mean
    used = min(e, 6) if case["runs"] else e * (1 - (1 - (0.9 if t > 1 else 1) / e) ** t)   # adapters in use, on average
    parts = len(_widths(case))
    return {"bytes": int(used * r * (parts * k + n) * 2) + t * k * 2 + 2 * t * n * size[case["out"]],
            "flops": int(2 * t * r * (parts * k + n))}


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


def exact(case, seed):
    kind = case["kind"]
    if kind == "norm":
        x, delta, w = _norm_inputs(case, seed)
        r = x.double() if delta is None else x.double() + delta.double()
        y = r * (r.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * (w.double() + case["offset"])
        if case["out"] == "f16":
            return [r, y]
        b = y.reshape(case["T"], -1, GROUP)
        d = b.abs().amax(-1, keepdim=True) / 127
        return [r, torch.where(b < 0, torch.ceil(b / d - 0.5), torch.floor(b / d + 0.5)) * d]
    if kind == "append":
        q, k, v, position, _, freq, _ = _append_inputs(case, seed)
        return [_rotated64(q, position, freq, case)[0],
                _exact_cached(_rotated64(k, position, freq, case)[0].to(torch.float16)),   # (the cache takes fp16 keys)
                _exact_cached(v)]
    if kind == "attn":
        _, lens, q, k, v = _attn_inputs(case, seed)
        nq, r, w = case["nq"], case["Hq"] // case["H"], case["window"]
        out = torch.empty(q.shape, dtype=torch.float64, device=DEV)
        at = 0
        for i, n in enumerate(lens):
            pos = torch.arange(n - nq, n, device=DEV)[:, None]
            t = torch.arange(n, device=DEV)[None, :]
            see = (t <= pos) & ((t > pos - w) | (t < case["sinks"]))
            some = torch.nonzero(see.any(0))[:, 0]
            for h in range(case["H"]):
                kk, vv = _exact_cached(k[at:at + n, h][some]), _exact_cached(v[at:at + n, h][some])
                for j in range(h * r, (h + 1) * r):
                    x = (q[i * nq:(i + 1) * nq, j].double() @ kk.t()) / math.sqrt(case["D"])
                    out[i * nq:(i + 1) * nq, j] = torch.softmax(x.masked_fill(~see[:, some], float("-inf")), -1) @ vv
            at += n
        return [out]
    x, ids, ranks, scales, ab, c = _lora_inputs(case, seed)
    out = c.double()
    at = 0
    for (a, b), n in zip(ab, _widths(case)):
        for e in range(case["E"]):
            rows = torch.nonzero(ids == e)[:, 0]
            if rows.numel():
                m = int(ranks[e])
                y = (x[rows].double() @ a[e, :m].double().t()) @ b[e, :, :m].double().t()
                out[rows, at:at + n] += float(scales[e]) * y
        at += n
    return [out]
