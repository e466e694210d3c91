#!/usr/bin/env python3
"""A mixture-of-experts decoder layer over 4-bit weights and a 4-bit key/value
cache, with every linear, the cache, attention, routing and experts' block
through the library:

    h = norm(x);  q k v = Wqkv h;  q, k rotated by position
    cache[slots] = k, v          kv4_store
    x += Wo attention(q, cache)  kv4_attention
    h = norm(x);  ids, weights = route(Wr h)      moe_route
    x += experts(h, ids, weights)                 moe_ffn

    python examples/moe_decoder.py [--streams 32] [--prompt 2000] [--steps 50]

takes in a prompt per stream, then decodes with one captured graph (lengths,
slots and positions are device memory, so the graph serves every step) and
prints the time of both.  Weights are random: this shows calls and times, not
language.  The norms and the rotation are torch.
"""
import argparse
import math
import os
import sys
import time

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "bus-fill_amd"))
import busfill as bf  # noqa: E402

PAGE = 64


class Shape:
    def __init__(self, width=5120, q_heads=40, kv_heads=8, dim=128, experts=64, chosen=8, ffn=1280):
        self.width, self.q_heads, self.kv_heads, self.dim = width, q_heads, kv_heads, dim
        self.experts, self.chosen, self.ffn = experts, chosen, ffn
        self.qkv = (q_heads + 2 * kv_heads) * dim


def random_q4_k(n, k, gen, device="cuda"):
    """n x k random weights of Q4_K blocks, as bytes: standard deviation about 1 / sqrt(k)."""
    nb, step = k // 256, 1 / (4.7 * 43 * math.sqrt(k))
    blk = torch.randint(0, 256, (n, nb, 144), generator=gen, device=device, dtype=torch.uint8)
    d = torch.full((n, nb, 1), step, device=device)
    blk[..., 0:4] = torch.cat([d, 7.5 * d], -1).half().view(torch.uint8)
    sc = torch.randint(32, 56, (n, nb, 8), generator=gen, device=device, dtype=torch.uint8)   # scales, and mins alike
    blk[..., 4:8] = (sc[..., :4] & 63) | (sc[..., 4:] >> 4 << 6)
    blk[..., 8:12] = blk[..., 4:8]
    blk[..., 12:16] = (sc[..., 4:] & 15) * 17
    return blk.reshape(n, nb * 144)


class Cache:
    """Pages for `streams` streams of up to `tokens` tokens, each stream's pages spread over the whole."""

    def __init__(self, shape, streams, tokens):
        self.per = (tokens + PAGE - 1) // PAGE
        pages = streams * self.per
        self.data = torch.empty(bf.kv4_bytes(pages, PAGE, shape.kv_heads, shape.dim), dtype=torch.uint8, device="cuda")
        self.c = bf.kv4_cache(self.data, pages, PAGE, shape.kv_heads, shape.dim)
        self.table = torch.arange(pages, dtype=torch.int32, device="cuda").reshape(self.per, streams).t().contiguous()
        self.tokens = self.per * PAGE

    def slots(self, stream, position):
        return self.table[stream, position // PAGE].long() * PAGE + position % PAGE


def norm(x):
    return (x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)).half()


def rotate(x, position):
    """Rotates the halves of each head of x [rows][heads][dim] (fp16) by its position."""
    half = x.shape[-1] // 2
    a = position.float()[:, None] * 10000.0 ** (-torch.arange(half, device=x.device) / half)
    c, s = a.cos()[:, None], a.sin()[:, None]
    p, q = x.float().split(half, -1)
    return torch.cat([p * c - q * s, q * c + p * s], -1).half()


class Batch:
    """The buffers of a call of the layer on `rows` rows of `streams` streams, up to most_kv cached tokens each."""

    def __init__(self, shape, rows, streams, max_q, most_kv):
        self.rows, self.streams, self.max_q, self.most_kv = rows, streams, max_q, most_kv
        f16 = lambda *n: torch.empty(*n, dtype=torch.float16, device="cuda")
        self.x = torch.empty(rows, shape.width, device="cuda")     # fp32 residual rows
        self.qkv, self.att = f16(rows, shape.qkv), f16(rows, shape.q_heads * shape.dim)
        self.y, self.logits = f16(rows, shape.width), torch.empty(rows, shape.experts, device="cuda")
        self.ids = torch.empty(rows, shape.chosen, dtype=torch.int32, device="cuda")
        self.weights = torch.empty(rows, shape.chosen, device="cuda")
        self.position = torch.zeros(rows, dtype=torch.int64, device="cuda")
        self.slots = torch.zeros(rows, dtype=torch.int64, device="cuda")
        self.q_start = torch.zeros(streams + 1, dtype=torch.int32, device="cuda")
        self.kv_len = torch.zeros(streams, dtype=torch.int32, device="cuda")


class Layer:
    def __init__(self, shape, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        s = self.shape = shape
        self.wqkv = random_q4_k(s.qkv, s.width, g)
        self.wo = random_q4_k(s.width, s.q_heads * s.dim, g)
        self.wr = random_q4_k(s.experts, s.width, g)
        self.gate = random_q4_k(s.experts * s.ffn, s.width, g)
        self.up = random_q4_k(s.experts * s.ffn, s.width, g)
        self.down = random_q4_k(s.experts * s.width, s.ffn, g)

    def __call__(self, cache, b):
        """b.x through the layer, in place; its keys and values into the cache."""
        s, n, h16 = self.shape, b.rows, bf.OUT_F16
        b.h1 = norm(b.x)
        bf.gemm(bf.Q4_K, self.wqkv, None, b.h1, b.qkv, n, s.qkv, s.width, otype=h16)
        heads = b.qkv.view(n, -1, s.dim)
        qk = s.q_heads + s.kv_heads
        heads[:, :qk] = rotate(heads[:, :qk], b.position)
        bf.kv4_store(cache.c, heads[:, s.q_heads], heads[:, qk], b.slots, n, ldk=s.qkv, ldv=s.qkv)
        bf.kv4_attention(cache.c, b.qkv, b.att, b.q_start, b.kv_len, cache.table, S=b.streams, T=n, q_heads=s.q_heads,
                         max_q=b.max_q, max_kv=b.most_kv, scale=s.dim ** -0.5, ldq=s.qkv, otype=h16)
        bf.gemm(bf.Q4_K, self.wo, None, b.att, b.y, n, s.width, s.q_heads * s.dim, otype=h16)
        b.x += b.y
        b.h2 = norm(b.x)
        bf.gemm(bf.Q4_K, self.wr, None, b.h2, b.logits, n, s.experts, s.width)
        bf.moe_route(b.logits, b.ids, b.weights, n, s.experts, s.chosen)
        bf.moe_ffn(bf.Q4_K, (self.gate, None), (self.up, None), (self.down, None), b.h2, b.ids, b.weights, b.y, T=n,
                   K=s.width, F=s.ffn, N=s.width, E=s.experts, k=s.chosen, otype=h16)
        b.x += b.y


def prompt(layer, cache, streams, x):
    """Takes in the same number of tokens for every stream: x [streams][tokens][width]."""
    n = x.shape[1]
    b = Batch(layer.shape, streams * n, streams, n, n)
    b.x.copy_(x.reshape(streams * n, -1))
    b.position.copy_(torch.arange(n).repeat(streams))
    stream = torch.arange(streams, device="cuda").repeat_interleave(n)
    b.slots.copy_(cache.slots(stream, b.position))
    b.q_start.copy_(torch.arange(streams + 1) * n)
    b.kv_len.fill_(n)
    layer(cache, b)
    return b


class Decoder:
    """Single tokens of every stream, as one captured graph."""

    def __init__(self, layer, cache, streams, length):
        self.b = b = Batch(layer.shape, streams, streams, 1, cache.tokens)
        b.q_start.copy_(torch.arange(streams + 1))
        self.cache, self.every = cache, torch.arange(streams, device="cuda")
        b.x.zero_()
        self.side = torch.cuda.Stream()
        self._at(length)
        torch.cuda.synchronize()
        with torch.cuda.stream(self.side):         # allocates the stream's workspace
            layer(cache, b)
        self.side.synchronize()
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph, stream=self.side):
            layer(cache, b)
        self._at(length)

    def _at(self, length):
        """The next token is at position `length` of every stream."""
        self.length = length
        self.b.position.fill_(length)
        self.b.slots.copy_(self.cache.slots(self.every, self.b.position))
        self.b.kv_len.fill_(length + 1)

    def step(self, x):
        self.b.x.copy_(x)
        self.graph.replay()
        self._at(self.length + 1)
        return self.b.x


def main():
    p = argparse.ArgumentParser()
    p.add_argument("--streams", type=int, default=32)
    p.add_argument("--prompt", type=int, default=2000)
    p.add_argument("--steps", type=int, default=50)
    a = p.parse_args()
    layer = Layer(Shape())
    s = layer.shape
    cache = Cache(s, a.streams, a.prompt + a.steps + 3)
    x = torch.randn(1, a.prompt, s.width, device="cuda")

    def timed(f):
        torch.cuda.synchronize()
        t = time.perf_counter()
        f()
        torch.cuda.synchronize()
        return time.perf_counter() - t

    one = Cache(s, 1, a.prompt)
    prompt(layer, one, 1, x)
    t = timed(lambda: prompt(layer, one, 1, x))
    print(f"prompt of {a.prompt} tokens: {t * 1e3:.2f} ms a layer")
    cache.data.random_(0, 64)                      # as if every stream had taken one in: finite scales, any codes
    d = Decoder(layer, cache, a.streams, a.prompt)
    tok = torch.randn(a.streams, s.width, device="cuda")
    d.step(tok)
    t = timed(lambda: [d.step(tok) for _ in range(a.steps)])
    print(f"{a.streams} streams from {a.prompt} tokens on: {t / a.steps * 1e6:.1f} us a step and layer")
    assert torch.isfinite(d.b.x).all()


if __name__ == "__main__":
    main()
