"""Low-rank adapters: a stream's workspace after a call of many rows, and a caller's of that
size, serve calls of fewer (run on an MI355X)."""
import pytest
import torch

import busfill as bf
from test_gpu_lora import Case

pytestmark = pytest.mark.gpu


def cases():
    return [Case(T, 5120, [512, 128, 128], 32, 64, otype=bf.OUT_F16) for T in (128, 32, 1)]


def test_captured_after_a_call_of_more_rows():
    """128 rows on a stream of its own, then 32 and one captured there."""
    most, *fewer = cases()
    st = torch.cuda.Stream()
    kw = most.device()
    y = torch.empty_like(most.dc)
    bf.lora(most.dx, most.dids, most.parts, most.dc, y, stream=st, **kw)
    torch.cuda.synchronize()
    most.check(y)
    for c in fewer:
        kw, y = c.device(), torch.zeros_like(c.c, device="cuda")
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            bf.lora(c.dx, c.dids, c.parts, c.dc, y, **kw)
        for _ in range(3):
            y.zero_()
            graph.replay()
            torch.cuda.synchronize()
            c.check(y)


def test_a_workspace_of_the_most_rows():
    most, *fewer = cases()
    kw = most.device()
    args = bf.lora_args(most.dx, most.dids, most.parts, most.dc, most.dc, **kw)
    n = bf.lora_workspace_bytes(args)
    ws = torch.full((n,), 0xFF, dtype=torch.uint8, device="cuda")
    for c in fewer:
        kw, y = c.device(), torch.empty_like(c.c, device="cuda")
        bf.lora_ws(bf.lora_args(c.dx, c.dids, c.parts, c.dc, y, **kw), ws, n)
        torch.cuda.synchronize()
        c.check(y)
