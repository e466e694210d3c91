"""The plans of the shapes in test_gpu_kv4_forms.py, on the CPU: each takes the
form that it is there for (bus-fill_amd/csrc/bf_kv4_plan.h compiled with g++)."""
import os
import shutil
import subprocess

import pytest

from test_gpu_kv4_forms import FORMS
from test_gpu_kv4_range import FORMS as RANGES

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SOURCE = r"""
#include <cstdio>
#include <cstdlib>
#include "bf_kv4_plan.h"
int main(int argc, char** argv) {
    int v[9];
    if (argc != 10) return 2;
    for (int i = 0; i < 9; i++) v[i] = std::atoi(argv[1 + i]);
    bf::Kv4Args a{};
    a.c = bf::Kv4Shape{1, 64, v[2], v[8]};
    a.S = v[0]; a.T = v[1]; a.q_heads = v[2] * v[3]; a.max_q = v[4]; a.max_kv = v[5]; a.causal = v[6]; a.window = v[7];
    const bf::Kv4Plan p = bf::plan_kv4(a, 256);
    std::printf("%d %d %d %d %d\n", p.prompt, p.chunk, p.splits, p.waves, p.row_tiles);
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    at = tmp_path_factory.mktemp("plan")
    (at / "plan.cpp").write_text(SOURCE)
    subprocess.run([gxx, "-O1", "-std=c++17", "-I", os.path.join(ROOT, "bus-fill_amd", "csrc"), str(at / "plan.cpp"), "-o",
                    str(at / "plan")], check=True)

    def run(S, T, heads, group, max_q, max_kv, window, dim):
        out = subprocess.run([str(at / "plan"), *map(str, (S, T, heads, group, max_q, max_kv, 1, window, dim))], check=True,
                             capture_output=True, text=True, timeout=60).stdout.split()
        return dict(zip(("prompt", "chunk", "splits", "waves", "row_tiles"), map(int, out)))
    return run


WANT = {
    "16-wave join": lambda p: p["splits"] > 32 and p["waves"] == 8,
    "16-wave join, shorter": lambda p: p["splits"] > 32,
    "chunks of four waves": lambda p: p["splits"] > 1 and p["waves"] == 4 and p["chunk"] == 20,
    "chunks of four waves, wide heads": lambda p: p["splits"] > 1 and p["waves"] == 4,
    "whole, eight waves": lambda p: p["splits"] == 1 and p["waves"] == 8 and 40 < p["chunk"] <= 256,
    "chunks in a window": lambda p: p["splits"] > 1 and p["chunk"] == 8,
    "chunks in a window, queries": lambda p: p["splits"] > 1 and p["row_tiles"] == 10,
    "chunks, queries": lambda p: p["splits"] > 1 and p["row_tiles"] > 1,
}


@pytest.mark.parametrize("form,dim", [(f, d) for f in FORMS for d in FORMS[f][5]])
def test_forms(plan, form, dim):
    lens, heads, group, nqs, window, _, most = FORMS[form]
    p = plan(len(lens), sum(nqs), heads, group, max(nqs), most, window, dim)
    assert not p["prompt"] and WANT[form](p), p


def test_ranges(plan):
    of = {f: plan(S, S * nq, heads, group, nq, n, 0, 128) for f, (S, n, heads, group, nq) in RANGES.items()}
    assert of["prompt"]["prompt"] == 1 and sum(p["prompt"] for p in of.values()) == 1
    assert of["whole"]["splits"] == 1 and of["eight waves"]["splits"] == 1 and of["eight waves"]["waves"] == 8
    assert of["chunks"]["splits"] > 1 and of["chunks"]["waves"] == 8
    assert of["four waves"]["splits"] > 1 and of["four waves"]["waves"] == 4
