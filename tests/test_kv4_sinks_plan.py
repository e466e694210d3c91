"""Attention with first tokens in sight, without a GPU: what it plans for where the window
covers the cache already.  tests/kv4_sinks_plan_check.cpp compiled with g++, and the entry
point's sizes."""
import os
import shutil
import subprocess

import pytest

import busfill as bf
from test_ops_abi import attention, cache

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_plans(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    exe = str(tmp_path / "kv4_sinks_plan_check")
    subprocess.run([gxx, "-O2", "-std=c++17", "-Wall", "-Wextra", "-Werror", "-I", os.path.join(ROOT, "bus-fill_amd", "csrc"),
                    os.path.join(ROOT, "tests", "kv4_sinks_plan_check.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr


@pytest.mark.parametrize("S,max_kv,window", [(8, 8000, 8000), (16, 1200, 4096), (2, 131072, 1 << 20)])
def test_first_tokens_inside_the_window_take_no_workspace(S, max_kv, window):
    c = cache(pages=1 << 16, kv_heads=8, head_dim=128)
    a = attention(S=S, T=S, q_heads=8, max_kv=max_kv, ldt=4096, window=window, ldq=1024, ldo=1024)
    sizes = [bf.kv4_attention_sinks_workspace_bytes(c, a, n) for n in (0, 4, 100, 4000, 1 << 30)]
    assert len(set(sizes)) == 1
    assert S != 16 or sizes[0] == 0                                # (a workgroup a sequence: 1200 tokens)
