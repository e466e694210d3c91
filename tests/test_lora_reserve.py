"""The low-rank adapters' workspace, without a GPU: a size that serves T rows serves
fewer.  tests/lora_reserve_check.cpp compiled with g++, and the entry point's sizes."""
import os
import shutil
import subprocess

import pytest

import busfill as bf
from test_layer_ops_abi import FAKE, lora

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_plan(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    exe = str(tmp_path / "lora_reserve_check")
    subprocess.run([gxx, "-O2", "-std=c++17", "-Wall", "-Wextra", "-Werror", "-I", os.path.join(ROOT, "bus-fill_amd", "csrc"),
                    os.path.join(ROOT, "tests", "lora_reserve_check.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr


@pytest.mark.parametrize("rank,adapters", [(64, 32), (16, 8), (128, 4)])
def test_fewer_rows_need_no_more(rank, adapters):
    """A query, key and value projection of 5120 columns and twice 1024."""
    slices = [(FAKE, FAKE, 5120, 0), (FAKE, FAKE, 1024, 5120), (FAKE, FAKE, 1024, 6144)]
    sizes = []
    for T in list(range(1, 700)) + [1152, 1200, 2000, 4000, 8000]:
        a, kept = lora(slices, T=T, K=5120, ldx=5120, ldc=7168, ldy=7168, rank=rank, adapters=adapters)
        sizes.append(bf.lora_workspace_bytes(a))
    assert sizes[0] > 0 and sizes == sorted(sizes)
