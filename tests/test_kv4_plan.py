"""The 4-bit cache's layout and the attention's plans (plain C++ headers under
bus-fill_amd/csrc) checked on the CPU: tests/kv4_plan_check.cpp compiled with g++."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def checker(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    exe = str(tmp_path_factory.mktemp("kv4") / "kv4_plan_check")
    subprocess.run([gxx, "-O2", "-std=c++17", "-Wall", "-Wextra", "-Werror",
                    "-I", os.path.join(ROOT, "bus-fill_amd", "csrc"),
                    os.path.join(ROOT, "tests", "kv4_plan_check.cpp"), "-o", exe], check=True)
    return exe


@pytest.mark.parametrize("part", ["layout", "plans"])
def test_kv4(checker, part):
    r = subprocess.run([checker, part], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr


def plan(checker, *shape):
    r = subprocess.run([checker, "plan", *map(str, shape)], capture_output=True, text=True, check=True, timeout=60)
    return tuple(map(int, r.stdout.split()))


@pytest.mark.parametrize("S,T,heads,group,max_q,max_kv,causal,window", [
    (8, 201, 40, 4, 50, 150, 1, 0), (4, 196, 40, 4, 70, 130, 0, 0), (4, 196, 64, 3, 70, 130, 1, 40),
    (4, 196, 32, 16, 70, 130, 1, 0), (4, 196, 48, 5, 70, 130, 1, 1), (4, 196, 32, 7, 70, 130, 1, 0),
    (1, 600, 16, 8, 600, 600, 1, 0), (2, 600, 8, 16, 300, 330, 1, 0), (1, 120, 128, 4, 120, 120, 1, 0),
    (1, 2000, 8, 5, 2000, 2000, 1, 0)])
def test_prompts_take_the_prompt_kernel(checker, S, T, heads, group, max_q, max_kv, causal, window):
    """The prompts of the GPU tests (and one of 2000 tokens, 40 heads over 8) take the kernel that they are there for."""
    assert plan(checker, S, T, heads, group, max_q, max_kv, causal, window)[0] == 1


def test_other_queries_do_not(checker):
    assert plan(checker, 1, 1000, 8, 5, 1000, 1000, 1, 0)[0] == 0
    assert plan(checker, 1, 512, 8, 5, 512, 8000, 1, 0)[0] == 0
    assert plan(checker, 32, 32, 8, 5, 1, 8000, 1, 0) == (0, 250, 1, 8)          # whole sequences
    assert plan(checker, 32, 32, 8, 4, 1, 8192, 1, 0) == (0, 256, 1, 8)
    assert plan(checker, 1, 1, 4, 8, 1, 131072, 1, 0) == (0, 64, 64, 8)          # as many chunks as CUs
    assert plan(checker, 20, 20, 8, 5, 1, 8000, 1, 0)[2:] == (13, 4)             # chunks that even out
