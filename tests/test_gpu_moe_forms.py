"""The experts' block in every form that the number of rows, experts and outputs
can select for few rows, against 64-bit references (tolerances: test_gpu_moe.py;
run on an MI355X)."""
import pytest
import torch

import busfill as bf
import oracle as O
from test_gpu_moe import QTS, Experts


def form(E, R, gu, T, k):
    """How the products of R weight rows an expert run below 24 slots an expert: parts along K, row tiles a pass, and
    whether a workgroup scans the slots itself (the rules of bus-fill_amd/csrc/bf_moe.hip)."""
    slots = T * k
    assert slots < 24 * E
    experts = min(E, slots)
    waves = (R + 15) // 16 * (2 if gu else 1) * experts
    ks = 4 if waves < 1536 else 2 if waves < 2 * 1536 else 1
    mt = 1 if slots <= 16 * E else 2
    return (2 if mt == 2 and ks == 4 else ks), mt, slots <= 1024


# E, K, F, N, T, k: gate and up's form, down's (its outputs off 16, or its slots, keep it from the whole-activation kernel)
SHAPES = [
    (48, 768, 768, 1040, 225, 4, (1, 2, True), (1, 2, True)),     # one wave a tile along K, three super-groups, two row tiles
    (64, 768, 512, 784, 300, 4, (1, 2, False), (1, 2, False)),    # ... by the plan's list
    (48, 256, 768, 1030, 100, 4, (1, 1, True), (1, 1, True)),     # one row tile, outputs off 16
    (64, 768, 512, 776, 260, 4, (1, 2, False), (1, 2, False)),
    (24, 768, 768, 1040, 130, 3, (2, 2, True), (2, 2, True)),     # two parts
    (24, 1280, 512, 1030, 90, 4, (2, 1, True), (2, 1, True)),     # two parts, five super-groups, one row tile
    (6, 768, 256, 200, 33, 4, (2, 2, True), (2, 2, True)),        # four parts would serve, two row tiles
    (64, 256, 768, 800, 1, 48, (1, 1, True), None),               # a row of 48 experts: down as one sum
    (6, 1280, 256, 40, 1, 6, (4, 1, True), None),                 # four parts, five super-groups
]


@pytest.mark.parametrize("E,K,F,N,T,k,gate,down", SHAPES)
def test_shapes_take_the_forms_that_they_are_there_for(E, K, F, N, T, k, gate, down):
    assert form(E, F, True, T, k) == gate
    if down:
        got = form(E, N, False, T, k)
        assert got == down and (N % 16 or got[1] == 2 or got[0] > 1)


@pytest.mark.gpu
@pytest.mark.parametrize("qt", QTS)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(map(str, s[:6])))
def test_few_rows(qt, shape):
    E, K, F, N, T, k, _, _ = shape
    x = Experts(qt, E, K, F, N, seed=3)
    x.check(T, k, otype=bf.OUT_F16 if qt == O.Q4_0 else bf.OUT_F32, workspace=qt == O.Q4_K)


@pytest.mark.gpu
@pytest.mark.parametrize("qt", QTS)
def test_few_rows_unevenly(qt):
    """Most slots on two experts (several passes of 32 rows and a rest), the others with one or none."""
    E, T, k = 48, 225, 4
    x = Experts(qt, E, 768, 768, 1040, seed=5)
    ids = torch.full((T, k), 7)
    ids[:, 1] = torch.where(torch.arange(T) % 3 == 0, 47, 7)
    ids[:, 2] = torch.arange(T) % 40
    ids[:, 3] = -1
    x.check(T, k, ids=ids)
