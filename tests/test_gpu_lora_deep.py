"""Low-rank adapters of many rows and a K of several thousand, against 64 bits (run on an
MI355X): up to eight pieces of K, and up to sixteen slabs of 320 a piece, the last of
them partial; ranks of one block, of several, and of the sums' join.

Tolerance: as tests/test_gpu_lora.py derives it."""
import pytest
import torch

import busfill as bf
from test_gpu_lora import Case

pytestmark = pytest.mark.gpu


class Deep(Case):
    def want(self):
        """Case.want, an adapter's rows at once."""
        y = self.c.double()
        tol = torch.zeros_like(y)
        for (a, b), n, at in zip(self.ab, self.widths, self.at):
            for e in range(self.adapters):
                rows = torch.nonzero(self.ids == e)[:, 0]
                if not rows.numel():
                    continue
                r = self.rank if self.ranks is None else min(max(int(self.ranks[e]), 0), self.rank)
                f = 1.0 if self.scales is None else float(self.scales[e])
                ar, br, x = a[e, :r].double(), b[e, :, :r].double(), self.x[rows].double()
                s, m = x @ ar.t(), x.abs() @ ar.abs().t()
                ds = (self.K / 32 + 40) * 2.0 ** -23 * m
                if r:
                    ds += 2.0 ** -21 * s.abs().amax(-1, keepdim=True)
                y[rows, at:at + n] += f * (s @ br.t())
                tol[rows, at:at + n] = abs(f) * ((ds + (r / 16 + 4) * 2.0 ** -23 * s.abs()) @ br.abs().t())
        tol = tol * (1 + 2.0 ** -10) + (2.0 ** -23 + (2.0 ** -11 if self.otype == bf.OUT_F16 else 0)) * y.abs() + 2.0 ** -24
        return y, tol


def mixed(T, E, seed=0):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(-1, E, (T,), generator=g)
    ids[T // 3:T // 2] = E // 2                                            # a run among them
    return ids.tolist()


@pytest.mark.parametrize("K", [5120, 5000])
@pytest.mark.parametrize("T", [129, 300, 2000])
@pytest.mark.parametrize("rank,otype", [(16, bf.OUT_F16), (64, bf.OUT_F32), (136, bf.OUT_F32)])
def test_pieces(T, K, rank, otype):
    Deep(T, K, [70], 9, rank, ids=mixed(T, 9), otype=otype).run(workspace=True)


def test_odd_ranks_of_their_own():
    Deep(700, 5000, [70, 12], 8, 64, ids=mixed(700, 8), ranks=[64, 1, 0, 7, 33, 16, 63, 48]).run()


@pytest.mark.parametrize("T,K,rank,E,widths", [
    (2112, 5000, 256, 7, [64, 10]),                # one piece of sixteen slabs, four blocks of ranks, joined
    (4160, 5000, 16, 9, [20, 30, 1, 16]),          # one piece
    (2000, 5120, 64, 6, [40, 20, 20]),             # two pieces of eight slabs
    (700, 17408, 64, 5, [33]),                     # eight pieces of seven
])
def test_long_pieces(T, K, rank, E, widths):
    Deep(T, K, widths, E, rank, ids=mixed(T, E), otype=bf.OUT_F32).run()


def test_same_bits_again():
    """Whatever the workspace held, and run after run."""
    c = Deep(600, 5000, [130], 9, 64, ids=mixed(600, 9))
    first = c.run().clone()
    assert torch.equal(first, c.run(workspace=True)) and torch.equal(first, c.run())
