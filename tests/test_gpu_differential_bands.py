"""Differential attention on bands that four latitudes share: any psi, partial groups and tiles, batches and heads that make eight, a NaN next to a band."""

import math

import pytest
import torch

from .test_gpu_differential import BF16, F16, F32, check, geometry, run, tensors

pytestmark = pytest.mark.gpu

WIDTHS = [(F32, 16, 32), (F32, 20, 36), (F32, 8, 16), (F32, 64, 128), (BF16, 16, 32), (BF16, 32, 64), (BF16, 64, 128), (F16, 32, 40), (BF16, 20, 36)]


def any_psi(ins, outs, seed):
    """Rows of points in no order, some of them twice, some rows empty, some long."""
    g = torch.Generator().manual_seed(seed)
    up = outs[1] > ins[1]
    rows, other = (ins, outs) if up else (outs, ins)
    n = other[0] * other[1]
    cols = []
    for r in range(rows[0]):
        few = torch.randint(0, n, (int(torch.randint(0, 40, (1,), generator=g)),), generator=g)
        start, length = int(torch.randint(0, other[1], (1,), generator=g)), int(torch.randint(1, other[1] + 1, (1,), generator=g))
        arc = (start + torch.arange(length)) % other[1] + other[1] * int(torch.randint(0, other[0], (1,), generator=g))
        cols.append([few, torch.cat([few, arc]), torch.cat([arc, few[:5], few[:5]]), few[:0]][r % 4])
    roff = torch.tensor([0] + [len(c) for c in cols]).cumsum(0)
    quad = torch.rand(ins[0], generator=g) + 0.05
    return quad, torch.cat(cols), roff


@pytest.mark.parametrize("dtype,d,cv", WIDTHS)
@pytest.mark.parametrize("ins,outs", [((6, 36), (6, 36)), ((7, 72), (5, 36)), ((5, 36), (7, 72)), ((9, 33), (9, 33))])
def test_any_psi(ins, outs, dtype, d, cv):
    check(ins, outs, 1, 2, d, cv, dtype, None, geo=any_psi(ins, outs, 3))


@pytest.mark.parametrize("dtype,d,cv", [(F32, 16, 32), (BF16, 32, 64)])
@pytest.mark.parametrize("B,nh", [(2, 4), (1, 8), (4, 4), (3, 3)])
def test_batches_times_heads(B, nh, dtype, d, cv):
    check((9, 50), (9, 50), B, nh, d, cv, dtype, 0.6)


@pytest.mark.parametrize("dtype,d,cv", [(F32, 16, 32), (F32, 32, 64), (BF16, 32, 64), (F16, 16, 32)])
@pytest.mark.parametrize("nlat", [1, 2, 3, 4, 5, 6])
def test_groups_that_are_not_full(nlat, dtype, d, cv):
    ins = (nlat, 40)
    geo = geometry(ins, ins, 1.2) if nlat > 1 else (torch.ones(1), torch.arange(-5, 6) % 40, torch.tensor([0, 11]))
    check(ins, ins, 2, 2, d, cv, dtype, 1.2, geo=geo)


@pytest.mark.parametrize("dtype,d,cv", [(F32, 16, 32), (BF16, 32, 64)])
def test_a_ring_that_only_one_of_four_sees(dtype, d, cv):
    """NaN in rows that the workgroup stages for one latitude: the other three are as without."""
    ins = (8, 48)
    quad, col, roff = geometry(ins, ins, 0.45)
    t = tensors(ins, ins, 1, 2, d, cv, dtype)
    want = run(*t, quad, col, roff, 2, ins, ins)
    k, v = t[0].clone(), t[1].clone()
    k[:, 0], v[:, 0] = math.nan, math.nan
    got = run(k, v, *t[2:], quad, col, roff, 2, ins, ins)
    sees = torch.tensor([bool((c < 48).any()) for c in col.split((roff[1:] - roff[:-1]).tolist())])
    assert sees.any() and not sees[:4].all()
    for n in ("y", "dq"):
        assert torch.isnan(got[n][:, sees]).all() and torch.equal(got[n][:, ~sees], want[n][:, ~sees])
