# A neighborhood's arcs may be listed in ascending columns or from their west ends on: the plan is the same.

import numpy as np
import pytest
import torch

from torch_harmonics_amd.plan import build_host_blob


def _csr(nlat, nlon_other, nlat_other, half, west_first):
    cols, off = [], [0]
    for r in range(nlat):
        for lat in range(nlat_other):
            m = half(r, lat)
            if m < 0:
                continue
            w = np.arange(nlon_other) if 2 * m + 1 >= nlon_other else np.arange(-m, m + 1) % nlon_other
            cols += (lat * nlon_other + (w if west_first else np.sort(w))).tolist()
        off.append(len(cols))
    return torch.tensor(cols), torch.tensor(off)


@pytest.mark.parametrize("ins, outs", [((5, 36), (5, 36)), ((7, 72), (4, 36)), ((4, 36), (7, 72)), ((3, 4), (3, 4)), ((2, 1), (2, 1))])
def test_order_of_an_arcs_columns_does_not_matter(ins, outs):
    up = outs[1] > ins[1]
    rows, other = (ins, outs) if up else (outs, ins)
    half = lambda r, lat: min(other[1], 3 + 2 * abs(r - lat)) if (r + lat) % 3 else -1 + (r + lat) % 2
    blobs = [build_host_blob(*_csr(rows[0], other[1], other[0], half, west), *ins, *outs).blob for west in (False, True)]
    assert torch.equal(*blobs)


def test_arcs_that_do_not_meet_stay_apart():
    # columns 10, 11 and 0, 1 of twelve meet; 9, 10 and 0, 1 do not; two arcs that overlap past a whole ring are not joined
    runs = lambda cols: build_host_blob(torch.tensor(cols), torch.tensor([0, len(cols)]), 1, 12, 1, 12).arrays()[1][:, 1:3].tolist()
    assert runs([10, 11, 0, 1]) == [[10, 4]] == runs([0, 1, 10, 11])
    assert sorted(runs([9, 10, 0, 1])) == [[0, 2], [9, 2]]
    assert sorted(runs([4, 5, 6, 7, 8, 9, 10, 11, 0, 1, 2, 3])) == [[4, 12]]
    assert sorted(runs([3, 4, 5, 6, 7, 8, 9, 10, 11, 0, 1, 2, 3])) == [[0, 4], [3, 9]]
