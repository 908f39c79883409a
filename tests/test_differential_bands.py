"""The bands that four latitudes share cover exactly the pairs of the CSR."""

import ctypes
import subprocess
import sys

import numpy as np
import pytest
import torch

from torch_harmonics_amd import _lib, precompute_neighborhood_s2
from torch_harmonics_amd.plan import build_host_blob

from .diff_util import mask_of


def quads(plan):
    h, PH = plan.header, _lib.PH
    ng, ns = (h[PH["NVOUT"]] + 3) // 4, (h[PH["NVIN"]] + 3) // 4
    at, blob = h[PH["QUADS"]], plan.blob.numpy()
    lists = [blob[at : at + 4 * ng].reshape(ng, 4), blob[at + 4 * ng : at + 4 * (ng + ns)].reshape(ns, 4)]
    at += 4 * (ng + ns)
    total = sum(int((t[:, 2] - t[:, 1]).sum()) for t in lists)
    assert (blob[at + 8 * total : at + 8 * total + 8] == 0).all() and at + 8 * total + 8 <= len(blob)
    return lists, blob[at : at + 8 * total].reshape(total, 8)


def pairs_of(groups, bands, nv, W, sigma, rho, shape):
    """How often each own point sees each other point, from the bands."""
    M = np.zeros(shape, dtype=np.int64)
    w = np.arange(W)
    for g, begin, end, zero in groups.tolist():
        assert zero == 0
        for band in bands[begin:end].tolist():
            lat, aux, ws, ln = band[:4]
            assert aux == lat // rho and 0 <= ws < W
            first, last, rings = [], [], False
            for i in range(4):
                vo, d, n = 4 * g + i, band[4 + i] >> 16, band[4 + i] & 0xFFFF
                if n == 0:
                    continue
                if n == 0xFFFF:  # the whole ring: positions 0 .. W, seen by all columns of a tile wherever it is
                    assert vo < nv and d == 0 and ln + 15 >= W
                    rings = True
                    own, other = np.meshgrid((vo // sigma) * sigma * W + vo % sigma + w * sigma, (lat // rho) * rho * W + lat % rho + w * rho)
                    np.add.at(M, (own, other), 1)
                    continue
                assert vo < nv and 0 <= d and d + n <= ln
                first.append(d), last.append(d + n)
                for t in range(d, d + n):
                    own = (vo // sigma) * sigma * W + vo % sigma + w * sigma
                    other = (lat // rho) * rho * W + lat % rho + (ws + t + w) % W * rho
                    np.add.at(M, (own, other), 1)
            if first:
                assert min(first) == 0 and (max(last) == ln or rings and ln == max(max(last), W - 15))
            else:
                assert rings and ln == max(1, W - 15)
    return M


@pytest.mark.parametrize(
    "ins,outs,theta",
    [((12, 24), (12, 24), 0.5), ((9, 17), (9, 17), 0.9), ((12, 24), (6, 12), 0.6), ((6, 12), (12, 24), 0.6), ((5, 11), (9, 33), 0.8), ((7, 8), (7, 8), 3.2), ((2, 4), (2, 4), 0.4), ((33, 16), (33, 16), 0.2), ((16, 48), (8, 16), 0.5), ((8, 16), (16, 48), 0.5)],
)
def test_bands_cover_exactly_the_pairs(ins, outs, theta):
    up = outs[1] > ins[1]
    col, roff, _ = precompute_neighborhood_s2(*((outs, ins) if up else (ins, outs)), theta_cutoff=theta)
    check(col, roff, ins, outs)


def check(col, roff, ins, outs):
    up = outs[1] > ins[1]
    plan = build_host_blob(col, roff, *ins, *outs)
    (gather, scatter), bands = quads(plan)
    W = min(ins[1], outs[1])
    qps, kps = (outs[1] // W, 1) if up else (1, ins[1] // W)
    want = mask_of(col, roff, *ins, *outs).numpy()
    for groups, nv, sigma, rho, T in ((gather, outs[0] * qps, qps, kps, want), (scatter, ins[0] * kps, kps, qps, want.T)):
        assert sorted(groups[:, 0].tolist()) == list(range((nv + 3) // 4))
        assert np.array_equal(pairs_of(groups, bands, nv, W, sigma, rho, T.shape), T)
    return [int((t[:, 2] - t[:, 1]).sum()) for t in (gather, scatter)]


def test_bands_of_any_csr():
    """Columns in no order, duplicates, gaps, empty rows."""
    gen = torch.Generator().manual_seed(5)
    for n in (3, 17, 60):
        rows = [torch.randint(0, 6 * 20, (int(torch.randint(0, n, (1,), generator=gen)),), generator=gen) for _ in range(6)]
        rows[2] = rows[2][:0]
        check(torch.cat(rows), torch.tensor([0] + list(np.cumsum([len(r) for r in rows]))), (6, 20), (6, 20))


def test_the_order_of_psi_does_not_matter():
    """Columns from the west of the meridian on, as arcs come out of an arc cosine, or ascending: as many bands.  (A full ring may start anywhere.)"""
    col, roff, _ = precompute_neighborhood_s2((12, 40), (12, 40), theta_cutoff=0.5)
    lat, lon = col // 40, col % 40
    moved = torch.cat([torch.tensor(sorted(c.tolist(), key=lambda x: (x // 40, (x % 40 + 20) % 40)), dtype=torch.int64) for c in col.split((roff[1:] - roff[:-1]).tolist())])
    assert not torch.equal(col, moved)
    assert check(col, roff, (12, 40), (12, 40)) == check(moved, roff, (12, 40), (12, 40))


@pytest.mark.parametrize(
    "dtype,d,cv,nlon,alignment,want",
    [("fp32", 16, 32, 40, 4, "split"), ("fp32", 16, 32, 31, 4, "vector"), ("fp32", 3, 32, 40, 4, "vector"), ("fp32", 64, 128, 40, 4, "split"), ("fp32", 68, 128, 40, 4, "vector"),
     ("bf16", 32, 64, 40, 16, "16bit"), ("bf16", 32, 64, 40, 8, "split"), ("bf16", 20, 36, 40, 16, "split"), ("fp16", 64, 128, 40, 16, "16bit"), ("fp16", 64, 128, 40, 8, "vector"), ("bf16", 16, 32, 16200, 16, "vector")],
)  # fmt: skip
def test_families_of_kernels(dtype, d, cv, nlon, alignment, want):
    """What a problem's widths, columns and alignment lead to; grids too wide for the bands' packed numbers have none."""
    lib = _lib.load()
    col, roff = torch.arange(-2, 3) % nlon, torch.tensor([0, 5, 5])
    plan = build_host_blob(col, roff, 2, nlon, 2, nlon)
    assert (plan.header[_lib.PH["QUADS"]] > 0) == (nlon < 0x3F00)
    shape = _lib.ShapeStruct(batch=1, num_heads=2, nlat_in=2, nlon_in=nlon, nlat_out=2, nlon_out=nlon, ck=d, cv=cv, dtype=["fp32", "bf16", "fp16"].index(dtype))
    rc = lib.s2attn_diff_family(ctypes.byref(plan.struct), ctypes.byref(shape), alignment)
    assert _lib.FAMILIES[_lib.check(rc, "family")] == want


def test_a_header_that_points_outside_the_plan_is_refused():
    lib = _lib.load()
    plan = build_host_blob(torch.arange(5), torch.tensor([0, 5, 5]), 2, 40, 2, 40)
    shape = _lib.ShapeStruct(batch=1, num_heads=2, nlat_in=2, nlon_in=40, nlat_out=2, nlon_out=40, ck=16, cv=32, dtype=0)
    bad = _lib.PlanStruct.make(plan.blob.data_ptr(), list(plan.header))
    for at in (-5, 3, int(plan.header[_lib.PH["TOTAL"]]) - 4):
        bad.header[_lib.PH["QUADS"]] = at
        assert lib.s2attn_diff_family(ctypes.byref(bad), ctypes.byref(shape), 16) == -1
        assert b"bands" in lib.s2attn_last_error()


def test_a_plan_that_memory_does_not_hold_is_an_error():
    """In a process of its own, whose memory is limited: an exception that left the C entry would end it."""
    code = """
import ctypes, resource
from torch_harmonics_amd import _lib
lib = _lib.load()
col, off = (ctypes.c_int64 * 1)(0), (ctypes.c_int64 * 2)(0, 1)
size = int(open("/proc/self/statm").read().split()[0]) * resource.getpagesize() + (256 << 20)
resource.setrlimit(resource.RLIMIT_AS, (size, size))
rc = lib.s2attn_plan_size(ctypes.cast(col, ctypes.c_void_p), ctypes.cast(off, ctypes.c_void_p), 1, 1, 1, 1 << 26, 2)
assert rc == -2 and b"plan" in lib.s2attn_last_error(), (rc, lib.s2attn_last_error())
print("refused")
"""
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and "refused" in out.stdout, out.stderr[-500:]
