"""Differential attention on the GPU against its definition in 64 bits: types, widths, grids, directions, points that see nothing, values that
are not finite, strides, streams, graphs."""

import math

import pytest
import torch

from .diff_util import HALF_STEP, assert_near, mask_of, reference
from torch_harmonics_amd import differential_s2_attention, neighborhood_s2_attention, precompute_latitudes, precompute_neighborhood_s2

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def geometry(ins, outs, theta, gi="equiangular", go="equiangular"):
    up = outs[1] % ins[1] == 0 and outs[1] != ins[1]
    args = (outs, ins, go, gi) if up else (ins, outs, gi, go)
    col, roff, _ = precompute_neighborhood_s2(*args, theta_cutoff=theta)
    quad = (2.0 * math.pi * precompute_latitudes(ins[0], grid=gi)[1].float() / ins[1]).contiguous()
    return quad, col, roff


def tensors(ins, outs, B, nh, d, cv, dtype, seed=0, lam_dtype=None, smooth=0.0):
    g = torch.Generator().manual_seed(seed)
    r = lambda hw, c: torch.randn(B, *hw, c, generator=g) + smooth * torch.randn(B, 1, 1, c, generator=g)  # noqa: E731
    k, v, q, dy = r(ins, 2 * nh * d), r(ins, nh * cv), r(outs, 2 * nh * d) / math.sqrt(d), torch.randn(B, *outs, nh * cv, generator=g)
    lam = torch.rand(nh, generator=g) * 1.4 - 0.5
    return *[t.to(dtype) for t in (k, v, q)], lam.to(lam_dtype or dtype), dy.to(dtype)


def run(k, v, q, lam, dy, quad, col, roff, nh, ins, outs):
    leaves = [t.detach().cuda().requires_grad_(True) for t in (k, v, q, lam)]
    y = differential_s2_attention(*leaves, quad.cuda(), col.cuda(), roff.cuda(), nh, ins[1], *outs)
    grads = torch.autograd.grad(y, leaves, dy.cuda())
    return dict(zip(("y", "dk", "dv", "dq", "dlam"), (y.detach(), *grads)))


def check(ins, outs, B, nh, d, cv, dtype, theta, lam_dtype=None, geo=None, **more):
    geo = geo or geometry(ins, outs, theta)
    t = tensors(ins, outs, B, nh, d, cv, dtype, lam_dtype=lam_dtype, **more)
    got = run(*t, *geo, nh, ins, outs)
    assert_near(got, reference(*t, geo[0], mask_of(*geo[1:], *ins, *outs), nh), dtype, lam_dtype)
    return got


GRIDS = {
    "self": ((12, 64), (12, 64), 0.5), "odd": ((9, 37), (9, 37), 0.7), "narrow": ((8, 11), (8, 11), 0.9), "down": ((14, 72), (7, 36), 0.6), "up": ((7, 36), (14, 72), 0.6),
    "down3": ((9, 99), (5, 33), 0.8), "up3": ((5, 33), (9, 99), 0.8), "wide": ((6, 160), (6, 160), 0.7), "point": ((1, 1), (1, 1), 1.0), "ring": ((2, 40), (2, 40), 0.3),
}  # fmt: skip


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("grid", GRIDS)
def test_grids_and_directions(grid, dtype):
    ins, outs, theta = GRIDS[grid]
    if grid == "point":
        geo = (torch.tensor([0.3]), torch.tensor([0]), torch.tensor([0, 1]))
        check(ins, outs, 2, 2, 16, 32, dtype, theta, geo=geo)
    else:
        check(ins, outs, 2, 2, 16, 32, dtype, theta)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("d,cv", [(1, 1), (3, 5), (4, 8), (8, 16), (8, 8), (12, 20), (16, 16), (20, 36), (24, 48), (24, 16), (32, 64), (32, 20), (8, 64), (40, 80), (64, 128), (64, 24), (16, 100), (96, 130), (256, 512)])
def test_head_widths(d, cv, dtype):
    check((7, 40), (7, 40), 1, 3 if d < 64 else 1, d, cv, dtype, 0.6)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("lam_dtype", [F32, BF16, F16])
def test_types_of_the_learned_weight(dtype, lam_dtype):
    check((6, 48), (6, 48), 2, 4, 16, 32, dtype, 0.8, lam_dtype=lam_dtype)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("d", [16, 32, 64, 20])
def test_smooth_fields(d, dtype):
    """Keys and values that share a large part: the sums of dS cancel, so the means have to fit the probabilities."""
    check((9, 64), (9, 64), 1, 2, d, 2 * d, dtype, 0.6, smooth=3.0)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("ins,outs", [((10, 64), (10, 64)), ((10, 64), (5, 32)), ((5, 32), (10, 64))])
def test_points_that_see_nothing(ins, outs, dtype):
    quad, col, roff = geometry(ins, outs, 0.7)
    nrow = roff.numel() - 1
    keep = torch.ones(nrow, dtype=torch.bool)
    keep[[0, nrow // 2]] = False  # rows of psi without an entry
    n = roff[1:] - roff[:-1]
    rows = torch.repeat_interleave(torch.arange(nrow), n)
    col, n = col[keep[rows]], torch.where(keep, n, torch.zeros_like(n))
    roff = torch.cat([torch.zeros(1, dtype=torch.int64), n.cumsum(0)])
    quad = quad.clone()
    quad[-4:] = 0.0  # latitudes of weight zero: some points see nothing else
    got = check(ins, outs, 2, 2, 16, 32, dtype, 0.7, geo=(quad, col, roff))
    M = mask_of(col, roff, *ins, *outs) * quad.double().repeat_interleave(ins[1])
    blind = (M.sum(1) == 0).view(*outs)
    assert blind.any() and (got["y"].cpu()[:, blind] == 0).all() and (got["dq"].cpu()[:, blind] == 0).all()


def test_psi_without_entries_and_empty_batches():
    quad, col, roff = geometry((6, 32), (6, 32), 0.5)
    t = tensors((6, 32), (6, 32), 1, 2, 8, 16, F32)
    got = run(*t, quad, col[:0], torch.zeros_like(roff), 2, (6, 32), (6, 32))
    assert all((x == 0).all() for x in got.values())
    t = tensors((6, 32), (6, 32), 0, 2, 8, 16, F32)
    got = run(*t, quad, col, roff, 2, (6, 32), (6, 32))
    assert got["y"].shape == (0, 6, 32, 32) and got["dk"].shape == (0, 6, 32, 32) and (got["dlam"] == 0).all()


def test_duplicate_entries_of_psi_count_twice():
    quad, col, roff = geometry((6, 40), (6, 40), 0.6)
    two = torch.cat([torch.cat([c, c[:3]]) for c in col.split((roff[1:] - roff[:-1]).tolist())])
    check((6, 40), (6, 40), 1, 2, 16, 32, F32, 0.6, geo=(quad, two, roff + 3 * torch.arange(roff.numel())))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_is_the_difference_of_two_attentions(dtype):
    """16-bit: each of the two, and their difference, is rounded once more there."""
    ins = outs = (12, 64)
    nh, d = 2, 32
    k, v, q, lam, dy = [t.cuda() for t in tensors(ins, outs, 1, nh, d, d, dtype)]
    geo = [t.cuda() for t in geometry(ins, outs, 0.5)]
    y = differential_s2_attention(k, v, q, lam, *geo, nh, ins[1], *outs)
    maps = lambda t, i: t.view(1, *ins, nh, 2, d)[..., i, :].reshape(1, *ins, nh * d).contiguous()  # noqa: E731
    one, two = [neighborhood_s2_attention(maps(k, i), v, maps(q, i), *geo, nh, ins[1], *outs).view(1, *outs, nh, d).double() for i in range(2)]
    want = (one - lam.double().view(nh, 1) * two).view(y.shape)
    M = mask_of(*[t.cpu() for t in geo[1:]], *ins, *outs)
    _, mag, kappa, _ = reference(k, v, q, lam, dy, geo[0], M, nh)["y"]
    u = HALF_STEP[dtype]
    bound = u * want.abs().cpu() + (32 if dtype == F32 else 12) * u * kappa * mag  # (both sides' bounds)
    assert ((y.double() - want).abs().cpu() <= bound).all()


@pytest.mark.parametrize("dtype,d", [(F32, 8), (F32, 16), (F32, 32), (F32, 20), (F32, 64), (BF16, 16), (BF16, 32), (BF16, 20), (F16, 32), (BF16, 64), (BF16, 3)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("where", ["k", "v", "q"])
def test_values_that_are_not_finite_reach_the_points_that_see_them_only(where, bad, dtype, d):
    ins = outs = (9, 80)
    quad, col, roff = geometry(ins, outs, 0.45)
    t = list(tensors(ins, outs, 1, 1, d, 2 * d, dtype))
    clean = run(*t, quad, col, roff, 1, ins, outs)
    point = (4, 33)
    x = t["kvq".index(where)]
    x[0, point[0], point[1], 0] = bad
    got = run(*t, quad, col, roff, 1, ins, outs)
    M = mask_of(col, roff, *ins, *outs) > 0
    at = point[0] * ins[1] + point[1]
    queries = M[:, at] if where != "q" else torch.arange(M.shape[0]) == at
    keys = M[queries].any(0)  # that a touched query sees
    if where == "v" and not math.isnan(bad):
        pass
    for n, seen in (("y", queries), ("dq", queries), ("dk", keys), ("dv", keys)):
        touched = ~torch.isfinite(got[n].cpu()).view(-1, got[n].shape[3]).all(1)
        assert not (touched & ~seen).any(), f"{n}: reaches points that do not see the value"
        same = (got[n] == clean[n]).cpu().view(-1, got[n].shape[3]).all(1)
        near = torch.isclose(got[n].float(), clean[n].float(), rtol=0.05, atol=0.05 * clean[n].float().abs().max().item()).cpu().view(-1, got[n].shape[3]).all(1)
        assert (near | seen).all(), f"{n}: {int((~(near | seen)).sum())} points that do not see the value changed ({int((same | seen).sum())} kept their bits)"
    if math.isnan(bad):
        y = got["y"].cpu().view(-1, got["y"].shape[3])
        assert torch.isnan(y[queries][:, 0]).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d", [16, 20, 32])
def test_strides(dtype, d):
    """Column blocks of a wider buffer are read in place, anything else is copied; gradients are those of the packed tensors."""
    ins = outs = (8, 48)
    nh, cv = 2, 2 * d
    geo = geometry(ins, outs, 0.6)
    k, v, q, lam, dy = tensors(ins, outs, 2, nh, d, cv, dtype)
    want = run(k, v, q, lam, dy, *geo, nh, ins, outs)
    buf = torch.cat([q, torch.full_like(q[..., :8], 7.0), k, v], 3).cuda().requires_grad_(True)
    n = 2 * nh * d
    qb, kb, vb = buf[..., :n], buf[..., n + 8 : 2 * n + 8], buf[..., 2 * n + 8 :]
    y = differential_s2_attention(kb, vb, qb, lam.cuda(), *[t.cuda() for t in geo], nh, ins[1], *outs)
    (g,) = torch.autograd.grad(y, buf, dy.cuda())
    assert torch.equal(y, want["y"]) and torch.equal(g[..., :n], want["dq"]) and torch.equal(g[..., n + 8 : 2 * n + 8], want["dk"]) and torch.equal(g[..., 2 * n + 8 :], want["dv"])
    odd = lambda t: t.cuda().permute(0, 3, 1, 2).contiguous().permute(0, 2, 3, 1)  # noqa: E731  channels first in memory
    shifted = lambda t: torch.cat([torch.zeros(1, dtype=t.dtype), t.flatten()]).cuda()[1:].view(t.shape)  # noqa: E731  no alignment beyond the element's
    for f in (odd, shifted):
        x = [f(t).detach().requires_grad_(True) for t in (k, v, q)]
        y = differential_s2_attention(*x, lam.cuda(), *[t.cuda() for t in geo], nh, ins[1], *outs)
        g = torch.autograd.grad(y, x, f(dy))
        ref = reference(k, v, q, lam, dy, geo[0], mask_of(*geo[1:], *ins, *outs), nh)
        assert_near(dict(y=y, dk=g[0], dv=g[1], dq=g[2]), ref, dtype)
    y = differential_s2_attention(*[t.cuda().requires_grad_(True) for t in (k, v, q)], lam.cuda(), *[t.cuda() for t in geo], nh, ins[1], *outs)
    y.sum().backward()  # (an expanded gradient)


@pytest.mark.parametrize("dtype,d", [(F32, 16), (BF16, 32), (F32, 3)])
def test_results_are_the_same_in_every_run(dtype, d):
    ins = outs = (32, 96)
    geo = geometry(ins, outs, 0.3)
    t = tensors(ins, outs, 2, 4, d, 2 * d, dtype)
    a, b = run(*t, *geo, 4, ins, outs), run(*t, *geo, 4, ins, outs)
    assert all(torch.equal(a[n], b[n]) for n in a)


@pytest.mark.parametrize("d", [8, 16, 32, 5])
def test_gradients_against_differences(d):
    """Central differences of <dy, f(x + e u)> along a random direction of each input.  Truncation: e^2 / 6 times the third derivative, of
    scores of unit size and directions of unit size per channel below 50 |f| per point; noise: 2^-20 / e of the sum's magnitude.  With e = 2^-7
    both stay below 2^-7 of the norm of the gradient times that of the direction."""
    ins = outs = (6, 40)
    nh, e = 2, 2.0**-7
    geo = geometry(ins, outs, 0.8)
    t = tensors(ins, outs, 1, nh, d, 2 * d, F32, seed=3)
    got = run(*t, *geo, nh, ins, outs)
    f = lambda x: differential_s2_attention(*[s.cuda() for s in x[:4]], *[s.cuda() for s in geo], nh, ins[1], *outs).double()  # noqa: E731
    gen = torch.Generator().manual_seed(11)
    for i, n in enumerate(("dk", "dv", "dq", "dlam")):
        u = torch.randn(t[i].shape, generator=gen)
        plus, minus = [[x + s * e * u if j == i else x for j, x in enumerate(t)] for s in (1, -1)]
        slope = ((f(plus) - f(minus)) * t[4].cuda().double()).sum().item() / (2 * e)
        want = (got[n].double().cpu() * u.double()).sum().item()
        assert abs(slope - want) <= 2.0**-7 * got[n].double().norm().item() * u.double().norm().item(), n


def test_only_the_gradients_asked_for():
    ins = outs = (6, 40)
    geo = geometry(ins, outs, 0.8)
    t = tensors(ins, outs, 1, 2, 16, 32, F32)
    want = run(*t, *geo, 2, ins, outs)
    for i, n in enumerate(("dk", "dv", "dq", "dlam")):
        x = [s.cuda().requires_grad_(j == i) for j, s in enumerate(t[:4])]
        y = differential_s2_attention(*x, *[s.cuda() for s in geo], 2, ins[1], *outs)
        (g,) = torch.autograd.grad(y, [x[i]], t[4].cuda())
        assert torch.equal(y, want["y"]) and torch.equal(g, want[n])
    with torch.no_grad():
        assert torch.equal(differential_s2_attention(*[s.cuda() for s in t[:4]], *[s.cuda() for s in geo], 2, ins[1], *outs), want["y"])


def test_changed_tensors_and_second_derivatives_are_refused():
    ins = outs = (6, 40)
    geo = [s.cuda() for s in geometry(ins, outs, 0.8)]
    x = [s.cuda().requires_grad_(True) for s in tensors(ins, outs, 1, 2, 16, 32, F32)[:4]]
    y = differential_s2_attention(*x, *geo, 2, ins[1], *outs)
    g = torch.autograd.grad(y.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated"):
        torch.autograd.grad(g[0].sum(), x[0])
    y = differential_s2_attention(*x, *geo, 2, ins[1], *outs)
    s = y.sum()
    y.detach().zero_()
    y = differential_s2_attention(*x, *geo, 2, ins[1], *outs)
    s = y.sum()
    y.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        s.backward()


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_autocast(dtype):
    ins = outs = (6, 40)
    geo = [s.cuda() for s in geometry(ins, outs, 0.8)]
    x = [s.cuda() for s in tensors(ins, outs, 1, 2, 16, 32, F32)[:4]]
    with torch.autocast("cuda", dtype=dtype):
        y = differential_s2_attention(*x, *geo, 2, ins[1], *outs)
    assert torch.equal(y, differential_s2_attention(*[s.to(dtype) for s in x[:3]], x[3], *geo, 2, ins[1], *outs)) and y.dtype == dtype


@pytest.mark.parametrize("dtype,d", [(F32, 16), (BF16, 32)])
def test_streams(dtype, d):
    """Two calls at once on two streams, and one on another stream than its tensors were made on."""
    ins = outs = (32, 96)
    geo = geometry(ins, outs, 0.3)
    a, b = [tensors(ins, outs, 2, 4, d, 2 * d, dtype, seed=s) for s in (1, 2)]
    want = [run(*t, *geo, 4, ins, outs) for t in (a, b)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [None, None]
    for _ in range(3):
        for i, t in enumerate((a, b)):
            with torch.cuda.stream(streams[i]):
                got[i] = run(*t, *geo, 4, ins, outs)
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(w[n], g[n]) for n in w)


def test_captured_graphs():
    """Forward and backward captured twice, replayed in turn with eager calls and new inputs between them."""
    ins = outs = (16, 64)
    nh, d = 2, 16
    geo = [s.cuda() for s in geometry(ins, outs, 0.5)]
    sets = [[s.cuda() for s in tensors(ins, outs, 1, nh, d, 2 * d, BF16, seed=i)] for i in range(4)]

    def step(x):
        leaves = [s.detach().requires_grad_(True) for s in x[:4]]
        y = differential_s2_attention(*leaves, *geo, nh, ins[1], *outs)
        return [y.detach(), *torch.autograd.grad(y, leaves, x[4])]

    want = [[s.clone() for s in step(x)] for x in sets]
    graphs = []
    for _ in range(2):
        held = [s.clone() for s in sets[0]]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(held)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(held)
        graphs.append((g, held, out))
    for turn in range(6):
        for n, (g, held, out) in enumerate(graphs):
            i = (turn + n) % len(sets)
            for s, x in zip(held, sets[i]):
                s.copy_(x)
            g.replay()
            eager = step(sets[(i + 1) % len(sets)])
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want[i]))
            assert all(torch.equal(a, b) for a, b in zip(eager, want[(i + 1) % len(sets)]))


def test_compiled_graph():
    ins = outs = (8, 48)
    geo = [s.cuda() for s in geometry(ins, outs, 0.6)]
    x = [s.cuda().requires_grad_(True) for s in tensors(ins, outs, 1, 2, 16, 32, F32)[:4]]
    f = lambda k, v, q, lam: differential_s2_attention(k, v, q, lam, *geo, 2, ins[1], *outs)  # noqa: E731
    want = f(*x)
    dy = torch.randn_like(want)
    grads = torch.autograd.grad(want, x, dy)
    got = torch.compile(f, backend="aot_eager", fullgraph=True)(*x)
    assert torch.equal(got, want) and all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(got, x, dy), grads))
    torch.library.opcheck(torch.ops.s2attn_kernels.differential_forward.default, (*x, *geo, 2, ins[1], *outs, True), test_utils=("test_schema", "test_faketensor"))


@pytest.mark.parametrize("dtype,d", [(BF16, 32), (BF16, 3)])
def test_offsets_past_32_bits(dtype, d):
    """A batch whose tensors hold more than 2^31 elements: its last entry as alone."""
    ins = outs = (16, 64)
    nh = 1
    n = ins[0] * ins[1] * 2 * d
    B = (2**31) // n + 3
    geo = [s.cuda() for s in geometry(ins, outs, 0.4)]
    k, v, q, lam, dy = [s.cuda() for s in tensors(ins, outs, 1, nh, d, 2 * d, dtype)]
    one = [s.requires_grad_(True) for s in (k, v, q)]
    y1 = differential_s2_attention(*one, lam, *geo, nh, ins[1], *outs)
    g1 = torch.autograd.grad(y1, one, dy)
    big = [s.detach().expand(B, -1, -1, -1).contiguous().requires_grad_(True) for s in one]
    y = differential_s2_attention(*big, lam, *geo, nh, ins[1], *outs)
    g = torch.autograd.grad(y, big, dy.expand(B, -1, -1, -1))
    assert torch.equal(y[-1], y1[0]) and all(torch.equal(a[-1], b[0]) for a, b in zip(g, g1)) and torch.equal(y[B // 2], y1[0])
