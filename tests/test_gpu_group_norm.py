"""The channels-last group norm on the GPU against its definition in 64 bits."""

import math

import pytest
import torch

from torch_harmonics_amd import group_norm_s2

from .diff_util import HALF_STEP, SUBNORMAL

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
EPS = 1e-5
U32 = 2.0**-24


def tensors(shape, dtype, pdtype=None, seed=0, offset=1.0, scale=1.0, ring=None):
    g = torch.Generator().manual_seed(seed)
    B, H, W, C = shape
    x = scale * torch.randn(shape, generator=g) + offset * torch.randn(C, generator=g)
    w, b = 1 + 0.3 * torch.randn(C, generator=g), 0.3 * torch.randn(C, generator=g)
    quad = None if ring is None else (torch.rand(H, generator=g) + 0.01 if ring == "some" else ring)
    return x.to(dtype), w.to(pdtype or dtype), b.to(pdtype or dtype), torch.randn(shape, generator=g).to(dtype), quad


def reference(x, w, b, dy, quad, G, activation):
    """{name: (value, bound on what fp32 arithmetic may be off by)}, in 64 bits.  dm, dz: the mean is off by at most eight half steps of its
    size and of the deviation's, 1 / std by eight, so z by sixteen of its summands' sizes; sigmoid and erf are 2^-21 off; the sums of the gradients
    add up to 64 half steps of the size of their summands, and what dz does to the slope of the activation (its curvature is below 1.2)."""
    x, dy = x.double(), dy.double()
    B, H, W, C = x.shape
    gamma, beta = [torch.full((C,), v, dtype=torch.float64) if t is None else t.double() for t, v in ((w, 1.0), (b, 0.0))]
    ring = torch.ones(H, dtype=torch.float64) if quad is None else quad.double()
    share = (ring / (ring.sum() * W * (C // G))).view(1, H, 1, 1, 1)
    xg = x.view(B, H, W, G, C // G)
    xm = torch.where(share > 0, xg, torch.zeros_like(xg))
    mean = (xm * share).sum((1, 2, 4), keepdim=True)
    var = ((xm - mean) ** 2 * share).sum((1, 2, 4), keepdim=True)
    r = (var + EPS).rsqrt()
    full = lambda t: t.expand(xg.shape).reshape(x.shape)  # noqa: E731
    xh = ((xg - mean) * r).reshape(x.shape)
    z = xh * gamma + beta
    # (a value far below the largest carries the largest's rounding in the mean: the deviation's size is the group's)
    ez = 16 * U32 * ((xh.abs() + 1 + full(mean.abs() * r)) * gamma.abs() + beta.abs())
    sg, phi = torch.sigmoid(z), 0.5 * torch.erfc(-z * math.sqrt(0.5))
    y, slope, curve = {
        "none": lambda: (z, torch.ones_like(z), torch.zeros_like(z)),
        "relu": lambda: (z.clamp(min=0), (z > 0).double(), (z.abs() <= ez).double() / ez),
        "silu": lambda: (z * sg, sg * (1 + z * (1 - sg)), torch.full_like(z, 1.2)),
        "gelu": lambda: (z * phi, phi + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi), torch.full_like(z, 1.2)),
    }[activation or "none"]()
    own = 2.0**-21 * (1 + z.abs()) if activation in ("silu", "gelu") else torch.zeros_like(z)
    dz = dy * slope
    edz = dy.abs() * (curve * ez + own)
    g = (dz * gamma).view(xg.shape)
    sums = lambda t: t.sum((1, 2, 4), keepdim=True)  # noqa: E731
    xhg = xh.view(xg.shape)
    A, E = sums(g), sums(g * xhg)
    dx = r * (g - share * (A + xhg * E))
    eg = (edz * gamma.abs()).view(xg.shape) + 64 * U32 * g.abs()
    ex = (ez / gamma.abs().clamp(min=1e-30)).view(xg.shape)  # of xhat
    edx = r * (eg + share * (sums(eg) + 64 * U32 * sums(g.abs()) + xhg.abs() * (sums(eg * xhg.abs()) + sums(g.abs() * ex) + 64 * U32 * sums((g * xhg).abs())) + ex * E.abs()))
    all_ = lambda t: t.sum((0, 1, 2))  # noqa: E731
    return dict(
        y=(y, 1.2 * ez + own), dx=(dx.view(x.shape), edx.view(x.shape) + 16 * U32 * dx.view(x.shape).abs()),
        dweight=(all_(dz * xh), all_(edz * xh.abs() + dz.abs() * ex.view(x.shape) + 64 * U32 * (dz * xh).abs())), dbias=(all_(dz), all_(edz + 64 * U32 * dz.abs())),
    )  # fmt: skip


def run(x, w, b, dy, quad, G, activation):
    leaves = {n: t.detach().cuda().requires_grad_(True) for n, t in (("x", x), ("weight", w), ("bias", b)) if t is not None}
    y = group_norm_s2(leaves["x"], G, leaves.get("weight"), leaves.get("bias"), quad_weights=None if quad is None else quad.cuda(), eps=EPS, activation=activation)
    grads = torch.autograd.grad(y, list(leaves.values()), dy.cuda())
    return {"y": y.detach(), **{"d" + n: g for n, g in zip(leaves, grads)}}


def assert_near(got, ref, dtype, pdtype=None):
    for n, t in got.items():
        want, bound = ref[n]
        dt = dtype if n in ("y", "dx") else pdtype or dtype
        t = t.detach().cpu().double()
        assert t.shape == want.shape and torch.isfinite(t).all(), n
        over = ((t - want).abs() - HALF_STEP[dt] * (want.abs() + bound) - bound - SUBNORMAL[dt]).max().item()
        assert over <= 0, f"{n}: off by {(t - want).abs().max().item():.3e}, {over:.3e} more than roundings explain"


def check(shape, G, dtype, activation=None, ring=None, pdtype=None, **more):
    t = tensors(shape, dtype, pdtype, ring=ring, **more)
    got = run(*t, G, activation)
    assert_near(got, reference(*t, G, activation), dtype, pdtype)
    return got


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("ring", [None, "some"])
@pytest.mark.parametrize("activation", [None, "relu", "silu", "gelu"])
def test_activations_and_weights(activation, ring, dtype):
    check((2, 12, 25, 48), 6, dtype, activation, ring)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize(
    "shape,G",
    [((1, 1, 1, 1), 1), ((1, 1, 1, 8), 2), ((3, 1, 1, 6), 3), ((1, 1, 7, 5), 5), ((2, 3, 5, 7), 1), ((1, 9, 17, 30), 3), ((1, 9, 17, 20), 5), ((2, 8, 16, 64), 64), ((1, 4, 8, 4096), 4), ((1, 3, 4, 3000), 1),
     ((1, 3, 4, 2500), 2), ((1, 2, 3, 2050), 41), ((1, 61, 122, 8), 2), ((40, 4, 8, 16), 2), ((1500, 2, 2, 8), 4), ((1, 128, 256, 12), 1), ((1, 90, 181, 96), 8), ((1, 1, 20000, 4), 1)],
)  # fmt: skip
def test_shapes(shape, G, dtype):
    check(shape, G, dtype, "silu", "some")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("pdtype", [F32, BF16, F16])
def test_types_of_the_parameters(dtype, pdtype):
    check((2, 8, 16, 32), 4, dtype, "gelu", None, pdtype)


@pytest.mark.parametrize("absent", [("w",), ("b",), ("w", "b")])
def test_without_parameters(absent):
    x, w, b, dy, quad = tensors((2, 8, 16, 32), F32)
    w, b = None if "w" in absent else w, None if "b" in absent else b
    got = run(x, w, b, dy, quad, 4, "silu")
    assert_near(got, reference(x, w, b, dy, quad, 4, "silu"), F32)
    assert set(got) == {"y", "dx"} | ({"dweight"} if w is not None else set()) | ({"dbias"} if b is not None else set())


@pytest.mark.parametrize("shape", [(1, 12, 25, 32), (1, 90, 180, 32)])
def test_offsets_and_outliers(shape):
    """A mean thousands of deviations away; a first value far from all others: no precision is lost to either."""
    check(shape, 4, F32, None, "some", offset=1e4)
    t = list(tensors(shape, F32))
    t[0][0, 0, 0, :] = 3e4
    assert_near(run(*t, 4, None), reference(*t, 4, None), F32)


def test_constant_fields():
    x, w, b, dy, _ = tensors((1, 6, 12, 16), F32)
    x = torch.full_like(x, 3.25)
    got = run(x, w, b, dy, None, 2, None)
    assert torch.equal(got["y"].cpu(), b.expand_as(x))
    assert_near(got, reference(x, w, b, dy, None, 2, None), F32)


def test_rings_of_weight_zero_are_left_out():
    ring = torch.tensor([0.0, 0.5, 1.0, 0.0, 2.0, 0.1])
    t = list(tensors((2, 6, 12, 16), F32, ring=ring))
    assert_near(run(*t, 4, "silu"), reference(*t, 4, "silu"), F32)
    clean = run(*t, 4, "silu")
    t[0][:, 3] = math.nan
    t[0][:, 0] = math.inf
    got = run(*t, 4, "silu")
    assert torch.equal(got["y"][:, [1, 2, 4, 5]], clean["y"][:, [1, 2, 4, 5]])
    t = list(tensors((2, 6, 12, 16), F32, ring=torch.zeros(6)))
    got = run(*t, 4, None)  # nothing to take a mean of: zero, and a variance of zero
    want = t[0] / math.sqrt(EPS) * t[1] + t[2]
    assert torch.allclose(got["y"].cpu(), want, rtol=1e-6, atol=1e-6)


def test_nan_stays_in_its_group_and_batch_entry():
    t = list(tensors((2, 8, 16, 24), F32))
    clean = run(*t, 4, "silu")
    t[0][1, 3, 5, 7] = math.nan
    got = run(*t, 4, "silu")
    for n in ("y", "dx"):
        assert torch.equal(got[n][0], clean[n][0]) and torch.equal(got[n][1][..., :6], clean[n][1][..., :6]) and torch.equal(got[n][1][..., 12:], clean[n][1][..., 12:])
        assert torch.isnan(got[n][1][..., 6:12]).all()
    assert torch.isnan(got["dweight"][6:12]).all() and torch.equal(got["dweight"][:6], clean["dweight"][:6])


def test_agrees_with_torch():
    x, w, b, dy, _ = [None if t is None else t.cuda() for t in tensors((2, 30, 61, 48), F32)]
    got = group_norm_s2(x, 6, w, b, eps=1e-3)
    want = torch.nn.functional.group_norm(x.permute(0, 3, 1, 2), 6, w, b, 1e-3).permute(0, 2, 3, 1)
    assert (got - want).abs().max() <= 64 * U32 * (1 + want.abs().max())


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides(dtype):
    x, w, b, dy, quad = tensors((2, 9, 20, 32), dtype, ring="some")
    want = run(x, w, b, dy, quad, 4, "silu")
    pw, pb, pq = w.cuda(), b.cuda(), quad.cuda()
    buf = torch.cat([torch.zeros_like(x[..., :8]), x, torch.zeros_like(x[..., :4])], 3).cuda().requires_grad_(True)
    y = group_norm_s2(buf[..., 8:40], 4, pw, pb, pq, EPS, "silu")
    (g,) = torch.autograd.grad(y, buf, dy.cuda())
    assert torch.equal(y, want["y"]) or torch.allclose(y.float(), want["y"].float(), rtol=2.0**-7, atol=1e-5)
    assert torch.allclose(g[..., 8:40].float(), want["dx"].float(), rtol=2.0**-6, atol=1e-4) and (g[..., :8] == 0).all()
    shifted = lambda t: torch.cat([torch.zeros(1, dtype=t.dtype), t.flatten()]).cuda()[1:].view(t.shape)  # noqa: E731
    first = lambda t: t.cuda().permute(0, 3, 1, 2).contiguous().permute(0, 2, 3, 1)  # noqa: E731
    for f in (shifted, first):
        leaf = f(x).detach().requires_grad_(True)
        y = group_norm_s2(leaf, 4, pw, pb, pq, EPS, "silu")
        (g,) = torch.autograd.grad(y, leaf, f(dy))
        ref = reference(x, w, b, dy, quad, 4, "silu")
        assert_near(dict(y=y, dx=g), ref, dtype)
    leaf = x.cuda().requires_grad_(True)
    group_norm_s2(leaf, 4, pw, pb, pq, EPS, "silu").sum().backward()


def test_only_the_gradients_asked_for():
    t = tensors((2, 9, 20, 32), F32)
    want = run(*t, 4, "gelu")
    for i, n in enumerate(("x", "weight", "bias")):
        s = [p.cuda().requires_grad_(j == i) for j, p in enumerate(t[:3])]
        y = group_norm_s2(s[0], 4, s[1], s[2], eps=EPS, activation="gelu")
        (g,) = torch.autograd.grad(y, [s[i]], t[3].cuda())
        assert torch.equal(g, want["d" + n]) and torch.equal(y, want["y"])
        s = [p.cuda().requires_grad_(True) for p in t[:3]]
        (g,) = torch.autograd.grad(group_norm_s2(s[0], 4, s[1], s[2], eps=EPS, activation="gelu"), [s[i]], t[3].cuda())
        assert torch.equal(g, want["d" + n])
    x = t[0].cuda().requires_grad_(True)
    y = group_norm_s2(x, 4, activation="silu")
    (g,) = torch.autograd.grad(y.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated"):
        torch.autograd.grad(g.sum(), x)
    x = t[0].cuda()
    bias = t[2].cuda().requires_grad_(True)  # no weight: the bias's place among the inputs moves
    (g,) = torch.autograd.grad(group_norm_s2(x, 4, None, bias, eps=EPS), [bias], t[3].cuda())
    assert torch.allclose(g, t[3].cuda().sum((0, 1, 2)), rtol=1e-5, atol=1e-4)


@pytest.mark.parametrize("activation", [None, "silu", "gelu"])
def test_gradients_against_differences(activation):
    """Central differences with e = 2^-6: truncation e^2 / 6 of a third derivative below 10 per unit direction, noise 2^-20 / e of the sum: below
    2^-8 of the norms' product."""
    t = tensors((1, 10, 21, 16), F32, ring="some", seed=5)
    got = run(*t, 4, activation)
    gen = torch.Generator().manual_seed(3)
    for i, n in enumerate(("x", "weight", "bias")):
        u = torch.randn(t[i].shape, generator=gen)
        f = []
        for s in (1, -1):
            p = [a + s * 2.0**-6 * u if j == i else a for j, a in enumerate(t[:3])]
            f.append((group_norm_s2(p[0].cuda(), 4, p[1].cuda(), p[2].cuda(), t[4].cuda(), EPS, activation).double() * t[3].cuda().double()).sum().item())
        slope = (f[0] - f[1]) / 2.0**-5
        want = (got["d" + n].cpu().double() * u.double()).sum().item()
        assert abs(slope - want) <= 2.0**-8 * got["d" + n].double().norm().item() * u.double().norm().item() + 1e-3 * abs(want)


@pytest.mark.parametrize("shape", [(1, 16, 32, 32), (2, 64, 130, 64)])
def test_runs_streams_and_graphs(shape):
    sets = [[None if p is None else p.cuda() for p in tensors(shape, BF16, seed=i, ring="some")] for i in range(3)]

    def step(t):
        leaves = [p.detach().requires_grad_(True) for p in t[:3]]
        y = group_norm_s2(leaves[0], 4, leaves[1], leaves[2], t[4], EPS, "silu")
        return [y.detach(), *torch.autograd.grad(y, leaves, t[3])]

    want = [[p.clone() for p in step(t)] for t in sets]
    assert all(torch.equal(a, b) for t, w in zip(sets, want) for a, b in zip(step(t), w))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [None, None]
    for _ in range(3):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i] = step(sets[i])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for i in range(2) for a, b in zip(got[i], want[i]))
    graphs = []
    for _ in range(2):
        held = [p.clone() for p in sets[0]]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(held)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(held)
        graphs.append((g, held, out))
    for turn in range(5):
        for n, (g, held, out) in enumerate(graphs):
            i = (turn + n) % 3
            for h, p in zip(held, sets[i]):
                h.copy_(p)
            g.replay()
            eager = step(sets[(i + 1) % 3])
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want[i])) and all(torch.equal(a, b) for a, b in zip(eager, want[(i + 1) % 3]))


def test_compiled_graph_and_empty_batches():
    t = [None if p is None else p.cuda() for p in tensors((2, 8, 16, 24), F32, ring="some")]
    leaves = [p.requires_grad_(True) for p in t[:3]]
    f = lambda x, w, b: group_norm_s2(x, 4, w, b, t[4], EPS, "gelu")  # noqa: E731
    want = f(*leaves)
    grads = torch.autograd.grad(want, leaves, t[3])
    got = torch.compile(f, backend="aot_eager", fullgraph=True)(*leaves)
    assert torch.equal(got, want) and all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(got, leaves, t[3]), grads))
    torch.library.opcheck(torch.ops.s2attn_kernels.group_norm_forward.default, (*[leaves[0], 4, leaves[1], leaves[2], t[4], EPS, 3],), test_utils=("test_schema", "test_faketensor"))
    x = torch.zeros(0, 8, 16, 24, device="cuda", requires_grad=True)
    y = group_norm_s2(x, 4, leaves[1], leaves[2])
    g = torch.autograd.grad(y.sum(), [x, leaves[1], leaves[2]])
    assert y.shape == x.shape and g[0].shape == x.shape and (g[1] == 0).all() and (g[2] == 0).all()


def test_offsets_past_32_bits():
    """More than 2^31 elements: a batch entry alone, and the last of a batch."""
    x = torch.randn(1, 64, 128, 64, device="cuda").to(BF16)
    dy = torch.randn(1, 64, 128, 64, device="cuda").to(BF16)
    B = 2**31 // x[0].numel() + 2
    leaf = x.requires_grad_(True)
    y1 = group_norm_s2(leaf, 4, activation="silu")
    (g1,) = torch.autograd.grad(y1, leaf, dy)
    big = x.detach().expand(B, -1, -1, -1).contiguous().requires_grad_(True)
    y = group_norm_s2(big, 4, activation="silu")
    (g,) = torch.autograd.grad(y, big, dy.expand(B, -1, -1, -1))
    near = lambda a, b: (a.float() - b.float()).abs().max() <= 2.0**-7 * b.float().abs().max()  # noqa: E731  (the sums are split another way)
    assert near(y[-1], y1[0]) and near(g[-1], g1[0]) and torch.equal(y[0], y[-1]) and torch.equal(g[0], g[-1])
    del big, y, g
    wide = torch.randn(1, 16, 32, 64, device="cuda").to(BF16).expand(1, -1, -1, -1)
    rows = torch.zeros(1, 4200, 8192, 64, device="cuda", dtype=BF16)
    rows[:, -16:, -32:] = wide
    ring = torch.zeros(4200, device="cuda")
    ring[-16:] = 1.0
    y = group_norm_s2(rows, 4, quad_weights=ring)
    xg = rows[:, -16:].double().view(16, 8192, 4, 16)
    mean, var = xg.mean((0, 1, 3)), xg.var((0, 1, 3), unbiased=False)
    want = ((xg - mean.view(4, 1)) / (var + 1e-5).sqrt().view(4, 1)).view(16, 8192, 64)
    assert (y[0, -16:].double() - want).abs().max() <= 2.0**-8 * want.abs().max() * 1.01
