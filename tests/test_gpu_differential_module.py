"""The differential layer and the group norm as modules: the operators in one run, against the same layer in 64 bits."""

import math

import pytest
import torch

from torch_harmonics_amd import DifferentialNeighborhoodAttentionS2, GroupNormS2, group_norm_s2, precompute_latitudes

from .diff_util import mask_of

pytestmark = pytest.mark.gpu


def plain(m, x, xk):
    """The layer from its formulas, with autograd, in the type of its inputs (CPU)."""
    p = {n: t.detach().cpu().to(x.dtype).requires_grad_(True) for n, t in m.named_parameters()}
    nh, B = m.num_heads, x.shape[0]
    nlat, nlon, nlat_in, nlon_in = m.nlat_out, m.nlon_out, m.nlat_in, m.nlon_in
    lin = lambda t, n: torch.einsum("bchw,oc->bhwo", t, p[n + "_weights"].flatten(1)) + (p[n + "_bias"] if n + "_bias" in p else 0)  # noqa: E731
    rms = lambda t, g: t * (t.square().mean(-1, keepdim=True) + torch.finfo(torch.float32).eps).rsqrt() * (1 + g)  # noqa: E731
    q, k, v = lin(x, "q").view(B, nlat * nlon, nh, 2, -1), lin(xk, "k").view(B, nlat_in * nlon_in, nh, 2, -1), lin(xk, "v").view(B, nlat_in * nlon_in, nh, -1)
    if m.q_norm_weights is not None:
        q, k = rms(q, p["q_norm_weights"]), rms(k, p["k_norm_weights"])
    M = mask_of(m.psi_col_idx, m.psi_roff_idx, nlat_in, nlon_in, nlat, nlon) * m.quad_weights.cpu().double().repeat_interleave(nlon_in)
    s = torch.einsum("bqhmc,bkhmc->bhmqk", q, k) * m.scale + torch.log(M).to(x.dtype)
    lam = torch.exp((p["lambda_q1"] * p["lambda_k1"]).sum(-1)) - torch.exp((p["lambda_q2"] * p["lambda_k2"]).sum(-1)) + m.lambda_init
    a = torch.softmax(s, -1)
    y = torch.einsum("bhqk,bkhc->bqhc", a[:, :, 0] - lam.view(1, nh, 1, 1) * a[:, :, 1], v)
    if m.norm == "group":
        w = precompute_latitudes(nlat, grid="equiangular")[1].to(x.dtype).repeat_interleave(nlon).view(1, -1, 1, 1)
        share = w / (w.sum() * y.shape[3])
        mean = (y * share).sum((1, 3), keepdim=True)
        y = (y - mean) * (((y - mean).square() * share).sum((1, 3), keepdim=True) + 1e-5).rsqrt()
        y = y.reshape(B, nlat * nlon, -1) * p["head_norm.weight"] + p["head_norm.bias"]
        act = {None: lambda t: t, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "relu": torch.relu}[m.activation]
        y = act(y) * (1 - m.lambda_init)
    elif m.norm == "rms":
        y = rms(y, p["head_norm_weights"]) * (1 - m.lambda_init)
    y = y.reshape(B, nlat, nlon, -1)
    out = torch.einsum("bhwc,oc->bohw", y, p["proj_weights"].flatten(1)) + (p["proj_bias"].view(-1, 1, 1) if "proj_bias" in p else 0)
    return out, p


@pytest.mark.parametrize("norm,activation,qknorm,bias", [("group", None, False, True), ("group", "silu", False, True), ("rms", None, True, True), (None, None, False, False), ("group", "gelu", True, False)])
@pytest.mark.parametrize("ins,outs", [((9, 64), (9, 64)), ((10, 80), (5, 40)), ((5, 40), (10, 80)), ((8, 15), (8, 15))])
def test_layer_in_fp32(ins, outs, norm, activation, qknorm, bias):
    """Every step is within 1e-5 of 64 bits relative to its largest values (the projections by torch, the attention and the norm by their own
    tests); four of them follow each other, and a norm divides by deviations that may be some tenths: 2e-4 of the largest value."""
    torch.manual_seed(3)
    m = DifferentialNeighborhoodAttentionS2(24, ins, outs, num_heads=2, theta_cutoff=0.8, k_channels=32, out_channels=32, norm=norm, activation=activation, use_qknorm=qknorm, bias=bias).cuda()
    with torch.no_grad():
        for n, p in m.named_parameters():
            if "bias" in n or "norm_weights" in n or n == "head_norm.weight":
                p.add_(0.2 * torch.randn_like(p))
    x, xk = torch.randn(2, 24, *outs), torch.randn(2, 24, *ins)
    want, p = plain(m, x.double().requires_grad_(True), xk.double() if ins != outs else x.double())
    a = x.cuda().requires_grad_(True)
    got = m(a) if ins == outs else m(a, xk.cuda(), xk.cuda())
    assert (got.detach().cpu().double() - want).abs().max() <= 2e-4 * want.abs().max()
    dy = torch.randn(want.shape)
    if ins == outs:
        xd = x.double().requires_grad_(True)
        want, p = plain(m, xd, xd)
    else:
        xd = x.double().requires_grad_(True)
        want, p = plain(m, xd, xk.double())
    names = [n for n in p]
    ref = torch.autograd.grad(want, [xd, *p.values()], dy.double(), allow_unused=True)
    own = torch.autograd.grad(got, [a, *[dict(m.named_parameters())[n] for n in names]], dy.cuda(), allow_unused=True)
    for n, g, r in zip(["x", *names], own, ref):
        if n == "k_bias" and not qknorm:  # (the softmax does not see it: zero up to rounding)
            continue
        # (a first-step bias or a lambda may be far smaller than the sums it comes from)
        scale = max(r.abs().max().item(), 1e-2 * ref[0].abs().max().item())
        assert (g.cpu().double() - r).abs().max().item() <= 1e-3 * scale, n


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("autocast", [True, False])
def test_layer_in_16_bits_trains(dtype, autocast):
    torch.manual_seed(3)
    m = DifferentialNeighborhoodAttentionS2(32, (12, 64), (12, 64), num_heads=2, theta_cutoff=0.5, k_channels=64, out_channels=64, activation="silu").cuda()
    x = torch.randn(2, 32, 12, 64, device="cuda")
    with torch.no_grad():
        want = m(x)
    if autocast:
        with torch.autocast("cuda", dtype=dtype):
            y = m(x)
    else:
        quad = m.quad_weights
        m = m.to(dtype)
        m.quad_weights = quad
        x = x.to(dtype)
        y = m(x)
    assert y.dtype == dtype and (y.float() - want).norm() <= (0.05 if dtype == torch.bfloat16 else 0.01) * want.norm()
    y.float().square().mean().backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() and p.grad.dtype == p.dtype for p in m.parameters())


def test_layer_under_compile_and_checkpoint():
    from torch.utils.checkpoint import checkpoint

    torch.manual_seed(3)
    m = DifferentialNeighborhoodAttentionS2(16, (8, 32), (8, 32), num_heads=2, theta_cutoff=0.8, activation="gelu").cuda()
    x = torch.randn(1, 16, 8, 32, device="cuda", requires_grad=True)
    want = torch.autograd.grad(m(x).square().sum(), [x, *m.parameters()])
    got = torch.autograd.grad(checkpoint(m, x, use_reentrant=False).square().sum(), [x, *m.parameters()])
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    got = torch.autograd.grad(torch.compile(m, backend="aot_eager")(x).square().sum(), [x, *m.parameters()])
    assert all(torch.allclose(a, b, rtol=1e-5, atol=1e-6 * a.abs().max().item()) for a, b in zip(want, got))


@pytest.mark.parametrize("fmt", [torch.contiguous_format, torch.channels_last])
@pytest.mark.parametrize("shape", [None, (12, 25)])
def test_norm_module(shape, fmt):
    torch.manual_seed(0)
    m = GroupNormS2(4, 32, shape, activation="silu").cuda()
    with torch.no_grad():
        m.weight.normal_()
        m.bias.normal_()
    x = torch.randn(2, 32, 12, 25, device="cuda").to(memory_format=fmt).requires_grad_(True)
    y = m(x)
    quad = None if shape is None else 2 * math.pi * precompute_latitudes(12, grid="equiangular")[1].float().cuda() / 25
    want = group_norm_s2(x.permute(0, 2, 3, 1).contiguous(), 4, m.weight, m.bias, quad, activation="silu").permute(0, 3, 1, 2)
    assert torch.equal(y, want) and y.is_contiguous(memory_format=fmt)
    dy = torch.randn_like(y)
    for a, b in zip(torch.autograd.grad(y, [x, m.weight, m.bias], dy), torch.autograd.grad(want, [x, m.weight, m.bias], dy)):
        assert torch.equal(a, b)
    if shape is None:
        assert torch.allclose(y, torch.nn.functional.silu(torch.nn.functional.group_norm(x, 4, m.weight, m.bias)), rtol=1e-4, atol=1e-5)
