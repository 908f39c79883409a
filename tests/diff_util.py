"""Differential attention in 64 bits from its definition (dense over the grid, small grids only), and what roundings may do to it."""

import math

import torch

from oracle import cpu_attention as oracle

HALF_STEP = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}


SUBNORMAL = {torch.float32: 1e-30, torch.bfloat16: 1e-30, torch.float16: 2.0**-25}  # half a step where values are subnormal


def mask_of(col, roff, Hi, Wi, Ho, Wo):
    """Boolean [Ho * Wo, Hi * Wi] and, for duplicate entries of psi, how often each pair occurs."""
    col, roff = col.cpu(), roff.cpu()
    M = torch.zeros(Ho * Wo, Hi * Wi, dtype=torch.float64)
    up = oracle.is_upsample(Wi, Wo)
    rows = torch.repeat_interleave(torch.arange(roff.numel() - 1), roff[1:] - roff[:-1])
    j = torch.arange(Wi if up else Wo)
    if up:
        ho, wo = col // Wo, col % Wo
        q = ho[:, None] * Wo + (wo[:, None] + (Wo // Wi) * j) % Wo
        k = rows[:, None] * Wi + j
    else:
        hi, wi = col // Wi, col % Wi
        q = rows[:, None] * Wo + j
        k = hi[:, None] * Wi + (wi[:, None] + (Wi // Wo) * j) % Wi
    M.view(-1).index_add_(0, (q * (Hi * Wi) + k).reshape(-1), torch.ones(q.numel(), dtype=torch.float64))
    return M


def reference(k, v, q, lam, dy, quad, M, nh):
    """Results and gradients in 64 bits, and for each the magnitude that a relative error of the probabilities, the products or the means
    multiplies: {name: (value, magnitude, kappa, size of the sums that g - D is the difference of)}.  All on the CPU."""
    k, v, q, lam, dy, quad = [t.detach().cpu().double() for t in (k, v, q, lam, dy, quad)]
    B, Hi, Wi, C = k.shape
    Ho, Wo = q.shape[1:3]
    d, cv = C // (2 * nh), v.shape[3] // nh
    K = k.view(B, Hi * Wi, nh, 2, d).permute(0, 2, 3, 1, 4)  # B nh 2 n d
    Q = q.view(B, Ho * Wo, nh, 2, d).permute(0, 2, 3, 1, 4)
    V = v.view(B, Hi * Wi, nh, 1, cv).permute(0, 2, 3, 1, 4)  # B nh 1 n cv
    G = dy.view(B, Ho * Wo, nh, 1, cv).permute(0, 2, 3, 1, 4)
    w = M * quad.repeat_interleave(Wi)[None, :]
    S = Q @ K.transpose(-1, -2)
    seen = w > 0
    top = torch.where(seen, S, torch.full_like(S, -math.inf)).amax(-1, keepdim=True)
    E = torch.where(seen, torch.exp(S - torch.where(top.isfinite(), top, torch.zeros_like(top))), torch.zeros_like(S)) * w
    Z = E.sum(-1, keepdim=True)
    P = torch.where(Z > 0, E / Z, torch.zeros_like(E))  # B nh 2 q n
    sign = torch.stack([torch.ones_like(lam), -lam], -1).view(1, nh, 2, 1, 1)
    Y2 = P @ V
    Y = (sign * Y2).sum(2)
    g = G @ V.transpose(-1, -2)  # B nh 1 q n
    D = (P * g).sum(-1, keepdim=True)
    dS = sign * P * (g - D)
    dQ, dK, dV = dS @ K, dS.transpose(-1, -2) @ Q, ((sign * P).sum(2, keepdim=True)).transpose(-1, -2) @ G
    dlam = -D[:, :, 1].sum((0, 2, 3))

    # the largest exponent's magnitude: a rounding of its operands is a relative error of as many roundings in a probability
    kappa = 1 + torch.where(seen, Q.abs() @ K.abs().transpose(-1, -2), torch.zeros_like(S)).amax().item()
    aP, spread = sign.abs() * P, (g - D).abs()
    mean_spread = (P * spread).sum(-1, keepdim=True)
    mag = sign.abs() * P * (spread + mean_spread)
    size = G.abs() @ V.abs().transpose(-1, -2)  # of the summands of g and, weighted, of D: what a rounding of a summand multiplies
    size = aP * (size + (P * size).sum(-1, keepdim=True))
    mags = dict(
        y=(aP @ V.abs()).sum(2), dq=mag @ K.abs(), dk=mag.transpose(-1, -2) @ Q.abs(), dv=(aP.transpose(-1, -2) @ G.abs()).sum(2),
        dlam=(mean_spread[:, :, 1] + (P[:, :, 1:2] @ V.abs() * G.abs()).sum(-1, keepdim=True)[:, :, 0]).sum((0, 2, 3)),
    )  # fmt: skip
    sizes = dict(y=0 * Y, dq=size @ K.abs(), dk=size.transpose(-1, -2) @ Q.abs(), dv=0 * dV[:, :, 0], dlam=0 * dlam)
    pack = lambda t, H, W: t.permute(0, 3, 1, 2, 4).reshape(B, H, W, -1) if t.dim() == 5 else t.permute(0, 2, 1, 3).reshape(B, H, W, -1)  # noqa: E731
    grids = dict(y=(Ho, Wo), dq=(Ho, Wo), dk=(Hi, Wi), dv=(Hi, Wi))
    values = dict(y=Y, dq=dQ, dk=dK, dv=dV[:, :, 0], dlam=dlam)
    out = {n: (t, mags[n], kappa, sizes[n]) if n == "dlam" else (pack(t, *grids[n]), pack(mags[n], *grids[n]), kappa, pack(sizes[n], *grids[n])) for n, t in values.items()}
    return out


def assert_near(got, ref, dtype, lam_dtype=None, slack=0.0):
    """16-bit storage: one rounding of the result, and of every probability (and dS) on the way into the matrix instructions, of the operands
    of the scores (each kappa roundings of a probability in all), and of y and y2 under the means: at most four times kappa of them, times
    the magnitude.  fp32: sums of up to a few hundred products in another order, products of three-term splits (2^-23), exp2 and
    log2 of one unit in the last place (2^-23), the exponent's own rounding (kappa): 16 half steps times kappa.  The sums <dy, v> and D in
    fp32: 16 half steps of the size of their summands, however small their difference is.  16-bit storage: D as first taken from the rounded y
    and y2 is off by one rounding of that size each, which is taken off again up to one rounding of the product: four of them squared."""
    u = HALF_STEP[dtype]
    per = 16 if dtype == torch.float32 else 4
    for n, t in got.items():
        want, mag, kappa, size = ref[n]
        t = t.detach().cpu().double()
        assert t.shape == want.shape, (n, t.shape, want.shape)
        uo = HALF_STEP[lam_dtype or dtype] if n == "dlam" else u
        bound = uo * want.abs() + per * u * kappa * mag + 16 * 2.0**-24 * (kappa * mag + size) + 4 * (0.0 if dtype == torch.float32 else u * u) * size + SUBNORMAL[dtype if n != 'dlam' else lam_dtype or dtype] + slack
        assert torch.isfinite(t).all(), f"{n}: not finite"
        over = ((t - want).abs() - bound).max().item()
        assert over <= 0, f"{n}: off by {(t - want).abs().max().item():.3e}, {over:.3e} more than roundings explain"
