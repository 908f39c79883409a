"""Differential attention without a GPU: what is refused, before anything is launched, and the shapes of its operators."""

import ctypes

import pytest
import torch

import torch_harmonics_amd as th
from torch_harmonics_amd import _lib, ops, plan


def _psi(ins=(6, 12), outs=(6, 12)):
    col, roff, _ = th.precompute_neighborhood_s2(ins, outs, theta_cutoff=0.6)
    return torch.ones(ins[0]), col, roff


def _args(device="meta", nh=2, ck=4, cv=6, dtype=torch.float32, grid=(6, 12)):
    q = torch.zeros(2, *grid, nh * 2 * ck, dtype=dtype, device=device)
    v = torch.zeros(2, *grid, nh * cv, dtype=dtype, device=device)
    quad, col, roff = _psi(grid, grid)
    return [q.clone(), v, q, torch.zeros(nh, dtype=dtype, device=device), quad.to(device), col.to(device), roff.to(device), nh, grid[1], *grid]


def test_shapes_on_meta_tensors():
    a = _args()
    y, y2, lse = ops.differential_forward(*a, True)
    assert y.shape == y2.shape == (2, 6, 12, 12) and lse.shape == (2, 2, 72, 2) and lse.dtype == torch.float32
    y, y2, lse = ops.differential_forward(*a, False)
    assert y.shape == (2, 6, 12, 12) and y2.numel() == lse.numel() == 0
    dk, dv, dq, dlam = ops.differential_backward(y, *a[:4], y, y, lse, *a[4:], [True, True])
    assert dk.shape == dq.shape == a[0].shape and dv.shape == a[1].shape and dlam.shape == (2,)
    dk, dv, dq, dlam = ops.differential_backward(y, *a[:4], y, y, lse, *a[4:], [False, False])
    assert dk.numel() == dv.numel() == dlam.numel() == 0 and dq.shape == a[0].shape


@pytest.mark.parametrize(
    "change,message",
    [
        (lambda a: a.__setitem__(0, a[0][..., :-1].contiguous()), "same channel count"),
        (lambda a: (a.__setitem__(0, a[0][..., :-2].contiguous()), a.__setitem__(2, a[2][..., :-2].contiguous())), "two maps per head"),
        (lambda a: a.__setitem__(1, a[1][..., :-1].contiguous()), "divisible by num_heads"),
        (lambda a: a.__setitem__(1, a[1].half()), "must match q dtype"),
        (lambda a: a.__setitem__(2, a[2][:1]), "share B"),
        (lambda a: a.__setitem__(3, a[3][:1]), "one number per head"),
        (lambda a: a.__setitem__(3, a[3].view(1, 2)), "one number per head"),
        (lambda a: a.__setitem__(3, a[3].long()), "unsupported dtype"),
        (lambda a: [a.__setitem__(i, a[i].double()) for i in range(3)], "fp32, bf16 and fp16"),
        (lambda a: a.__setitem__(4, a[4][:-1]), "quad_weights must have nlat_in"),
        (lambda a: a.__setitem__(7, 0), "num_heads must be positive"),
        (lambda a: a.__setitem__(8, 7), "integer multiple"),
        (lambda a: a.__setitem__(9, 5), "extents do not match"),
        (lambda a: a.__setitem__(6, a[6].int()), "must be int64"),
        (lambda a: a.__setitem__(2, a[2][0]), "4-dimensional"),
        (lambda a: None, "only run on a ROCm GPU"),
    ],
)
def test_refusals(change, message):
    a = _args("cpu")
    change(a)
    with pytest.raises(RuntimeError, match=message):
        th.differential_s2_attention(*a)
    with pytest.raises(RuntimeError, match=message):
        ops.differential_forward(*a, True)


def test_entry_points_refuse_bad_arguments_before_touching_the_gpu():
    lib = _lib.load()
    quad, col, roff = _psi()
    p = plan.build_host_blob(col, roff, 6, 12, 6, 12)  # (host memory: never read on the device, every call is refused)
    at = ctypes.c_void_p(4096)
    shape = lambda **kw: _lib.ShapeStruct(**{**dict(batch=1, num_heads=2, nlat_in=6, nlon_in=12, nlat_out=6, nlon_out=12, ck=4, cv=8, dtype=0), **kw})  # noqa: E731

    def forward(sh=None, plan_=p, k=at, lam=at, lam_dtype=0, y=at, y2=None, lse=None):
        return lib.s2attn_diff_forward(k, at, at, lam, lam_dtype, at, y, y2, lse, ctypes.byref(plan_.struct) if plan_ else None, ctypes.byref(sh) if sh else None, None)

    def backward(sh=None, dk=at, dv=at, dq=at, ws=at, y2=at, lse=at):
        return lib.s2attn_diff_backward(at, at, at, at, 0, at, at, y2, lse, at, dk, dv, dq, at, ws, ctypes.byref(p.struct), ctypes.byref(sh or shape()), None)

    def says(rc, code, text):
        assert rc == code and text in lib.s2attn_last_error().decode(), (rc, lib.s2attn_last_error())

    says(forward(), -1, "shape is null")
    says(forward(shape(), None), -1, "plan is null")
    says(forward(shape(), k=None), -1, "null tensor")
    says(forward(shape(), lam=None), -1, "null tensor")
    says(forward(shape(), y=None), -1, "null tensor")
    says(forward(shape(), lam_dtype=5), -1, "dtype code 5 of lam")
    says(forward(shape(), y2=at), -1, "together or not at all")
    says(forward(shape(), y2=at, lse=ctypes.c_void_p(4100)), -1, "8-byte aligned")
    says(forward(shape(ck=0)), -1, "1 to 256 channels")
    says(forward(shape(ck=257)), -2, "1 to 256 channels")
    says(forward(shape(cv=513)), -2, "above 512")
    says(forward(shape(batch=0)), -1, "must be positive")
    says(forward(shape(dtype=3)), -1, "dtype code")
    says(forward(shape(ld_q=12)), -1, "point stride")
    says(forward(shape(nlat_out=5)), -1, "plan was built for")
    says(backward(dk=None), -1, "together or not at all")
    says(backward(dq=None), -1, "null tensor")
    says(backward(ws=None), -1, "null tensor")
    says(backward(ws=ctypes.c_void_p(4104)), -1, "16-byte")
    says(backward(y2=None), -1, "null tensor")
    says(lib.s2attn_diff_backward_workspace_bytes(ctypes.byref(shape(ck=300))), -2, "1 to 256")
    assert lib.s2attn_diff_backward_workspace_bytes(ctypes.byref(shape())) == 2 * 72 * 20


def test_module_state_and_refusals():
    m = th.DifferentialNeighborhoodAttentionS2(16, (8, 16), (8, 16), num_heads=2, use_qknorm=True)
    assert m.scale == 1 / 2 and m.q_norm_weights.shape == (4,) and m.lambda_q1.shape == (2, 4) and m.learned_lambda().shape == (2,)
    base = th.NeighborhoodAttentionS2(16, (8, 16), (8, 16), num_heads=2)
    assert set(base.state_dict()) <= set(m.state_dict())
    assert set(m.state_dict()) - set(base.state_dict()) == {"lambda_q1", "lambda_k1", "lambda_q2", "lambda_k2", "q_norm_weights", "k_norm_weights", "head_norm.weight", "head_norm.bias"}
    with pytest.raises(ValueError, match="two maps per head"):
        th.DifferentialNeighborhoodAttentionS2(12, (8, 16), (8, 16), num_heads=4)
    with pytest.raises(ValueError, match="unknown norm"):
        th.DifferentialNeighborhoodAttentionS2(16, (8, 16), (8, 16), norm="layer")
    with pytest.raises(ValueError, match="part of the group norm"):
        th.DifferentialNeighborhoodAttentionS2(16, (8, 16), (8, 16), norm="rms", activation="silu")
    with pytest.raises(RuntimeError, match="only run on a ROCm GPU"):
        m(torch.zeros(1, 16, 8, 16))
    with pytest.raises(RuntimeError, match="query latitudes"):
        m(torch.zeros(1, 16, 9, 16))
    with pytest.raises(ValueError, match="divides num_channels"):
        th.GroupNormS2(3, 16)
    with pytest.raises(ValueError, match="unknown activation"):
        th.GroupNormS2(4, 16, activation="tanh")
    n = th.GroupNormS2(4, 16, (8, 16))
    assert abs(n.quad_weights.sum().item() * 16 - 12.566371) < 1e-4 and set(n.state_dict()) == {"weight", "bias"}
    with pytest.raises(RuntimeError, match="input longitudes"):
        n(torch.zeros(1, 16, 8, 15))
    with pytest.raises(RuntimeError, match="input channels"):
        n(torch.zeros(1, 15, 8, 16))
