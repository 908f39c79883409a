"""The group norm without a GPU: what is refused, and the shapes of its operators."""

import ctypes

import pytest
import torch

import torch_harmonics_amd as th
from torch_harmonics_amd import _lib, ops


def test_shapes_on_meta_tensors():
    x, w = torch.zeros(2, 3, 4, 6, device="meta", dtype=torch.bfloat16), torch.zeros(6, device="meta")
    y, stats = ops.group_norm_forward(x, 3, w, w, None, 1e-5, 2)
    assert y.shape == x.shape and y.dtype == x.dtype and stats.shape == (2, 3, 3) and stats.dtype == torch.float32
    dx, dw, db = ops.group_norm_backward(y, x, 3, w, None, None, stats, 1e-5, 2, [True, True, True])
    assert dx.shape == x.shape and dw.shape == (6,) and dw.dtype == torch.float32 and db.numel() == 0


@pytest.mark.parametrize(
    "kw,message",
    [
        (dict(num_groups=4), "4 groups do not divide 6"),
        (dict(num_groups=0), "0 groups"),
        (dict(x=torch.zeros(2, 3, 6)), "4-dimensional"),
        (dict(x=torch.zeros(2, 3, 4, 6, dtype=torch.float64)), "unsupported dtype"),
        (dict(weight=torch.ones(5)), "one number per channel"),
        (dict(bias=torch.ones(6, 1)), "one number per channel"),
        (dict(weight=torch.ones(6), bias=torch.ones(6).half()), "share a dtype"),
        (dict(weight=torch.ones(6).long()), "unsupported dtype"),
        (dict(quad_weights=torch.ones(4)), "quad_weights must have nlat = 3"),
        (dict(eps=-1.0), "eps must not be negative"),
        (dict(eps=float("nan")), "eps must not be negative"),
        (dict(), "only run on a ROCm GPU"),
    ],
)
def test_refusals(kw, message):
    args = dict(x=torch.zeros(2, 3, 4, 6), num_groups=3)
    args.update(kw)
    with pytest.raises(RuntimeError, match=message):
        th.group_norm_s2(**args)


def test_unknown_activations():
    with pytest.raises(ValueError, match="unknown activation 'tanh'"):
        th.group_norm_s2(torch.zeros(2, 3, 4, 6), 3, activation="tanh")


def test_entry_points_refuse_bad_arguments_before_touching_the_gpu():
    lib = _lib.load()
    at = ctypes.c_void_p(4096)
    good = dict(batch=1, nlat=3, nlon=4, channels=6, groups=3, dtype=0, param_dtype=0, activation=0, eps=1e-5, x=at, y=at, stats=at, dy=at, dx=at, workspace=at)

    def says(code, text, backward=False, **kw):
        n = _lib.GroupNormStruct(**{**good, **kw})
        f = lib.s2attn_group_norm_backward if backward else lib.s2attn_group_norm
        assert f(ctypes.byref(n), None) == code and text in lib.s2attn_last_error().decode(), lib.s2attn_last_error()

    says(-1, "must be positive", batch=0)
    says(-1, "must be positive", channels=0)
    says(-1, "do not divide", groups=4)
    says(-1, "dtype code 7", dtype=7)
    says(-1, "of the parameters", param_dtype=-1)
    says(-1, "unknown activation 9", activation=9)
    says(-1, "eps", eps=-1.0)
    says(-1, "point stride", ld_x=5)
    says(-2, "2^31 points", nlat=1 << 16, nlon=1 << 16)
    says(-1, "null tensor", x=None)
    says(-1, "null tensor", stats=None)
    says(-1, "null tensor", workspace=None)
    says(-1, "null tensor", True, dy=None)
    assert lib.s2attn_group_norm(None, None) == -1
    n = _lib.GroupNormStruct(**{**good, "dx": None})
    assert lib.s2attn_group_norm_backward(ctypes.byref(n), None) == 0  # nothing asked for, nothing launched
    assert lib.s2attn_group_norm_workspace_bytes(ctypes.byref(_lib.GroupNormStruct(**{**good, "groups": 4})), 0) == -1
