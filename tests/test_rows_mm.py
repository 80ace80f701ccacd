"""What the entries of the float products refuse, and their workspaces, without a GPU."""
if __name__ == "__main__":  # `python tests/<file>.py`, as the reference runs its tests
    import sys as _sys

    import pytest as _pytest
    _sys.exit(_pytest.main([__file__, "-q"]))
import ctypes

import pytest

from jjjetson_ops_amd import capi

A = 4096  # an address that is never read: every call here is refused, or ends where no device is found
F32, F16, BF16 = capi.DTYPE_F32, capi.DTYPE_F16, capi.DTYPE_BF16
BIG = 1 << 62


def _linear(x=A, x_stride=64, w=A, bias=A, residual=A, r_stride=32, y=A, y_stride=32, pre=A, dtype=BF16, act=1, K=64,
            N=32, T=5, ws=A, ws_bytes=BIG):
    return capi.lib().linear_rows_forward_device(None, x, x_stride, w, bias, residual, r_stride, y, y_stride, pre, dtype,
                                                 act, K, N, T, ws, ws_bytes)


def _linear_back(g=A, g_stride=32, x=A, x_stride=64, w=A, pre=A, gx=A, gx_stride=64, gw=A, gb=A, dtype=BF16, gd=BF16,
                 act=1, K=64, N=32, T=5, ws=A, ws_bytes=BIG):
    return capi.lib().linear_rows_backward_device(None, g, g_stride, x, x_stride, w, pre, gx, gx_stride, gw, gb, dtype, gd,
                                                  act, K, N, T, ws, ws_bytes)


def _grouped(x=A, w=A, offsets=A, E=4, y=A, dtype=F16, K=64, N=32, R=9, ws=A, ws_bytes=BIG):
    return capi.lib().mat_mul_rows_grouped_device(None, x, w, offsets, E, y, dtype, K, N, R, ws, ws_bytes)


def _grouped_back(g=A, x=A, w=A, offsets=A, E=4, gx=A, gw=A, dtype=F16, gd=F16, K=64, N=32, R=9, ws=A, ws_bytes=BIG):
    return capi.lib().mat_mul_rows_grouped_backward_device(None, g, x, w, offsets, E, gx, gw, dtype, gd, K, N, R, ws,
                                                           ws_bytes)


def _swiglu(x=A, wg=A, wu=A, offsets=A, E=4, both=A, mid=A, dtype=F32, H=64, I=32, R=9, ws=A, ws_bytes=BIG):
    return capi.lib().moe_rows_gate_up_swiglu_device(None, x, wg, wu, offsets, E, both, mid, dtype, H, I, R, ws, ws_bytes)


def _swiglu_back(g=A, both=A, x=A, wg=A, wu=A, offsets=A, E=4, gx=A, gwg=A, gwu=A, dtype=F16, gd=F16, H=64, I=32, R=9,
                 ws=A, ws_bytes=BIG):
    return capi.lib().moe_rows_gate_up_swiglu_backward_device(None, g, both, x, wg, wu, offsets, E, gx, gwg, gwu, dtype, gd,
                                                              H, I, R, ws, ws_bytes)


REFUSED = [
    # sizes and types
    *[(_linear, {n: v}) for n in "KNT" for v in (0, -1, (1 << 28) + 1)],
    *[(_linear_back, {n: v}) for n in "KNT" for v in (0, -1, (1 << 28) + 1)],
    *[(f, {n: v}) for f in (_grouped, _grouped_back) for n in "KNR" for v in (0, -1, (1 << 28) + 1)],
    *[(f, {n: v}) for f in (_swiglu, _swiglu_back) for n in "HIR" for v in (0, -1, (1 << 28) + 1)],
    *[(f, {"E": v}) for f in (_grouped, _grouped_back, _swiglu, _swiglu_back) for v in (0, -1, 4097)],
    *[(f, {"dtype": v}) for f in (_linear, _linear_back, _grouped, _grouped_back, _swiglu, _swiglu_back) for v in (-1, 3)],
    *[(f, {"act": v}) for f in (_linear, _linear_back) for v in (-1, 5)],
    *[(f, {"dtype": BF16, "gd": F16}) for f in (_linear_back, _grouped_back, _swiglu_back)],
    *[(f, {"dtype": F32, "gd": BF16}) for f in (_linear_back, _grouped_back, _swiglu_back)],
    (_linear, {"K": 1 << 21, "N": 1 << 20, "x_stride": 1 << 21, "y_stride": 1 << 20, "r_stride": 1 << 20}),
    (_grouped, {"K": 1 << 20, "N": 1 << 19}),
    # pointers
    *[(_linear, {n: None}) for n in ("x", "w", "y")], *[(_linear, {n: A + 1}) for n in ("x", "w", "bias", "residual", "y", "pre")],
    *[(_linear_back, {n: None}) for n in ("g", "x", "w", "pre")],
    *[(_linear_back, {n: A + 1}) for n in ("g", "x", "w", "pre", "gx", "gw", "gb")],
    (_linear_back, {"gx": None, "gw": None, "gb": None}), (_linear_back, {"gw": A + 2, "gd": F32}),
    *[(_grouped, {n: None}) for n in ("x", "w", "offsets", "y")],
    *[(_grouped, {n: A + 1}) for n in ("x", "w", "y")], (_grouped, {"offsets": A + 2}),
    *[(_grouped_back, {n: None}) for n in ("g", "x", "w", "offsets")], (_grouped_back, {"gx": None, "gw": None}),
    *[(_swiglu, {n: None}) for n in ("x", "wg", "wu", "offsets", "mid")], (_swiglu, {"both": A + 2}),
    *[(_swiglu_back, {n: None}) for n in ("g", "both", "x", "wg", "wu", "offsets", "gwg", "gwu")],
    (_swiglu_back, {"gx": None, "gwg": None, "gwu": None}),
    # strides
    (_linear, {"x_stride": 63}), (_linear, {"y_stride": 31}), (_linear, {"r_stride": -32}), (_linear, {"x_stride": 1 << 40}),
    (_linear_back, {"g_stride": 31}), (_linear_back, {"x_stride": 0}), (_linear_back, {"gx_stride": 63}),
    # workspaces
    (_linear_back, {"ws": None}), (_linear_back, {"ws_bytes": 511}), (_linear_back, {"ws": A + 16}),
    (_swiglu_back, {"ws": None}), (_swiglu_back, {"ws_bytes": 0}), (_swiglu_back, {"ws": A + 128}),
]


@pytest.mark.parametrize("call,change", REFUSED, ids=lambda v: v.__name__[1:] if callable(v) else "-".join(map(str, v.items())))
def test_refused(call, change):
    assert call(**change) == capi.JJO_ERR_INVALID_ARG
    assert capi.lib().jjo_last_error()


def test_what_only_a_gradient_needs_may_be_missing():
    """Arguments that pass the checks end where no device is found (or are not run here at all)."""
    import torch
    if torch.cuda.is_available():
        pytest.skip("the addresses are not real")
    ok = capi.JJO_ERR_NO_DEVICE
    assert _linear(bias=None, residual=None, r_stride=0, pre=None, act=0) in (ok, capi.JJO_ERR_HIP)
    assert _linear(T=1, x_stride=0, y_stride=-3) in (ok, capi.JJO_ERR_HIP)
    assert _linear_back(w=None, gx=None, gx_stride=0) in (ok, capi.JJO_ERR_HIP)
    assert _linear_back(x=None, x_stride=0, gw=None) in (ok, capi.JJO_ERR_HIP)
    assert _linear_back(pre=None, act=0) in (ok, capi.JJO_ERR_HIP)
    assert _grouped_back(w=None, gx=None, gd=F32) in (ok, capi.JJO_ERR_HIP)
    assert _swiglu_back(x=None, gwg=None, gwu=None) in (ok, capi.JJO_ERR_HIP)


def test_workspace_bytes():
    assert capi.linear_rows_workspace_bytes(BF16, 4096, 11008, 1) == 0
    assert capi.linear_rows_workspace_bytes(BF16, 0, 11008, 1) == -1
    assert capi.linear_rows_workspace_bytes(3, 64, 64, 1) == -1
    assert capi.grouped_mat_mul_rows_workspace_bytes(F16, 64, 64, 8, 0) == -1
    for d, es, planes in ((F32, 4, 1), (F16, 2, 2), (BF16, 2, 3)):
        # at least the gradient through the activation, and through SwiGLU, in all its planes
        assert capi.linear_rows_backward_workspace_bytes(d, 64, 512, 100) >= planes * es * 51200
        assert capi.moe_gate_up_swiglu_rows_backward_workspace_bytes(d, 64, 512, 100, 4) >= planes * es * 102400
    most = 1 << 28
    for f in (capi.linear_rows_workspace_bytes, capi.linear_rows_backward_workspace_bytes):
        assert f(BF16, most, most, most) == -1
        assert f(BF16, 1 << 12, 1 << 12, most) >= 0
    for f in (capi.grouped_mat_mul_rows_workspace_bytes, capi.grouped_mat_mul_rows_backward_workspace_bytes,
              capi.moe_gate_up_swiglu_rows_workspace_bytes, capi.moe_gate_up_swiglu_rows_backward_workspace_bytes):
        assert f(BF16, 1 << 12, 1 << 12, most, 4096) >= 0
        assert f(BF16, most, most, 1, 1) == -1


def test_wrappers_check_tensors():
    """The Python side's own checks, on tensors that are not on a device."""
    torch = pytest.importorskip("torch")
    x, w, y = torch.zeros(3, 8), torch.zeros(4, 8), torch.zeros(3, 4)
    with pytest.raises(ValueError, match="dtype"):
        capi.linear_rows(x, w.half(), y, 8, 4, 3)
    with pytest.raises(ValueError, match="too small"):
        capi.linear_rows(x, w, y, 8, 4, 4)
    with pytest.raises(ValueError, match="too small"):
        capi.linear_rows(x, w, y, 8, 4, 3, bias=torch.zeros(3))
    with pytest.raises(ValueError, match="float32"):
        capi.linear_rows_backward(y.half(), x.half(), w.half(), x.half(), w.bfloat16(), None, 8, 4, 3)
    with pytest.raises(ValueError, match="one dtype"):
        capi.linear_rows_backward(y.half(), x.half(), w.half(), None, w.half(), torch.zeros(4), 8, 4, 3)
    with pytest.raises(ValueError, match="must be float32, float16"):
        capi.linear_rows(x.double(), w.double(), y.double(), 8, 4, 3)
    offsets = torch.tensor([0, 1, 3])
    with pytest.raises(ValueError, match="expert_offsets"):
        capi.grouped_mat_mul_rows(x, torch.zeros(2, 4, 8), offsets, y, 8, 4, 3)
    with pytest.raises(ValueError, match="w is too small"):
        capi.grouped_mat_mul_rows(x, w, offsets.int(), y, 8, 4, 3)
    with pytest.raises(ValueError, match="gate_up is too small"):
        capi.moe_gate_up_swiglu_rows(x, torch.zeros(2, 4, 8), torch.zeros(2, 4, 8), offsets.int(), 2, y, 8, 4, 3, gate_up=y)
