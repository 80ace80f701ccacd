"""Workspaces of the float products' backward passes: what a call uses, and nothing for terms that it does not ask for;
without a GPU."""
if __name__ == "__main__":  # `python tests/<file>.py`, as the reference runs its tests
    import sys as _sys

    import pytest as _pytest
    _sys.exit(_pytest.main([__file__, "-q"]))
import pytest

from jjjetson_ops_amd import capi

A = 4096  # an address that is never read
F32, F16, BF16 = capi.DTYPE_F32, capi.DTYPE_F16, capi.DTYPE_BF16
SIZE = {F32: 4, F16: 2, BF16: 2}
TERMS = {F32: 1, F16: 2, BF16: 3}


def _refused(rc):
    if rc == capi.JJO_ERR_INVALID_ARG:
        return True
    assert rc in (capi.JJO_ERR_NO_DEVICE, capi.JJO_ERR_HIP), rc
    return False


def _linear(d, gd, act, K, N, T, ws, gx=A, gw=A, gb=A):
    return _refused(capi.lib().linear_rows_backward_device(None, A, N, A, K, A, A, gx, K, gw, gb, d, gd, act, K, N, T,
                                                           A if ws else None, ws))


def _swiglu(d, gd, H, I, R, E, ws, gx=A, gw=A):
    return _refused(capi.lib().moe_rows_gate_up_swiglu_backward_device(None, A, A, A, A, A, A, E, gx, gw, gw, d, gd, H, I, R,
                                                                       A if ws else None, ws))


def _skip_on_a_gpu():
    import torch
    if torch.cuda.is_available():
        pytest.skip("the addresses are not real")


@pytest.mark.parametrize("d,gd", [(F32, F32), (F16, F16), (F16, F32), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("K,N,T", [(64, 512, 100), (4096, 4096, 2048), (4096, 128256, 4096), (7, 5, 3)])
def test_linear(d, gd, K, N, T):
    _skip_on_a_gpu()
    most = capi.linear_rows_backward_workspace_bytes(d, K, N, T)
    gz = SIZE[d] * T * N
    without = capi.linear_rows_backward_workspace_bytes(d, K, N, T, activation=capi.ACT_NONE, grad_dtype=gd)
    for act in (capi.ACT_NONE, capi.ACT_SILU):
        need = capi.linear_rows_backward_workspace_bytes(d, K, N, T, activation=act, grad_dtype=gd)
        terms = 0 if act == capi.ACT_NONE else TERMS[d] if gd != d else 1
        assert 0 < need <= most and terms * gz <= need - without <= terms * (gz + 255)
        assert not _linear(d, gd, act, K, N, T, need) and _linear(d, gd, act, K, N, T, need - 256)
    # what only a gradient that is not asked for uses
    assert not _linear(d, gd, capi.ACT_NONE, K, N, T, without, gw=None) and without < 2 * gz + (1 << 28)
    one = capi.linear_rows_backward_workspace_bytes(d, K, N, T, activation=capi.ACT_SILU, grad_dtype=d)
    assert not _linear(d, gd, capi.ACT_SILU, K, N, T, one, gw=None)


def test_nothing_is_needed_where_nothing_is_kept():
    """One product over many tiles, no activation, no bias: no workspace at all."""
    _skip_on_a_gpu()
    assert not _linear(BF16, BF16, capi.ACT_NONE, 4096, 4096, 2048, 0, gb=None)
    assert _linear(BF16, BF16, capi.ACT_SILU, 4096, 4096, 2048, 0, gb=None)


@pytest.mark.parametrize("d,gd", [(F32, F32), (F16, F16), (F16, F32), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("H,I,R,E", [(64, 512, 100, 4), (4096, 14336, 2048, 8), (7, 5, 3, 2)])
def test_swiglu(d, gd, H, I, R, E):
    _skip_on_a_gpu()
    need = capi.moe_gate_up_swiglu_rows_backward_workspace_bytes(d, H, I, R, E, grad_dtype=gd)
    one = capi.moe_gate_up_swiglu_rows_backward_workspace_bytes(d, H, I, R, E, grad_dtype=d)
    gz, more = SIZE[d] * 2 * R * I, (TERMS[d] if gd != d else 1) - 1
    assert more * gz <= need - one <= more * (gz + 255) and gz <= one
    assert need <= capi.moe_gate_up_swiglu_rows_backward_workspace_bytes(d, H, I, R, E)
    assert not _swiglu(d, gd, H, I, R, E, need) and _swiglu(d, gd, H, I, R, E, need - 256)
    assert not _swiglu(d, gd, H, I, R, E, one, gw=None) and _swiglu(d, gd, H, I, R, E, gz - 1, gx=None)


def test_refused():
    f, g = capi.lib().linear_rows_backward_workspace_bytes_for, capi.lib().moe_rows_gate_up_swiglu_backward_workspace_bytes_for
    assert f(BF16, F16, 0, 64, 64, 1) == f(BF16, BF16, 5, 64, 64, 1) == f(BF16, BF16, -1, 64, 64, 1) == -1
    assert f(3, 3, 0, 64, 64, 1) == f(BF16, BF16, 0, 0, 64, 1) == f(BF16, BF16, 0, 64, 64, -1) == -1
    assert g(BF16, F16, 64, 64, 8, 4) == g(F32, BF16, 64, 64, 8, 4) == g(BF16, BF16, 64, 64, 8, 0) == g(F16, F16, 0, 64, 8, 4) == -1
    most = 1 << 28
    for d in (F32, F16, BF16):
        assert f(d, F32, 4, most, most, most) == g(d, F32, most, most, most, 4096) == -1
        assert f(d, F32, 4, 1 << 12, 1 << 12, most) > 0 and g(d, F32, 1 << 12, 1 << 12, most, 4096) > 0
