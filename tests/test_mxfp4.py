"""MXFP4 and sorted-row entries without a GPU: sizes, refusals, and what the native binding reads
from its arguments (stand-ins for device tensors)."""
if __name__ == "__main__":  # `python tests/<file>.py`, as the reference runs its tests
    import sys as _sys

    import pytest as _pytest
    _sys.exit(_pytest.main([__file__, "-q"]))
import ctypes

import numpy as np
import pytest
import torch

import _mxfp4 as mx
from jjjetson_ops_amd import capi

P = ctypes.c_void_p
A, A8, W = P(16), P(8), P(256)
BAD = capi.JJO_ERR_INVALID_ARG


def test_bytes():
    assert capi.mxfp4_bytes(3, 64) == 3 * 2 * 17
    assert capi.mxfp4_bytes(1 << 20, 1 << 14) == (1 << 34) // 32 * 17
    for rows, cols in ((0, 32), (1, 0), (1, 33), (-1, 32), (1 << 60, 32)):
        assert capi.mxfp4_bytes(rows, cols) == -1
    assert capi.moe_ffn_mxfp4_workspace_bytes(4, 64, 32, 8, 2) > 0
    for bad in ((0, 64, 32, 8, 2), (4, 48, 32, 8, 2), (4, 64, 40, 8, 2), (4, 64, 32, 8, 9), (4, 64, 32, 1025, 2),
                (4, 64, 32, 64, 33)):
        assert capi.moe_ffn_mxfp4_workspace_bytes(*bad) == -1


def _calls():
    L = capi.lib()
    f32, bad = capi.DTYPE_F32, 3
    q, d = L.quantize_mxfp4_device, L.dequantize_mxfp4_device
    mm, lin, grp = L.mat_mul_mxfp4_device, L.linear_mxfp4_forward_device, L.mat_mul_mxfp4_grouped_device
    gu, ffn = L.moe_mxfp4_gate_up_swiglu_device, L.moe_mxfp4_ffn_forward_device
    dis, disb = L.moe_dispatch_rows_device, L.moe_dispatch_rows_backward_device
    com, comb = L.moe_combine_rows_device, L.moe_combine_rows_backward_device
    return {
        "q null": lambda: q(None, None, f32, 32, A, 1, 32),
        "q dtype": lambda: q(None, A, bad, 32, A, 1, 32),
        "q cols": lambda: q(None, A, f32, 48, A, 1, 48),
        "q one launch": lambda: q(None, A, f32, 1 << 15, A, 1 << 20, 1 << 15),
        "dq one launch": lambda: d(None, A, A, f32, 1 << 15, 1 << 20, 1 << 15),
        "q rows": lambda: q(None, A, f32, 32, A, 0, 32),
        "q aligned": lambda: q(None, A8, f32, 32, A, 1, 32),
        "q stride below": lambda: q(None, A, f32, 28, A, 2, 32),
        "q stride unaligned": lambda: q(None, A, capi.DTYPE_BF16, 36, A, 2, 32),
        "q grid": lambda: q(None, A, f32, 32, A, 1 << 40, 32),
        "d null": lambda: d(None, A, None, f32, 32, 1, 32),
        "d cols": lambda: d(None, A, A, f32, 31, 1, 31),
        "mm null": lambda: mm(A, None, A, f32, 32, 4, 1, None),
        "mm K": lambda: mm(A, A, A, f32, 48, 4, 1, None),
        "mm N": lambda: mm(A, A, A, f32, 32, 0, 1, None),
        "mm aligned": lambda: mm(A8, A, A, f32, 32, 4, 1, None),
        "mm dtype": lambda: mm(A, A, A, -1, 32, 4, 1, None),
        "mm batch": lambda: mm(A, A, A, f32, 32, 4, (1 << 28) + 1, None),
        "linear ws": lambda: lin(None, None, A, f32, A, A, f32, 32, 4, 2),
        "linear dtype": lambda: lin(None, A, A, bad, A, A, f32, 32, 4, 2),
        "linear K": lambda: lin(None, A, A, f32, A, A, f32, 33, 4, 2),
        "linear T": lambda: lin(None, A, A, f32, A, A, f32, 32, 4, 0),
        "grouped offsets": lambda: grp(A, A, None, 8, None, A, f32, 32, 4, 4, None),
        "grouped experts": lambda: grp(A, A, A, 4097, None, A, f32, 32, 4, 4, None),
        "gate_up I": lambda: gu(None, A, A, A, A, 8, A, 32, 40, 4),
        "gate_up w_up": lambda: gu(None, A, A8, A, A, 8, A, 32, 32, 4),
        "ffn dtype": lambda: ffn(None, A, A, A, A, A, A, bad, 4, 32, 32, 8, 2, W, 1 << 30),
        "ffn ws": lambda: ffn(None, A, A, A, A, A, A, f32, 4, 32, 32, 8, 2, W, 16),
        "ffn ws aligned": lambda: ffn(None, A, A, A, A, A, A, f32, 4, 32, 32, 8, 2, A, 1 << 30),
        "ffn null": lambda: ffn(None, A, None, A, A, A, A, f32, 4, 32, 32, 8, 2, W, 1 << 30),
        "ffn top_k": lambda: ffn(None, A, A, A, A, A, A, f32, 4, 32, 32, 2, 3, W, 1 << 30),
        "dispatch null": lambda: dis(None, A, A, f32, 4, 2, 32, 8, A, A, None, A),
        "dispatch top_k": lambda: dis(None, A, A, f32, 4, 33, 32, 64, A, A, A, A),
        "dispatch experts": lambda: dis(None, A, A, f32, 4, 2, 32, 1025, A, A, A, A),
        "dispatch tokens": lambda: dis(None, A, A, f32, 0, 2, 32, 8, A, A, A, A),
        "dispatch routes": lambda: dis(None, A, A, f32, 1 << 23, 32, 32, 64, A, A, A, A),
        "dispatch_backward": lambda: disb(None, A, f32, A, None, 4, 32, 2),
        "combine hidden": lambda: com(None, A, f32, A, A, A, 4, 0, 2),
        "combine null": lambda: com(None, A, f32, A, None, A, 4, 32, 2),
        "combine_backward": lambda: comb(None, A, A, f32, A, A, A, None, 4, 32, 2),
        "combine_backward dtype": lambda: comb(None, A, A, bad, A, A, A, A, 4, 32, 2),
    }


@pytest.mark.parametrize("name", sorted(_calls()))
def test_refused_before_a_device_is_touched(name):
    assert _calls()[name]() == BAD, capi.lib().jjo_last_error()
    assert capi.lib().jjo_last_error()


class Fake:
    """What the binding reads of a device tensor."""

    def __init__(self, dtype=torch.float32, n=1 << 20, device=0, contiguous=True):
        self.dtype, self._n, self._device, self._c, self.is_cuda = dtype, n, device, contiguous, device >= 0

    def numel(self):
        return self._n

    def element_size(self):
        return torch.empty(0, dtype=self.dtype).element_size()

    def is_contiguous(self):
        return self._c

    def get_device(self):
        return self._device

    def data_ptr(self):
        return 0x1000

    def dim(self):
        return 1


@pytest.fixture
def on_device_0(monkeypatch):
    monkeypatch.setattr(capi, "_current_device", lambda: 0)


F32, U8, I32 = torch.float32, torch.uint8, torch.int32


@pytest.mark.parametrize("bad,text", [(Fake(device=-1), "must be a device tensor"),
                                      (Fake(contiguous=False), "must be contiguous"),
                                      (Fake(device=1), "is on device 1, the current device is 0"),
                                      (Fake(dtype=torch.float64), "must be float32, float16 or bfloat16"),
                                      (Fake(n=3), "is too small")])
def test_wrapper_refuses_tensors(bad, text, on_device_0):
    with pytest.raises(ValueError, match="y " + text):
        capi.mat_mul_mxfp4(Fake(U8), Fake(U8), bad, 32, 4, 1, stream=0)


def test_wrapper_refuses_sizes(on_device_0):
    t, u, i = Fake(), Fake(U8), Fake(I32)
    small, short = Fake(U8, n=16), Fake(I32, n=1)
    for call, text in ((lambda: capi.quantize_mxfp4(t, small, 1, 32, stream=0), "out is too small"),
                       (lambda: capi.dequantize_mxfp4(small, t, 1, 32, stream=0), "q is too small"),
                       (lambda: capi.linear_mxfp4(t, u, t, 32, 4, 2, ws=small, stream=0), "ws is smaller"),
                       (lambda: capi.linear_mxfp4(t, small, t, 32, 4, 2, ws=u, stream=0), "w is too small"),
                       (lambda: capi.grouped_mat_mul_mxfp4(u, u, short, t, 32, 4, 2, stream=0), "expert_offsets"),
                       (lambda: capi.grouped_mat_mul_mxfp4(u, u, Fake(I32, n=9), t, 32, 4, 2, route_dst=short, stream=0),
                        "route_dst"),
                       (lambda: capi.moe_gate_up_swiglu_mxfp4(u, u, u, short, 8, u, 32, 32, 2, stream=0), "offsets"),
                       (lambda: capi.moe_ffn_mxfp4(t, Fake(n=3), u, u, u, t, 4, 32, 32, 8, 2, u, stream=0), "logits"),
                       (lambda: capi.moe_ffn_mxfp4(t, t, u, u, u, Fake(torch.float16), 4, 32, 32, 8, 2, u, stream=0),
                        "y must have"),
                       (lambda: capi.moe_dispatch_rows(short, t, t, i, i, i, 4, 2, 32, 8, stream=0), "ids"),
                       (lambda: capi.moe_dispatch_rows(i, t, Fake(n=9), i, i, i, 4, 2, 32, 8, stream=0), "x_sorted"),
                       (lambda: capi.moe_dispatch_rows_backward(t, t, t, 4, 32, 2, stream=0), "dst_of_route"),
                       (lambda: capi.moe_combine_rows(t, i, i, t, 4, 32, 2, stream=0), "weights"),
                       (lambda: capi.moe_combine_rows_backward(t, t, i, t, t, Fake(n=1), 4, 32, 2, stream=0),
                        "grad_weights")):
        with pytest.raises(ValueError, match=text):
            call()
    with pytest.raises(TypeError, match="M must be an int"):
        capi._entry(capi._MAT_MUL, "x", 0, u, u, t, 0, 32, 4, 1.0)
    with pytest.raises(ValueError, match="M is out of range"):
        capi._entry(capi._MAT_MUL, "x", 0, u, u, t, 0, 32, 4, 1 << 31)
    with pytest.raises(capi.JJOError) as e:
        capi.mat_mul_mxfp4(u, u, t, 48, 4, 1, stream=0)
    assert e.value.code == BAD and "ncols_k=48" in str(e.value)


def test_scattered_outputs_need_a_row(on_device_0):
    """With route_dst the rows of y are the table's to name, but there is at least one."""
    u, i = Fake(U8), Fake(I32, n=9)
    for n in (0, 3):
        with pytest.raises(ValueError, match="y is too small"):
            capi.grouped_mat_mul_mxfp4(u, u, i, Fake(n=n), 32, 4, 2, route_dst=i, stream=0)


def test_oracle_of_the_format():
    """The oracle's rounding against the nearest of all e2m1 values, ties to the even code."""
    v = np.concatenate([np.linspace(-8, 8, 4097), np.array(mx.BOUNDS), np.nextafter(mx.BOUNDS, 0)])
    got = mx.values(mx.round_codes(v))
    d = np.abs(np.abs(v)[:, None] - mx.E2M1[None, :])
    best = d.min(1)
    for a, g, b, row in zip(v, got, best, d):
        assert abs(abs(a) - abs(g)) == b
        ties = np.flatnonzero(row == b)
        assert len(ties) == 1 or mx.E2M1.tolist().index(abs(g)) % 2 == 0
    x = np.array([[2.0 ** -126] + [0.0] * 31 + [6.0] * 32 + [np.inf] + [1.0] * 31 + [np.nan] + [1.0] * 31 + [0.0] * 32])
    code, s = mx.quantize(x)
    assert s[0].tolist() == [0, 127, 255, 255, 0] and code[0, 0] == 4 and code[0, 32] == 7
    assert np.array_equal(mx.unpack(mx.pack(code, s), 1, 160)[0], code)
