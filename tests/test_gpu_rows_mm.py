"""Products of float matrices (linear with epilogue, experts' products, gate|up with SwiGLU) and their gradients
against 64 bits."""
if __name__ == "__main__":  # `python tests/<file>.py`, as the reference runs its tests
    import sys as _sys

    import pytest as _pytest
    _sys.exit(_pytest.main([__file__, "-q"]))
import pytest
import torch

import _rows_mm as R
from jjjetson_ops_amd import capi

pytestmark = pytest.mark.gpu
DTYPE_NAMES = ("bf16", "f16", "f32")
CODES = {"f32": capi.DTYPE_F32, "f16": capi.DTYPE_F16, "bf16": capi.DTYPE_BF16}
# K, N, T: one of everything, odd ones, multiples of a piece and not, around the tiles and stages
SIZES = [(1, 1, 1), (7, 5, 3), (64, 64, 1), (64, 16, 2), (40, 72, 17), (65, 129, 63), (128, 128, 128), (200, 136, 257),
         (136, 264, 130), (513, 257, 5), (1408, 520, 33), (2048, 256, 300)]


def _activations(seed, rows, cols, dtype):
    x = R.randn(seed, rows, cols, scale=0.5)
    x[:, cols // 2] *= 8.0
    return x.to(dtype)


def _linear_case(name, K, N, T, act, bias, residual, keep, dev_x=None, dev_y=None):
    d = R.DTYPES[name]
    x = _activations(1, T, K, d) if dev_x is None else dev_x
    w = R.randn(2, N, K, dtype=d, scale=K ** -0.5)
    b = R.randn(3, N, dtype=d) if bias else None
    r = R.randn(4, T, N, dtype=d) if residual else None
    y = torch.empty(T, N, dtype=d, device="cuda") if dev_y is None else dev_y
    pre = torch.empty(T, N, dtype=d, device="cuda") if keep else None
    ws = R.workspace(capi.linear_rows_workspace_bytes(CODES[name], K, N, T))
    capi.linear_rows(x, w, y, K, N, T, bias=b, residual=r, activation=R.ACTS[act], pre=pre, ws=ws)
    ref, bound, z, ez = R.linear(x, w, b, r, act)
    R.check(y, ref, bound, "y")
    if keep:
        R.check(pre, z, ez, "pre")


@pytest.mark.parametrize("K,N,T", SIZES)
@pytest.mark.parametrize("name", DTYPE_NAMES)
def test_linear(dev, name, K, N, T):
    _linear_case(name, K, N, T, "none", False, False, False)
    _linear_case(name, K, N, T, "silu", True, True, True)


@pytest.mark.parametrize("act", list(R.ACTS))
@pytest.mark.parametrize("name", DTYPE_NAMES)
def test_linear_activations(dev, name, act):
    _linear_case(name, 96, 200, 37, act, True, False, True)


@pytest.mark.parametrize("K,N,T", [(64, 8, 9), (200, 136, 70), (61, 33, 40)])
@pytest.mark.parametrize("name", DTYPE_NAMES)
def test_linear_strides(dev, name, K, N, T):
    """Slices of wider matrices, at an odd place too; the columns beside y's stay as they were; the residual in place."""
    d = R.DTYPES[name]
    for at, more in ((0, 8), (8, 24), (3, 13)):
        wide_x = _activations(1, T, K + more, d)
        wide_y = torch.full((T, N + more), 7.0, dtype=d, device="cuda")
        _linear_case(name, K, N, T, "gelu", True, False, True, wide_x[:, at:at + K], wide_y[:, at:at + N])
        assert (wide_y[:, :at] == 7.0).all() and (wide_y[:, at + N:] == 7.0).all()
    x, w, y = _activations(1, T, K, d), R.randn(2, N, K, dtype=d, scale=K ** -0.5), R.randn(5, T, N, dtype=d)
    ref, bound, _, _ = R.linear(x, w, None, y.clone(), "relu")
    capi.linear_rows(x, w, y, K, N, T, residual=y, activation=capi.ACT_RELU,
                     ws=R.workspace(capi.linear_rows_workspace_bytes(CODES[name], K, N, T)))
    R.check(y, ref, bound, "in place")


def _linear_back(name, K, N, T, act, wide, want="xwb"):
    d = R.DTYPES[name]
    x, w = _activations(1, T, K, d), R.randn(2, N, K, dtype=d, scale=K ** -0.5)
    g, pre = R.randn(3, T, N, dtype=d, scale=0.1), R.randn(4, T, N, dtype=d, scale=1.5)
    gd = torch.float32 if wide else d
    gx = torch.empty(T, K, dtype=d, device="cuda") if "x" in want else None
    gw = torch.empty(N, K, dtype=gd, device="cuda") if "w" in want else None
    gb = torch.empty(N, dtype=gd, device="cuda") if "b" in want else None
    ws = R.workspace(capi.linear_rows_backward_workspace_bytes(CODES[name], K, N, T))
    capi.linear_rows_backward(g, x if "w" in want else None, w if "x" in want else None, gx, gw, gb, K, N, T,
                              activation=R.ACTS[act], pre=None if act == "none" else pre, ws=ws)
    gz, e32, e = R.gz_of(g, pre, act, d)
    if gx is not None:
        R.check(gx, *R.mm_of(gz, e, w.t()), "grad_x")
    if gw is not None:
        # a sum over the parts of a split gradient has up to three times the additions
        _, _, ew = R.gz_of(g, pre, act, d, wide)
        ref, bound = R.mm_of(gz.t(), ew.t(), x.t())
        R.check(gw, ref, 3 * bound if wide else bound, "grad_w")
    if gb is not None:
        R.check(gb, gz.sum(0), 1.01 * (e32.sum(0) + (T + 2) * 2.0 ** -23 * gz.abs().sum(0)), "grad_b")


@pytest.mark.parametrize("K,N,T", SIZES)
@pytest.mark.parametrize("name", DTYPE_NAMES)
def test_linear_backward(dev, name, K, N, T):
    _linear_back(name, K, N, T, "none", True)
    _linear_back(name, K, N, T, "gelu_tanh", False)
    _linear_back(name, K, N, T, "gelu", True)


@pytest.mark.parametrize("act", list(R.ACTS))
@pytest.mark.parametrize("want", ["x", "w", "b", "xw", "wb"])
def test_linear_backward_parts(dev, act, want):
    _linear_back("bf16", 96, 136, 70, act, False, want)


@pytest.mark.parametrize("K,N,T", [(64, 8, 9), (200, 136, 70), (61, 33, 40)])
@pytest.mark.parametrize("name", DTYPE_NAMES)
def test_linear_backward_strides(dev, name, K, N, T):
    """Slices of wider gradients and inputs; the columns beside grad_x stay as they were."""
    d = R.DTYPES[name]
    w = R.randn(2, N, K, dtype=d, scale=K ** -0.5)
    for at, more in ((0, 8), (8, 24), (3, 13)):
        x, g = _activations(1, T, K + more, d)[:, at:at + K], R.randn(3, T, N + more, dtype=d, scale=0.1)[:, at:at + N]
        wide = torch.full((T, K + more), 7.0, dtype=d, device="cuda")
        gx, gw, gb = wide[:, at:at + K], torch.empty_like(w), torch.empty(N, dtype=d, device="cuda")
        ws = R.workspace(capi.linear_rows_backward_workspace_bytes(CODES[name], K, N, T))
        for act in ("none", "relu"):
            pre = None if act == "none" else R.randn(4, T, N, dtype=d)
            capi.linear_rows_backward(g, x, w, gx, gw, gb, K, N, T, activation=R.ACTS[act], pre=pre, ws=ws)
            gz, e32, e = R.gz_of(g, pre, act, d)
            R.check(gx, *R.mm_of(gz, e, w.t()), "grad_x")
            R.check(gw, *R.mm_of(gz.t(), e.t(), x.t()), "grad_w")
            R.check(gb, gz.sum(0), 1.01 * (e32.sum(0) + (T + 2) * 2.0 ** -23 * gz.abs().sum(0)), "grad_b")
            assert (wide[:, :at] == 7.0).all() and (wide[:, at + K:] == 7.0).all()


def test_gradients_beyond_fp16(dev):
    """A gradient that fp16 cannot hold is infinite in the fp32 gradients of the weights, and nothing beside it is lost."""
    T, K, N = 40, 64, 72
    x, g, pre = R.randn(1, T, K, dtype=torch.float16), R.randn(2, T, N, dtype=torch.float16), R.randn(3, T, N, dtype=torch.float16)
    g[5, 7], pre[5, 7] = 60000.0, 1.6  # times gelu'(1.6) = 1.12
    x[5] = x[5].abs() + 1
    gw = torch.empty(N, K, dtype=torch.float32, device="cuda")
    ws = R.workspace(capi.linear_rows_backward_workspace_bytes(CODES["f16"], K, N, T))
    capi.linear_rows_backward(g, x, None, None, gw, None, K, N, T, activation=capi.ACT_GELU, pre=pre, ws=ws)
    assert torch.isinf(gw[7]).all() and torch.isfinite(gw[:7]).all() and torch.isfinite(gw[8:]).all()


COUNTS = [[1], [0, 3, 0], [5, 0, 1, 64, 0, 65, 2, 0], [128, 129, 0, 7], [0] * 63 + [2], [3] * 70, [300, 1, 0, 20]]
# K, N of the experts
GROUPED = [(64, 64), (72, 40), (33, 17), (200, 136), (512, 264)]


@pytest.mark.parametrize("counts", COUNTS, ids=lambda c: "-".join(map(str, c[:8])))
@pytest.mark.parametrize("K,N", GROUPED)
@pytest.mark.parametrize("name", DTYPE_NAMES)
def test_grouped(dev, name, K, N, counts):
    """The products, their gradients, and SwiGLU with its; rows behind the last expert's are neither read (NaN) nor
    written."""
    d, E, n = R.DTYPES[name], len(counts), sum(counts)
    rows, offsets = n + 3, R.offsets_of(counts)
    ends = offsets.tolist()

    def padded(t):
        t[n:] = float("nan")
        return t
    x = padded(_activations(1, rows, K, d))
    w, w2 = (R.randn(s, E, N, K, dtype=d, scale=K ** -0.5) for s in (2, 3))
    y, mid = (torch.full((rows, N), 7.0, dtype=d, device="cuda") for _ in range(2))
    both = torch.full((rows, 2 * N), 7.0, dtype=d, device="cuda")
    ws = R.workspace(capi.grouped_mat_mul_rows_workspace_bytes(CODES[name], K, N, rows, E))
    capi.grouped_mat_mul_rows(x, w, offsets, y, K, N, rows, ws=ws)
    ws = R.workspace(capi.moe_gate_up_swiglu_rows_workspace_bytes(CODES[name], K, N, rows, E))
    capi.moe_gate_up_swiglu_rows(x, w, w2, offsets, E, mid, K, N, rows, gate_up=both, ws=ws)
    bare = torch.full_like(mid, 7.0)
    capi.moe_gate_up_swiglu_rows(x, w, w2, offsets, E, bare, K, N, rows, ws=ws)
    assert torch.equal(mid, bare)

    g = padded(R.randn(5, rows, N, dtype=d, scale=0.1))
    saved = padded(R.randn(6, rows, 2 * N, dtype=d, scale=1.5))
    gx, sx = (torch.full((rows, K), 7.0, dtype=d, device="cuda") for _ in range(2))
    gw, sg = torch.empty_like(w), torch.empty(E, N, K, dtype=torch.float32, device="cuda")
    su = torch.empty_like(sg)
    ws = R.workspace(capi.grouped_mat_mul_rows_backward_workspace_bytes(CODES[name], K, N, rows, E))
    capi.grouped_mat_mul_rows_backward(g, x, w, offsets, gx, gw, K, N, rows, ws=ws)
    ws = R.workspace(capi.moe_gate_up_swiglu_rows_backward_workspace_bytes(CODES[name], K, N, rows, E))
    capi.moe_gate_up_swiglu_rows_backward(g, saved, x, w, w2, offsets, E, sx, sg, su, K, N, rows, ws=ws)
    for t in (y, mid, both, gx, sx):
        assert (t[n:] == 7.0).all()
    for e in range(E):
        a, b = ends[e], ends[e + 1]
        if a == b:
            assert (gw[e] == 0).all() and (sg[e] == 0).all() and (su[e] == 0).all()
            continue
        xs, gs = x[a:b], g[a:b]
        z, ez = R.mm(xs, w[e])
        R.check(y[a:b], z, ez, f"y {e}")
        up, eu = R.mm(xs, w2[e])
        R.check(both[a:b], torch.cat([z, up], 1), torch.cat([ez, eu], 1), f"gate|up {e}")
        s = R.act(z, "silu")
        es = 1.13 * ez + 2.0 ** -19 * z.abs().clamp(min=1.0)
        R.check(mid[a:b], s * up, 1.01 * (es * up.abs() + s.abs() * eu + es * eu + 2.0 ** -23 * (s * up).abs()), f"mid {e}")
        zero = torch.zeros_like(gs, dtype=torch.float64)
        R.check(gx[a:b], *R.mm_of(gs, zero, w[e].t()), f"grad_x {e}")
        R.check(gw[e], *R.mm_of(gs.t(), zero.t(), xs.t()), f"grad_w {e}")
        gg, eg, gu, egu = R.swiglu_back(gs, saved[a:b, :N], saved[a:b, N:], d)
        ra, ea = R.mm_of(gg, eg, w[e].t())
        rb, eb = R.mm_of(gu, egu, w2[e].t())
        # one sum of 2 N products: twice the additions
        R.check(sx[a:b], ra + rb, 2 * (ea + eb), f"swiglu grad_x {e}")
        _, eg, _, egu = R.swiglu_back(gs, saved[a:b, :N], saved[a:b, N:], d, True)
        for got, gz, ez in ((sg[e], gg, eg), (su[e], gu, egu)):  # fp32: sums over all parts of the gradient
            ref, bound = R.mm_of(gz.t(), ez.t(), xs.t())
            R.check(got, ref, 3 * bound, f"grad_w_gate, grad_w_up {e}")
