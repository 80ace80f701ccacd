"""Float products through the public entries where precision or a kernel's way differs: the terms of a gradient that
is split for fp32 weights' gradients, epilogues and saved sums on every tile, rows that are not 16-byte aligned."""
if __name__ == "__main__":  # `python tests/<file>.py`, as the reference runs its tests
    import sys as _sys

    import pytest as _pytest
    _sys.exit(_pytest.main([__file__, "-q"]))
import pytest
import torch

import _rows_mm as R
import _rows_paths as P
from jjjetson_ops_amd import capi

pytestmark = pytest.mark.gpu
CODES = {"f32": capi.DTYPE_F32, "f16": capi.DTYPE_F16, "bf16": capi.DTYPE_BF16}


def _kept(gz, dtype):
    """What two terms of fp16, the second times 2^11, or three of bf16 keep of a gradient: half a step of each term,
    2^-11 * 2^-11 or 2^-8 * 2^-8 * 2^-8 of the value; fp16's last term has steps of 2^-24 times 2^-11 at the least."""
    if dtype == torch.float16:
        return (2.0 ** -22 * gz.abs()).clamp(min=2.0 ** -36)
    return 2.0 ** -24 * gz.abs()


def _added(gz, dtype):
    """What an addition may be off by, per unit of x: 2^-23 of the product.  The matrix unit does not normalize fp16's
    subnormals: a product of one is exact, but is aligned for an addition by the exponents that its operands have,
    and so cut as one of 2^-14 would be, 2^-23 * 2^-14 (g of 1e-5 and of 1e-6 show it with grad_y's own product: one
    token is exact, two are off by up to 2^-39 |x|, of either size)."""
    return 2.0 ** -23 * (gz.abs().clamp(min=2.0 ** -14) if dtype == torch.float16 else gz.abs())


@pytest.mark.parametrize("scale", [1.0, 1e-2, 1e-3, 1e-4, 1e-5])
@pytest.mark.parametrize("name", ["f16", "bf16"])
def test_terms_keep_their_bits(dev, name, scale):
    """fp32 weights' gradients from gradients of any size: two tokens, so that the error is that of gz, 2^-19 of the
    derivative at |z| < 2 (its own fp32), and of up to six products.  fp16's grad_y has its own steps below 2^-14 and is
    taken as it is."""
    d, T, K, N = R.DTYPES[name], 2, 72, 520
    x = R.randn(1, T, K, dtype=d)
    g, pre = R.randn(2, T, N, scale=scale).to(d), R.randn(3, T, N, dtype=d).clamp(-2, 2)
    gw = torch.empty(N, K, dtype=torch.float32, device="cuda")
    ws = R.workspace(capi.linear_rows_backward_workspace_bytes(CODES[name], K, N, T))
    for act in ("gelu", "gelu_tanh", "silu"):
        capi.linear_rows_backward(g, x, None, None, gw, None, K, N, T, activation=R.ACTS[act], pre=pre, ws=ws)
        gz, e32, _ = R.gz_of(g, pre, act, d)
        ref = gz.t() @ x.double()
        bound = (e32 + _kept(gz, d) + 10 * _added(gz, d)).t() @ x.double().abs()
        R.check(gw, ref, bound, f"{act} grad_w")
    # SwiGLU: both halves, one expert with a row of its own
    rows, E = 3, 3
    offsets = R.offsets_of([1, 0, 2])
    xs, gm = R.randn(4, rows, K, dtype=d), R.randn(5, rows, N, scale=scale).to(d)
    both = R.randn(6, rows, 2 * N, dtype=d).clamp(-2, 2)
    gg, gu = (torch.empty(E, N, K, dtype=torch.float32, device="cuda") for _ in range(2))
    ws = R.workspace(capi.moe_gate_up_swiglu_rows_backward_workspace_bytes(CODES[name], K, N, rows, E))
    capi.moe_gate_up_swiglu_rows_backward(gm, both, xs, None, None, offsets, E, None, gg, gu, K, N, rows, ws=ws)
    gate, up, g64 = both[:, :N].double(), both[:, N:].double(), gm.double()
    for got, gz, at_one in ((gg, g64 * up * R.slope(gate, "silu"), g64 * up), (gu, g64 * R.act(gate, "silu"), g64)):
        e = at_one.abs() * 2.0 ** -19 * gate.abs().clamp(min=1.0) + _kept(gz, d)
        for k, (a, b) in enumerate(((0, 1), (1, 1), (1, 3))):
            xe = xs[a:b].double()
            R.check(got[k], gz[a:b].t() @ xe, (e + 10 * _added(gz, d))[a:b].t() @ xe.abs(), f"expert {k}")


@pytest.mark.parametrize("name", list(R.DTYPES))
def test_relu_lets_nothing_through_where_it_is_zero(dev, name):
    """Infinite and NaN gradients at z <= 0 are zeros behind relu; at z > 0 they stay, and so does a NaN of z."""
    d, T, K, N = R.DTYPES[name], 5, 24, 40
    x, w, g = R.randn(1, T, K, dtype=d), R.randn(2, N, K, dtype=d), R.randn(3, T, N, dtype=d)
    pre = R.randn(4, T, N, dtype=d)
    pre[0, :4] = torch.tensor([0.0, -1.0, -0.0, float("-inf")])
    g[0, :4] = torch.tensor([float("inf"), float("-inf"), float("nan"), float("inf")])
    pre[1, 7], g[1, 7], pre[2, 8] = 1.0, float("inf"), float("nan")
    gx, gw, gb = torch.empty_like(x), torch.empty_like(w), torch.empty(N, dtype=d, device="cuda")
    ws = R.workspace(capi.linear_rows_backward_workspace_bytes(CODES[name], K, N, T))
    capi.linear_rows_backward(g, x, w, gx, gw, gb, K, N, T, activation=capi.ACT_RELU, pre=pre, ws=ws)
    assert gb[7] == float("inf") and gb[8].isnan() and not torch.isfinite(gx[1:3]).any()
    gz = torch.where(pre > 0, g, 0.0).double()
    zero = torch.zeros_like(gz)
    rows, cols = [0, 3, 4], [n for n in range(N) if n not in (7, 8)]
    R.check(gx[rows], *R.mm_of(gz[rows], zero[rows], w.t()), "grad_x")
    R.check(gw[cols], *R.mm_of(gz.t()[cols], zero.t()[cols], x.t()), "grad_w")
    R.check(gb[cols], gz.sum(0)[cols], (T + 2) * 2.0 ** -23 * gz.abs().sum(0)[cols], "grad_b")


@pytest.mark.parametrize("name", list(R.DTYPES))
def test_gelu_keeps_its_lower_tail(dev, name):
    """gelu and its derivative from z = -12 to 12: relative to the normal distribution's tail, not to 1.  Its error: that of
    erfc's argument x = z / sqrt 2, 2^-23.6 of itself (constant and product), which erfc's slope makes 2 x^2 = 144 times
    as much, 2^-16.4; that of e^(-x^2)'s argument, rounded twice, 72 * 2^-23 = 2^-16.8; of the fit 2^-19.8 (erfcf: 16
    ulp) and a few more steps: 2^-15 in all.  fp16 and its subnormals end at z = -5.5."""
    d = R.DTYPES[name]
    z = torch.linspace(-12, 12, 4801, device="cuda").to(d)
    N, x, y = z.numel(), torch.ones(1, 1, dtype=d, device="cuda"), torch.empty(1, z.numel(), dtype=d, device="cuda")
    capi.linear_rows(x, z.view(-1, 1).contiguous(), y, 1, N, 1, activation=capi.ACT_GELU)
    z64 = z.double()
    tail = 0.5 * torch.special.erfc(-z64 * 0.5 ** 0.5)
    R.check(y[0], z64 * tail, 2.0 ** -15 * (z64 * tail).abs(), "gelu")
    gb = torch.empty(N, dtype=torch.float32, device="cuda")
    ws = R.workspace(capi.linear_rows_backward_workspace_bytes(CODES[name], 1, N, 1))
    capi.linear_rows_backward(torch.ones_like(y), None, None, None, None, gb, 1, N, 1, activation=capi.ACT_GELU, pre=z, ws=ws)
    density = z64 * torch.exp(-0.5 * z64 * z64) / (2 * torch.pi) ** 0.5
    R.check(gb, tail + density, 2.0 ** -15 * (tail + density.abs()), "its derivative")


@pytest.mark.parametrize("name", list(R.DTYPES))
@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
def test_activations_far_out(dev, name, act):
    """Any finite z: the activation and its derivative end as z and 1 above, 0 and 0 below."""
    d = R.DTYPES[name]
    most = torch.finfo(d).max
    z = torch.tensor([s * v for v in (100.0, 1e4, 6e4, 1e13, 2e19, 1e30, most) if v <= most for s in (1, -1)], device="cuda").to(d)
    N, x, y = z.numel(), torch.ones(1, 1, dtype=d, device="cuda"), torch.empty(1, z.numel(), dtype=d, device="cuda")
    capi.linear_rows(x, z.view(-1, 1).contiguous(), y, 1, N, 1, activation=R.ACTS[act])
    assert torch.equal(y[0], z.clamp(min=0.0))
    gb = torch.empty(N, dtype=torch.float32, device="cuda")
    ws = R.workspace(capi.linear_rows_backward_workspace_bytes(CODES[name], 1, N, 1))
    capi.linear_rows_backward(torch.ones_like(y), None, None, None, None, gb, 1, N, 1, activation=R.ACTS[act], pre=z, ws=ws)
    assert torch.equal(gb, (z > 0).float())


@pytest.mark.parametrize("act", list(R.ACTS))
@pytest.mark.parametrize("sizes", [s[0] for s in P.LINEAR], ids=lambda s: "-".join(map(str, s)))
def test_epilogues_of_every_tile(dev, sizes, act):
    """Bias, activation, residual and the kept sums together, and each alone, on every tile and behind slices."""
    name, K, N, T = sizes
    d = R.DTYPES[name]
    x, w = R.randn(1, T, K, dtype=d), R.randn(2, N, K, dtype=d, scale=K ** -0.5)
    bias, residual = R.randn(3, N, dtype=d), R.randn(4, T, N, dtype=d)
    ws = R.workspace(capi.linear_rows_workspace_bytes(CODES[name], K, N, T))
    for b, r, keep in ((bias, residual, True), (None, None, False), (bias, None, False), (None, residual, False)):
        y = torch.empty(T, N, dtype=d, device="cuda")
        pre = torch.empty_like(y) if keep else None
        capi.linear_rows(x, w, y, K, N, T, bias=b, residual=r, activation=R.ACTS[act], pre=pre, ws=ws)
        ref, bound, z, ez = R.linear(x, w, b, r, act)
        R.check(y, ref, bound, "y")
        if keep:
            R.check(pre, z, ez, "pre")


@pytest.mark.parametrize("sizes", [s[0] for s in P.SWIGLU_FORWARD], ids=lambda s: "-".join(map(str, s[:3])))
def test_swiglu_of_every_tile(dev, sizes):
    """mid alone, and with the saved gate|up, the same bits; rows behind the last expert's as they were."""
    name, H, I, counts = sizes
    d, E, n = R.DTYPES[name], len(counts), sum(counts)
    offsets = R.offsets_of(counts)
    ends = offsets.tolist()
    x = R.randn(1, n + 5, H, dtype=d)
    wg, wu = (R.randn(s, E, I, H, dtype=d, scale=H ** -0.5) for s in (2, 3))
    mid, bare = (torch.full((n + 5, I), 7.0, dtype=d, device="cuda") for _ in range(2))
    both = torch.full((n + 5, 2 * I), 7.0, dtype=d, device="cuda")
    ws = R.workspace(capi.moe_gate_up_swiglu_rows_workspace_bytes(CODES[name], H, I, n + 5, E))
    capi.moe_gate_up_swiglu_rows(x, wg, wu, offsets, E, mid, H, I, n + 5, gate_up=both, ws=ws)
    capi.moe_gate_up_swiglu_rows(x, wg, wu, offsets, E, bare, H, I, n + 5, ws=ws)
    assert torch.equal(mid, bare) and (mid[n:] == 7.0).all() and (both[n:] == 7.0).all()
    for e in range(E):
        a, b = ends[e], ends[e + 1]
        z, ez = R.mm(x[a:b], wg[e])
        up, eu = R.mm(x[a:b], wu[e])
        R.check(both[a:b, :I], z, ez, f"gate {e}")
        R.check(both[a:b, I:], up, eu, f"up {e}")
        s, es = R.act(z, "silu"), 1.13 * ez + 2.0 ** -19 * z.abs().clamp(min=1.0)
        R.check(mid[a:b], s * up, 1.01 * (es * up.abs() + s.abs() * eu + es * eu + 2.0 ** -23 * (s * up).abs()), f"mid {e}")


def _terms(name):
    return {"f16": 2, "bf16": 3}.get(name, 1)


def _split_sum(gz, e, x, terms, d):
    """gz^T . x of a split gradient that is off by e, and its bound: one sum of `terms` parts of each product."""
    x = x.double()
    n = terms * x.shape[0] + 2
    return gz.t() @ x, (e + _kept(gz, d) + n * _added(gz, d)).t() @ x.abs()


@pytest.mark.parametrize("sizes", [s[0] for s in P.WEIGHTS] + [("bf16", 515, 333, 500), ("f16", 515, 333, 500), ("f16", 33, 1407, 70),
                                                               ("bf16", 1407, 33, 70)],
                         ids=lambda s: "-".join(map(str, s)))
def test_terms_on_every_tile(dev, sizes):
    """fp32 weights' gradients of 16 bits, a term's sums of several stages and a part of one."""
    name, K, N, T = sizes
    d = R.DTYPES[name]
    x, g, pre = R.randn(1, T, K, dtype=d), R.randn(2, T, N, dtype=d, scale=0.1), R.randn(3, T, N, dtype=d).clamp(-2, 2)
    gw = torch.empty(N, K, dtype=torch.float32, device="cuda")
    ws = R.workspace(capi.linear_rows_backward_workspace_bytes(CODES[name], K, N, T))
    capi.linear_rows_backward(g, x, None, None, gw, None, K, N, T, activation=capi.ACT_SILU, pre=pre, ws=ws)
    gz, e32, _ = R.gz_of(g, pre, "silu", d)
    R.check(gw, *_split_sum(gz, e32, x, _terms(name), d), "grad_w")


@pytest.mark.parametrize("sizes", [s[0] for s in P.SWIGLU_WEIGHTS] + [("f16", 515, 333, (200, 1, 0, 131)),
                                                                      ("bf16", 333, 515, (1, 0, 70, 261))],
                         ids=lambda s: "-".join(map(str, s[:3])))
def test_terms_of_both_halves_on_every_tile(dev, sizes):
    name, H, I, counts = sizes
    d, E, n = R.DTYPES[name], len(counts), sum(counts)
    offsets = R.offsets_of(counts)
    ends = offsets.tolist()
    x, gm = R.randn(1, n + 5, H, dtype=d), R.randn(2, n + 5, I, dtype=d, scale=0.1)
    both = R.randn(3, n + 5, 2 * I, dtype=d).clamp(-2, 2)
    wg, wu = (R.randn(s, E, I, H, dtype=d, scale=I ** -0.5) for s in (4, 5))
    gx = torch.full((n + 5, H), 7.0, dtype=d, device="cuda")
    gg, gu = (torch.empty(E, I, H, dtype=torch.float32, device="cuda") for _ in range(2))
    ws = R.workspace(capi.moe_gate_up_swiglu_rows_backward_workspace_bytes(CODES[name], H, I, n + 5, E))
    capi.moe_gate_up_swiglu_rows_backward(gm, both, x, wg, wu, offsets, E, gx, gg, gu, H, I, n + 5, ws=ws)
    assert (gx[n:] == 7.0).all()
    for e in range(E):
        a, b = ends[e], ends[e + 1]
        gate, up, g64 = both[a:b, :I].double(), both[a:b, I:].double(), gm[a:b].double()
        big = 2.0 ** -19 * gate.abs().clamp(min=1.0)
        for got, gz, e32 in ((gg[e], g64 * up * R.slope(gate, "silu"), (g64 * up).abs() * big),
                             (gu[e], g64 * R.act(gate, "silu"), g64.abs() * big)):
            R.check(got, *_split_sum(gz, e32, x[a:b], _terms(name), d), f"expert {e}")
        ga, ea, gb, eb = R.swiglu_back(gm[a:b], both[a:b, :I], both[a:b, I:], d)
        (ra, ba), (rb, bb) = R.mm_of(ga, ea, wg[e].t()), R.mm_of(gb, eb, wu[e].t())
        R.check(gx[a:b], ra + rb, 2 * (ba + bb), f"grad_x {e}")


# Rows that are not 16-byte aligned: few and many tiles, slices, several stages, edges inside a piece of 16 bytes
ODD = [(1031, 515, 40), (4095, 129, 70), (2047, 1407, 130), (515, 4095, 33), (1025, 3, 300), (3, 1025, 300), (9, 9, 9), (64, 63, 65)]


@pytest.mark.parametrize("K,N,T", ODD)
@pytest.mark.parametrize("name", list(R.DTYPES))
def test_odd_rows(dev, name, K, N, T):
    d = R.DTYPES[name]
    x, w = R.randn(1, T, K, dtype=d), R.randn(2, N, K, dtype=d, scale=K ** -0.5)
    g, pre = R.randn(3, T, N, dtype=d, scale=0.1), R.randn(4, T, N, dtype=d).clamp(-2, 2)
    bias, residual = R.randn(5, N, dtype=d), R.randn(6, T, N, dtype=d)
    y, z_kept, gx = torch.empty(T, N, dtype=d, device="cuda"), torch.empty(T, N, dtype=d, device="cuda"), torch.empty_like(x)
    gb, narrow = (torch.empty(N, dtype=torch.float32, device="cuda"), torch.empty(N, K, dtype=d, device="cuda"))
    wide = torch.empty(N, K, dtype=torch.float32, device="cuda")
    ws = R.workspace(capi.linear_rows_workspace_bytes(CODES[name], K, N, T))
    capi.linear_rows(x, w, y, K, N, T, bias=bias, residual=residual, activation=capi.ACT_GELU, pre=z_kept, ws=ws)
    ref, bound, z, ez = R.linear(x, w, bias, residual, "gelu")
    R.check(y, ref, bound, "y")
    R.check(z_kept, z, ez, "pre")
    ws = R.workspace(capi.linear_rows_backward_workspace_bytes(CODES[name], K, N, T))
    capi.linear_rows_backward(g, x, w, gx, wide, gb, K, N, T, activation=capi.ACT_SILU, pre=pre, ws=ws)
    capi.linear_rows_backward(g, x, None, None, narrow, None, K, N, T, ws=ws)
    gz, e32, e = R.gz_of(g, pre, "silu", d)
    R.check(gx, *R.mm_of(gz, e, w.t()), "grad_x")
    if name == "f32":
        R.check(wide, *R.mm_of(gz.t(), e.t(), x.t()), "grad_w")
    else:
        R.check(wide, *_split_sum(gz, e32, x, _terms(name), d), "grad_w")
    R.check(narrow, *R.mm(g.t(), x.t()), "grad_w of grad_y itself")
    R.check(gb, gz.sum(0), 1.01 * (e32.sum(0) + (T + 2) * 2.0 ** -23 * gz.abs().sum(0)), "grad_b")


@pytest.mark.parametrize("K,N", [(2047, 333), (333, 1407), (65, 9), (1031, 1031)])
@pytest.mark.parametrize("name", list(R.DTYPES))
def test_odd_rows_of_experts(dev, name, K, N):
    """The experts' products, SwiGLU and their gradients, rows of ragged experts that no 16-byte alignment has; what is
    behind the last row of x and of the gradients is not read (NaN) and not written."""
    d, counts = R.DTYPES[name], [5, 0, 130, 1, 64, 0, 200, 17]
    E, n, rows = len(counts), sum(counts), sum(counts) + 3
    offsets = R.offsets_of(counts)
    ends = offsets.tolist()
    x, g, both = R.randn(1, rows, K, dtype=d), R.randn(2, rows, N, dtype=d), R.randn(3, rows, 2 * N, dtype=d).clamp(-2, 2)
    for t in (x, g, both):
        t[n:] = float("nan")
    w, w2 = (R.randn(s, E, N, K, dtype=d, scale=K ** -0.5) for s in (4, 5))
    y, mid = (torch.full((rows, N), 7.0, dtype=d, device="cuda") for _ in range(2))
    gx, sx = (torch.full((rows, K), 7.0, dtype=d, device="cuda") for _ in range(2))
    gw, sg, su = (torch.empty(E, N, K, dtype=d, device="cuda") for _ in range(3))
    need = max(f(CODES[name], K, N, rows, E) for f in (
        capi.grouped_mat_mul_rows_workspace_bytes, capi.grouped_mat_mul_rows_backward_workspace_bytes,
        capi.moe_gate_up_swiglu_rows_workspace_bytes, capi.moe_gate_up_swiglu_rows_backward_workspace_bytes))
    ws = R.workspace(need)
    capi.grouped_mat_mul_rows(x, w, offsets, y, K, N, rows, ws=ws)
    capi.moe_gate_up_swiglu_rows(x, w, w2, offsets, E, mid, K, N, rows, ws=ws)
    capi.grouped_mat_mul_rows_backward(g, x, w, offsets, gx, gw, K, N, rows, ws=ws)
    capi.moe_gate_up_swiglu_rows_backward(g, both, x, w, w2, offsets, E, sx, sg, su, K, N, rows, ws=ws)
    for t in (y, mid, gx, sx):
        assert (t[n:] == 7.0).all()
    for e in range(E):
        a, b = ends[e], ends[e + 1]
        if a == b:
            assert (gw[e] == 0).all() and (sg[e] == 0).all() and (su[e] == 0).all()
            continue
        z, ez = R.mm(x[a:b], w[e])
        up, eu = R.mm(x[a:b], w2[e])
        R.check(y[a:b], z, ez, f"y {e}")
        s, es = R.act(z, "silu"), 1.13 * ez + 2.0 ** -19 * z.abs().clamp(min=1.0)
        R.check(mid[a:b], s * up, 1.01 * (es * up.abs() + s.abs() * eu + es * eu + 2.0 ** -23 * (s * up).abs()), f"mid {e}")
        R.check(gx[a:b], *R.mm(g[a:b], w[e].t()), f"grad_x {e}")
        R.check(gw[e], *R.mm(g[a:b].t(), x[a:b].t()), f"grad_w {e}")
        ga, ea, gb, eb = R.swiglu_back(g[a:b], both[a:b, :N], both[a:b, N:], d)
        (ra, ba), (rb, bb) = R.mm_of(ga, ea, w[e].t()), R.mm_of(gb, eb, w2[e].t())
        R.check(sx[a:b], ra + rb, 2 * (ba + bb), f"swiglu grad_x {e}")
        R.check(sg[e], *R.mm_of(ga.t(), ea.t(), x[a:b].t()), f"grad_w_gate {e}")
        R.check(su[e], *R.mm_of(gb.t(), eb.t(), x[a:b].t()), f"grad_w_up {e}")


@pytest.mark.parametrize("name", list(R.DTYPES))
def test_odd_places(dev, name):
    """Sizes of whole pieces at odd addresses and strides: slices of wider matrices, on every tile that is chosen by the
    sizes alone; what is beside the outputs stays as it was."""
    d = R.DTYPES[name]
    for K, N, T in ((264, 520, 100), (2056, 264, 77), (136, 5128, 1990)):
        x = R.randn(1, T, K + 5, dtype=d)[:, 3:3 + K]
        w = R.randn(2, N * K + 1, dtype=d, scale=K ** -0.5)[1:].view(N, K)
        wide = torch.full((T, N + 3), 7.0, dtype=d, device="cuda")
        y = wide[:, 1:1 + N]
        ws = R.workspace(capi.linear_rows_workspace_bytes(CODES[name], K, N, T))
        capi.linear_rows(x, w, y, K, N, T, activation=capi.ACT_SILU, ws=ws)
        ref, bound, _, _ = R.linear(x, w, None, None, "silu")
        R.check(y, ref, bound, "y")
        assert (wide[:, :1] == 7.0).all() and (wide[:, 1 + N:] == 7.0).all()
        g = R.randn(3, T, N + 7, dtype=d, scale=0.1)[:, 1:1 + N]
        wide = torch.full((T, K + 3), 7.0, dtype=d, device="cuda")
        gx, gw = wide[:, 1:1 + K], torch.full((N * K + 2,), 7.0, dtype=d, device="cuda")
        ws = R.workspace(capi.linear_rows_backward_workspace_bytes(CODES[name], K, N, T))
        capi.linear_rows_backward(g, x, w, gx, gw[1:-1].view(N, K), None, K, N, T, ws=ws)
        R.check(gx, *R.mm(g, w.t()), "grad_x")
        R.check(gw[1:-1].view(N, K), *R.mm(g.t(), x.t()), "grad_w")
        assert (wide[:, :1] == 7.0).all() and (wide[:, 1 + K:] == 7.0).all() and gw[0] == 7.0 and gw[-1] == 7.0


@pytest.mark.parametrize("K,N,T", [(136, 264, 70), (4096, 520, 64), (515, 333, 40)])
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("name", list(R.DTYPES))
def test_workspaces_of_a_call_are_enough(dev, name, wide, K, N, T):
    """Gradients with the workspace of just their activation and type: the same bits as with the largest, and nothing
    behind it is written."""
    d, gd = R.DTYPES[name], torch.float32 if wide else R.DTYPES[name]
    code, g_code = CODES[name], CODES["f32"] if wide else CODES[name]
    counts = [T // 2, 0, T - T // 2]
    offsets, E = R.offsets_of(counts), 3
    x, g, pre = R.randn(1, T, K, dtype=d), R.randn(2, T, N, dtype=d), R.randn(3, T, N, dtype=d)
    w, both = R.randn(4, E, N, K, dtype=d), R.randn(5, T, 2 * N, dtype=d)

    def linear(act, ws):
        out = torch.empty(T, K, dtype=d, device="cuda"), torch.empty(N, K, dtype=gd, device="cuda"), torch.empty(N, dtype=gd, device="cuda")
        capi.linear_rows_backward(g, x, w[0], *out, K, N, T, activation=act, pre=pre, ws=ws)
        return out

    def experts(ws):
        out = torch.empty(T, K, dtype=d, device="cuda"), *(torch.empty(E, N, K, dtype=gd, device="cuda") for _ in range(2))
        capi.moe_gate_up_swiglu_rows_backward(g, both, x, w, w, offsets, E, *out, K, N, T, ws=ws)
        return out
    most = R.workspace(capi.linear_rows_backward_workspace_bytes(code, K, N, T))
    cases = [(lambda ws, act=act: linear(act, ws), most,
              capi.linear_rows_backward_workspace_bytes(code, K, N, T, activation=act, grad_dtype=g_code))
             for act in (capi.ACT_NONE, capi.ACT_GELU)]
    most = R.workspace(capi.moe_gate_up_swiglu_rows_backward_workspace_bytes(code, K, N, T, E))
    cases.append((experts, most, capi.moe_gate_up_swiglu_rows_backward_workspace_bytes(code, K, N, T, E, grad_dtype=g_code)))
    for call, largest, need in cases:
        guarded = torch.full((need + 1024,), 0x5a, dtype=torch.uint8, device="cuda")
        for a, b in zip(call(largest), call(guarded[:need])):
            assert torch.equal(a, b)
        assert (guarded[need:] == 0x5a).all()


@pytest.mark.parametrize("name", list(R.DTYPES))
def test_rows_far_apart(dev, name):
    """Strides of 8 MiB and more, at which a tile's offsets leave 32 bits."""
    d, K, N, T = R.DTYPES[name], 72, 40, 5
    stride = (1 << 23) // d.itemsize
    for step in (stride - 8, stride, stride + 8, stride + 3):
        far = torch.zeros(T, step, dtype=d, device="cuda")
        x, w = far[:, :K], R.randn(2, N, K, dtype=d)
        x.copy_(R.randn(1, T, K, dtype=d))
        y, g = torch.empty(T, N, dtype=d, device="cuda"), R.randn(3, T, N, dtype=d)
        ws = R.workspace(capi.linear_rows_workspace_bytes(CODES[name], K, N, T))
        capi.linear_rows(x, w, y, K, N, T, ws=ws)
        R.check(y, *R.mm(x, w), "y")
        gw = torch.empty(N, K, dtype=torch.float32, device="cuda")
        ws = R.workspace(capi.linear_rows_backward_workspace_bytes(CODES[name], K, N, T))
        capi.linear_rows_backward(g, x, None, None, gw, None, K, N, T, ws=ws)
        R.check(gw, *R.mm(g.t(), x.t()), "grad_w")


@pytest.mark.parametrize("K,N,T", [(4104, 2056, 100), (4096, 2048, 100), (4104, 4104, 60), (1408, 520, 40)])
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("name", ["bf16", "f16"])
def test_weights_gradients_at_any_place(dev, name, wide, K, N, T):
    """Outputs of the large tiles at places of one element after the other, aligned operands: the same bits as aligned, and
    nothing beside them is written."""
    d = R.DTYPES[name]
    gd = torch.float32 if wide else d
    x, g, pre = R.randn(1, T, K, dtype=d), R.randn(2, T, N, dtype=d), R.randn(3, T, N, dtype=d)
    ws = R.workspace(capi.linear_rows_backward_workspace_bytes(CODES[name], K, N, T))
    want = torch.empty(N, K, dtype=gd, device="cuda")
    capi.linear_rows_backward(g, x, None, None, want, None, K, N, T, activation=capi.ACT_RELU, pre=pre, ws=ws)
    for at in (1, 2, 3, 8, 32):
        buf = torch.full((N * K + 64,), 7.0, dtype=gd, device="cuda")
        capi.linear_rows_backward(g, x, None, None, buf[at:at + N * K].view(N, K), None, K, N, T, activation=capi.ACT_RELU, pre=pre,
                                  ws=ws)
        assert torch.equal(buf[at:at + N * K].view(N, K), want)
        assert (buf[:at] == 7.0).all() and (buf[at + N * K:] == 7.0).all()
