"""Float products through the public entries where precision or a kernel's way differs: the terms of a gradient that
is split for fp32 weights' gradients."""
if __name__ == "__main__":  # `python tests/<file>.py`, as the reference runs its tests
    import sys as _sys

    import pytest as _pytest
    _sys.exit(_pytest.main([__file__, "-q"]))
import pytest
import torch

import _rows_mm as R
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
