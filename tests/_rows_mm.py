"""The products of float matrices in 64 bits, and how far 32-bit sums may be from them.

A sum of n products in fp32: each product (exact for 16-bit operands) and addition is off by at most
2^-23 of its result if the matrix unit chops, so the sum by at most (n + 2) * 2^-23 * S, S the sum
of the products' magnitudes.  A result rounded to its type is off by half its eps (and by half the smallest
subnormal of fp16).  Activations have slopes of at most 1.13 and derivatives that change by at most 1.2 per unit;
they are computed within 2^-19 of max(|z|, 1) (exp2 and the reciprocal 1 ulp each, an argument of up to 64
times log2 e rounded once: 2^-24 * 92 of the exponential, under 2^-17 of a term that is then below e^-64; 8 ulp
where the argument is small).
"""
import math

import torch

ACTS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def act(z, name):
    f = torch.nn.functional
    return {"none": lambda v: v, "relu": f.relu, "gelu": f.gelu, "gelu_tanh": lambda v: f.gelu(v, approximate="tanh"),
            "silu": f.silu}[name](z)


def slope(z, name):
    z = z.detach().clone().requires_grad_(True)
    return torch.autograd.grad(act(z, name).sum(), z)[0]


def mm(a, b):
    """(a . b^T, the bound of its fp32 sum's error) of float matrices [m, k] and [n, k] in 64 bits."""
    a, b = a.double(), b.double()
    return a @ b.t(), (a.shape[1] + 2) * 2.0 ** -23 * (a.abs() @ b.abs().t())


def rounding(ref, dtype):
    tiny = {torch.float16: 2.0 ** -25}.get(dtype, 2.0 ** -134)
    return torch.finfo(dtype).eps / 2 * ref.abs() + tiny


def check(got, ref, bound, what):
    """|got - ref| <= bound + the rounding of got's type (of a value already off by bound)."""
    limit = bound + rounding(ref.abs() + bound, got.dtype)
    off = (got.double() - ref).abs()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    worst = (off / limit).max().item() if off.numel() else 0.0
    assert (off <= limit).all(), f"{what}: {int((off > limit).sum())} of {off.numel()} outside, worst {worst:.2f} of the limit"


def linear(x, w, bias, residual, name):
    z, e = mm(x, w)
    if bias is not None:
        z, e = z + bias.double(), e + 2.0 ** -23 * (z.abs() + bias.double().abs())
    y, ey = z, e
    if name != "none":
        y, ey = act(z, name), 1.13 * e + 2.0 ** -19 * z.abs().clamp(min=1.0)
    if residual is not None:
        y, ey = y + residual.double(), ey + 2.0 ** -23 * (y.abs() + residual.double().abs())
    return y, ey, z, e


def kept(x, dtype, wide):
    """The error of a gradient x that is rounded to dtype; wide: and of what that left, rounded again (bf16: twice)."""
    left = rounding(x, dtype)
    for _ in range(0 if not wide else {torch.float16: 1, torch.bfloat16: 2}.get(dtype, 0)):
        left = rounding(left, dtype)
    return left


def gz_of(g, pre, name, dtype, wide=False):
    """The gradient through an activation, its error in fp32, and that once it is rounded to dtype."""
    g = g.double()
    if name == "none":
        return g, torch.zeros_like(g), torch.zeros_like(g)
    gz = g * slope(pre.double(), name)
    fp32 = g.abs() * 2.0 ** -19 * pre.double().abs().clamp(min=1.0)
    return gz, fp32, fp32 + kept(gz.abs() + fp32, dtype, wide)


def mm_of(a, ea, b):
    """a . b^T where a is off by ea."""
    ref, e = mm(a, b)
    return ref, 1.01 * e + ea @ b.double().abs().t()


def swiglu_back(g, gate, up, dtype, wide=False):
    """Gradients of gate and up, each with its error once rounded."""
    g, gate, up = g.double(), gate.double(), up.double()
    gg, gu = g * up * slope(gate, "silu"), g * act(gate, "silu")
    big = gate.abs().clamp(min=1.0)
    eg, eu = (g * up).abs() * 2.0 ** -19 * big, g.abs() * 2.0 ** -19 * big
    return gg, eg + kept(gg.abs() + eg, dtype, wide), gu, eu + kept(gu.abs() + eu, dtype, wide)


def workspace(n):
    return torch.empty(n, dtype=torch.uint8, device="cuda") if n > 0 else None


def randn(seed, *shape, dtype=torch.float32, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def offsets_of(counts):
    return torch.tensor([0] + list(counts), dtype=torch.int32, device="cuda").cumsum(0).to(torch.int32)
