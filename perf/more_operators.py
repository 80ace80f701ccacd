"""Products with float weights, as they are measured: a linear layer with bias, activation and residual,
the experts' products of rows sorted by expert, and their gate|up projection with SwiGLU, each with its
gradients.

A case is one pass through one of them, as an inference engine or a training step with fp32, fp16 or bf16
weights makes it.  Layer sizes are those of perf/cases.py, perf/operators.py and the tests (hidden 2048
and 4096, intermediate 1408, 11008 and 14336).

Where `own` is false a pass is computed in elementary torch operations in 32 bits; where it is true, by
the framework's entries.  Both read the same state.

    linear       y = act(x W^T + b) + r                    x [T][K], W [N][K], b [N], r and y [T][N]
    linear_grad  gz = gy act'(x W^T + b), gx = gz W, gW = gz^T x, gb = the columns' sums of gz
    grouped      y[p] = x[p] W[e]^T for the rows p of expert e, rows sorted by expert
    grouped_grad gx[p] = gy[p] W[e], gW[e] = the sum over e's rows of gy[p]^T x[p]
    swiglu       mid[p] = silu(x[p] Wg[e]^T) * (x[p] Wu[e]^T)
    swiglu_grad  from the gradient of mid and the saved gate|up: gx, gWg, gWu
"""
import math

import torch

own = False

ROTATE_BYTES = 512 << 20  # weights of one state that is bound by reading them, as perf/cases.py
SMALL_ROWS = 64  # up to this many rows for a matrix reading it is what a product costs
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ACTIVATIONS = ("none", "relu", "gelu", "gelu_tanh", "silu")


def _linear(name, kind, tokens, k, n, dtype, act, bias, residual=False, wide=False):
    return {"name": name, "kind": kind, "tokens": tokens, "k": k, "n": n, "dtype": dtype, "act": act, "bias": bias,
            "residual": residual, "wide": wide}


def _experts(name, kind, tokens, padded, experts, top_k, k, n, dtype, wide=False):
    return {"name": name, "kind": kind, "tokens": tokens, "padded": padded, "experts": experts, "top_k": top_k,
            "k": k, "n": n, "dtype": dtype, "wide": wide}


def listed():
    return [
        # One token through the MLP's gate projection: decode, the weights are read once.
        _linear("linear1_k4096_n11008_bf16", "linear", 1, 4096, 11008, "bf16", "silu", False),
        # Twenty-four sequences decoded together through a down projection onto the residual stream.
        _linear("linear24_k11008_n4096_f16", "linear", 24, 11008, 4096, "f16", "none", True, True),
        # An engine that keeps fp32 weights, a prompt of an odd length.
        _linear("linear333_k2048_n1408_f32", "linear", 333, 2048, 1408, "f32", "gelu", True, True),
        # A long prompt of an odd length through an up projection: the largest forward linear.
        _linear("linear2047_k4096_n14336_bf16", "linear", 2047, 4096, 14336, "bf16", "gelu_tanh", True),
        # The gradients of a small layer, an odd number of tokens.
        _linear("linear_grad777_k1408_n2048_f16", "linear_grad", 777, 1408, 2048, "f16", "gelu", True),
        # The gradients of a projection, a training batch; the weights' gradients in fp32.
        _linear("linear_grad2048_k4096_n4096_bf16", "linear_grad", 2048, 4096, 4096, "bf16", "silu", True, wide=True),
        # Four decoded tokens through the experts' down projection.
        _experts("grouped4_e8_k14336_n4096_bf16", "grouped", 4, 0, 8, 2, 14336, 4096, "bf16"),
        # A batch of prompt tokens through many small experts.
        _experts("grouped200_e64_k2048_n1408_f16", "grouped", 200, 0, 64, 8, 2048, 1408, "f16"),
        # A padded training batch, many small experts, the gradients of rows and weights.
        _experts("grouped_grad2048_e64_k1408_n2048_bf16", "grouped_grad", 2048, 100, 64, 8, 1408, 2048, "bf16"),
        # One token through its eight small experts of 64: the smallest call.
        _experts("swiglu1_e64_k2048_n1408_bf16", "swiglu", 1, 0, 64, 8, 2048, 1408, "bf16"),
        # A prompt through the experts' gate|up projection.
        _experts("swiglu1023_e8_k4096_n14336_bf16", "swiglu", 1023, 0, 8, 2, 4096, 14336, "bf16"),
        # A training step's gradients of the gate|up projection: the largest.
        _experts("swiglu_grad1024_e8_k4096_n14336_bf16", "swiglu_grad", 1024, 0, 8, 2, 4096, 14336, "bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def _size(rng, lo, hi):
    """A layer size: mostly a multiple of 64, sometimes of 8, now and then any number."""
    v, step = _log(rng, lo, hi), rng.choice((64, 64, 64, 8, 1))
    return max(lo, v // step * step)


def draw(rng):
    kind = rng.choice(("linear", "linear", "linear_grad", "grouped", "grouped_grad", "swiglu", "swiglu_grad"))
    dtype, wide = rng.choice(("f32", "f16", "bf16", "bf16")), rng.random() < 0.5
    # Multiply-adds of one product: the largest listed cases', fewer in fp32.
    most = (8 if dtype == "f32" else 64) << 30
    k, n = _size(rng, 256, 11008), _size(rng, 256, 14336)
    if kind in ("linear", "linear_grad"):
        tokens = _log(rng, 1, min(4096, most // (k * n)))
        if kind == "linear" and rng.random() < 0.2:
            tokens = 1
        return {"kind": kind, "tokens": tokens, "k": k, "n": n, "dtype": dtype, "act": rng.choice(ACTIVATIONS),
                "bias": rng.random() < 0.5, "residual": kind == "linear" and rng.random() < 0.5,
                "wide": kind == "linear_grad" and wide}
    experts, top_k = rng.choice(((8, 2), (16, 2), (16, 4), (64, 8)))
    n = max(256, min(n, 8 * 4096 * 14336 // (experts * k) // 8 * 8))
    tokens = _log(rng, 1, min(4096, most // (k * n * top_k)))
    return {"kind": kind, "tokens": tokens, "padded": rng.choice((0, tokens // 16)), "experts": experts,
            "top_k": top_k, "k": k, "n": n, "dtype": dtype, "wide": kind.endswith("grad") and wide}


# ------------------------------------------------------------------------- inputs
def _gen(seed, what):
    return torch.Generator(device="cuda").manual_seed(1000003 * int(seed) + what)


def _randn(seed, what, dtype, scale, *shape):
    return (torch.randn(*shape, generator=_gen(seed, what), device="cuda") * scale).to(DTYPES[dtype])


def _weights(seed, what, dtype, *shape):
    return _randn(seed, what, dtype, 0.02, *shape)


def _activation(rows, k, seed, dtype):
    """Hidden states: N(0, 1) with one channel in a thousand twenty times larger."""
    g = _gen(seed, 1)
    x = torch.randn(rows, k, generator=g, device="cuda")
    x[:, torch.randperm(k, generator=g, device="cuda")[:max(1, k // 1000)]] *= 20.0
    return x.to(DTYPES[dtype])


def _ends(case, seed):
    """Rows of each expert from the router of the unpadded tokens, some experts liked better than others."""
    g = _gen(seed, 2)
    logits = torch.randn(case["tokens"] - case["padded"], case["experts"], generator=g, device="cuda")
    logits += 0.5 * torch.randn(case["experts"], generator=g, device="cuda")
    ids = torch.topk(logits, case["top_k"], dim=1).indices
    return torch.bincount(ids.reshape(-1), minlength=case["experts"]).cumsum(0).tolist()


def _extra(case, seed):
    """Bias and residual, where the layer has them."""
    t, n, dtype = case["tokens"], case["n"], case["dtype"]
    return (_randn(seed, 4, dtype, 0.5, n) if case["bias"] else None,
            _randn(seed, 5, dtype, 1.0, t, n) if case["residual"] else None)


def _rotated(mats, rows, state):
    size = sum(m.numel() * m.element_size() for m in mats)
    copies = max(1, math.ceil(ROTATE_BYTES / size)) if rows <= SMALL_ROWS else 1
    return state | {"w": [mats] + [[m.clone() for m in mats] for _ in range(copies - 1)], "at": 0}


def _inputs(case, seed):
    """The tensors of a pass without the weights: x and, for gradients, that of the output and what was saved."""
    t, k, n, dtype = case["tokens"], case["k"], case["n"], case["dtype"]
    if case["kind"] in ("linear", "linear_grad"):
        out = {"x": _activation(t, k, seed, dtype)}
        if case["kind"] == "linear_grad":
            out["g"] = _randn(seed, 6, dtype, 0.05, t, n)
            out["pre"] = None if case["act"] == "none" else _randn(seed, 7, dtype, 1.5, t, n)
        return out
    r = t * case["top_k"]
    out = {"x": _activation(r, k, seed, dtype)}
    if case["kind"].endswith("grad"):
        out["g"] = _randn(seed, 6, dtype, 0.05, r, n)
    if case["kind"] == "swiglu_grad":
        out["gate_up"] = _randn(seed, 7, dtype, 1.5, r, 2 * n)
    return out


def _mats(case, seed):
    k, n, dtype = case["k"], case["n"], case["dtype"]
    if case["kind"] in ("linear", "linear_grad"):
        return [_weights(seed, 3, dtype, n, k)]
    return [_weights(seed, what, dtype, case["experts"], n, k)
            for what in ((3, 8) if case["kind"].startswith("swiglu") else (3,))]


def prepare(case, seed):
    t, k, n, kind = case["tokens"], case["k"], case["n"], case["kind"]
    dtype, grad = DTYPES[case["dtype"]], torch.float32 if case["wide"] else DTYPES[case["dtype"]]
    state = {"case": case} | _inputs(case, seed)
    if kind in ("linear", "linear_grad"):
        rows = t
        state["bias"], state["residual"] = _extra(case, seed)
        if kind == "linear":
            state["y"] = torch.empty(t, n, dtype=dtype, device="cuda")
        else:
            state |= {"gx": torch.empty(t, k, dtype=dtype, device="cuda"),
                      "gw": [torch.empty(n, k, dtype=grad, device="cuda")],
                      "gb": torch.empty(n, dtype=grad, device="cuda") if case["bias"] else None}
    else:
        r, e = t * case["top_k"], case["experts"]
        rows = r // e
        ends = _ends(case, seed)
        state |= {"ends": ends, "offsets": torch.tensor([0] + ends, dtype=torch.int32, device="cuda")}
        if kind.endswith("grad"):  # rows behind the last expert's stay as they are: zeros
            state |= {"gx": torch.zeros(r, k, dtype=dtype, device="cuda"),
                      "gw": [torch.empty(e, n, k, dtype=grad, device="cuda") for _ in range(2 if kind[0] == "s" else 1)]}
        else:
            state["y"] = torch.zeros(r, n, dtype=dtype, device="cuda")
    if own:
        state["ws"] = torch.empty(max(256, _workspace(case)), dtype=torch.uint8, device="cuda")
    return _rotated(_mats(case, seed), rows, state)


# --------------------------------------------------------------------- plain forms
def _erf(z):
    return torch.erf(z * math.sqrt(0.5))


def _tanh(z):
    return torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z))


def _act(z, act):
    if act == "relu":
        return torch.clamp(z, min=0.0)
    if act == "gelu":
        return 0.5 * z * (1.0 + _erf(z))
    if act == "gelu_tanh":
        return 0.5 * z * (1.0 + _tanh(z))
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    return z


def _slope(z, act):
    if act == "relu":
        return (z > 0.0).float()
    if act == "gelu":
        return 0.5 * (1.0 + _erf(z)) + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    if act == "gelu_tanh":
        th = _tanh(z)
        return 0.5 * (1.0 + th) + 0.5 * z * (1.0 - th * th) * math.sqrt(2.0 / math.pi) * (1.0 + 0.134145 * z * z)
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return s * (1.0 + z * (1.0 - s))
    return torch.ones_like(z)


def _plain(state, w):
    case, kind, x = state["case"], state["case"]["kind"], state["x"].float()
    if kind == "linear":
        z = x @ w[0].float().t()
        if state["bias"] is not None:
            z = z + state["bias"].float()
        y = _act(z, case["act"])
        if state["residual"] is not None:
            y = y + state["residual"].float()
        return y.to(state["x"].dtype)
    if kind == "linear_grad":
        gz = state["g"].float()
        if state["pre"] is not None:
            gz = gz * _slope(state["pre"].float(), case["act"])
        out = [(gz @ w[0].float()).to(state["x"].dtype), (gz.t() @ x).to(state["gw"][0].dtype)]
        return out + ([gz.sum(0).to(state["gb"].dtype)] if case["bias"] else [])
    n = case["n"]
    if kind == "swiglu_grad":
        gate, up, gm = state["gate_up"][:, :n].float(), state["gate_up"][:, n:].float(), state["g"].float()
        grads = [gm * up * _slope(gate, "silu"), gm * _act(gate, "silu")]
    elif kind == "grouped_grad":
        grads = [state["g"].float()]
    rows = torch.zeros_like(state["gx"] if kind.endswith("grad") else state["y"])
    gws = [torch.zeros_like(m) for m in state["gw"]] if kind.endswith("grad") else []
    first = 0
    for e, end in enumerate(state["ends"]):
        mine, first = slice(first, end), end
        if mine.start == end:
            continue
        if kind == "grouped":
            rows[mine] = (x[mine] @ w[0][e].float().t()).to(rows.dtype)
        elif kind == "swiglu":
            rows[mine] = (_act(x[mine] @ w[0][e].float().t(), "silu") * (x[mine] @ w[1][e].float().t())).to(rows.dtype)
        else:
            rows[mine] = sum(g[mine] @ m[e].float() for g, m in zip(grads, w)).to(rows.dtype)
            for g, gw in zip(grads, gws):
                gw[e] = (g[mine].t() @ x[mine]).to(gw.dtype)
    return [rows] + gws


# --------------------------------------------------------------------------- pass
def _workspace(case):
    from jjjetson_ops_amd import capi
    d = {"f32": capi.DTYPE_F32, "f16": capi.DTYPE_F16, "bf16": capi.DTYPE_BF16}[case["dtype"]]
    t, k, n, kind = case["tokens"], case["k"], case["n"], case["kind"]
    if kind == "linear":
        return capi.linear_rows_workspace_bytes(d, k, n, t)
    if kind == "linear_grad":
        return capi.linear_rows_backward_workspace_bytes(d, k, n, t)
    size = {"grouped": capi.grouped_mat_mul_rows_workspace_bytes,
            "grouped_grad": capi.grouped_mat_mul_rows_backward_workspace_bytes,
            "swiglu": capi.moe_gate_up_swiglu_rows_workspace_bytes,
            "swiglu_grad": capi.moe_gate_up_swiglu_rows_backward_workspace_bytes}[kind]
    return size(d, k, n, t * case["top_k"], case["experts"])


def _call(state, w):
    from jjjetson_ops_amd import capi
    case, kind, x, ws = state["case"], state["case"]["kind"], state["x"], state["ws"]
    t, k, n = case["tokens"], case["k"], case["n"]
    if kind in ("linear", "linear_grad"):
        act = {"none": capi.ACT_NONE, "relu": capi.ACT_RELU, "gelu": capi.ACT_GELU, "gelu_tanh": capi.ACT_GELU_TANH,
               "silu": capi.ACT_SILU}[case["act"]]
        if kind == "linear":
            capi.linear_rows(x, w[0], state["y"], k, n, t, bias=state["bias"], residual=state["residual"],
                             activation=act, ws=ws)
            return state["y"]
        capi.linear_rows_backward(state["g"], x, w[0], state["gx"], state["gw"][0], state["gb"], k, n, t,
                                  activation=act, pre=state["pre"], ws=ws)
        return [state["gx"], state["gw"][0]] + ([state["gb"]] if case["bias"] else [])
    r, e, offsets = t * case["top_k"], case["experts"], state["offsets"]
    if kind == "grouped":
        capi.grouped_mat_mul_rows(x, w[0], offsets, state["y"], k, n, r, ws=ws)
        return [state["y"]]
    if kind == "swiglu":
        capi.moe_gate_up_swiglu_rows(x, w[0], w[1], offsets, e, state["y"], k, n, r, ws=ws)
        return [state["y"]]
    if kind == "grouped_grad":
        capi.grouped_mat_mul_rows_backward(state["g"], x, w[0], offsets, state["gx"], state["gw"][0], k, n, r, ws=ws)
    else:
        capi.moe_gate_up_swiglu_rows_backward(state["g"], state["gate_up"], x, w[0], w[1], offsets, e, state["gx"],
                                              state["gw"][0], state["gw"][1], k, n, r, ws=ws)
    return [state["gx"]] + state["gw"]


def run(state):
    w = state["w"][state["at"]]
    state["at"] = (state["at"] + 1) % len(state["w"])
    return _call(state, w) if own else _plain(state, w)


# --------------------------------------------------------------------- what it needs
def work(case):
    t, k, n, kind, size = case["tokens"], case["k"], case["n"], case["kind"], 4 if case["dtype"] == "f32" else 2
    wide = 4 if case["wide"] else size
    if kind == "linear":
        return {"bytes": size * (t * k + n * k + t * n * (1 + case["residual"]) + n * case["bias"]),
                "flops": 2 * t * k * n}
    if kind == "linear_grad":
        return {"bytes": size * (2 * t * k + n * k + t * n * (1 + (case["act"] != "none"))) + wide * n * (k + case["bias"]),
                "flops": 4 * t * k * n}
    e, top_k, live = case["experts"], case["top_k"], case["tokens"] - case["padded"]
    r, mats = live * top_k, 2 if kind.startswith("swiglu") else 1
    active = e * (1.0 - (1.0 - top_k / e) ** live)  # experts with a row, for a balanced router
    if not kind.endswith("grad"):
        return {"bytes": int(size * (active * mats * n * k + r * (k + n))), "flops": 2 * mats * r * k * n}
    saved = 2 if mats == 2 else 0  # gate|up
    return {"bytes": int(size * (active * mats * n * k + r * (2 * k + (1 + saved) * n)) + wide * e * mats * n * k),
            "flops": 4 * mats * r * k * n}


# -------------------------------------------------------------------------- in 64 bits
def _exact_act(z, act):
    f = torch.nn.functional
    return {"none": lambda v: v, "relu": f.relu, "gelu": f.gelu, "gelu_tanh": lambda v: f.gelu(v, approximate="tanh"),
            "silu": f.silu}[act](z)


def exact(case, seed):
    kind, act = case["kind"], case.get("act")
    v = {name: None if m is None else m.double() for name, m in _inputs(case, seed).items()}
    mats = _mats(case, seed)
    if kind == "linear":
        bias, residual = _extra(case, seed)
        z = torch.matmul(mats[0].double(), v["x"].t()).t()
        z = _exact_act(z if bias is None else z + bias.double(), act)
        return z if residual is None else z + residual.double()
    if kind == "linear_grad":
        if v["pre"] is not None:  # the activation's gradient by differentiation
            pre = v["pre"].requires_grad_(True)
            v["g"], = torch.autograd.grad(_exact_act(pre, act), pre, v["g"])
        gb = [torch.matmul(torch.ones(1, case["tokens"], dtype=torch.float64, device="cuda"), v["g"])[0]]
        return [torch.matmul(v["g"], mats[0].double()), torch.matmul(v["x"].t(), v["g"]).t()] + (gb if case["bias"] else [])
    n, r = case["n"], case["tokens"] * case["top_k"]
    starts = [0] + _ends(case, seed)
    if kind == "swiglu_grad":
        both = v["gate_up"].requires_grad_(True)
        gate, up = both.split(n, dim=1)
        grads = torch.autograd.grad(torch.nn.functional.silu(gate) * up, both, v["g"])[0].split(n, dim=1)
    else:
        grads = [v["g"]] if kind == "grouped_grad" else []
    rows = torch.zeros(r, case["k"] if grads else n, dtype=torch.float64, device="cuda")
    gws = [torch.zeros(case["experts"], n, case["k"], dtype=torch.float64, device="cuda") for _ in grads]
    for e in range(case["experts"]):
        a, b = starts[e], starts[e + 1]
        if a == b:
            continue
        outs = [torch.matmul(m[e].double(), v["x"][a:b].t()).t() for m in mats] if not grads else []
        if kind == "grouped":
            rows[a:b] = outs[0]
        elif kind == "swiglu":
            rows[a:b] = torch.nn.functional.silu(outs[0]) * outs[1]
        for g, m, gw in zip(grads, mats, gws):
            rows[a:b] += torch.matmul(g[a:b], m[e].double())
            gw[e] = torch.matmul(v["x"][a:b].t(), g[a:b]).t()
    return [rows] + gws
