"""The microscaled 4-bit (MXFP4) operators and the rows sorted by expert, as they are measured.

A case is one pass through an operator, as an inference engine with MXFP4 weights or a
training step of its router makes it: the quantizer and its inverse, a linear layer, the
mixture-of-experts FFN, token rows to their experts and back, and the gradients of the last
two.  Layer sizes are those of perf/cases.py, bench.py and the tests (hidden 2048 and 4096,
intermediate 1408, 11008 and 14336).

Where `own` is false a pass is computed in elementary torch operations in 32 bits; where it
is true, by the framework's entries.  Both read the same state.

MXFP4 matrix [rows][cols], cols % 32 == 0: rows * cols / 2 bytes of e2m1 codes (element 2j of
a row in the low nibble of its byte j), then rows * cols / 32 scale bytes s; a value is
e2m1 * 2^(s - 127).  A block of 32 takes 2^(floor(log2 max|x|) - 2) and rounds to nearest,
ties to even, at most 6.
"""
import math

import torch

own = False

ROTATE_BYTES = 512 << 20  # weights of one state that is bound by reading them, as perf/cases.py
SMALL_TOKENS = 64  # up to this many tokens reading the weights is what a linear layer costs
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _quantize(name, rows, cols, dtype):
    return {"name": name, "kind": "quantize", "rows": rows, "cols": cols, "dtype": dtype}


def _linear(name, tokens, k, n, dtype):
    return {"name": name, "kind": "linear", "tokens": tokens, "k": k, "n": n, "dtype": dtype}


def _ffn(name, tokens, experts, top_k, hidden, inter, dtype):
    return {"name": name, "kind": "ffn", "tokens": tokens, "experts": experts, "top_k": top_k, "hidden": hidden,
            "inter": inter, "dtype": dtype}


def _rows(name, kind, tokens, padded, experts, top_k, hidden, dtype):
    return {"name": name, "kind": kind, "tokens": tokens, "padded": padded, "experts": experts, "top_k": top_k,
            "hidden": hidden, "dtype": dtype}


def listed():
    return [
        # One token's hidden state to MXFP4 and back to values: the smallest call, launch-bound.
        _quantize("token_k4096_f32", 1, 4096, "f32"),
        # Loading a checkpoint: a bf16 projection to MXFP4 (and its values read back).
        _quantize("load_14336x4096_bf16", 14336, 4096, "bf16"),
        # One token through the MLP's up projection, in the engine's fp32.
        _linear("decode_k4096_n11008_f32", 1, 4096, 11008, "f32"),
        # Twenty-four sequences decoded together, long rows.
        _linear("batch24_k11008_n4096_bf16", 24, 11008, 4096, "bf16"),
        # A long prompt of an odd length through an up projection: the largest linear.
        _linear("prompt2047_k4096_n14336_bf16", 2047, 4096, 14336, "bf16"),
        # Four tokens through a mixture-of-experts FFN: decode, most experts' weights read.
        _ffn("moe4_e8_h4096_i14336_bf16", 4, 8, 2, 4096, 14336, "bf16"),
        # A batch of prompt tokens through many small experts, a few routes for each.
        _ffn("moe100_e64_h2048_i1408_bf16", 100, 64, 8, 2048, 1408, "bf16"),
        # A prompt through the mixture-of-experts FFN: the largest FFN.
        _ffn("moe512_e8_h4096_i14336_bf16", 512, 8, 2, 4096, 14336, "bf16"),
        # Four decoded tokens' rows to their experts: launch-bound.
        _rows("sort4_e8_h4096_f32", "sort", 4, 0, 8, 2, 4096, "f32"),
        # A padded training batch, many experts: the gradient of the rows that were sorted.
        _rows("sort_grad2048_e64_h2048_bf16", "sort_grad", 2048, 100, 64, 8, 2048, "bf16"),
        # A prompt of an odd length back to token order.
        _rows("join777_e8_h4096_bf16", "join", 777, 0, 8, 2, 4096, "bf16"),
        # The gradients of the experts' rows and of the router's weights, a long batch.
        _rows("join_grad8192_e8_h4096_bf16", "join_grad", 8192, 0, 8, 2, 4096, "bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("quantize", "linear", "linear", "ffn", "ffn", "sort", "sort_grad", "join", "join_grad"))
    dtype = rng.choice(("f32", "f16", "bf16"))
    if kind == "quantize":
        cols = 32 * _log(rng, 4, 448)
        return {"kind": kind, "rows": _log(rng, 1, 14336 * 4096 // cols // (2 if dtype == "f32" else 1)), "cols": cols,
                "dtype": dtype}
    if kind == "linear":
        k = 32 * _log(rng, 32, 448)
        n = _log(rng, 1024, 14336)
        most = min(2047, 2047 * 4096 * 14336 // (k * n))
        tokens = 1 if rng.random() < 0.25 else _log(rng, 1, most)
        return {"kind": kind, "tokens": tokens, "k": k, "n": n, "dtype": dtype}
    experts, top_k = rng.choice(((8, 2), (16, 2), (16, 4), (64, 8)))
    if kind == "ffn":
        hidden = 32 * _log(rng, 32, 128)
        inter = 32 * _log(rng, 32, min(448, 8 * 128 * 448 // (experts * hidden // 32)))
        most = min(512, 1024 * 4096 * 14336 // (top_k * hidden * inter))
        return {"kind": kind, "tokens": _log(rng, 1, most), "experts": experts, "top_k": top_k, "hidden": hidden,
                "inter": inter, "dtype": rng.choice(("f16", "bf16"))}
    hidden = _log(rng, 256, 7168)
    tokens = _log(rng, 1, min(8192, 8192 * 4096 * 2 // (hidden * top_k * (2 if dtype == "f32" else 1))))
    return {"kind": kind, "tokens": tokens, "padded": rng.choice((0, tokens // 16)), "experts": experts,
            "top_k": top_k, "hidden": hidden, "dtype": dtype}


# ------------------------------------------------------------------------- inputs
def _gen(seed, what):
    return torch.Generator(device="cuda").manual_seed(1000003 * int(seed) + what)


def _weights(rows, cols, seed, what):
    return torch.randn(rows, cols, generator=_gen(seed, what), device="cuda") * 0.02


def _activation(tokens, k, seed, dtype):
    """Hidden states: N(0, 1) with one channel in a thousand twenty times larger."""
    g = _gen(seed, 1)
    x = torch.randn(tokens, k, generator=g, device="cuda")
    x[:, torch.randperm(k, generator=g, device="cuda")[:max(1, k // 1000)]] *= 20.0
    return x.to(DTYPES[dtype])


def _logits(case, seed):
    return torch.randn(case["tokens"], case["experts"], generator=_gen(seed, 2), device="cuda")


def _routing(case, seed):
    """Expert ids [T][top_k] (distinct per token, -1 for a padded token) and weights that sum to 1."""
    top, ids = torch.topk(_logits(case, seed), case["top_k"], dim=1)
    ids = ids.to(torch.int32)
    ids[case["tokens"] - case["padded"]:] = -1
    return ids.contiguous(), torch.softmax(top, dim=1)


def _gradient(rows, hidden, seed, what, dtype):
    return (torch.randn(rows, hidden, generator=_gen(seed, what), device="cuda") * 0.05).to(DTYPES[dtype])


def prepare(case, seed):
    kind, dtype = case["kind"], DTYPES[case["dtype"]]
    if kind == "quantize":
        rows, cols = case["rows"], case["cols"]
        return {"case": case, "x": _weights(rows, cols, seed, 3).to(dtype),
                "q": torch.empty(rows * cols // 32 * 17, dtype=torch.uint8, device="cuda"),
                "y": torch.empty(rows, cols, dtype=dtype, device="cuda")}
    if kind == "linear":
        t, k, n = case["tokens"], case["k"], case["n"]
        w = _pack(_weights(n, k, seed, 3))
        copies = max(1, math.ceil(ROTATE_BYTES / w.numel())) if t <= SMALL_TOKENS else 1
        return {"case": case, "w": [w] + [w.clone() for _ in range(copies - 1)], "at": 0,
                "x": _activation(t, k, seed, case["dtype"]),
                "ws": torch.empty(t * k + 32 * t * n + (1 << 20), dtype=torch.uint8, device="cuda"),
                "y": torch.empty(t, n, dtype=dtype, device="cuda")}
    if kind == "ffn":
        t, e, top_k, h, i = (case[v] for v in ("tokens", "experts", "top_k", "hidden", "inter"))
        mats = [_pack(_weights(e * rows, cols, seed, what)) for rows, cols, what in ((i, h, 100), (i, h, 300), (h, i, 500))]
        copies = max(1, math.ceil(ROTATE_BYTES / sum(m.numel() for m in mats)))
        room = 16 * t * top_k * (h + 2 * i + 8) + (1 << 20)  # more than every intermediate in 32 bits
        return {"case": case, "w": [mats] + [[m.clone() for m in mats] for _ in range(copies - 1)], "at": 0,
                "x": _activation(t, h, seed, case["dtype"]), "logits": _logits(case, seed),
                "ws": torch.empty(room, dtype=torch.uint8, device="cuda"),
                "y": torch.empty(t, h, dtype=dtype, device="cuda")}
    t, e, top_k, h = (case[v] for v in ("tokens", "experts", "top_k", "hidden"))
    r = t * top_k
    ids, share = _routing(case, seed)
    state = {"case": case, "ids": ids, "share": share}
    if kind == "sort":  # rows behind the last sorted one stay as they are: zeros
        state |= {"x": _activation(t, h, seed, case["dtype"]), "rows": torch.zeros(r, h, dtype=dtype, device="cuda"),
                  "offsets": torch.zeros(e + 1, dtype=torch.int32, device="cuda"),
                  "src": torch.zeros(r, dtype=torch.int32, device="cuda"),
                  "dst": torch.zeros(t, top_k, dtype=torch.int32, device="cuda")}
        return state
    state["dst"] = _sorted(ids, e)[2]
    if kind == "sort_grad":
        return state | {"g": _gradient(r, h, seed, 5, case["dtype"]), "gx": torch.empty(t, h, dtype=dtype, device="cuda")}
    state["e"] = _gradient(r, h, seed, 6, case["dtype"])
    if kind == "join":
        return state | {"y": torch.empty(t, h, dtype=dtype, device="cuda")}
    return state | {"g": _gradient(t, h, seed, 7, case["dtype"]), "ge": torch.zeros(r, h, dtype=dtype, device="cuda"),
                    "gw": torch.empty(t, top_k, dtype=torch.float32, device="cuda")}


# --------------------------------------------------------------------- plain forms
def _codes(x):
    """e2m1 codes [rows, cols] (uint8, sign in bit 3) and scale bytes [rows, cols/32] of fp32 x."""
    g = x.reshape(x.shape[0], -1, 32)
    amax = g.abs().amax(dim=2)
    shared = ((amax.view(torch.int32) >> 23) - 127 - 2).clamp(min=-127)  # exponent bits of a float >= 0
    v = g.abs() * ((127 - shared) << 23).view(torch.float32)[..., None]
    code = (v > 0.25).to(torch.uint8)
    code += v >= 0.75
    code += v > 1.25
    code += v >= 1.75
    code += v > 2.5
    code += v >= 3.5
    code += v > 5.0
    code += 8 * torch.signbit(g)
    return code.reshape(x.shape), (shared + 127).to(torch.uint8)


def _pack(x):
    code, scale = _codes(x)
    return torch.cat([(code[:, 0::2] | (code[:, 1::2] << 4)).reshape(-1), scale.reshape(-1)])


def _decode(code, scale):
    """The values in fp32: a code's magnitude is half of 0, 1, 2, 3, 4, 6, 8, 12."""
    m = code & 7
    twice = torch.where(m < 4, m, torch.where(m < 6, 2 * m - 4, 4 * m - 16)).to(torch.float32)
    twice = torch.where(code >= 8, -twice, twice)
    return (twice.reshape(*scale.shape, 32) * torch.exp2(scale.double() - 128.0).float()[..., None]).reshape(code.shape)


def _unpack(q, rows, cols):
    b = q[:rows * cols // 2].reshape(rows, cols // 2)
    code = torch.stack([b & 15, b >> 4], dim=2).reshape(rows, cols)
    return _decode(code, q[rows * cols // 2:].reshape(rows, cols // 32))


def _rounded(x):
    """What MXFP4 holds of x, in fp32."""
    return _decode(*_codes(x))


def _sorted(ids, experts):
    """Offsets of the experts, the route at each sorted row (0 behind the last) and each route's row (-1: none)."""
    flat = ids.reshape(-1)
    live = (flat >= 0) & (flat < experts)
    key = torch.where(live, flat, experts)
    order = torch.argsort(key, stable=True)
    at = torch.arange(flat.numel(), device=flat.device)
    offsets = (key[None, :] < torch.arange(experts + 1, device=flat.device)[:, None]).sum(1)
    dst = torch.empty_like(order)
    dst[order] = at
    return (offsets.to(torch.int32), torch.where(at < offsets[-1], order, 0).to(torch.int32),
            torch.where(live, dst, -1).to(torch.int32).reshape(ids.shape))


def _plain_ffn(state, w):
    case, x = state["case"], _rounded(state["x"].float())
    e, top_k, h, i = (case[v] for v in ("experts", "top_k", "hidden", "inter"))
    top, ids = torch.sort(state["logits"], dim=1, descending=True, stable=True)
    top, ids = top[:, :top_k], ids[:, :top_k]
    share = torch.exp(top - top[:, :1])
    share = share / share.sum(1, keepdim=True)
    offsets, src, dst = _sorted(ids, e)
    src, dst = src.long(), dst.reshape(-1).long()
    expert = ids.reshape(-1)[src]
    at = torch.arange(src.numel(), device=src.device) - offsets[expert]
    # The experts' rows side by side, each padded to the longest.
    longest = int((offsets[1:] - offsets[:-1]).max())
    xs = torch.zeros(e, h, longest, device=x.device)
    xs[expert, :, at] = x[src // top_k]
    gate = torch.bmm(_unpack(w[0], e * i, h).reshape(e, i, h), xs)
    up = torch.bmm(_unpack(w[1], e * i, h).reshape(e, i, h), xs)
    mid = _rounded((gate / (1.0 + torch.exp(-gate)) * up)[expert, :, at])
    ms = torch.zeros(e, i, longest, device=x.device)
    ms[expert, :, at] = mid
    down = torch.bmm(_unpack(w[2], e * h, i).reshape(e, h, i), ms)[expert, :, at]
    return (share[..., None] * down[dst].reshape(-1, top_k, h)).sum(1).to(state["x"].dtype)


def _plain(state):
    case, kind = state["case"], state["case"]["kind"]
    if kind == "quantize":
        return _rounded(state["x"].float()).to(state["x"].dtype)
    if kind == "linear":
        w = state["w"][state["at"]]
        state["at"] = (state["at"] + 1) % len(state["w"])
        return (_rounded(state["x"].float()) @ _unpack(w, case["n"], case["k"]).t()).to(state["x"].dtype)
    if kind == "ffn":
        w = state["w"][state["at"]]
        state["at"] = (state["at"] + 1) % len(state["w"])
        return _plain_ffn(state, w)
    if kind == "sort":
        offsets, src, dst = _sorted(state["ids"], case["experts"])
        live = torch.arange(src.numel(), device=src.device) < offsets[-1]
        rows = state["x"][src.long() // case["top_k"]]
        return [torch.where(live[:, None], rows, 0), offsets, src, dst]
    dst = state["dst"].long()
    live = (dst >= 0)[..., None]
    if kind == "sort_grad":
        return torch.where(live, state["g"][dst.clamp(min=0)].float(), 0.0).sum(1).to(state["g"].dtype)
    rows = torch.where(live, state["e"][dst.clamp(min=0)].float(), 0.0)
    if kind == "join":
        return (state["share"][..., None] * rows).sum(1).to(state["e"].dtype)
    g = state["g"].float()[:, None, :]
    ge = torch.zeros(dst.numel() + 1, case["hidden"], dtype=state["e"].dtype, device=g.device)  # the last: dropped routes
    ge[torch.where(dst < 0, dst.numel(), dst)] = (state["share"][..., None] * g).to(ge.dtype)
    return [ge[:-1], (g * rows).sum(2)]


# --------------------------------------------------------------------------- pass
def _call(state):
    from jjjetson_ops_amd import capi
    case, kind = state["case"], state["case"]["kind"]
    if kind == "quantize":
        capi.quantize_mxfp4(state["x"], state["q"], case["rows"], case["cols"])
        capi.dequantize_mxfp4(state["q"], state["y"], case["rows"], case["cols"])
        return state["y"]
    if kind == "linear":
        w = state["w"][state["at"]]
        state["at"] = (state["at"] + 1) % len(state["w"])
        capi.linear_mxfp4(state["x"], w, state["y"], case["k"], case["n"], case["tokens"], ws=state["ws"])
        return state["y"]
    if kind == "ffn":
        w = state["w"][state["at"]]
        state["at"] = (state["at"] + 1) % len(state["w"])
        capi.moe_ffn_mxfp4(state["x"], state["logits"], w[0], w[1], w[2], state["y"], case["tokens"], case["hidden"],
                           case["inter"], case["experts"], case["top_k"], state["ws"])
        return state["y"]
    t, top_k, h = case["tokens"], case["top_k"], case["hidden"]
    if kind == "sort":
        capi.moe_dispatch_rows(state["ids"], state["x"], state["rows"], state["offsets"], state["src"], state["dst"],
                               t, top_k, h, case["experts"])
        return [state["rows"], state["offsets"], state["src"], state["dst"]]
    if kind == "sort_grad":
        capi.moe_dispatch_rows_backward(state["g"], state["dst"], state["gx"], t, h, top_k)
        return state["gx"]
    if kind == "join":
        capi.moe_combine_rows(state["e"], state["dst"], state["share"], state["y"], t, h, top_k)
        return state["y"]
    capi.moe_combine_rows_backward(state["g"], state["e"], state["dst"], state["share"], state["ge"], state["gw"],
                                   t, h, top_k)
    return [state["ge"], state["gw"]]


def run(state):
    return _call(state) if own else _plain(state)


# --------------------------------------------------------------------- what it needs
def work(case):
    kind, size = case["kind"], 4 if case["dtype"] == "f32" else 2
    if kind == "quantize":
        values = case["rows"] * case["cols"]
        return {"bytes": values * (2 * size) + values // 32 * 17, "flops": 0}
    if kind == "linear":
        t, k, n = case["tokens"], case["k"], case["n"]
        return {"bytes": n * k // 32 * 17 + size * t * (k + n), "flops": 2 * t * k * n}
    t, e, top_k, h = (case[v] for v in ("tokens", "experts", "top_k", "hidden"))
    if kind == "ffn":
        i = case["inter"]
        active = e * (1.0 - (1.0 - top_k / e) ** t)  # experts with a route, for a balanced router
        return {"bytes": int(active * 3 * h * i // 32 * 17) + t * (2 * size * h + 4 * e), "flops": 6 * t * top_k * h * i}
    live, r = t - case["padded"], t * top_k
    if kind == "sort":
        return {"bytes": size * h * live * (1 + top_k) + 4 * (3 * r + e + 1), "flops": 0}
    if kind == "join_grad":
        return {"bytes": size * h * live * (1 + 2 * top_k) + 12 * r, "flops": 3 * live * top_k * h}
    return {"bytes": size * h * (live * top_k + t) + 8 * r, "flops": 2 * live * top_k * h}


# -------------------------------------------------------------------------- in 64 bits
def _exact_mx(x):
    """The nearest multiples of e2m1's steps in fp64, from the logarithms of the values."""
    g = x.double().reshape(*x.shape[:-1], -1, 32)
    unit = torch.exp2(torch.floor(torch.log2(g.abs().amax(-1, keepdim=True))).clamp(min=-125.0) - 2.0)
    v = g / unit
    step = torch.exp2(torch.floor(torch.log2(v.abs())).clamp(0.0, 2.0) - 1.0)
    return ((torch.round(v / step) * step).clamp(-6.0, 6.0) * unit).reshape(x.shape)


def _exact_ffn(case, seed):
    e, top_k, h, i = (case[v] for v in ("experts", "top_k", "hidden", "inter"))
    x = _exact_mx(_activation(case["tokens"], h, seed, case["dtype"]))
    top, ids = torch.topk(_logits(case, seed).double(), top_k, dim=1)
    share = torch.softmax(top, dim=1)
    gates, ups, downs = (_weights(e * rows, cols, seed, what).reshape(e, rows, cols)
                         for rows, cols, what in ((i, h, 100), (i, h, 300), (h, i, 500)))
    y = torch.zeros(case["tokens"], h, dtype=torch.float64, device="cuda")
    for expert in range(e):
        tok, slot = torch.nonzero(ids == expert, as_tuple=True)
        if tok.numel():
            gate, up = x[tok] @ _exact_mx(gates[expert]).t(), x[tok] @ _exact_mx(ups[expert]).t()
            mid = _exact_mx(gate * torch.sigmoid(gate) * up)
            y.index_add_(0, tok, share[tok, slot][:, None] * (mid @ _exact_mx(downs[expert]).t()))
    return y


def exact(case, seed):
    kind = case["kind"]
    if kind == "quantize":
        return _exact_mx(_weights(case["rows"], case["cols"], seed, 3).to(DTYPES[case["dtype"]]))
    if kind == "linear":
        return (_exact_mx(_activation(case["tokens"], case["k"], seed, case["dtype"]))
                @ _exact_mx(_weights(case["n"], case["k"], seed, 3)).t())
    if kind == "ffn":
        return _exact_ffn(case, seed)
    t, e, top_k, h = (case[v] for v in ("tokens", "experts", "top_k", "hidden"))
    r = t * top_k
    ids, share = _routing(case, seed)
    ids, share = ids.reshape(-1).cpu().tolist(), share.double().reshape(-1, 1)
    order = sorted((expert, route) for route, expert in enumerate(ids) if 0 <= expert < e)
    route = torch.tensor([v for _, v in order], device="cuda")
    n = route.numel()
    if kind == "sort":
        rows = torch.zeros(r, h, dtype=torch.float64, device="cuda")
        rows[:n] = _activation(t, h, seed, case["dtype"]).double()[route // top_k]
        return [rows, None, None, None]
    if kind == "sort_grad":
        g = _gradient(r, h, seed, 5, case["dtype"]).double()
        return torch.zeros(t, h, dtype=torch.float64, device="cuda").index_add_(0, route // top_k, g[:n])
    rows = _gradient(r, h, seed, 6, case["dtype"]).double()[:n]
    if kind == "join":
        y = torch.zeros(t, h, dtype=torch.float64, device="cuda")
        return y.index_add_(0, route // top_k, share[route] * rows)
    g = _gradient(t, h, seed, 7, case["dtype"]).double()[route // top_k]
    ge, gw = torch.zeros(r, h, dtype=torch.float64, device="cuda"), torch.zeros(r, dtype=torch.float64, device="cuda")
    ge[:n] = share[route] * g
    gw[route] = (g * rows).sum(1)
    return [ge, gw.reshape(t, top_k)]
