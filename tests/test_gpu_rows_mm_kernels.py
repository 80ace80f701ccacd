"""Every kernel of the float products by name, the limits of their addressing, and a MoE layer of them: captured, on
other streams, with its gradients."""
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
TILES = [capi.ROWS_TILE_64, capi.ROWS_TILE_128, capi.ROWS_TILE_160, capi.ROWS_TILE_256]


def _part_bytes(slices, outputs):
    return torch.empty(max(256, 4 * slices * outputs), dtype=torch.uint8, device="cuda") if slices > 1 else None


def _forward(name, kernel, slices, cols, rows, sums, counts=None):
    d = R.DTYPES[name]
    E = 1 if counts is None else len(counts)
    w = R.randn(1, E, cols, sums, dtype=d, scale=sums ** -0.5)
    w2 = R.randn(2, E, cols, sums, dtype=d, scale=sums ** -0.5)
    x = R.randn(3, rows, sums, dtype=d)
    offsets = None if counts is None else R.offsets_of(counts)
    ends = [0, rows] if counts is None else offsets.tolist()
    y, mid = (torch.full((rows, cols), 7.0, dtype=d, device="cuda") for _ in range(2))
    capi.rows_kernel(capi.ROWS_FORWARD, kernel, w, x, y, cols, rows, sums, offsets=offsets, slices=slices,
                     ws=_part_bytes(slices, rows * cols))
    capi.rows_kernel(capi.ROWS_SWIGLU, kernel, w, x, mid, cols, rows, sums, p2=w2, offsets=offsets, slices=slices,
                     ws=_part_bytes(slices, 2 * rows * cols))
    for e in range(E):
        a, b = ends[e], ends[e + 1]
        z, ez = R.mm(x[a:b], w[e])
        R.check(y[a:b], z, ez, f"y {e}")
        up, eu = R.mm(x[a:b], w2[e])
        s, es = R.act(z, "silu"), 1.13 * ez + 2.0 ** -19 * z.abs().clamp(min=1.0)
        R.check(mid[a:b], s * up, 1.01 * (es * up.abs() + s.abs() * eu + es * eu + 2.0 ** -23 * (s * up).abs()), f"mid {e}")
    assert (y[ends[-1]:] == 7.0).all() and (mid[ends[-1]:] == 7.0).all()


def _backward(name, kernel, slices, cols, rows, sums, halves, counts=None):
    """form 2: rows x (halves * sums) times halves matrices [sums][cols]; form 3: [sums][halves * rows]^T [sums][cols]."""
    d = R.DTYPES[name]
    E = 1 if counts is None else len(counts)
    if counts is None or kernel is not None:
        n = rows if counts is None else sum(counts)
        offsets = None if counts is None else R.offsets_of(counts)
        ends = [0, n] if counts is None else offsets.tolist()
        ws = [R.randn(4 + h, E, sums, cols, dtype=d, scale=sums ** -0.5) for h in range(halves)]
        g = R.randn(6, n, halves * sums, dtype=d)
        y = torch.empty(n, cols, dtype=d, device="cuda")
        capi.rows_kernel(capi.ROWS_INPUT, kernel, ws[0], g, y, cols, n, sums, p2=ws[1] if halves == 2 else None,
                         offsets=offsets, slices=slices, ws=_part_bytes(slices, n * cols))
        for e in range(E):
            a, b = ends[e], ends[e + 1]
            parts = [R.mm(g[a:b, h * sums:(h + 1) * sums], ws[h][e].t()) for h in range(halves)]
            R.check(y[a:b], sum(p[0] for p in parts), halves * sum(p[1] for p in parts), f"input {e}")
    if kernel == capi.ROWS_TILE_160:
        return
    n = sums if counts is None else sum(counts)
    offsets = None if counts is None else R.offsets_of(counts)
    ends = [0, n] if counts is None else offsets.tolist()
    x, g = R.randn(7, n, cols, dtype=d), R.randn(8, n, halves * rows, dtype=d)
    gw = [torch.empty(E, rows, cols, dtype=d, device="cuda") for _ in range(halves)]
    capi.rows_kernel(capi.ROWS_WEIGHT, kernel, x, g, gw[0], cols, rows, n, y2=gw[1] if halves == 2 else None,
                     offsets=offsets, slices=slices, ws=_part_bytes(slices, E * halves * rows * cols))
    for h in range(halves):
        for e in range(E):
            a, b = ends[e], ends[e + 1]
            ref, bound = R.mm(g[a:b, h * rows:(h + 1) * rows].t(), x[a:b].t())
            R.check(gw[h][e], ref, bound, f"weight {h} {e}")


@pytest.mark.parametrize("slices", [1, 3])
@pytest.mark.parametrize("kernel", TILES)
@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
def test_tiles(dev, name, kernel, slices):
    """Several tiles each way with ragged edges, a stage that ends inside, experts with and without rows; the order in
    blocks of eight row tiles, and more than 64 experts."""
    _forward(name, kernel, slices, 520, 333, 200)
    _forward(name, kernel, slices, 264, 330, 72, [0, 161, 1, 0, 160])
    _forward(name, kernel, slices, 72, 230, 136, [3] * 70 + [0, 17])
    _backward(name, kernel, slices, 520, 333, 200, 2)
    _backward(name, kernel, slices, 264, 136, 72, 1, [0, 161, 1, 0, 160])
    _backward(name, kernel, slices, 72, 136, 264, 2, [3] * 70 + [0, 17])


@pytest.mark.parametrize("kernel", [capi.ROWS_TILE_64, capi.ROWS_TILE_256])
def test_many_tiles(dev, kernel):
    """More tiles than workgroups at once: a stream over several tiles, chunks that XCDs take in turn."""
    _forward("bf16", kernel, 1, 4096, 2600, 128)
    _backward("bf16", kernel, 1, 2304, 1100, 264, 2, [0, 5, 130, 64, 65])
    _backward("bf16", kernel, 1, 256, 2400, 72, 1, [1] * 100 + [0] * 3 + [70])


@pytest.mark.parametrize("kernel,cols,rows", [(capi.ROWS_TILE_64, 520, 500), (capi.ROWS_TILE_256, 1800, 1700)])
def test_many_experts_of_unlike_rows(dev, kernel, cols, rows):
    """Weights' gradients of experts taken by their rows, some of them alike, the first and last without."""
    _backward("bf16", kernel, 1, cols, rows, 72, 1, [0, 5, 130, 64, 5, 300, 0, 1] + [33, 7, 64] * 5 + [0])


@pytest.mark.parametrize("waves", [1, 2, 5, 8])
@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
def test_direct(dev, name, waves):
    for cols, rows, sums in ((40, 3, 200), (17, 40, 61), (264, 16, 2056), (8, 1, 1)):
        _forward(name, capi.ROWS_DIRECT + waves, 1, cols, rows, sums)
    _forward(name, capi.ROWS_DIRECT + waves, 1, 48, 60, 136, [1, 0, 16, 17, 0, 20])


@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
def test_sums_do_not_depend_on_neighbours(dev, name):
    """A row's results are the same bits alone and among others, where the same kernel runs."""
    d, K, N = R.DTYPES[name], 200, 136
    x, w = R.randn(1, 300, K, dtype=d), R.randn(2, N, K, dtype=d)
    y, one = torch.empty(300, N, dtype=d, device="cuda"), torch.empty(40, N, dtype=d, device="cuda")
    capi.rows_kernel(capi.ROWS_FORWARD, capi.ROWS_TILE_128, w, x, y, N, 300, K)
    capi.rows_kernel(capi.ROWS_FORWARD, capi.ROWS_TILE_128, w, x[250:290], one, N, 40, K)
    assert torch.equal(one, y[250:290])


@pytest.mark.parametrize("name", ["bf16", "f32"])
def test_values_that_are_no_numbers_stay_in_their_rows(dev, name):
    """Infinities and NaN of one expert's row reach its own output row and its expert's gradient only; rows that share
    a stage, and the stage's end, take nothing from them."""
    d, K, N, counts = R.DTYPES[name], 72, 136, [5, 7, 30]
    offsets, n = R.offsets_of(counts), sum(counts)
    x, w, g = R.randn(1, n, K, dtype=d), R.randn(2, 3, N, K, dtype=d, scale=0.1), R.randn(3, n, N, dtype=d)
    clean = [torch.empty(n, N, dtype=d, device="cuda"), torch.empty(n, K, dtype=d, device="cuda"), torch.empty_like(w)]
    dirty = [torch.empty_like(t) for t in clean]
    for outs, poison in ((clean, False), (dirty, True)):
        if poison:
            x[6, 3], x[7, 10], g[6, 2] = float("nan"), float("inf"), float("inf")
        capi.grouped_mat_mul_rows(x, w, offsets, outs[0], K, N, n,
                                  ws=R.workspace(capi.grouped_mat_mul_rows_workspace_bytes(CODES[name], K, N, n, 3)))
        capi.grouped_mat_mul_rows_backward(
            g, x, w, offsets, outs[1], outs[2], K, N, n,
            ws=R.workspace(capi.grouped_mat_mul_rows_backward_workspace_bytes(CODES[name], K, N, n, 3)))
    others = [i for i in range(n) if i not in (6, 7)]
    assert torch.equal(clean[0][others], dirty[0][others]) and not torch.isfinite(dirty[0][6:8]).any()
    others = [i for i in range(n) if i != 6]
    assert torch.equal(clean[1][others], dirty[1][others]) and not torch.isfinite(dirty[1][6]).any()
    assert torch.equal(clean[2][[0, 2]], dirty[2][[0, 2]])
    assert not torch.isfinite(dirty[2][1, :, 3]).any() and torch.isfinite(dirty[2][1, :2, 20:]).all()


def test_offsets_are_clamped(dev):
    """A malformed table drops rows or takes some twice; nothing outside the buffers is touched."""
    K, N, rows = 64, 64, 40
    d = torch.bfloat16
    x, w = R.randn(1, rows, K, dtype=d), R.randn(2, 3, N, K, dtype=d)
    for table in ([0, 10, 5, 2 ** 31 - 1], [-5, 3, -2 ** 31, 40], [0, 100, 200, 300], [40, 40, 40, 40], [0, 40, 40, 40]):
        offsets = torch.tensor(table, dtype=torch.int32, device="cuda")
        y = torch.full((rows + 64, N), 7.0, dtype=d, device="cuda")
        gw = torch.full((5, N, K), 7.0, dtype=d, device="cuda")
        gx = torch.full((rows + 64, K), 7.0, dtype=d, device="cuda")
        for kernel in TILES + [capi.ROWS_DIRECT + 2]:
            capi.rows_kernel(capi.ROWS_FORWARD, kernel, w, x, y, N, rows, K, offsets=offsets)
        for kernel in TILES:
            capi.rows_kernel(capi.ROWS_INPUT, kernel, w, x, gx, K, rows, N, offsets=offsets)
            if kernel != capi.ROWS_TILE_160:
                capi.rows_kernel(capi.ROWS_WEIGHT, kernel, x, x, gw, K, N, rows, offsets=offsets)
        torch.cuda.synchronize()
        assert (y[rows:] == 7.0).all() and (gw[3:] == 7.0).all() and (gx[rows:] == 7.0).all()


def test_more_than_32_bits(dev):
    """Outputs, rows and weights beyond 2^31 elements: their last ones are right."""
    d, K, N, T = torch.bfloat16, 64, 40000, 66000
    x, w = R.randn(1, T, K, dtype=d), R.randn(2, N, K, dtype=d, scale=0.1)
    y = torch.empty(T, N, dtype=d, device="cuda")
    ws = capi.linear_rows_workspace_bytes(capi.DTYPE_BF16, K, N, T)
    capi.linear_rows(x, w, y, K, N, T, residual=y.zero_(), activation=capi.ACT_SILU, ws=R.workspace(ws))
    ref, bound, _, _ = R.linear(x[-300:], w, None, None, "silu")
    R.check(y[-300:], ref, bound + 2.0 ** -23 * ref.abs(), "y")
    # ... as the gradient of a product with long rows
    gx, gw = torch.empty(T, K, dtype=d, device="cuda"), torch.empty(N, K, dtype=torch.float32, device="cuda")
    need = capi.linear_rows_backward_workspace_bytes(capi.DTYPE_BF16, K, N, T)
    capi.linear_rows_backward(y, x, w, gx, gw, None, K, N, T, ws=R.workspace(need))
    R.check(gx[-300:], *R.mm(y[-300:], w.t()), "grad_x")
    R.check(gw[-300:], *R.mm(y[:, -300:].t(), x.t()), "grad_w")


def _layer(name, T, H, I, E, top_k, seed):
    d = R.DTYPES[name]
    ids = torch.topk(R.randn(seed, T, E), top_k, dim=1).indices.to(torch.int32).contiguous()
    ids[-1] = -1  # a padded token
    return {"d": d, "code": CODES[name], "sizes": (T, H, I, E, top_k), "ids": ids,
            "share": torch.softmax(R.randn(seed + 1, T, top_k), dim=1), "x": R.randn(seed + 2, T, H, dtype=d),
            "wg": R.randn(seed + 3, E, I, H, dtype=d, scale=H ** -0.5),
            "wu": R.randn(seed + 4, E, I, H, dtype=d, scale=H ** -0.5),
            "wd": R.randn(seed + 5, E, H, I, dtype=d, scale=I ** -0.5), "gy": R.randn(seed + 6, T, H, dtype=d, scale=0.1)}


def _buffers(s):
    T, H, I, E, top_k = s["sizes"]
    r, d, code = T * top_k, s["d"], s["code"]
    z = lambda *shape, dtype=d: torch.zeros(*shape, dtype=dtype, device="cuda")  # noqa: E731
    i32 = torch.int32
    need = max(capi.moe_gate_up_swiglu_rows_workspace_bytes(code, H, I, r, E),
               capi.grouped_mat_mul_rows_workspace_bytes(code, I, H, r, E),
               capi.grouped_mat_mul_rows_backward_workspace_bytes(code, I, H, r, E),
               capi.moe_gate_up_swiglu_rows_backward_workspace_bytes(code, H, I, r, E))
    return {"xs": z(r, H), "offsets": z(E + 1, dtype=i32), "src": z(r, dtype=i32), "dst": z(T, top_k, dtype=i32),
            "gate_up": z(r, 2 * I), "mid": z(r, I), "down": z(r, H), "y": z(T, H), "g_down": z(r, H),
            "g_share": z(T, top_k, dtype=torch.float32), "g_mid": z(r, I), "g_wd": torch.empty_like(s["wd"]), "g_xs": z(r, H),
            "g_wg": torch.empty_like(s["wg"]), "g_wu": torch.empty_like(s["wu"]), "g_x": z(T, H),
            "ws": torch.empty(max(need, 256), dtype=torch.uint8, device="cuda")}


def _step(s, b, stream=None):
    """A MoE layer forward and backward, as a training step calls it."""
    T, H, I, E, top_k = s["sizes"]
    r, ws = T * top_k, b["ws"]
    capi.moe_dispatch_rows(s["ids"], s["x"], b["xs"], b["offsets"], b["src"], b["dst"], T, top_k, H, E, stream=stream)
    capi.moe_gate_up_swiglu_rows(b["xs"], s["wg"], s["wu"], b["offsets"], E, b["mid"], H, I, r, gate_up=b["gate_up"], ws=ws,
                                 stream=stream)
    capi.grouped_mat_mul_rows(b["mid"], s["wd"], b["offsets"], b["down"], I, H, r, ws=ws, stream=stream)
    capi.moe_combine_rows(b["down"], b["dst"], s["share"], b["y"], T, H, top_k, stream=stream)
    capi.moe_combine_rows_backward(s["gy"], b["down"], b["dst"], s["share"], b["g_down"], b["g_share"], T, H, top_k,
                                   stream=stream)
    capi.grouped_mat_mul_rows_backward(b["g_down"], b["mid"], s["wd"], b["offsets"], b["g_mid"], b["g_wd"], I, H, r, ws=ws,
                                       stream=stream)
    capi.moe_gate_up_swiglu_rows_backward(b["g_mid"], b["gate_up"], b["xs"], s["wg"], s["wu"], b["offsets"], E, b["g_xs"],
                                          b["g_wg"], b["g_wu"], H, I, r, ws=ws, stream=stream)
    capi.moe_dispatch_rows_backward(b["g_xs"], b["dst"], b["g_x"], T, H, top_k, stream=stream)


OUTPUTS = ("y", "g_share", "g_wd", "g_wg", "g_wu", "g_x")


def _reference(s):
    """The layer and its gradients in 64 bits, by differentiation."""
    T, H, I, E, top_k = s["sizes"]
    leaves = {k: s[k].double().requires_grad_(True) for k in ("x", "share", "wg", "wu", "wd")}
    y = torch.zeros(T, H, dtype=torch.float64, device="cuda")
    for e in range(E):
        tok, slot = torch.nonzero(s["ids"] == e, as_tuple=True)
        xe = leaves["x"][tok]
        mid = torch.nn.functional.silu(xe @ leaves["wg"][e].t()) * (xe @ leaves["wu"][e].t())
        y = y.index_add(0, tok, leaves["share"][tok, slot][:, None] * (mid @ leaves["wd"][e].t()))
    y.backward(s["gy"].double())
    return {"y": y.detach(), "g_share": leaves["share"].grad, "g_wd": leaves["wd"].grad, "g_wg": leaves["wg"].grad,
            "g_wu": leaves["wu"].grad, "g_x": leaves["x"].grad}


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("sizes", [(37, 96, 72, 5, 2), (300, 264, 136, 8, 3), (1, 64, 64, 4, 2)])
def test_moe_layer(dev, name, sizes):
    """Dispatch, gate|up, down, combine and all gradients together.  Each of the chain's up to five roundings to the
    layer's type is off by half a step, eps / 2 (and each of its fp32 sums of n terms by n 2^-23, n at most 264 here); to
    first order the errors of independent steps add, in the 2-norm over a result, at most to their sum times
    the sum of magnitudes over the result's own norm: 2 for sums of products of both signs, whose terms
    are of random sign."""
    s = _layer(name, *sizes, seed=11)
    b = _buffers(s)
    _step(s, b)
    ref = _reference(s)
    eps = torch.finfo(s["d"]).eps / 2
    limit = 2 * (5 * eps + 3 * 300 * 2.0 ** -23)
    for k in OUTPUTS:
        norm = ref[k].norm()
        off = (b[k].double() - ref[k]).norm()
        assert off <= limit * norm, (k, (off / norm).item() if norm > 0 else off.item(), limit)


def test_captured_and_replayed(dev):
    """Two captured layers that share a workspace, replayed with eager work and new inputs between."""
    layers = [_layer("bf16", 200, 136, 264, 8, 2, seed=21), _layer("bf16", 77, 136, 264, 8, 2, seed=31)]
    bufs = [_buffers(s) for s in layers]
    ws = max((b["ws"] for b in bufs), key=torch.Tensor.numel)
    for b in bufs:
        b["ws"] = ws
    for s, b in zip(layers, bufs):  # kernels are loaded before the capture
        _step(s, b)
    torch.cuda.synchronize()
    graphs = []
    for s, b in zip(layers, bufs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            _step(s, b)
        graphs.append(g)
    for turn in range(4):
        for k, s in enumerate(layers):
            s["x"].copy_(R.randn(100 + 10 * turn + k, *s["x"].shape, dtype=s["d"]))
            s["gy"].copy_(R.randn(200 + 10 * turn + k, *s["gy"].shape, dtype=s["d"], scale=0.1))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        got = [{k: b[k].clone() for k in OUTPUTS} for b in bufs]
        for s, b, have in zip(layers, bufs, got):
            for k in OUTPUTS:
                b[k].zero_()
            _step(s, b)
            torch.cuda.synchronize()
            for k in OUTPUTS:
                assert torch.equal(b[k], have[k]), (turn, k)


def test_streams(dev):
    """Two layers on two streams at once, each with its own workspace; the same bits as one after the other."""
    layers = [_layer("f16", 260, 264, 136, 8, 2, seed=41), _layer("f16", 130, 264, 136, 8, 2, seed=51)]
    bufs = [_buffers(s) for s in layers]
    for s, b in zip(layers, bufs):
        _step(s, b)
    torch.cuda.synchronize()
    want = [{k: b[k].clone() for k in OUTPUTS} for b in bufs]
    streams = [torch.cuda.Stream() for _ in layers]
    for _ in range(3):
        for b in bufs:
            for k in OUTPUTS:
                b[k].zero_()
        torch.cuda.synchronize()
        for s, b, st in zip(layers, bufs, streams):
            _step(s, b, stream=st)
        torch.cuda.synchronize()
        for b, w in zip(bufs, want):
            for k in OUTPUTS:
                assert torch.equal(b[k], w[k]), k


def test_gradients_against_differences(dev):
    """The linear layer's gradients against central differences of its own forward pass (fp32).  A step h of 2^-6 along a
    random direction: the difference is off by h^2 / 6 of a third derivative (below 4 for these activations at |z| < 4, times
    the direction's cube) and by the forward's rounding, 2^-20 of the loss's magnitude, over h."""
    T, K, N, h = 24, 40, 56, 2.0 ** -6
    x, w, b, g = R.randn(1, T, K), R.randn(2, N, K, scale=K ** -0.5), R.randn(3, N, scale=0.1), R.randn(4, T, N)
    for act in ("gelu", "gelu_tanh", "silu"):
        code = R.ACTS[act]
        pre, gx, gw, gb = (torch.empty(*s, device="cuda") for s in ((T, N), (T, K), (N, K), (N,)))
        y = torch.empty(T, N, device="cuda")
        ws = R.workspace(max(capi.linear_rows_workspace_bytes(0, K, N, T), capi.linear_rows_backward_workspace_bytes(0, K, N, T)))

        def loss(x_, w_, b_):
            capi.linear_rows(x_, w_, y, K, N, T, bias=b_, activation=code, ws=ws, pre=pre)
            return (g.double() * y.double()).sum().item()
        base = loss(x, w, b)
        capi.linear_rows_backward(g, x, w, gx, gw, gb, K, N, T, activation=code, pre=pre, ws=ws)
        size = (g.double() * y.double()).abs().sum().item()
        for t, grad, k in ((x, gx, 0), (w, gw, 1), (b, gb, 2)):
            v = R.randn(9 + k, *t.shape)
            v /= v.norm()
            at = [x, w, b]
            sides = []
            for sign in (1, -1):
                at[k] = t + sign * h * v
                sides.append(loss(*at))
            slope = (sides[0] - sides[1]) / (2 * h)
            moved = (x @ v.t() if k == 1 else v @ w.t() if k == 0 else v.expand(T, N)).double().abs()
            limit = h * h / 6 * 4 * (g.double().abs() * moved ** 3).sum().item() + 2 * 2.0 ** -20 * size / (2 * h)
            assert abs(slope - (grad.double() * v.double()).sum().item()) <= limit, (act, k, slope, base, limit)


def test_tensors_of_the_host_and_others_are_refused(dev):
    x, w, y = torch.zeros(3, 8), torch.zeros(4, 8, device="cuda"), torch.zeros(3, 4, device="cuda")
    with pytest.raises(ValueError, match="device tensor"):
        capi.linear_rows(x, w, y, 8, 4, 3)
    with pytest.raises(ValueError, match="contiguous"):
        capi.linear_rows(x.cuda(), w.t().contiguous().t(), y, 8, 4, 3)
    with pytest.raises(ValueError, match="do not overlap"):
        capi.linear_rows(x.cuda()[0].expand(3, 8), w, y, 8, 4, 3)
    with pytest.raises(capi.JJOError) as e:
        capi.linear_rows_backward(y, x.cuda(), w, None, w, None, 8, 4, 3, activation=capi.ACT_RELU, ws=None, pre=y)
    assert e.value.code == capi.JJO_ERR_INVALID_ARG
