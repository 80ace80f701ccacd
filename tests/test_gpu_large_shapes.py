"""MXFP4 and sorted-row calls at the limits that their entries document."""
if __name__ == "__main__":  # `python tests/<file>.py`, as the reference runs its tests
    import sys as _sys

    import pytest as _pytest
    _sys.exit(_pytest.main([__file__, "-q"]))
import pytest
import torch

import _mxfp4 as mx
from jjjetson_ops_amd import capi
from test_gpu_mxfp4 import _close_dev, _product, _values, note

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _memory():
    """Tens of gigabytes a test: given back before the next."""
    torch.cuda.empty_cache()
    yield
    torch.cuda.empty_cache()


def test_combine_backward_of_all_routes(dev):
    """2^26 routes of rows that a whole wave shares: one grid of a wave per route would have 2^32
    threads.  grad_expert_out is one fp32 product.  grad_weights: a lane or thread has at most one
    piece of four values (H <= 256), then at most eight additions in turn, 2^-24 each."""
    T, k, H = 1 << 21, 32, 129
    R = T * k
    note(f"combine backward T={T} k={k} H={H}")
    gen = torch.Generator(device=dev).manual_seed(1)
    gy = torch.randn(T, H, device=dev, generator=gen)
    w = torch.rand(T, k, device=dev, generator=gen)
    rows = torch.empty(R, H, device=dev)
    for part in rows.split(1 << 22):
        part.normal_(generator=gen)
    ge = torch.full((R, H), float("nan"), device=dev)
    gw = torch.full((T, k), float("nan"), device=dev)
    dst = torch.arange(R - 1, -1, -1, dtype=torch.int32, device=dev)
    capi.moe_combine_rows_backward(gy, rows, dst, w, ge, gw, T, H, k)
    step = 1 << 15
    for t in range(0, T, step):
        g = gy[t:t + step].double()[:, None]
        sl = slice(R - (t + step) * k, R - t * k)  # the tokens' routes, the last one first
        e, got = (a[sl].flip(0).view(step, k, H) for a in (rows, ge))
        terms = g * e.double()
        bad = ~((gw[t:t + step].double() - terms.sum(2)).abs() <= 12 * 2.0 ** -24 * terms.abs().sum(2))
        assert not bad.any(), (t, bad.nonzero()[:4].tolist())
        want = w[t:t + step].double()[..., None] * g
        bad = ~((got.double() - want).abs() <= mx.HALF_STEP["f32"] * want.abs() + mx.TINY["f32"])
        assert not bad.any(), (t, bad.nonzero()[:4].tolist())


def _codes(gen, rows, cols, dev):
    """Random codes under one scale, 1: a product is a whole number of quarters, 144 at most, so a sum of
    up to 2^16 of them is exact in fp32 in any order."""
    half = rows * cols // 2
    q = torch.randint(0, 256, (rows * cols // 32 * 17,), dtype=torch.uint8, device=dev, generator=gen)
    q[half:] = 127
    return q


def _rows_of(q, rows, cols, first, n):
    """The values (fp64) of rows first.. of a matrix under one scale."""
    table = torch.from_numpy(mx.values(torch.arange(16, dtype=torch.uint8).numpy())).to(q.device)
    b = q[first * cols // 2:(first + n) * cols // 2].view(n, cols // 2).int()
    return torch.stack([table[b & 15], table[b >> 4]], 2).view(n, cols)


def test_mat_mul_of_short_rows_and_many_outputs(dev):
    """2^33 outputs of K = 32: 16 tokens x 32 rows a workgroup would be a grid of 2^32 threads.  The sums
    are exact, so the outputs are the fp64 products rounded once."""
    K, N, M = 32, 8200, (1 << 20) + 5
    note(f"mat_mul K={K} N={N} M={M}")
    gen = torch.Generator(device=dev).manual_seed(2)
    w, x = _codes(gen, N, K, dev), _codes(gen, M, K, dev)
    y = torch.full((M, N), float("nan"), dtype=torch.bfloat16, device=dev)
    capi.mat_mul_mxfp4(w, x, y, K, N, M)
    wv = _rows_of(w, N, K, 0, N).float().t().contiguous()
    step = 1 << 15
    for t in range(0, M, step):
        n = min(step, M - t)
        assert torch.equal(y[t:t + n], (_rows_of(x, M, K, t, n).float() @ wv).bfloat16()), t


def test_mat_mul_of_most_weight_rows(dev):
    """2^28 weight rows, 16 a workgroup: as many workgroups of 256 threads would be 2^32."""
    K, N = 32, 1 << 28
    note(f"mat_mul K={K} N={N} M=1")
    gen = torch.Generator(device=dev).manual_seed(4)
    w, x = _codes(gen, N, K, dev), _codes(gen, 1, K, dev)
    xv = _rows_of(x, 1, K, 0, 1)
    for call in ("mat_mul", "linear"):
        y = torch.full((1, N), float("nan"), device=dev)
        if call == "mat_mul":
            capi.mat_mul_mxfp4(w, x, y, K, N, 1)
        else:  # the row's largest code is 6 or 4, so its quantized form is the row itself
            assert xv.abs().max() >= 4
            capi.linear_mxfp4(xv.float(), w, y, K, N, 1)
        step = 1 << 22
        for n in range(0, N, step):
            assert torch.equal(y[0, n:n + step].double(), (_rows_of(w, N, K, n, step) * xv).sum(1)), (call, n)


def test_gate_up_of_short_rows_and_many_outputs(dev):
    """The same for gate|up: equal rows give equal bytes, whichever launch they are in."""
    K, I, E, base_rows = 32, 8224, 2, 1 << 11
    R = 1 << 20
    note(f"gate_up K={K} I={I} R={R}")
    gen = torch.Generator(device=dev).manual_seed(3)
    wg, wu = _codes(gen, E * I, K, dev), _codes(gen, E * I, K, dev)
    few = _codes(gen, base_rows, K, dev)
    half = base_rows * K // 2
    x = torch.cat([few[:half].repeat(R // base_rows), few[half:].repeat(R // base_rows)])

    def run(q, rows):
        mid = torch.full((capi.mxfp4_bytes(rows, I),), 0x5A, dtype=torch.uint8, device=dev)
        off = torch.tensor([0, rows // 2, rows], dtype=torch.int32, device=dev)
        capi.moe_gate_up_swiglu_mxfp4(wg, wu, q, off, E, mid, K, I, rows)
        n = rows * I // 2
        return mid[:n].view(rows, I // 2), mid[n:].view(rows, I // 32)

    two = torch.cat([few[:half], few[:half], few[half:], few[half:]])  # each expert has every row once
    small = run(two, 2 * base_rows)
    for got, want in zip(run(x, R), small):
        for e in range(E):
            g = got[e * R // 2:(e + 1) * R // 2].view(-1, base_rows, got.shape[1])
            for part in g:
                assert torch.equal(part, want[e * base_rows:(e + 1) * base_rows])


def test_ffn_of_tokens_beyond_4_gib(dev):
    """More than 4 GiB of MXFP4 tokens, whose rows gate|up gathers: tokens of the first rows, around the
    middle and of the last rows against the public stages on these tokens alone.  One scale for
    tokens and for gate and up: their sums are exact, so the intermediate bytes do not depend on
    the tile."""
    T, H, I, E, k = (1 << 20) + 3, 8192, 4096, 4, 2
    note(f"ffn T={T} H={H} I={I} E={E} k={k}")
    gen = torch.Generator(device=dev).manual_seed(5)
    wg, wu = _codes(gen, E * I, H, dev), _codes(gen, E * I, H, dev)
    for w in (wg, wu):
        w[E * I * H // 2:] = 119  # sums of some 2^14 quarters, times 2^-8
    wd = _codes(gen, E * H, I, dev)
    wd[E * H * I // 2:] = 110
    few = 1 << 10
    values = _rows_of(_codes(gen, few, H, dev), few, H, 0, few).bfloat16()
    values.view(few, -1, 32)[..., 5] = 6.0  # every block's scale is 1
    x = torch.empty(T, H, dtype=torch.bfloat16, device=dev)
    for t in range(0, T, few):
        x[t:t + few] = values[:min(few, T - t)]
    logits = torch.randn(T, E, device=dev, generator=gen)
    y = torch.full((T, H), float("nan"), dtype=torch.bfloat16, device=dev)
    ws = torch.empty(capi.moe_ffn_mxfp4_workspace_bytes(T, H, I, E, k), dtype=torch.uint8, device=dev)
    capi.moe_ffn_mxfp4(x, logits, wg, wu, wd, y, T, H, I, E, k, ws)
    del ws
    for part in y.split(1 << 16):
        assert not part.isnan().any()

    at = torch.cat([torch.arange(64), torch.arange(T // 2 - 64, T // 2 + 64), torch.arange(T - 64, T)]).to(dev)
    n, i32 = len(at), dict(dtype=torch.int32, device=dev)
    R = n * k
    share, ids, off = torch.empty(n, k, device=dev), torch.empty(n, k, **i32), torch.empty(E + 1, **i32)
    src, dst = torch.empty(R, **i32), torch.empty(R, **i32)
    rows = torch.empty(R, H, dtype=torch.bfloat16, device=dev)
    xq, mid = (torch.empty(capi.mxfp4_bytes(R, c), dtype=torch.uint8, device=dev) for c in (H, I))
    capi.moe_top_k(logits[at].contiguous(), share, ids, n, E, k)
    capi.moe_dispatch_rows(ids, x[at].contiguous(), rows, off, src, dst, n, k, H, E)
    capi.quantize_mxfp4(rows, xq, R, H)
    capi.moe_gate_up_swiglu_mxfp4(wg, wu, xq, off, E, mid, H, I, R)
    o, midv, wdv = off.tolist(), _values(mid, R, I), _values(wd, E * H, I)
    eo, eb = (torch.zeros(R, H, dtype=torch.float64, device=dev) for _ in range(2))
    for e in range(E):
        q = slice(o[e], o[e + 1])
        eo[q], eb[q] = _product(midv[q], wdv[e * H:(e + 1) * H])
    d, w = dst.long().view(n, k), share.double()[..., None]
    exp = (w * eo[d]).sum(1)
    bound = (w * (eb[d] + k * 2.0 ** -23 * eo[d].abs())).sum(1)
    _close_dev(y[at], exp, bound + mx.HALF_STEP["bf16"] * (exp.abs() + bound) + mx.TINY["bf16"])


@pytest.mark.parametrize("T,k,E,H", [(1 << 21, 32, 1000, 8), (1 << 23, 8, 3, 1), (1 << 23, 1, 64, 40)])
def test_rows_of_most_routes(T, k, E, H, dev):
    """The most tokens and the most routes, there and back: the sort against torch's stable one, whole
    numbers as rows, so that their sums are exact."""
    R = T * k
    note(f"rows T={T} k={k} E={E} H={H}")
    gen = torch.Generator(device=dev).manual_seed(6)
    ids = torch.randint(-1, E, (T, k), dtype=torch.int32, device=dev, generator=gen)  # -1: dropped
    x = torch.randint(-4, 5, (T, H), device=dev, generator=gen).bfloat16()
    rows = torch.full((R, H), 7.0, dtype=torch.bfloat16, device=dev)
    off, src, dst = (torch.full((n,), -5, dtype=torch.int32, device=dev) for n in (E + 1, R, R))
    capi.moe_dispatch_rows(ids, x, rows, off, src, dst, T, k, H, E)
    key, order = torch.where(ids < 0, E, ids).view(-1).sort(stable=True)
    live = int((key < E).sum())
    assert torch.equal(off.long(), torch.searchsorted(key[:live], torch.arange(E + 1, device=dev, dtype=torch.int32)))
    assert torch.equal(src[:live].long(), order[:live]) and (src[live:] == -5).all()
    want = torch.full((R,), -1, dtype=torch.int32, device=dev)
    want[order[:live]] = torch.arange(live, dtype=torch.int32, device=dev)
    assert torch.equal(dst, want)
    del key, want
    step = 1 << 22
    for p in range(0, live, step):
        n = min(step, live - p)
        assert torch.equal(rows[p:p + n], x[order[p:p + n] // k])
    assert (rows[live:] == 7.0).all()
    del order, src
    counts = (ids >= 0).sum(1, keepdim=True)
    back, y = torch.full_like(x, float("nan")), torch.full_like(x, float("nan"))
    capi.moe_dispatch_rows_backward(rows, dst, back, T, H, k)
    assert torch.equal(back.float(), (x.float() * counts).bfloat16().float())
    w = torch.full((T, k), 0.5, device=dev)
    capi.moe_combine_rows(rows, dst, w, y, T, H, k)
    assert torch.equal(y.float(), (x.float() * counts * 0.5).bfloat16().float())
    gw = torch.full((T, k), float("nan"), device=dev)
    ge = torch.full_like(rows, 7.0)
    capi.moe_combine_rows_backward(x, rows, dst, w, ge, gw, T, H, k)
    assert torch.equal(gw, (x.float() ** 2).sum(1, keepdim=True) * (ids >= 0))
    assert torch.equal(ge[:live], rows[:live] * 0.5) and (ge[live:] == 7.0).all()


def test_quantize_of_most_values(dev):
    """2^35 - 2^23 values in one call and back: rows that repeat give bytes that repeat, and one more row
    of blocks is refused."""
    rows, cols, few = (1 << 20) - (1 << 8), 1 << 15, 1 << 8
    note(f"quantize {rows}x{cols}")
    gen = torch.Generator(device=dev).manual_seed(7)
    some = torch.randn(few, cols, device=dev, generator=gen).bfloat16()
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device=dev)
    x.view(-1, few, cols)[:] = some
    q = torch.empty(capi.mxfp4_bytes(rows, cols), dtype=torch.uint8, device=dev)
    capi.quantize_mxfp4(x, q, rows, cols)
    q0 = torch.empty(capi.mxfp4_bytes(few, cols), dtype=torch.uint8, device=dev)
    capi.quantize_mxfp4(some, q0, few, cols)
    half, half0 = rows * cols // 2, few * cols // 2
    for got, want in ((q[:half], q0[:half0]), (q[half:], q0[half0:])):
        for part in got.view(-1, want.numel()).split(256):
            assert (part == want).all()
    back0 = torch.empty_like(some)
    capi.dequantize_mxfp4(q0, back0, few, cols)
    x.fill_(float("nan"))
    capi.dequantize_mxfp4(q, x, rows, cols)
    for part in x.view(-1, few * cols).split(256):
        assert (part == back0.view(-1)).all()
    with pytest.raises(capi.JJOError, match="exceeds one launch"):
        capi._check(capi.lib().quantize_mxfp4_device(None, x.data_ptr(), capi.DTYPE_BF16, cols, q.data_ptr(), rows + 1,
                                                     cols), "quantize_mxfp4_device")
