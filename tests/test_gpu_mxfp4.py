"""MXFP4 operators against fp64: bytes of the quantizer, products in every kernel's range, the
grouped forms, SwiGLU, the FFN as a whole and as the run of its public stages."""
if __name__ == "__main__":  # `python tests/<file>.py`, as the reference runs its tests
    import sys as _sys

    import pytest as _pytest
    _sys.exit(_pytest.main([__file__, "-q"]))
import sys

import numpy as np
import pytest
import torch

import _mxfp4 as mx
from jjjetson_ops_amd import capi

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def note(msg):
    print(f"[case] {msg}", flush=True)
    sys.stdout.flush()


def _host(t):
    torch.cuda.synchronize()
    return t.double().cpu().numpy()


def _rand(rng, rows, cols, dtype="f32", scale=1.0):
    """Values with a different magnitude per block, rounded to dtype."""
    x = rng.standard_normal((rows, cols)) * scale * np.exp2(rng.integers(-6, 7, (rows, 1)))
    x[rng.random((rows, cols)) < 0.02] *= 20
    return torch.from_numpy(x).to(DT[dtype])


def _mx(rng, rows, cols, dev, scale=0.05):
    """(device MXFP4 matrix, its values in fp64)."""
    q = mx.pack(*mx.quantize(rng.standard_normal((rows, cols)) * scale))
    return torch.from_numpy(q).to(dev), mx.dequantize(q, rows, cols)


def _close(got, exp, bound):
    bad = ~(np.abs(got - exp) <= bound)
    assert not bad.any(), (int(bad.sum()), np.abs(got - exp)[bad].max(), bound[bad].min(), np.argwhere(bad)[:4].tolist())


# ------------------------------------------------------------------------- quantizer
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("rows,cols", [(1, 32), (1, 4096), (3, 96), (17, 160), (130, 2048), (5, 11008)])
def test_quantize_bytes(rows, cols, dtype, dev):
    note(f"quantize {rows}x{cols} {dtype}")
    rng = np.random.default_rng(rows + cols)
    x = _rand(rng, rows, cols, dtype)
    q = torch.full((capi.mxfp4_bytes(rows, cols) + 16,), 0xA5, dtype=torch.uint8, device=dev)
    capi.quantize_mxfp4(x.to(dev), q, rows, cols)
    exp = mx.pack(*mx.quantize(x.double().numpy()))
    got = q.cpu().numpy()
    assert np.array_equal(got[:-16], exp) and (got[-16:] == 0xA5).all()
    y = torch.empty(rows, cols, dtype=DT[dtype], device=dev)
    capi.dequantize_mxfp4(q, y, rows, cols)
    want = torch.from_numpy(mx.dequantize(exp, rows, cols)).to(DT[dtype])
    assert torch.equal(y.cpu(), want)


def test_quantize_borders(dev):
    """Every border between two codes, at exponents down to the subnormals and up to the top,
    zeros of both signs, NaN and infinities; every scale byte back to values."""
    note("quantize borders")
    m = np.array([0.0, 0.1, 0.25, 0.5, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.9], np.float32)
    m = np.concatenate([m, np.nextafter(m, np.float32(0)), np.nextafter(m, np.float32(9))])
    rows = []
    for e in (-150, -149, -135, -128, -127, -126, -125, -60, 0, 60, 124):
        for v in m:
            row = np.zeros(32, np.float32)
            row[0], row[1], row[2] = np.ldexp(np.float32(4), e), np.ldexp(v, e), -np.ldexp(v, e)
            rows.append(row)
    rows.append(np.where(np.arange(32) % 2, -0.0, 0.0).astype(np.float32))
    for bad in (np.inf, -np.inf, np.nan, -np.nan):
        row = np.linspace(-3, 3, 32, dtype=np.float32)
        row[7] = bad
        rows.append(row)
    x = np.stack(rows)
    q = torch.empty(capi.mxfp4_bytes(len(x), 32), dtype=torch.uint8, device=dev)
    capi.quantize_mxfp4(torch.from_numpy(x).to(dev), q, len(x), 32)
    code, s = mx.unpack(q.cpu().numpy(), len(x), 32)
    want_code, want_s = mx.quantize(x)
    assert np.array_equal(s, want_s)
    assert np.array_equal(code, want_code)
    all_q = mx.pack(np.tile(np.arange(32, dtype=np.uint8) % 16, (256, 1)), np.arange(256, dtype=np.uint8)[:, None])
    for dtype in DT:
        y = torch.empty(256, 32, dtype=DT[dtype], device=dev)
        capi.dequantize_mxfp4(torch.from_numpy(all_q).to(dev), y, 256, 32)
        want = torch.from_numpy(mx.dequantize(all_q, 256, 32)).to(torch.float32).to(DT[dtype])
        assert torch.equal(y.cpu().nan_to_num(nan=7.0), want.nan_to_num(nan=7.0)) and torch.equal(y.cpu().isnan(), want.isnan())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_quantize_strided(dtype, dev):
    """Rows of a wider tensor, read and written; what lies between them stays."""
    note(f"quantize strided {dtype}")
    wide = _rand(np.random.default_rng(5), 37, 512, dtype).to(dev)
    x = wide[:, 64:64 + 224]
    q = torch.empty(capi.mxfp4_bytes(37, 224), dtype=torch.uint8, device=dev)
    capi.quantize_mxfp4(x, q, 37, 224)
    exp = mx.pack(*mx.quantize(x.double().cpu().numpy()))
    assert np.array_equal(q.cpu().numpy(), exp)
    back = torch.full_like(wide, 9.0)
    capi.dequantize_mxfp4(q, back[:, 64:64 + 224], 37, 224)
    want = torch.full((37, 512), 9.0, dtype=DT[dtype])
    want[:, 64:64 + 224] = torch.from_numpy(mx.dequantize(exp, 37, 224)).to(DT[dtype])
    assert torch.equal(back.cpu(), want)
    for bad in (wide.t(), wide[:, ::2]):
        with pytest.raises(ValueError, match="contiguous"):
            capi.quantize_mxfp4(bad, q, 32, 32)
    with pytest.raises(capi.JJOError, match="16-byte aligned"):
        capi.quantize_mxfp4(wide[:, 1:225], q, 37, 224)


# -------------------------------------------------------------------------- products
SHAPES = [(32, 1, 1), (32, 16, 1), (128, 5, 2), (160, 33, 3), (4096, 96, 1), (4096, 100, 4), (1056, 130, 16),
          (992, 64, 17), (2048, 256, 24), (11008, 48, 7), (512, 200, 33), (1024, 257, 64), (160, 70, 65),
          (640, 300, 100), (4096, 256, 129), (256, 1000, 255), (1312, 520, 300), (2048, 512, 600), (288, 8300, 2050),
          (800, 4200, 4111)]


@pytest.mark.parametrize("K,N,M", SHAPES)
def test_mat_mul(K, N, M, dev):
    note(f"mat_mul K={K} N={N} M={M}")
    rng = np.random.default_rng(K + 7 * N + M)
    w, wv = _mx(rng, N, K, dev)
    x, xv = _mx(rng, M, K, dev, 1.0)
    exp, bound = xv @ wv.T, mx.sum_bound(xv, wv)
    for dtype in DT:
        y = torch.full((M * N + 8,), 3.0, dtype=DT[dtype], device=dev)
        capi.mat_mul_mxfp4(w, x, y, K, N, M)
        got = _host(y)
        assert (got[M * N:] == 3.0).all()
        _close(got[:M * N].reshape(M, N), exp, bound + mx.rounding(np.abs(exp) + bound, dtype))


@pytest.mark.parametrize("K,N,M", [(64, 40, 2), (4096, 64, 1), (512, 96, 150)])
def test_mat_mul_extreme_scales(K, N, M, dev):
    """Blocks of very different magnitudes, a NaN block, and zero blocks."""
    note(f"mat_mul scales K={K} N={N} M={M}")
    rng = np.random.default_rng(K + N)
    wq, xq = (mx.quantize(rng.standard_normal((n, K)) * np.exp2(rng.integers(-30, 30, (n, 1)))) for n in (N, M))
    wq[1][:, 0] = rng.integers(90, 160, N)
    xq[1][:, -1] = rng.integers(90, 160, M)
    wq[0][1, :32] = 0
    wq[1][3, 1] = 255
    w, x = mx.pack(*wq), mx.pack(*xq)
    wv, xv = mx.dequantize(w, N, K), mx.dequantize(x, M, K)
    y = torch.empty(M, N, dtype=torch.float32, device=dev)
    capi.mat_mul_mxfp4(torch.from_numpy(w).to(dev), torch.from_numpy(x).to(dev), y, K, N, M)
    got = _host(y)
    assert np.isnan(got[:, 3]).all()
    keep = np.arange(N) != 3
    _close(got[:, keep], xv @ wv[keep].T, mx.sum_bound(xv, wv[keep]) + 2.0 ** -140)


@pytest.mark.parametrize("din,dout", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f32"), ("f32", "bf16")])
@pytest.mark.parametrize("K,N,T", [(32, 8, 1), (4096, 200, 1), (14336, 64, 1), (20480, 48, 1), (1056, 100, 1),
                                   (96, 33, 2), (2048, 128, 5), (160, 250, 40), (1024, 300, 200)])
def test_linear(K, N, T, din, dout, dev):
    note(f"linear K={K} N={N} T={T} {din}->{dout}")
    rng = np.random.default_rng(K + N + T)
    w, wv = _mx(rng, N, K, dev)
    x = _rand(rng, T, K, din)
    xv = mx.dequantize(mx.pack(*mx.quantize(x.double().numpy())), T, K)
    ws = torch.full((max(16, capi.linear_mxfp4_workspace_bytes(K, T)),), 0xFF, dtype=torch.uint8, device=dev)
    y = torch.full((T, N), float("nan"), dtype=DT[dout], device=dev)
    capi.linear_mxfp4(x.to(dev), w, y, K, N, T, ws=ws)
    exp, bound = xv @ wv.T, mx.sum_bound(xv, wv)
    _close(_host(y), exp, bound + mx.rounding(np.abs(exp) + bound, dout))


# --------------------------------------------------------------------------- grouped
def _offsets(rng, E, R, skew):
    if skew == "one":
        counts = np.zeros(E, int)
        counts[E // 2] = R
    else:
        counts = rng.multinomial(R, rng.dirichlet(np.full(E, 0.5 if skew == "skewed" else 50.0)))
    return np.concatenate([[0], np.cumsum(counts)])


GROUPED = [(3, 64, 40, 1, "even"), (8, 256, 96, 5, "skewed"), (8, 512, 130, 40, "even"), (5, 160, 64, 100, "one"),
           (70, 128, 32, 200, "skewed"), (4, 1056, 256, 300, "even"), (8, 512, 160, 1000, "skewed"),
           (300, 64, 32, 64, "even"), (64, 288, 1056, 9500, "even"), (64, 256, 1030, 9500, "skewed")]


@pytest.mark.parametrize("E,K,N,R,skew", GROUPED)
def test_grouped(E, K, N, R, skew, dev):
    """Sorted rows, some of them behind the last expert's (not written), with and without
    a scatter of the output rows."""
    note(f"grouped E={E} K={K} N={N} R={R} {skew}")
    rng = np.random.default_rng(E + K + R)
    w, wv = _mx(rng, E * N, K, dev)
    x, xv = _mx(rng, R, K, dev, 1.0)
    live = R - R // 8
    off = _offsets(rng, E, live, skew)
    exp, bound = np.full((R, N), 5.0), np.zeros((R, N))
    for e in range(E):
        rows, we = slice(off[e], off[e + 1]), wv[e * N:(e + 1) * N]
        exp[rows], bound[rows] = xv[rows] @ we.T, mx.sum_bound(xv[rows], we)
    od = torch.from_numpy(off.astype(np.int32)).to(dev)
    y = torch.full((R, N), 5.0, device=dev)
    capi.grouped_mat_mul_mxfp4(w, x, od, y, K, N, R)
    _close(_host(y), exp, bound)
    perm = rng.permutation(R).astype(np.int32)
    y2 = torch.full((R, N), 5.0, dtype=torch.bfloat16, device=dev)
    capi.grouped_mat_mul_mxfp4(w, x, od, y2, K, N, R, route_dst=torch.from_numpy(perm).to(dev))
    _close(_host(y2)[perm], exp, bound + mx.rounding(np.abs(exp) + bound, "bf16"))


def _check_swiglu(mid, g, u, dg, du):
    """The MXFP4 bytes of silu(g) * u where g and u are known to dg and du: the scale is that of
    a maximum within the error, and each value lies between the roundings of the
    ends of its interval.  silu's slope is at most 1.1; six fp32 operations follow."""
    rows, cols = g.shape
    with np.errstate(over="ignore"):
        silu = g / (1 + np.exp(-g))
    v = silu * u
    d = 1.1 * dg * (np.abs(u) + du) + np.abs(silu) * du + 8 * 2.0 ** -24 * np.abs(v) + 2.0 ** -126
    code, s = mx.unpack(mid, rows, cols)
    lo, hi = (np.abs(v) - d).clip(0).reshape(rows, -1, 32).max(2), (np.abs(v) + d).reshape(rows, -1, 32).max(2)
    assert ((s >= mx.scale_byte(lo)) & (s <= mx.scale_byte(hi))).all()
    sc = np.repeat(mx.scale_value(s), 32, 1)
    got = mx.values(code)
    assert (got >= mx.values(mx.round_codes((v - d) / sc))).all()
    assert (got <= mx.values(mx.round_codes((v + d) / sc))).all()


@pytest.mark.parametrize("E,K,I,R,skew", [(3, 64, 32, 1, "even"), (8, 512, 96, 12, "skewed"), (4, 160, 160, 50, "even"),
                                          (4, 1056, 128, 300, "even"), (8, 512, 224, 1000, "skewed"),
                                          (70, 128, 32, 200, "skewed"), (64, 288, 544, 9500, "even"),
                                          (64, 256, 512, 9500, "skewed")])
def test_gate_up_swiglu(E, K, I, R, skew, dev):
    note(f"gate_up E={E} K={K} I={I} R={R}")
    rng = np.random.default_rng(E + K + R + I)
    wg, wgv = _mx(rng, E * I, K, dev)
    wu, wuv = _mx(rng, E * I, K, dev)
    x, xv = _mx(rng, R, K, dev, 1.0)
    live = R - R // 8
    off = _offsets(rng, E, live, skew)
    g, u, dg, du = (np.zeros((R, I)) for _ in range(4))
    for e in range(E):
        rows, we = slice(off[e], off[e + 1]), slice(e * I, (e + 1) * I)
        g[rows], dg[rows] = xv[rows] @ wgv[we].T, mx.sum_bound(xv[rows], wgv[we])
        u[rows], du[rows] = xv[rows] @ wuv[we].T, mx.sum_bound(xv[rows], wuv[we])
    mid = torch.full((capi.mxfp4_bytes(R, I) + 16,), 0x5A, dtype=torch.uint8, device=dev)
    capi.moe_gate_up_swiglu_mxfp4(wg, wu, x, torch.from_numpy(off.astype(np.int32)).to(dev), E, mid, K, I, R)
    got = mid.cpu().numpy()
    code, s = mx.unpack(got, R, I)
    assert (got[-16:] == 0x5A).all() and (s[live:] == 0x5A).all()  # rows of no expert stay
    _check_swiglu(mx.pack(code[:live], s[:live]), g[:live], u[:live], dg[:live], du[:live])


def _ffn_case(rng, T, H, I, E, dev, dtype):
    mats = [_mx(rng, rows, cols, dev)[0] for rows, cols in ((E * I, H), (E * I, H), (E * H, I))]
    x = _rand(rng, T, H, dtype).to(dev)
    return mats, x, torch.from_numpy(rng.standard_normal((T, E)).astype(np.float32)).to(dev)


FFN = [(1, 64, 32, 4, 1, "f32"), (1, 512, 256, 8, 2, "bf16"), (4, 1024, 512, 8, 2, "bf16"), (16, 160, 96, 64, 8, "f32"),
       (33, 512, 224, 8, 2, "f16"), (100, 256, 128, 64, 8, "bf16"), (300, 512, 416, 8, 2, "f32"),
       (700, 256, 256, 4, 2, "bf16"), (3, 128, 64, 300, 32, "f32"), (2100, 256, 128, 8, 2, "bf16"),
       (600, 128, 64, 300, 8, "f32")]


@pytest.mark.parametrize("T,H,I,E,k,dtype", FFN)
def test_ffn_is_the_run_of_its_stages(T, H, I, E, k, dtype, dev):
    """The FFN's output against the public stages in turn: top-k, rows to their experts,
    quantizer, gate|up with SwiGLU, down, combine; and the last two against fp64."""
    note(f"ffn T={T} H={H} I={I} E={E} k={k} {dtype}")
    mats, x, logits = _ffn_case(np.random.default_rng(T + H + E), T, H, I, E, dev, dtype)
    _check_ffn(mats, x, logits, T, H, I, E, k, dtype, dev)


def _check_ffn(mats, x, logits, T, H, I, E, k, dtype, dev):
    wg, wu, wd = mats
    R = T * k
    y = torch.full((T, H), float("nan"), dtype=DT[dtype], device=dev)
    ws = torch.full((capi.moe_ffn_mxfp4_workspace_bytes(T, H, I, E, k),), 0xFF, dtype=torch.uint8, device=dev)
    capi.moe_ffn_mxfp4(x, logits, wg, wu, wd, y, T, H, I, E, k, ws)

    i32 = dict(dtype=torch.int32, device=dev)
    share, ids, off = torch.empty(T, k, device=dev), torch.empty(T, k, **i32), torch.empty(E + 1, **i32)
    src, dst = torch.empty(R, **i32), torch.empty(R, **i32)
    rows = torch.empty(R, H, dtype=DT[dtype], device=dev)
    xq = torch.empty(capi.mxfp4_bytes(R, H), dtype=torch.uint8, device=dev)
    mid = torch.empty(capi.mxfp4_bytes(R, I), dtype=torch.uint8, device=dev)
    out = torch.empty(R, H, device=dev)
    capi.moe_top_k(logits, share, ids, T, E, k)
    capi.moe_dispatch_rows(ids, x, rows, off, src, dst, T, k, H, E)
    capi.quantize_mxfp4(rows, xq, R, H)
    capi.moe_gate_up_swiglu_mxfp4(wg, wu, xq, off, E, mid, H, I, R)
    capi.grouped_mat_mul_mxfp4(wd, mid, off, out, I, H, R)
    y2 = torch.empty(T, H, device=dev)
    capi.moe_combine_rows(out, dst, share, y2, T, H, k)
    assert torch.equal(y, y2.to(DT[dtype]))

    midv, wdv = mx.dequantize(mid.cpu().numpy(), R, I), mx.dequantize(wd.cpu().numpy(), E * H, I)
    o, d, w = off.cpu().numpy(), dst.cpu().numpy().reshape(T, k), _host(share)
    eo, eb = np.zeros((R, H)), np.zeros((R, H))
    for e in range(E):
        r = slice(o[e], o[e + 1])
        eo[r], eb[r] = midv[r] @ wdv[e * H:(e + 1) * H].T, mx.sum_bound(midv[r], wdv[e * H:(e + 1) * H])
    exp = (w[..., None] * eo[d]).sum(1)
    bound = (w[..., None] * (eb[d] + k * 2.0 ** -23 * np.abs(eo[d]))).sum(1)
    _close(_host(y), exp, bound + mx.rounding(np.abs(exp) + bound, dtype))


def test_ffn_same_expert_for_all_and_for_none(dev):
    """Every token to one expert (the others have no rows), and logits of -infinity."""
    note("ffn one expert")
    T, H, I, E, k = 40, 128, 64, 8, 2
    rng = np.random.default_rng(3)
    (wg, wu, wd), x, logits = _ffn_case(rng, T, H, I, E, dev, "f32")
    logits[:, 5], logits[:, 2] = 30.0, 20.0
    logits[7] = float("-inf")
    logits[7, 1] = 0.0
    _check_ffn((wg, wu, wd), x, logits, T, H, I, E, k, "f32", dev)


# ------------------------------------------------- large products, every tile; the oracle on the GPU
def _values(q, rows, cols):
    """The values of an MXFP4 matrix without NaN blocks, in fp64."""
    half = rows * cols // 2
    table = torch.from_numpy(mx.values(np.arange(16, dtype=np.uint8))).to(q.device)
    b = q[:half].view(rows, cols // 2).int()
    v = torch.stack([table[b & 15], table[b >> 4]], 2).view(rows, cols // 32, 32)
    v *= torch.exp2(q[half:rows * cols // 32 * 17].view(rows, cols // 32, 1).double() - 127)
    return v.view(rows, cols)


def _bytes(gen, rows, cols, dev, scale=119):
    """Random codes under scales of seven magnitudes, and their values in fp64."""
    half = rows * cols // 2
    q = torch.randint(0, 256, (rows * cols // 32 * 17,), dtype=torch.uint8, device=dev, generator=gen)
    q[half:] = scale + q[half:] % 7
    return q, _values(q, rows, cols)


def _product(x, w):
    """x . w^T and the bound of its fp32 sum (sum_bound)."""
    return x @ w.t().contiguous(), (x.shape[1] // 32 + 8) * 2.0 ** -23 * (x.abs() @ w.abs().t().contiguous())


def _close_dev(got, exp, bound):
    bad = ~((got.double() - exp).abs() <= bound)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist(), (got.double() - exp).abs().max().item())


# With 256 CUs: tiles of 32, 64, 96 and 128 tokens cut along K, then whole, then 160, 192 and 256; a last block, a
# last pair of stages and row and token tiles that are not full.
@pytest.mark.parametrize("K,N,M", [(2080, 8264, 50), (2336, 16424, 33), (2080, 16424, 70), (2048, 16420, 100),
                                   (544, 16424, 16), (1056, 16424, 50), (608, 16420, 90), (768, 16424, 127),
                                   (544, 14344, 625), (544, 14341, 700), (800, 14339, 1000), (2080, 16423, 70),
                                   (1056, 16417, 50)])
def test_mat_mul_tiles(K, N, M, dev):
    note(f"mat_mul tiles K={K} N={N} M={M}")
    gen = torch.Generator(device=dev).manual_seed(K + N + M)
    w, wv = _bytes(gen, N, K, dev)
    x, xv = _bytes(gen, M, K, dev)
    exp, bound = _product(xv, wv)
    for dtype in DT:
        y = torch.full((M * N + 8,), 3.0, dtype=DT[dtype], device=dev)
        capi.mat_mul_mxfp4(w, x, y, K, N, M)
        assert (y[M * N:] == 3.0).all()
        _close_dev(y[:M * N].view(M, N), exp, bound + mx.HALF_STEP[dtype] * (exp.abs() + bound) + mx.TINY[dtype])


# (E, K, values a row of the two matrices together, rows): the same tiles for an expert's rows.
TILES = [(4, 2080, 4160, 48), (4, 2336, 4160, 160), (4, 2080, 4160, 256), (4, 2048, 4160, 400), (4, 544, 4160, 48),
         (4, 1056, 4160, 160), (4, 608, 4160, 256), (4, 768, 4160, 400), (8, 544, 8192, 1030), (8, 544, 8192, 1240),
         (8, 800, 8192, 1600), (4, 2080, 4160, 16)]


def _uneven(E, R):
    """Ranges of rows: one expert has none, one the most, and some rows belong to no expert."""
    share = np.full(E, (R - R // 16) // E)
    share[1] += share[2] - share[2] // 2
    share[2] //= 2
    share[3] += share[0]
    share[0] = 0
    return np.concatenate([[0], np.cumsum(share)])


@pytest.mark.parametrize("E,K,N,R", TILES)
def test_grouped_tiles(E, K, N, R, dev):
    note(f"grouped tiles E={E} K={K} N={N} R={R}")
    gen = torch.Generator(device=dev).manual_seed(K + N + R)
    w, wv = _bytes(gen, E * N, K, dev)
    x, xv = _bytes(gen, R, K, dev)
    off = _uneven(E, R)
    exp = torch.full((R, N), 5.0, dtype=torch.float64, device=dev)
    bound = torch.zeros_like(exp)
    for e in range(E):
        r = slice(off[e], off[e + 1])
        exp[r], bound[r] = _product(xv[r], wv[e * N:(e + 1) * N])
    od = torch.from_numpy(off.astype(np.int32)).to(dev)
    y = torch.full((R, N), 5.0, device=dev)
    capi.grouped_mat_mul_mxfp4(w, x, od, y, K, N, R)
    _close_dev(y, exp, bound)


@pytest.mark.parametrize("E,K,N,R", TILES)
def test_gate_up_swiglu_tiles(E, K, N, R, dev):
    I = N // 2
    note(f"gate_up tiles E={E} K={K} I={I} R={R}")
    gen = torch.Generator(device=dev).manual_seed(K + N + R)
    (wg, wgv), (wu, wuv) = (_bytes(gen, E * I, K, dev) for _ in range(2))
    x, xv = _bytes(gen, R, K, dev)
    off = _uneven(E, R)
    live = off[-1]
    g, u, dg, du = (torch.zeros(live, I, dtype=torch.float64, device=dev) for _ in range(4))
    for e in range(E):
        r, we = slice(off[e], off[e + 1]), slice(e * I, (e + 1) * I)
        g[r], dg[r] = _product(xv[r], wgv[we])
        u[r], du[r] = _product(xv[r], wuv[we])
    mid = torch.full((capi.mxfp4_bytes(R, I) + 16,), 0x5A, dtype=torch.uint8, device=dev)
    capi.moe_gate_up_swiglu_mxfp4(wg, wu, x, torch.from_numpy(off.astype(np.int32)).to(dev), E, mid, K, I, R)
    got = mid.cpu().numpy()
    code, s = mx.unpack(got, R, I)
    assert (got[-16:] == 0x5A).all() and (s[live:] == 0x5A).all()  # rows of no expert stay
    _check_swiglu(mx.pack(code[:live], s[:live]), *(t.cpu().numpy() for t in (g, u, dg, du)))


@pytest.mark.parametrize("T,H,I,E,k,dtype", [(500, 4096, 4096, 8, 2, "bf16"), (400, 4096, 8224, 6, 2, "f32"),
                                             (1100, 2048, 5600, 12, 2, "f16")])
def test_ffn_down_in_slices(T, H, I, E, k, dtype, dev):
    """Experts with many rows and few tiles: the down product in two slices of K, added by the
    combine, against fp64 from the intermediate on."""
    note(f"ffn slices T={T} H={H} I={I} E={E} k={k} {dtype}")
    gen = torch.Generator(device=dev).manual_seed(T)
    R = T * k
    wg, wu = (_bytes(gen, E * I, H, dev, 116)[0] for _ in range(2))
    wd = _bytes(gen, E * H, I, dev)[0]
    x = torch.randn(T, H, device=dev, generator=gen).to(DT[dtype])
    logits = torch.randn(T, E, device=dev, generator=gen)
    n = capi.moe_ffn_mxfp4_workspace_bytes(T, H, I, E, k)
    assert n > 2 * R * H * 4 + capi.mxfp4_bytes(T, H) + capi.mxfp4_bytes(R, I)  # two slices
    ws = torch.full((n,), 0xFF, dtype=torch.uint8, device=dev)
    y = torch.full((T, H), float("nan"), dtype=DT[dtype], device=dev)
    capi.moe_ffn_mxfp4(x, logits, wg, wu, wd, y, T, H, I, E, k, ws)

    i32 = dict(dtype=torch.int32, device=dev)
    share, ids, off = torch.empty(T, k, device=dev), torch.empty(T, k, **i32), torch.empty(E + 1, **i32)
    src, dst = torch.empty(R, **i32), torch.empty(R, **i32)
    rows = torch.empty(R, H, dtype=DT[dtype], device=dev)
    xq = torch.empty(capi.mxfp4_bytes(R, H), dtype=torch.uint8, device=dev)
    mid = torch.empty(capi.mxfp4_bytes(R, I), dtype=torch.uint8, device=dev)
    capi.moe_top_k(logits, share, ids, T, E, k)
    capi.moe_dispatch_rows(ids, x, rows, off, src, dst, T, k, H, E)
    capi.quantize_mxfp4(rows, xq, R, H)
    capi.moe_gate_up_swiglu_mxfp4(wg, wu, xq, off, E, mid, H, I, R)
    o, midv, wdv = off.tolist(), _values(mid, R, I), _values(wd, E * H, I)
    eo, eb = (torch.zeros(R, H, dtype=torch.float64, device=dev) for _ in range(2))
    for e in range(E):
        q = slice(o[e], o[e + 1])
        eo[q], eb[q] = _product(midv[q], wdv[e * H:(e + 1) * H])
    d, w = dst.long().view(T, k), share.double()[..., None]
    exp = (w * eo[d]).sum(1)
    bound = (w * (eb[d] + k * 2.0 ** -23 * eo[d].abs())).sum(1)
    _close_dev(y, exp, bound + mx.HALF_STEP[dtype] * (exp.abs() + bound) + mx.TINY[dtype])


@pytest.mark.parametrize("M", [1, 7, 40])
def test_mat_mul_offsets_beyond_32_bits(M, dev):
    """A weight of 4.7 GB: its first and last rows."""
    K, N = 16384, 540_000
    note(f"mat_mul offsets K={K} N={N} M={M}")
    gen = torch.Generator(device=dev).manual_seed(M)
    half = N * (K // 2)
    w = torch.randint(0, 256, (N * (K // 32) * 17,), dtype=torch.uint8, device=dev, generator=gen)
    w[half:] = 119 + w[half:] % 7
    x, xv = _bytes(gen, M, K, dev)
    y = torch.full((M, N), float("nan"), device=dev)
    capi.mat_mul_mxfp4(w, x, y, K, N, M)
    rows = 64
    for n0 in (0, N - rows):
        codes, scales = w[n0 * (K // 2):(n0 + rows) * (K // 2)], w[half + n0 * (K // 32):half + (n0 + rows) * (K // 32)]
        wv = mx.dequantize(torch.cat([codes, scales]).cpu().numpy(), rows, K)
        exp, bound = _product(xv, torch.from_numpy(wv).to(dev))
        _close_dev(y[:, n0:n0 + rows], exp, bound)
    assert not y.isnan().any()


# ---------------------------------------------------------------- graphs and streams
def _replays_match(fn, outs, dev, n=3):
    fn()
    torch.cuda.synchronize()
    eager = [o.clone() for o in outs]
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            fn()
    for _ in range(n):
        for o in outs:
            o.zero_()
        torch.randn(1 << 20, device=dev).sum().item()
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, eager):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("T", [1, 3, 40, 300])
def test_graph(T, dev):
    note(f"mxfp4 graph T={T}")
    H, I, E, k = 256, 160, 8, 2
    rng = np.random.default_rng(T)
    (wg, wu, wd), x, logits = _ffn_case(rng, T, H, I, E, dev, "bf16")
    ws = torch.empty(capi.moe_ffn_mxfp4_workspace_bytes(T, H, I, E, k), dtype=torch.uint8, device=dev)
    lw = torch.empty(max(16, capi.linear_mxfp4_workspace_bytes(H, T)), dtype=torch.uint8, device=dev)
    y, z = torch.empty(T, H, dtype=torch.bfloat16, device=dev), torch.empty(T, E * I, device=dev)

    def step():
        capi.moe_ffn_mxfp4(x, logits, wg, wu, wd, y, T, H, I, E, k, ws)
        capi.linear_mxfp4(y, wg, z, H, E * I, T, ws=lw)

    _replays_match(step, [y, z], dev)


@pytest.mark.parametrize("T,H,I", [(300, 544, 576), (500, 4096, 4096)])
def test_graph_tiles(T, H, I, dev):
    """The tiled kernels, the two-launch routing and the sliced down product; two graphs of one
    workspace, replayed in turn."""
    note(f"mxfp4 graph tiles T={T} H={H}")
    E, k = 8, 2
    gen = torch.Generator(device=dev).manual_seed(T)
    wg, wu, wd = (_bytes(gen, rows, cols, dev, 116)[0] for rows, cols in ((E * I, H), (E * I, H), (E * H, I)))
    xs = [torch.randn(T, H, device=dev, generator=gen).bfloat16() for _ in range(2)]
    logits = torch.randn(T, E, device=dev, generator=gen)
    ws = torch.empty(capi.moe_ffn_mxfp4_workspace_bytes(T, H, I, E, k), dtype=torch.uint8, device=dev)
    lw = torch.empty(capi.linear_mxfp4_workspace_bytes(H, T), dtype=torch.uint8, device=dev)
    ys, zs = [torch.empty_like(x) for x in xs], [torch.empty(T, E * I, device=dev) for _ in xs]

    def step(i):
        capi.moe_ffn_mxfp4(xs[i], logits, wg, wu, wd, ys[i], T, H, I, E, k, ws)
        capi.linear_mxfp4(ys[i], wg, zs[i], H, E * I, T, ws=lw)

    for i in range(2):
        step(i)
    torch.cuda.synchronize()
    eager = [t.clone() for t in ys + zs]
    s, graphs = torch.cuda.Stream(), []
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i], stream=s):
            step(i)
    for _ in range(3):
        for t in ys + zs:
            t.zero_()
        ws.fill_(0xFF)
        torch.cuda.synchronize()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for a, b in zip(ys + zs, eager):
            assert torch.equal(a, b)


def test_streams(dev):
    """Two streams at once, each with its own workspace, give what one call alone gives."""
    note("mxfp4 streams")
    K, N, T = 2048, 1024, 40
    rng = np.random.default_rng(1)
    w, _ = _mx(rng, N, K, dev)
    xs = [_rand(rng, T, K).to(dev) for _ in range(2)]
    n = capi.linear_mxfp4_workspace_bytes(K, T)
    want = []
    for x in xs:
        y = torch.empty(T, N, device=dev)
        capi.linear_mxfp4(x, w, y, K, N, T, ws=torch.empty(n, dtype=torch.uint8, device=dev))
        want.append(y)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    wss, ys = [torch.empty(n, dtype=torch.uint8, device=dev) for _ in xs], [torch.empty(T, N, device=dev) for _ in xs]
    torch.cuda.synchronize()
    for _ in range(10):
        for s, x, ws, y in zip(streams, xs, wss, ys):
            capi.linear_mxfp4(x, w, y, K, N, T, ws=ws, stream=s)
    torch.cuda.synchronize()
    for a, b in zip(ys, want):
        assert torch.equal(a, b)
