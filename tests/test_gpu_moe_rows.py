"""Token rows to their experts and back, and the gradients, against fp64."""
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
# tokens, top_k, hidden, experts, dtype, dropped: the one-launch dispatch (up to 4096 routes) and the
# sort before it, rows in pieces of 16 bytes with and without a rest, shorter than one, and longer than
# a workgroup's pieces.
CASES = [(1, 1, 1, 1, "f32", "none"), (1, 2, 4096, 8, "f32", "none"), (4, 2, 4096, 8, "bf16", "some"),
         (5, 3, 7, 4, "bf16", "some"), (33, 8, 130, 64, "f16", "some"), (100, 1, 5, 3, "f32", "none"),
         (512, 8, 96, 64, "bf16", "padded"), (513, 8, 64, 1024, "f32", "some"), (2000, 4, 33, 5, "f16", "padded"),
         (700, 32, 40, 40, "bf16", "some"), (64, 2, 20000, 8, "bf16", "none"), (9, 2, 256, 8, "f32", "all"),
         (3000, 2, 8, 1, "f32", "none"), (5000, 2, 514, 1000, "bf16", "padded"), (8200, 1, 9, 1024, "bf16", "some"),
         (65, 3, 2049, 16, "f16", "some"), (40, 2, 4095, 8, "f32", "padded"), (2200, 3, 1031, 16, "bf16", "some"),
         (70001, 2, 3, 2, "f16", "padded")]


def note(msg):
    print(f"[case] {msg}", flush=True)
    sys.stdout.flush()


def _ids(rng, T, k, E, dropped):
    ids = np.stack([rng.permutation(max(E, k))[:k] % E for _ in range(T)]).astype(np.int32)
    if dropped == "some":
        ids[rng.random((T, k)) < 0.2] = rng.choice([-1, E, -2 ** 31, 2 ** 31 - 1])
    elif dropped == "padded":
        ids[T - T // 10:] = -1
    elif dropped == "all":
        ids[:] = -1
    return ids


def _sorted(ids, E):
    flat = ids.reshape(-1)
    live = (flat >= 0) & (flat < E)
    order = np.array(sorted(np.flatnonzero(live), key=lambda r: (flat[r], r)), dtype=np.int64)
    dst = np.full(flat.size, -1, np.int64)
    dst[order] = np.arange(order.size)
    return np.searchsorted(flat[order], np.arange(E + 1)) if order.size else np.zeros(E + 1, int), order, dst


def _host(t):
    torch.cuda.synchronize()
    return t.double().cpu().numpy()


def _close(got, exp, bound):
    bad = ~(np.abs(got - exp) <= bound)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4].tolist())


@pytest.mark.parametrize("T,k,H,E,dtype,dropped", CASES)
def test_dispatch(T, k, H, E, dtype, dropped, dev):
    note(f"dispatch T={T} k={k} H={H} E={E} {dtype} {dropped}")
    rng = np.random.default_rng(T + H)
    ids, R = _ids(rng, T, k, E, dropped), T * k
    x = torch.from_numpy(rng.standard_normal((T, H))).to(DT[dtype])
    off, order, dst = _sorted(ids, E)
    rows = torch.full((R, H), 7.0, dtype=DT[dtype], device=dev)
    o = torch.full((E + 1,), -5, dtype=torch.int32, device=dev)
    s, d = (torch.full((R,), -5, dtype=torch.int32, device=dev) for _ in range(2))
    capi.moe_dispatch_rows(torch.from_numpy(ids).to(dev), x.to(dev), rows, o, s, d, T, k, H, E)
    assert np.array_equal(o.cpu().numpy(), off)
    assert np.array_equal(d.cpu().numpy(), dst)
    assert np.array_equal(s.cpu().numpy()[:order.size], order) and (s.cpu().numpy()[order.size:] == -5).all()
    want = torch.full((R, H), 7.0, dtype=DT[dtype])
    want[:order.size] = x[torch.from_numpy(order // k)]
    assert torch.equal(rows.cpu(), want)


@pytest.mark.parametrize("T,k,H,E,dtype,dropped", CASES)
def test_dispatch_backward_and_combine(T, k, H, E, dtype, dropped, dev):
    """Sums over k in fp32, each product and addition off by at most 2^-24 of its magnitude, then
    one rounding to the rows' type."""
    note(f"join T={T} k={k} H={H} E={E} {dtype} {dropped}")
    rng = np.random.default_rng(T + H + 1)
    ids, R = _ids(rng, T, k, E, dropped), T * k
    dst = _sorted(ids, E)[2].reshape(T, k)
    rows = torch.from_numpy(rng.standard_normal((R, H))).to(DT[dtype])
    share = torch.from_numpy(rng.random((T, k))).float()
    live = (dst >= 0)[..., None]
    taken = np.where(live, rows.double().numpy()[dst.clip(0)], 0.0)
    dd, rd = torch.from_numpy(dst.astype(np.int32)).to(dev), rows.to(dev)
    for w in (None, share.double().numpy()):
        y = torch.full((T, H), float("nan"), dtype=DT[dtype], device=dev)
        if w is None:
            capi.moe_dispatch_rows_backward(rd, dd, y, T, H, k)
        else:
            capi.moe_combine_rows(rd, dd, share.to(dev), y, T, H, k)
        terms = taken if w is None else w[..., None] * taken
        exp, mag = terms.sum(1), np.abs(terms).sum(1)
        bound = k * 2.0 ** -24 * mag
        _close(_host(y), exp, bound + mx.rounding(np.abs(exp) + bound, dtype))


@pytest.mark.parametrize("T,k,H,E,dtype,dropped", CASES)
def test_combine_backward(T, k, H, E, dtype, dropped, dev):
    """grad_expert_out: one fp32 product, rounded to the rows' type.  grad_weights: a thread has pieces
    of at most eight values, one of every 256, so at most H/256 + 8 products in turn, then eight
    additions, 2^-24 each."""
    note(f"join grad T={T} k={k} H={H} E={E} {dtype} {dropped}")
    rng = np.random.default_rng(T + H + 2)
    ids, R = _ids(rng, T, k, E, dropped), T * k
    dst = _sorted(ids, E)[2].reshape(T, k)
    rows, g = (torch.from_numpy(rng.standard_normal((n, H))).to(DT[dtype]) for n in (R, T))
    share = torch.from_numpy(rng.random((T, k))).float()
    ge = torch.full((R, H), 7.0, dtype=DT[dtype], device=dev)
    gw = torch.full((T, k), float("nan"), device=dev)
    capi.moe_combine_rows_backward(g.to(dev), rows.to(dev), torch.from_numpy(dst.astype(np.int32)).to(dev),
                                   share.to(dev), ge, gw, T, H, k)
    gd, w = g.double().numpy(), share.double().numpy()
    exp = np.full((R, H), 7.0)
    t, j = np.nonzero(dst >= 0)
    exp[dst[t, j]] = w[t, j][:, None] * gd[t]
    off = 2.0 ** -24 * np.abs(exp)
    off[np.setdiff1d(np.arange(R), dst)] = 0.0
    _close(_host(ge), exp, off + mx.rounding(np.abs(exp) + off, dtype))
    terms = np.where((dst >= 0)[..., None], gd[:, None, :] * rows.double().numpy()[dst.clip(0)], 0.0)
    _close(_host(gw), terms.sum(2), (H // 256 + 17) * 2.0 ** -24 * np.abs(terms).sum(2))


@pytest.mark.parametrize("T,k,H,dtype", [(300, 4, 1024, "bf16"), (300, 4, 1024, "f16"), (200, 3, 512, "f32"),
                                         (64, 2, 1000, "bf16"), (40, 3, 514, "bf16"), (50, 2, 4096, "f32"),
                                         (50, 2, 1032, "f16"), (30, 2, 33, "f32"), (9, 8, 7, "f16")])
def test_combine_backward_weights(T, k, H, dtype, dev):
    """grad_weights within the roundings of either kernel, 2^-24 of the magnitudes each, V values a
    piece (8, or 4 of fp32).  Up to 128 pieces a wave or part of one has the row: at most two pieces a
    lane, 2 V products added in turn, then at most six steps of lanes.  Longer, a workgroup: a thread
    has every 256th piece, then six steps and two for the waves."""
    note(f"join grad weights T={T} k={k} H={H} {dtype}")
    rng = np.random.default_rng(T + H + 3)
    V, R = (4 if dtype == "f32" else 8), T * k
    dst = rng.permutation(R).astype(np.int32).reshape(T, k)
    rows, g = (torch.from_numpy(rng.standard_normal((n, H))).to(DT[dtype]) for n in (R, T))
    ge = torch.empty(R, H, dtype=DT[dtype], device=dev)
    gw = torch.full((T, k), float("nan"), device=dev)
    capi.moe_combine_rows_backward(g.to(dev), rows.to(dev), torch.from_numpy(dst).to(dev), torch.rand(T, k, device=dev),
                                   ge, gw, T, H, k)
    terms = g.double().numpy()[:, None, :] * rows.double().numpy()[dst]
    roundings = 2 * V + 6 if H <= 128 * V else -(-H // (256 * V)) * V + 8
    _close(_host(gw), terms.sum(2), roundings * 2.0 ** -24 * np.abs(terms).sum(2))


def test_gradients_against_differences(dev):
    """The combine is linear in the rows and in the weights, the dispatch in x: a difference of the
    forward pass along a direction is the gradient's product with it, up to the fp32 rounding
    of the two passes."""
    note("rows differences")
    T, k, H, E = 40, 4, 72, 16
    rng = np.random.default_rng(11)
    R = T * k
    ids = torch.from_numpy(_ids(rng, T, k, E, "some")).to(dev)
    i32 = dict(dtype=torch.int32, device=dev)
    off, src, dst = torch.empty(E + 1, **i32), torch.empty(R, **i32), torch.empty(R, **i32)

    def dispatch(x):
        rows = torch.zeros(R, H, device=dev)
        capi.moe_dispatch_rows(ids, x, rows, off, src, dst, T, k, H, E)
        return rows

    def combine(rows, w):
        y = torch.empty(T, H, device=dev)
        capi.moe_combine_rows(rows, dst, w, y, T, H, k)
        return y

    x, dx, gy = (torch.randn(T, H, device=dev) for _ in range(3))
    rows, drows = dispatch(x), torch.randn(R, H, device=dev)
    w, dw = torch.rand(T, k, device=dev), torch.randn(T, k, device=dev)
    n = int(off[-1])
    drows[n:] = 0
    ge, gw, gx = torch.zeros(R, H, device=dev), torch.empty(T, k, device=dev), torch.empty(T, H, device=dev)
    capi.moe_combine_rows_backward(gy, rows, dst, w, ge, gw, T, H, k)
    capi.moe_dispatch_rows_backward(ge, dst, gx, T, H, k)
    d = torch.float64

    def along(f0, f1, g, direction):
        diff = (gy.to(d) * (f1.to(d) - f0.to(d))).sum().item()
        pred = (g.to(d) * direction.to(d)).sum().item()
        # k + 1 roundings of each pass and the gradient's (H/256 + 11), of terms below the sum of the
        # magnitudes, and the rounding of the moved point itself
        mag = (gy.to(d).abs() * (f0.to(d).abs() + f1.to(d).abs())).sum().item() + (g.to(d).abs() * direction.to(d).abs()).sum().item()
        assert abs(diff - pred) <= 32 * k * 2.0 ** -24 * mag

    y = combine(rows, w)
    along(y, combine(rows + drows, w), ge, drows)
    along(y, combine(rows, w + dw), gw, dw)
    along(y, combine(dispatch(x + dx), w), gx, dx)


def test_graph(dev):
    """Dispatch, combine and both gradients captured together, replayed on changed tables."""
    note("rows graph")
    for T in (6, 2500):
        k, H, E = 2, 96, 8
        rng = np.random.default_rng(T)
        R = T * k
        ids = torch.from_numpy(_ids(rng, T, k, E, "some")).to(dev)
        x, gy = torch.randn(T, H, device=dev), torch.randn(T, H, device=dev)
        w = torch.rand(T, k, device=dev)
        i32 = dict(dtype=torch.int32, device=dev)
        off, src, dst = torch.zeros(E + 1, **i32), torch.zeros(R, **i32), torch.zeros(R, **i32)
        rows, ge = torch.zeros(R, H, device=dev), torch.zeros(R, H, device=dev)
        y, gx, gw = torch.zeros(T, H, device=dev), torch.zeros(T, H, device=dev), torch.zeros(T, k, device=dev)
        outs = [off, src, dst, rows, y, ge, gw, gx]

        def step():
            capi.moe_dispatch_rows(ids, x, rows, off, src, dst, T, k, H, E)
            capi.moe_combine_rows(rows, dst, w, y, T, H, k)
            capi.moe_combine_rows_backward(gy, rows, dst, w, ge, gw, T, H, k)
            capi.moe_dispatch_rows_backward(ge, dst, gx, T, H, k)

        step()
        s = torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                step()
        for seed in range(3):
            ids.copy_(torch.from_numpy(_ids(np.random.default_rng(100 + seed), T, k, E, "some")))
            for o in outs:
                o.zero_()
            step()
            torch.cuda.synchronize()
            eager = [o.clone() for o in outs]
            for o in outs:
                o.zero_()
            torch.randn(1 << 20, device=dev).sum().item()
            g.replay()
            torch.cuda.synchronize()
            for a, b in zip(outs, eager):
                assert torch.equal(a, b)


def test_rows_beyond_32_bits(dev):
    """Sorted rows of 4.6 GB, there and back: with one expert's rows behind the other's, the sum of
    a token's eight equal rows is exact."""
    T, k, H, E = 70_000, 8, 4096, 16
    note(f"rows offsets T={T} k={k} H={H}")
    gen = torch.Generator(device=dev).manual_seed(1)
    R = T * k
    x = torch.randn(T, H, device=dev, dtype=torch.bfloat16, generator=gen)
    ids = torch.argsort(torch.rand(T, E, device=dev, generator=gen), 1)[:, :k].int().contiguous()
    rows = torch.empty(R, H, dtype=torch.bfloat16, device=dev)
    off, src, dst = (torch.empty(n, dtype=torch.int32, device=dev) for n in (E + 1, R, R))
    capi.moe_dispatch_rows(ids, x, rows, off, src, dst, T, k, H, E)
    want = torch.argsort(ids.view(-1).long() * R + torch.arange(R, device=dev))
    assert torch.equal(src.long(), want)
    assert torch.equal(off.long(), torch.searchsorted(ids.view(-1).sort()[0].long(), torch.arange(E + 1, device=dev)))
    for p in range(0, R, 70_000):
        assert torch.equal(rows[p:p + 70_000], x[want[p:p + 70_000] // k])
    back = torch.empty(T, H, dtype=torch.bfloat16, device=dev)
    capi.moe_dispatch_rows_backward(rows, dst, back, T, H, k)
    assert torch.equal(back, x * 8)
