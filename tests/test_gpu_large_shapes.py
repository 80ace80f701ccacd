"""MXFP4 and sorted-row calls at the limits that their entries document."""
if __name__ == "__main__":  # `python tests/<file>.py`, as the reference runs its tests
    import sys as _sys

    import pytest as _pytest
    _sys.exit(_pytest.main([__file__, "-q"]))
import pytest
import torch

import _mxfp4 as mx
from jjjetson_ops_amd import capi
from test_gpu_mxfp4 import note

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
