"""The MXFP4 MoE FFN where its kernels change: every tile of the gathered rows, and the routing's
launches."""
if __name__ == "__main__":  # `python tests/<file>.py`, as the reference runs its tests
    import sys as _sys

    import pytest as _pytest
    _sys.exit(_pytest.main([__file__, "-q"]))
import numpy as np
import pytest
import torch

import test_gpu_mxfp4 as base

pytestmark = pytest.mark.gpu


def _close_f16(got, exp, bound, close=base._close):
    """Within the bound for fp16 outputs: the largest value is 65504 and the step there 32, so what is
    65520 or more rounds to infinity, and what comes that far within the bound may."""
    over = (np.abs(exp) + bound >= 65520) & np.isinf(got) & (np.signbit(got) == np.signbit(exp))
    assert over[np.abs(exp) - bound >= 65520].all()
    close(np.where(over, 0.0, got), np.where(over, 0.0, exp), bound)


def _check(T, H, I, E, k, dtype, dev, monkeypatch, uneven):
    base.note(f"ffn T={T} H={H} I={I} E={E} k={k} {dtype}")
    rng = np.random.default_rng(T + H + I + E)
    mats, x, logits = base._ffn_case(rng, T, H, I, E, dev, dtype)
    if uneven:
        logits += torch.from_numpy(rng.standard_normal(E).astype(np.float32)).to(dev)
    if dtype == "f16":
        monkeypatch.setattr(base, "_close", _close_f16)
    base._check_ffn(mats, x, logits, T, H, I, E, k, dtype, dev)


# With 256 CUs, the tile of gate|up: 32, 64, 96 and 128 tokens cut along K, then whole, then 160, 192 and 256; a last
# block, a last pair of stages and tiles that are not full.
@pytest.mark.parametrize("T,H,I,E,k,dtype", [(263, 2080, 288, 4, 3, "bf16"), (100, 2048, 1024, 8, 2, "f32"),
                                             (701, 2080, 288, 4, 2, "f16"), (200, 2048, 1024, 8, 2, "bf16"),
                                             (455, 2080, 800, 4, 2, "bf16"), (701, 2080, 800, 4, 2, "f32"),
                                             (131, 544, 288, 4, 3, "f32"), (701, 544, 288, 4, 2, "bf16"),
                                             (455, 544, 800, 4, 2, "f16"), (701, 544, 800, 4, 2, "bf16"),
                                             (701, 544, 2080, 4, 2, "f32"), (601, 544, 2080, 8, 2, "bf16"),
                                             (455, 544, 2080, 8, 3, "f16")])
def test_gathered_tiles(T, H, I, E, k, dtype, dev, monkeypatch):
    """gate|up reads a route's row by its token; the stages it is compared with read sorted
    copies of the rows.  Experts of very different shares."""
    _check(T, H, I, E, k, dtype, dev, monkeypatch, True)


# 65 to 256 experts in one launch (up to 512 routes); 512 and 513, 4096 and 4097 routes.
@pytest.mark.parametrize("T,H,I,E,k,dtype", [(1, 64, 32, 128, 4, "bf16"), (64, 96, 64, 128, 8, "f32"),
                                             (17, 64, 32, 256, 8, "f16"), (30, 64, 32, 65, 17, "bf16"),
                                             (256, 64, 32, 8, 2, "bf16"), (171, 64, 32, 100, 3, "f32"),
                                             (2048, 64, 32, 32, 2, "f32"), (241, 64, 32, 32, 17, "bf16")])
def test_routing_launches(T, H, I, E, k, dtype, dev, monkeypatch):
    _check(T, H, I, E, k, dtype, dev, monkeypatch, False)
