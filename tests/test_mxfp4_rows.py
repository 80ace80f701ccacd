"""Which rows the MXFP4 quantizer and its inverse take from a tensor (no GPU: what the wrappers hand on)."""
if __name__ == "__main__":  # `python tests/<file>.py`, as the reference runs its tests
    import sys as _sys

    import pytest as _pytest
    _sys.exit(_pytest.main([__file__, "-q"]))
import pytest
import torch

from jjjetson_ops_amd import capi

# shape, rows, cols, the row stride: rows of a wider tensor as of its slice; values in order where it is flat, has
# rows of that length or is read as rows of another length.
CASES = [((4, 64), 4, 32, 64), ((9, 96), 4, 32, 96), ((2, 4, 64), 8, 32, 64), ((4, 64), 4, 64, 64), ((256,), 4, 64, 64),
         ((4, 64), 8, 32, 32), ((4, 64), 2, 128, 128), ((2, 2, 64), 4, 64, 64), ((1, 256), 4, 64, 64), ((8, 64), 2, 64, 64)]


@pytest.mark.parametrize("shape,rows,cols,stride", CASES)
def test_row_stride(shape, rows, cols, stride, monkeypatch):
    calls = []
    monkeypatch.setattr(capi, "_entry", lambda which, where, stream, *args: calls.append(args))
    x, q = torch.zeros(shape), torch.zeros(1024, dtype=torch.uint8)
    capi.quantize_mxfp4(x, q, rows, cols)
    assert calls.pop()[:3] == (x, capi.DTYPE_F32, stride)
    capi.dequantize_mxfp4(q, x, rows, cols)
    assert calls.pop()[1:4] == (x, capi.DTYPE_F32, stride)


def test_too_small():
    for shape in ((3, 64), (1, 100), (100,)):
        with pytest.raises(ValueError, match="x is too small"):
            capi.quantize_mxfp4(torch.zeros(shape), torch.zeros(1024, dtype=torch.uint8), 7, 32)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_wider_tensor_is_its_slice(dtype, dev):
    wide = torch.randn(37, 512, device=dev).to(dtype)
    qs = [torch.empty(capi.mxfp4_bytes(37, 224), dtype=torch.uint8, device=dev) for _ in range(2)]
    backs = [torch.full_like(wide, 9.0) for _ in range(2)]
    for x, back, q in ((wide, backs[0], qs[0]), (wide[:, :224], backs[1][:, :224], qs[1])):
        capi.quantize_mxfp4(x, q, 37, 224)
        capi.dequantize_mxfp4(q, back, 37, 224)
    assert torch.equal(*qs) and torch.equal(*backs)
