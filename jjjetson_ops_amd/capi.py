"""ctypes binding of the C ABI (include/jjjetson_ops_amd.h) for device tensors.

These wrappers take torch device tensors (HIP memory) and launch on torch's
current stream, so ``torch.cuda.Event`` timing brackets exactly the kernels.
The shared library must have been built (``python -m jjjetson_ops_amd.build``);
loading fails loudly otherwise — there is no CPU fallback.
"""
from __future__ import annotations

import ctypes
import os
from pathlib import Path

LIB_PATH = Path(__file__).resolve().with_name("libjjjetson_ops_amd.so")

JJO_OK = 0
JJO_ERR_INVALID_ARG = 1
JJO_ERR_HIP = 2
JJO_ERR_NO_DEVICE = 3

ALGO_AUTO = 0
ALGO_GEMV = 1
ALGO_MFMA = 2
ALGO_SKINNY = 3
ALGO_SKINNY_LDS = 4
ALGO_MFMA64 = 5
ALGO_MFMA32 = 6
ALGO_MFMA_W32 = 7
KERNEL_KSLICE = 16  # + tile form 0..3 (mm_auto_kernel, mm_kernel), column tiles (grouped_auto_kernel)

QK = 32
QSUPER = 128
Q8_BLOCK_BYTES = 144
Q4_BLOCK_BYTES = 18

# Every symbol include/jjjetson_ops_amd.h declares.
EXPORTED_SYMBOLS = (
    "jjo_last_error",
    "jjo_version",
    "q8_1_output_bytes",
    "q8_1",
    "q8_1_device",
    "parse_q8_1_output",
    "mat_mul_q4_0_q8_1",
    "mat_mul_q4_0_q8_1_device",
    "mat_mul_q4_0_q8_1_f32_device",
    "mat_mul_q4_0_q8_1_device_algo",
    "mat_mul_q4_0_q8_1_block_sums_device",
    "mat_mul_q4_0_q8_1_grouped_device",
    "mat_mul_q4_0s_q8_1_grouped_device",
    "jjo_mm_auto_kernel",
    "jjo_grouped_auto_kernel",
    "jjo_grouped_kernel_device",
    "jjo_mm_kernel_device",
    "jjo_read_floor_device",
    "linear_q4_0_workspace_bytes",
    "linear_q4_0_forward_device",
    "linear_q4_0s_forward_device",
    "linear_q4_0_forward_host",
    "linear_q4_0_noalloc_max_bytes",
    "linear_q4_0_forward_device_noalloc",
    "moe_top_k_device",
    "moe_dispatch_q8_1_device",
    "moe_q4_0_gate_up_device",
    "moe_q4_0_gate_up_swiglu_q8_1_device",
    "swiglu_quantize_q8_1_device",
    "moe_combine_device",
    "moe_q4_0_ffn_workspace_bytes",
    "moe_q4_0_ffn_forward_device",
    "moe_q4_0s_ffn_forward_device",
    "q4_0_bytes",
    "quantize_q4_0_host",
    "quantize_q4_0_device",
    "safetensors_read_file_q4_0",
    "jjo_host_tensors_free",
    "jjo_host_tensors_find",
    "safetensors_write_file_q4_0",
    "safetensors_quantize_q4_0",
    "q4_0_split_bytes",
    "q4_0_to_split",
    "q4_0_from_split",
    "q4_0_to_split_device",
    "mat_mul_q4_0s_q8_1_device",
    "mat_mul_q4_0s_q8_1_f32_device",
    "mxfp4_bytes",
    "quantize_mxfp4_device",
    "dequantize_mxfp4_device",
    "mat_mul_mxfp4_device",
    "linear_mxfp4_workspace_bytes",
    "linear_mxfp4_forward_device",
    "mat_mul_mxfp4_grouped_device",
    "moe_mxfp4_gate_up_swiglu_device",
    "moe_mxfp4_ffn_workspace_bytes",
    "moe_mxfp4_ffn_forward_device",
    "moe_dispatch_rows_device",
    "moe_dispatch_rows_backward_device",
    "moe_combine_rows_device",
    "moe_combine_rows_backward_device",
    "linear_rows_workspace_bytes",
    "linear_rows_forward_device",
    "linear_rows_backward_workspace_bytes",
    "linear_rows_backward_workspace_bytes_for",
    "linear_rows_backward_device",
    "mat_mul_rows_grouped_workspace_bytes",
    "mat_mul_rows_grouped_device",
    "mat_mul_rows_grouped_backward_workspace_bytes",
    "mat_mul_rows_grouped_backward_device",
    "moe_rows_gate_up_swiglu_workspace_bytes",
    "moe_rows_gate_up_swiglu_device",
    "moe_rows_gate_up_swiglu_backward_workspace_bytes",
    "moe_rows_gate_up_swiglu_backward_workspace_bytes_for",
    "moe_rows_gate_up_swiglu_backward_device",
    "jjo_rows_kernel_device",
)

DTYPE_F32 = 0
DTYPE_F16 = 1
DTYPE_BF16 = 2

ACT_NONE = 0
ACT_RELU = 1
ACT_GELU = 2
ACT_GELU_TANH = 3
ACT_SILU = 4

MX_BLOCK_BYTES = 17

WEIGHT_DTYPE_F32 = 0
WEIGHT_DTYPE_Q4_0 = 1


class HostTensor(ctypes.Structure):
    """jjo_host_tensor (include/jjjetson_ops_amd.h)."""
    _fields_ = [
        ("name", ctypes.c_char_p),
        ("data", ctypes.c_void_p),
        ("dims", ctypes.POINTER(ctypes.c_int64)),
        ("ndim", ctypes.c_int),
        ("dtype", ctypes.c_int),
        ("nbytes", ctypes.c_int64),
    ]


class JJOError(RuntimeError):
    """A non-zero status from the C ABI."""

    def __init__(self, code: int, where: str, msg: str):
        super().__init__(f"{where}: status {code}: {msg}")
        self.code = code


_lib = None


def lib() -> ctypes.CDLL:
    global _lib
    if _lib is None:
        if not LIB_PATH.exists():
            raise ImportError(
                f"{LIB_PATH} is missing: build it with `python -m jjjetson_ops_amd.build` "
                "(there is no CPU fallback for this path)")
        L = ctypes.CDLL(str(LIB_PATH))
        vp, i64p, i32, i64 = ctypes.c_void_p, ctypes.POINTER(ctypes.c_int64), ctypes.c_int, ctypes.c_int64
        L.jjo_last_error.restype = ctypes.c_char_p
        L.jjo_last_error.argtypes = []
        L.jjo_version.restype = ctypes.c_char_p
        L.jjo_version.argtypes = []
        L.q8_1_output_bytes.restype = i64
        L.q8_1_output_bytes.argtypes = [i64p, i32]
        L.q8_1.restype = i32
        L.q8_1.argtypes = [vp, vp, i64p, i32]
        L.q8_1_device.restype = i32
        L.q8_1_device.argtypes = [vp, vp, i64p, i32, vp]
        L.parse_q8_1_output.restype = None
        L.parse_q8_1_output.argtypes = [vp, vp, vp, vp, i64]
        L.mat_mul_q4_0_q8_1.restype = i32
        L.mat_mul_q4_0_q8_1.argtypes = [vp, vp, vp, vp, i64p, i32, i32, i32]
        L.mat_mul_q4_0_q8_1_device.restype = i32
        L.mat_mul_q4_0_q8_1_device.argtypes = [vp, vp, vp, i32, i32, i32, vp]
        L.mat_mul_q4_0_q8_1_f32_device.restype = i32
        L.mat_mul_q4_0_q8_1_f32_device.argtypes = [vp, vp, vp, vp, i32, i32, i32, vp]
        L.mat_mul_q4_0_q8_1_device_algo.restype = i32
        L.mat_mul_q4_0_q8_1_device_algo.argtypes = [vp, vp, vp, i32, i32, i32, i32, vp]
        L.mat_mul_q4_0_q8_1_block_sums_device.restype = i32
        L.mat_mul_q4_0_q8_1_block_sums_device.argtypes = [vp, vp, vp, i32, i32, i32, vp]
        L.mat_mul_q4_0_q8_1_grouped_device.restype = i32
        L.mat_mul_q4_0_q8_1_grouped_device.argtypes = [vp, vp, vp, i32, vp, vp, i32, i32, i32, vp]
        L.mat_mul_q4_0s_q8_1_grouped_device.restype = i32
        L.mat_mul_q4_0s_q8_1_grouped_device.argtypes = [vp, vp, vp, i32, vp, vp, i32, i32, i32, vp]
        L.jjo_mm_auto_kernel.restype = i32
        L.jjo_mm_auto_kernel.argtypes = [i32, i32, i32, i32]
        L.jjo_grouped_auto_kernel.restype = i32
        L.jjo_grouped_auto_kernel.argtypes = [i32, i32, i32, i32]
        L.jjo_grouped_kernel_device.restype = i32
        L.jjo_grouped_kernel_device.argtypes = [vp, vp, vp, i32, vp, vp, i32, i32, i32, i32, i32, vp]
        L.jjo_mm_kernel_device.restype = i32
        L.jjo_mm_kernel_device.argtypes = [vp, vp, vp, i32, i32, i32, i32, i32, vp]
        L.jjo_read_floor_device.restype = i32
        L.jjo_read_floor_device.argtypes = [vp, i64, vp, vp]
        L.linear_q4_0_workspace_bytes.restype = i64
        L.linear_q4_0_workspace_bytes.argtypes = [i32, i32]
        L.linear_q4_0_forward_device.restype = i32
        L.linear_q4_0_forward_device.argtypes = [vp, vp, vp, vp, vp, i32, i32, i32]
        L.linear_q4_0s_forward_device.restype = i32
        L.linear_q4_0s_forward_device.argtypes = [vp, vp, vp, vp, vp, i32, i32, i32]
        L.linear_q4_0_noalloc_max_bytes.restype = i64
        L.linear_q4_0_noalloc_max_bytes.argtypes = []
        L.linear_q4_0_forward_device_noalloc.restype = i32
        L.linear_q4_0_forward_device_noalloc.argtypes = [vp, vp, vp, vp, i32, i32, i32]
        L.linear_q4_0_forward_host.restype = i32
        L.linear_q4_0_forward_host.argtypes = [vp, vp, vp, i32, i32, i32]
        L.moe_top_k_device.restype = i32
        L.moe_top_k_device.argtypes = [vp, vp, vp, vp, i32, i32, i32]
        L.moe_dispatch_q8_1_device.restype = i32
        L.moe_dispatch_q8_1_device.argtypes = [vp, vp, vp, i32, i32, i32, i32, vp, vp, vp, vp]
        L.moe_q4_0_gate_up_device.restype = i32
        L.moe_q4_0_gate_up_device.argtypes = [vp, vp, vp, vp, vp, i32, vp, i32, i32, i32]
        L.moe_q4_0_gate_up_swiglu_q8_1_device.restype = i32
        L.moe_q4_0_gate_up_swiglu_q8_1_device.argtypes = [vp, vp, vp, vp, vp, i32, vp, i32, i32, i32]
        L.swiglu_quantize_q8_1_device.restype = i32
        L.swiglu_quantize_q8_1_device.argtypes = [vp, vp, vp, vp, i32, i32]
        L.moe_combine_device.restype = i32
        L.moe_combine_device.argtypes = [vp, vp, vp, vp, vp, i32, i32, i32]
        L.moe_q4_0_ffn_workspace_bytes.restype = i64
        L.moe_q4_0_ffn_workspace_bytes.argtypes = [i32, i32, i32, i32, i32]
        L.moe_q4_0_ffn_forward_device.restype = i32
        L.moe_q4_0_ffn_forward_device.argtypes = [vp, vp, vp, vp, vp, vp, vp, i32, i32, i32, i32, i32, vp, i64]
        L.moe_q4_0s_ffn_forward_device.restype = i32
        L.moe_q4_0s_ffn_forward_device.argtypes = [vp, vp, vp, vp, vp, vp, vp, i32, i32, i32, i32, i32, vp, i64]
        L.q4_0_bytes.restype = i64
        L.q4_0_bytes.argtypes = [i64, i64]
        L.quantize_q4_0_host.restype = i32
        L.quantize_q4_0_host.argtypes = [vp, vp, i64, i64, i32]
        L.quantize_q4_0_device.restype = i32
        L.quantize_q4_0_device.argtypes = [vp, vp, vp, i64, i64]
        ht_p = ctypes.POINTER(HostTensor)
        L.safetensors_read_file_q4_0.restype = i32
        L.safetensors_read_file_q4_0.argtypes = [ctypes.c_char_p, ctypes.POINTER(ht_p), ctypes.POINTER(i32)]
        L.jjo_host_tensors_free.restype = None
        L.jjo_host_tensors_free.argtypes = [ht_p, i32]
        L.jjo_host_tensors_find.restype = ht_p
        L.jjo_host_tensors_find.argtypes = [ht_p, i32, ctypes.c_char_p]
        L.safetensors_write_file_q4_0.restype = i32
        L.safetensors_write_file_q4_0.argtypes = [ctypes.c_char_p, ht_p, i32]
        L.safetensors_quantize_q4_0.restype = i32
        L.safetensors_quantize_q4_0.argtypes = [ctypes.c_char_p, ctypes.c_char_p,
                                                ctypes.POINTER(ctypes.c_char_p), i32, i32]
        L.q4_0_split_bytes.restype = i64
        L.q4_0_split_bytes.argtypes = [i64, i64]
        L.q4_0_to_split.restype = i32
        L.q4_0_to_split.argtypes = [vp, vp, i64, i64]
        L.q4_0_from_split.restype = i32
        L.q4_0_from_split.argtypes = [vp, vp, i64, i64]
        L.q4_0_to_split_device.restype = i32
        L.q4_0_to_split_device.argtypes = [vp, vp, i32, i32, vp]
        L.mat_mul_q4_0s_q8_1_device.restype = i32
        L.mat_mul_q4_0s_q8_1_device.argtypes = [vp, vp, vp, i32, i32, i32, vp]
        L.mat_mul_q4_0s_q8_1_f32_device.restype = i32
        L.mat_mul_q4_0s_q8_1_f32_device.argtypes = [vp, vp, vp, vp, i32, i32, i32, vp]
        L.mxfp4_bytes.restype = i64
        L.mxfp4_bytes.argtypes = [i64, i64]
        L.quantize_mxfp4_device.restype = i32
        L.quantize_mxfp4_device.argtypes = [vp, vp, i32, i64, vp, i64, i64]
        L.dequantize_mxfp4_device.restype = i32
        L.dequantize_mxfp4_device.argtypes = [vp, vp, vp, i32, i64, i64, i64]
        L.mat_mul_mxfp4_device.restype = i32
        L.mat_mul_mxfp4_device.argtypes = [vp, vp, vp, i32, i32, i32, i32, vp]
        L.linear_mxfp4_workspace_bytes.restype = i64
        L.linear_mxfp4_workspace_bytes.argtypes = [i32, i32]
        L.linear_mxfp4_forward_device.restype = i32
        L.linear_mxfp4_forward_device.argtypes = [vp, vp, vp, i32, vp, vp, i32, i32, i32, i32]
        L.mat_mul_mxfp4_grouped_device.restype = i32
        L.mat_mul_mxfp4_grouped_device.argtypes = [vp, vp, vp, i32, vp, vp, i32, i32, i32, i32, vp]
        L.moe_mxfp4_gate_up_swiglu_device.restype = i32
        L.moe_mxfp4_gate_up_swiglu_device.argtypes = [vp, vp, vp, vp, vp, i32, vp, i32, i32, i32]
        L.moe_mxfp4_ffn_workspace_bytes.restype = i64
        L.moe_mxfp4_ffn_workspace_bytes.argtypes = [i32, i32, i32, i32, i32]
        L.moe_mxfp4_ffn_forward_device.restype = i32
        L.moe_mxfp4_ffn_forward_device.argtypes = [vp, vp, vp, vp, vp, vp, vp, i32, i32, i32, i32, i32, i32, vp, i64]
        L.moe_dispatch_rows_device.restype = i32
        L.moe_dispatch_rows_device.argtypes = [vp, vp, vp, i32, i32, i32, i32, i32, vp, vp, vp, vp]
        L.moe_dispatch_rows_backward_device.restype = i32
        L.moe_dispatch_rows_backward_device.argtypes = [vp, vp, i32, vp, vp, i32, i32, i32]
        L.moe_combine_rows_device.restype = i32
        L.moe_combine_rows_device.argtypes = [vp, vp, i32, vp, vp, vp, i32, i32, i32]
        L.moe_combine_rows_backward_device.restype = i32
        L.moe_combine_rows_backward_device.argtypes = [vp, vp, vp, i32, vp, vp, vp, vp, i32, i32, i32]
        L.jjo_rows_kernel_device.restype = i32
        L.jjo_rows_kernel_device.argtypes = [vp, i32, i32, i32, i32, vp, vp, vp, vp, i32, vp, vp, i32, i32, i32, vp, i64]
        for name in ("linear_rows", "linear_rows_backward"):
            f = getattr(L, name + "_workspace_bytes")
            f.restype, f.argtypes = i64, [i32, i32, i32, i32]
        for name in ("mat_mul_rows_grouped", "mat_mul_rows_grouped_backward", "moe_rows_gate_up_swiglu",
                     "moe_rows_gate_up_swiglu_backward"):
            f = getattr(L, name + "_workspace_bytes")
            f.restype, f.argtypes = i64, [i32, i32, i32, i32, i32]
        for name in ("linear_rows_backward", "moe_rows_gate_up_swiglu_backward"):
            f = getattr(L, name + "_workspace_bytes_for")
            f.restype, f.argtypes = i64, [i32, i32, i32, i32, i32, i32]
        L.linear_rows_forward_device.restype = i32
        L.linear_rows_forward_device.argtypes = [vp, vp, i64, vp, vp, vp, i64, vp, i64, vp, i32, i32, i32, i32, i32,
                                                 vp, i64]
        L.linear_rows_backward_device.restype = i32
        L.linear_rows_backward_device.argtypes = [vp, vp, i64, vp, i64, vp, vp, vp, i64, vp, vp, i32, i32, i32, i32,
                                                  i32, i32, vp, i64]
        L.mat_mul_rows_grouped_device.restype = i32
        L.mat_mul_rows_grouped_device.argtypes = [vp, vp, vp, vp, i32, vp, i32, i32, i32, i32, vp, i64]
        L.mat_mul_rows_grouped_backward_device.restype = i32
        L.mat_mul_rows_grouped_backward_device.argtypes = [vp, vp, vp, vp, vp, i32, vp, vp, i32, i32, i32, i32, i32,
                                                           vp, i64]
        L.moe_rows_gate_up_swiglu_device.restype = i32
        L.moe_rows_gate_up_swiglu_device.argtypes = [vp, vp, vp, vp, vp, i32, vp, vp, i32, i32, i32, i32, vp, i64]
        L.moe_rows_gate_up_swiglu_backward_device.restype = i32
        L.moe_rows_gate_up_swiglu_backward_device.argtypes = [vp, vp, vp, vp, vp, vp, vp, i32, vp, vp, vp, i32, i32,
                                                              i32, i32, i32, vp, i64]
        _lib = L
    return _lib


def _check(rc: int, where: str) -> None:
    if rc != JJO_OK:
        raise JJOError(rc, where, lib().jjo_last_error().decode(errors="replace"))


def _dims(dims) -> tuple:
    d = (ctypes.c_int64 * len(dims))(*[int(v) for v in dims])
    return d, len(dims)


def version() -> str:
    return lib().jjo_version().decode()


def q8_1_output_bytes(dims) -> int:
    d, n = _dims(dims)
    return int(lib().q8_1_output_bytes(d, n))


_torch = None


def _current_stream() -> int:
    """The current torch stream of the current device, as an address."""
    global _torch
    if _torch is None:
        import torch
        _torch = torch
    return _torch._C._cuda_getCurrentRawStream(_torch.cuda.current_device())


def _stream(stream) -> int:
    if stream is None:
        return _current_stream()
    if isinstance(stream, int):
        return stream
    return stream.cuda_stream


def _dev(t, name: str) -> int:
    if not t.is_cuda:
        raise ValueError(f"{name} must be a device tensor")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t.data_ptr()


_linear_native = None


def _linear(split: bool, x, w, y, in_features, out_features, num_tokens, ws, stream) -> int:
    """The two linear entries through the native binding (csrc/bind_linear.cpp)."""
    global _linear_native
    if _linear_native is None:
        lib()  # the same loud failure where nothing is built
        from ._linear import linear
        _linear_native = linear
    rc = _linear_native(split, _current_stream, x, w, y, in_features, out_features, num_tokens, ws, stream)
    if rc is None:  # an argument that only ctypes converts (a c_int, _as_parameter_) or refuses (ArgumentError)
        fn = lib().linear_q4_0s_forward_device if split else lib().linear_q4_0_forward_device
        rc = fn(_stream(stream), None if ws is None else _dev(ws, "ws"), _dev(x, "x"), _dev(w, "w"), _dev(y, "y"),
                in_features, out_features, num_tokens)
    return rc


def quantize_q8_1(x, out, dims=None, stream=None) -> None:
    """Device quantize: x fp32 (dim0 = K fastest), out uint8 of q8_1_output_bytes(dims)."""
    import torch
    if x.dtype != torch.float32 or out.dtype != torch.uint8:
        raise ValueError("x must be float32 and out uint8")
    if dims is None:
        dims = [x.shape[-1], x.numel() // x.shape[-1]]
    need = q8_1_output_bytes(dims)
    if need < 0:
        raise ValueError(f"invalid dims {dims}")
    if out.numel() < need or x.numel() < int(__import__("math").prod(dims)):
        raise ValueError("buffer too small for dims")
    d, n = _dims(dims)
    _check(lib().q8_1_device(_dev(x, "x"), _dev(out, "out"), d, n, _stream(stream)), "q8_1_device")


def mat_mul(w, xq, y, K: int, N: int, M: int, algo: int = ALGO_AUTO, stream=None) -> None:
    """y[M, N] (fp32) = Q4_0 w [N, K/32 blocks] x Q8_1 xq (quantizer layout, M tokens)."""
    import torch
    if y.dtype != torch.float32:
        raise ValueError("y must be float32")
    if w.numel() * w.element_size() < N * (K // QK) * Q4_BLOCK_BYTES:
        raise ValueError("weight buffer too small")
    if xq.numel() * xq.element_size() < M * (K // QSUPER) * Q8_BLOCK_BYTES:
        raise ValueError("Q8_1 buffer too small")
    if y.numel() < M * N:
        raise ValueError("output buffer too small")
    _check(lib().mat_mul_q4_0_q8_1_device_algo(_dev(w, "w"), _dev(xq, "xq"), _dev(y, "y"), K, N, M, algo,
                                               _stream(stream)), "mat_mul_q4_0_q8_1_device")


def mat_mul_f32(w, x, xq, y, K: int, N: int, M: int, stream=None) -> None:
    """Quantize fp32 x [M, K] (into xq, may be None when M == 1) and y[M, N] = W . x."""
    import torch
    if x.dtype != torch.float32 or y.dtype != torch.float32:
        raise ValueError("x and y must be float32")
    if x.numel() < M * K or y.numel() < M * N:
        raise ValueError("x or y too small")
    if xq is not None and xq.numel() * xq.element_size() < M * (K // QSUPER) * Q8_BLOCK_BYTES:
        raise ValueError("Q8_1 workspace too small")
    if w.numel() * w.element_size() < N * (K // QK) * Q4_BLOCK_BYTES:
        raise ValueError("weight buffer too small")
    xqp = _dev(xq, "xq") if xq is not None else ctypes.c_void_p(0)
    _check(lib().mat_mul_q4_0_q8_1_f32_device(_dev(w, "w"), _dev(x, "x"), xqp, _dev(y, "y"), K, N, M,
                                              _stream(stream)), "mat_mul_q4_0_q8_1_f32_device")


# ---------------------------------------------------------------- split weight layout
def q4_0_to_split_host(w, nrows: int, ncols_k: int):
    """Host repack: uint8 block_q4_0 rows -> split layout (a new uint8 ndarray)."""
    import numpy as np
    w = np.ascontiguousarray(w, dtype=np.uint8).reshape(-1)
    n = int(lib().q4_0_split_bytes(nrows, ncols_k))
    if n < 0 or w.size < n:
        raise ValueError("invalid shape or weight buffer too small")
    out = np.empty(n, np.uint8)
    _check(lib().q4_0_to_split(w.ctypes.data, out.ctypes.data, nrows, ncols_k), "q4_0_to_split")
    return out


def q4_0_from_split_host(ws, nrows: int, ncols_k: int):
    """Host inverse repack: split layout -> block_q4_0 rows (a new uint8 ndarray)."""
    import numpy as np
    ws = np.ascontiguousarray(ws, dtype=np.uint8).reshape(-1)
    n = int(lib().q4_0_split_bytes(nrows, ncols_k))
    if n < 0 or ws.size < n:
        raise ValueError("invalid shape or weight buffer too small")
    out = np.empty(n, np.uint8)
    _check(lib().q4_0_from_split(ws.ctypes.data, out.ctypes.data, nrows, ncols_k), "q4_0_from_split")
    return out


def q4_0_to_split(w, out, nrows: int, ncols_k: int, stream=None) -> None:
    """Device repack of block_q4_0 rows (w) into the split layout (out, 16-byte aligned)."""
    n = nrows * (ncols_k // QK) * Q4_BLOCK_BYTES
    if w.numel() * w.element_size() < n or out.numel() * out.element_size() < n:
        raise ValueError("buffer too small")
    _check(lib().q4_0_to_split_device(_dev(w, "w"), _dev(out, "out"), nrows, ncols_k, _stream(stream)),
           "q4_0_to_split_device")


def mat_mul_split(ws, xq, y, K: int, N: int, M: int, stream=None) -> None:
    """y[M, N] = split-layout Q4_0 ws x Q8_1 xq (quantizer layout)."""
    if ws.numel() * ws.element_size() < N * (K // QK) * Q4_BLOCK_BYTES:
        raise ValueError("weight buffer too small")
    if xq.numel() * xq.element_size() < M * (K // QSUPER) * Q8_BLOCK_BYTES or y.numel() < M * N:
        raise ValueError("Q8_1 or output buffer too small")
    _check(lib().mat_mul_q4_0s_q8_1_device(_dev(ws, "w"), _dev(xq, "xq"), _dev(y, "y"), K, N, M, _stream(stream)),
           "mat_mul_q4_0s_q8_1_device")


def mat_mul_split_f32(ws, x, xq, y, K: int, N: int, M: int, stream=None) -> None:
    """Quantize fp32 x [M, K] (into xq, may be None when M == 1) and y = split W . x."""
    import torch
    if x.dtype != torch.float32 or y.dtype != torch.float32:
        raise ValueError("x and y must be float32")
    if x.numel() < M * K or y.numel() < M * N:
        raise ValueError("x or y too small")
    if xq is not None and xq.numel() * xq.element_size() < M * (K // QSUPER) * Q8_BLOCK_BYTES:
        raise ValueError("Q8_1 workspace too small")
    if ws.numel() * ws.element_size() < N * (K // QK) * Q4_BLOCK_BYTES:
        raise ValueError("weight buffer too small")
    xqp = _dev(xq, "xq") if xq is not None else ctypes.c_void_p(0)
    _check(lib().mat_mul_q4_0s_q8_1_f32_device(_dev(ws, "w"), _dev(x, "x"), xqp, _dev(y, "y"), K, N, M,
                                               _stream(stream)), "mat_mul_q4_0s_q8_1_f32_device")


def block_sums(w, xq, out, K: int, N: int, M: int, stream=None) -> None:
    """int32 out[M, N, K/32] per-block integer dots."""
    import torch
    if out.dtype != torch.int32 or out.numel() < M * N * (K // QK):
        raise ValueError("out must be int32 with M*N*K/32 elements")
    _check(lib().mat_mul_q4_0_q8_1_block_sums_device(_dev(w, "w"), _dev(xq, "xq"), _dev(out, "out"), K, N, M,
                                                     _stream(stream)), "block_sums")


def grouped_mat_mul(w, xq, expert_offsets, y, K: int, N: int, n_routes: int, route_dst=None,
                    stream=None, split: bool = False) -> None:
    """One-launch MoE expert GEMM over routes sorted by expert (see the C header);
    split: w holds the stacked experts repacked into the split layout."""
    _grouped(w, xq, expert_offsets, y, K, N, n_routes, route_dst, stream, split, 0)


def grouped_kernel(w, xq, expert_offsets, y, K: int, N: int, n_routes: int, kernel: int, route_dst=None,
                   stream=None, split: bool = False) -> None:
    """jjo_grouped_kernel_device: grouped_mat_mul on one of the kernels that grouped_auto_kernel
    names (but ALGO_GEMV)."""
    _grouped(w, xq, expert_offsets, y, K, N, n_routes, route_dst, stream, split, kernel)


def _grouped(w, xq, expert_offsets, y, K, N, n_routes, route_dst, stream, split, kernel) -> None:
    import torch
    n_experts = expert_offsets.numel() - 1
    if expert_offsets.dtype != torch.int32:
        raise ValueError("expert_offsets must be int32")
    if route_dst is not None and (route_dst.dtype != torch.int32 or route_dst.numel() < n_routes):
        raise ValueError("route_dst must be int32 with n_routes entries")
    if w.numel() * w.element_size() < n_experts * N * (K // QK) * Q4_BLOCK_BYTES:
        raise ValueError("weight buffer too small for all experts")
    rd = _dev(route_dst, "route_dst") if route_dst is not None else ctypes.c_void_p(0)
    if kernel:
        _check(lib().jjo_grouped_kernel_device(_dev(w, "w"), _dev(xq, "xq"), _dev(expert_offsets, "offsets"), n_experts,
                                               rd, _dev(y, "y"), K, N, n_routes, int(split), kernel, _stream(stream)),
               "jjo_grouped_kernel_device")
        return
    fn = lib().mat_mul_q4_0s_q8_1_grouped_device if split else lib().mat_mul_q4_0_q8_1_grouped_device
    _check(fn(_dev(w, "w"), _dev(xq, "xq"), _dev(expert_offsets, "offsets"), n_experts, rd, _dev(y, "y"), K, N,
              n_routes, _stream(stream)), "grouped_mat_mul")


def mm_auto_kernel(K: int, N: int, M: int, split: bool = False) -> int:
    """jjo_mm_auto_kernel: the kernel the matmul entries run for this shape (ALGO_* or
    KERNEL_KSLICE + tile form)."""
    k = int(lib().jjo_mm_auto_kernel(K, N, M, int(split)))
    if k < 0:
        _check(JJO_ERR_INVALID_ARG, "jjo_mm_auto_kernel")
    return k


def grouped_auto_kernel(K: int, N: int, n_routes: int, n_experts: int) -> int:
    """jjo_grouped_auto_kernel: ALGO_GEMV, ALGO_MFMA or KERNEL_KSLICE + column tiles."""
    k = int(lib().jjo_grouped_auto_kernel(K, N, n_routes, n_experts))
    if k < 0:
        _check(JJO_ERR_INVALID_ARG, "jjo_grouped_auto_kernel")
    return k


def mm_kernel(w, xq, y, K: int, N: int, M: int, kernel: int, split: bool = False, stream=None) -> None:
    """jjo_mm_kernel_device: mat_mul / mat_mul_split on a chosen tiled or K-sliced kernel."""
    import torch
    if y.dtype != torch.float32:
        raise ValueError("y must be float32")
    if w.numel() * w.element_size() < N * (K // QK) * Q4_BLOCK_BYTES:
        raise ValueError("weight buffer too small")
    if xq.numel() * xq.element_size() < M * (K // QSUPER) * Q8_BLOCK_BYTES:
        raise ValueError("Q8_1 buffer too small")
    if y.numel() < M * N:
        raise ValueError("output buffer too small")
    _check(lib().jjo_mm_kernel_device(_dev(w, "w"), _dev(xq, "xq"), _dev(y, "y"), K, N, M, int(split), kernel,
                                      _stream(stream)), "jjo_mm_kernel_device")


def read_floor(src, nbytes: int, out, stream=None) -> None:
    """jjo_read_floor_device: one plain read of nbytes of a device tensor."""
    _check(lib().jjo_read_floor_device(_dev(src, "src"), int(nbytes), _dev(out, "out"), _stream(stream)),
           "jjo_read_floor_device")


def parse_q8_1(raw, n_blocks: int):
    """Host parse through the C ABI: returns (qs int8[n,128], d f32[n,4], s f32[n,4])."""
    import numpy as np
    raw = np.ascontiguousarray(raw, dtype=np.uint8)
    if raw.size < n_blocks * Q8_BLOCK_BYTES:
        raise ValueError("raw buffer too small")
    qs = np.empty((n_blocks, 128), np.int8)
    d = np.empty((n_blocks, 4), np.float32)
    s = np.empty((n_blocks, 4), np.float32)
    lib().parse_q8_1_output(raw.ctypes.data, qs.ctypes.data, d.ctypes.data, s.ctypes.data, n_blocks)
    return qs, d, s


# ---------------------------------------------------------------- engine linear
def linear_q4_0(x, w, y, in_features: int, out_features: int, num_tokens: int, ws=None, stream=None) -> None:
    """linear_q4_0_forward_device: y [T, out] = x [T, in] . dequant(w [out, in/32 blocks]).T"""
    rc = _linear(False, x, w, y, in_features, out_features, num_tokens, ws, stream)
    if rc != JJO_OK:
        _check(rc, "linear_q4_0_forward_device")


def linear_q4_0_split(x, ws_split, y, in_features: int, out_features: int, num_tokens: int, ws=None,
                      stream=None) -> None:
    """linear_q4_0s_forward_device: linear_q4_0 on weights repacked into the split layout."""
    rc = _linear(True, x, ws_split, y, in_features, out_features, num_tokens, ws, stream)
    if rc != JJO_OK:
        _check(rc, "linear_q4_0s_forward_device")


def linear_q4_0_noalloc(x, w, y, in_features: int, out_features: int, num_tokens: int, stream=None) -> None:
    """linear_q4_0_forward_device_noalloc: as linear_q4_0 with the library's static
    Q8_1 buffer instead of a workspace (calls on one device must not overlap)."""
    _check(lib().linear_q4_0_forward_device_noalloc(_stream(stream), _dev(x, "x"), _dev(w, "w"), _dev(y, "y"),
                                                    in_features, out_features, num_tokens),
           "linear_q4_0_forward_device_noalloc")


def linear_q4_0_noalloc_max_bytes() -> int:
    return int(lib().linear_q4_0_noalloc_max_bytes())


def linear_q4_0_workspace_bytes(in_features: int, num_tokens: int) -> int:
    return int(lib().linear_q4_0_workspace_bytes(in_features, num_tokens))


# ---------------------------------------------------------------- MoE FFN
def moe_top_k(logits, weights, ids, num_tokens: int, num_experts: int, top_k: int, stream=None) -> None:
    _check(lib().moe_top_k_device(_stream(stream), _dev(logits, "logits"), _dev(weights, "weights"),
                                  _dev(ids, "ids"), num_tokens, num_experts, top_k), "moe_top_k_device")


def moe_dispatch(ids, offsets, src_route, dst_of_route, num_tokens: int, top_k: int, hidden: int,
                 num_experts: int, xq=None, xq_perm=None, stream=None) -> None:
    _check(lib().moe_dispatch_q8_1_device(_stream(stream), _dev(ids, "ids"), None if xq is None else _dev(xq, "xq"),
                                          num_tokens, top_k, hidden, num_experts, _dev(offsets, "offsets"),
                                          _dev(src_route, "src_route"), _dev(dst_of_route, "dst_of_route"),
                                          None if xq_perm is None else _dev(xq_perm, "xq_perm")),
           "moe_dispatch_q8_1_device")


def moe_gate_up(w_gate, w_up, xq_perm, offsets, num_experts: int, gate_up, hidden: int, inter: int,
                n_routes: int, stream=None) -> None:
    _check(lib().moe_q4_0_gate_up_device(_stream(stream), _dev(w_gate, "w_gate"), _dev(w_up, "w_up"),
                                         _dev(xq_perm, "xq_perm"), _dev(offsets, "offsets"), num_experts,
                                         _dev(gate_up, "gate_up"), hidden, inter, n_routes),
           "moe_q4_0_gate_up_device")


def moe_gate_up_swiglu(w_gate, w_up, xq_perm, offsets, num_experts: int, mid_q, hidden: int, inter: int,
                       n_routes: int, stream=None) -> None:
    _check(lib().moe_q4_0_gate_up_swiglu_q8_1_device(_stream(stream), _dev(w_gate, "w_gate"), _dev(w_up, "w_up"),
                                                     _dev(xq_perm, "xq_perm"), _dev(offsets, "offsets"), num_experts,
                                                     _dev(mid_q, "mid_q"), hidden, inter, n_routes),
           "moe_q4_0_gate_up_swiglu_q8_1_device")


def swiglu_quantize(gate_up, mid_q, rows: int, inter: int, mid_f32=None, stream=None) -> None:
    _check(lib().swiglu_quantize_q8_1_device(_stream(stream), _dev(gate_up, "gate_up"), _dev(mid_q, "mid_q"),
                                             None if mid_f32 is None else _dev(mid_f32, "mid_f32"), rows, inter),
           "swiglu_quantize_q8_1_device")


def moe_combine(expert_out, dst_of_route, weights, y, num_tokens: int, hidden: int, top_k: int,
                stream=None) -> None:
    _check(lib().moe_combine_device(_stream(stream), _dev(expert_out, "expert_out"),
                                    _dev(dst_of_route, "dst_of_route"), _dev(weights, "weights"), _dev(y, "y"),
                                    num_tokens, hidden, top_k), "moe_combine_device")


def moe_ffn_workspace_bytes(num_tokens: int, hidden: int, inter: int, num_experts: int, top_k: int) -> int:
    return int(lib().moe_q4_0_ffn_workspace_bytes(num_tokens, hidden, inter, num_experts, top_k))


def moe_ffn(x, logits, w_gate, w_up, w_down, y, num_tokens: int, hidden: int, inter: int, num_experts: int,
            top_k: int, ws, stream=None, split: bool = False) -> None:
    """The Q4_0 MoE FFN; split: the three expert weight buffers are in the split layout."""
    fn = lib().moe_q4_0s_ffn_forward_device if split else lib().moe_q4_0_ffn_forward_device
    _check(fn(_stream(stream), _dev(x, "x"), _dev(logits, "logits"), _dev(w_gate, "w_gate"), _dev(w_up, "w_up"),
              _dev(w_down, "w_down"), _dev(y, "y"), num_tokens, hidden, inter, num_experts, top_k, _dev(ws, "ws"),
              ws.numel() * ws.element_size()),
           "moe_q4_0s_ffn_forward_device" if split else "moe_q4_0_ffn_forward_device")


# ---------------------------------------------------------------- MXFP4 and sorted rows
# The entries of csrc/bind_linear.cpp by their places in its table.
(_QUANTIZE, _DEQUANTIZE, _MAT_MUL, _LINEAR, _GROUPED, _GATE_UP, _FFN, _DISPATCH, _DISPATCH_BACKWARD, _COMBINE,
 _COMBINE_BACKWARD, _LINEAR_ROWS, _LINEAR_ROWS_BACKWARD, _ROWS_GROUPED, _ROWS_GROUPED_BACKWARD, _ROWS_GATE_UP,
 _ROWS_GATE_UP_BACKWARD) = range(17)
_entry_native = None
_dtypes = None


def _entry(which: int, where: str, stream, *args) -> None:
    """A C entry through the native binding: tensors must be contiguous and on the current device."""
    global _entry_native
    if _entry_native is None:
        lib()  # the same loud failure where nothing is built
        from ._linear import entry
        _entry_native = entry
    rc = _entry_native(which, _stream_of, _current_device, stream, *args)
    if rc != JJO_OK:
        _check(rc, where)


def _current_device() -> int:
    return _torch.cuda.current_device()


def _stream_of(device: int) -> int:
    return _torch._C._cuda_getCurrentRawStream(device)


def _load_torch() -> None:
    global _dtypes, _torch
    import torch
    _torch = torch
    _dtypes = {torch.float32: DTYPE_F32, torch.float16: DTYPE_F16, torch.bfloat16: DTYPE_BF16}


def _dtype(t, name: str) -> int:
    """JJO_DTYPE_* of a float32, float16 or bfloat16 tensor."""
    if _dtypes is None:
        _load_torch()
    d = _dtypes.get(t.dtype)
    if d is None:
        raise ValueError(f"{name} must be float32, float16 or bfloat16")
    return d


def _same_dtype(name: str, d: int, t) -> None:
    if _dtypes.get(t.dtype) != d:
        raise ValueError(f"{name} must have the dtype of the other rows")


def _room(name: str, t, n: int) -> None:
    """t holds at least n elements."""
    if t.numel() < n:
        raise ValueError(f"{name} is too small: {t.numel()} elements, need {n}")


def _mx_room(name: str, t, rows: int, cols: int) -> None:
    """t holds a [rows, cols] MXFP4 matrix (an invalid shape is the entry's to refuse)."""
    if t.numel() * t.element_size() < rows * (cols // QK) * MX_BLOCK_BYTES:
        raise ValueError(f"{name} is too small for a [{rows}, {cols}] MXFP4 matrix")


def _typed(name: str, t, dtype, n: int) -> None:
    if t.dtype != dtype or t.numel() < n:
        raise ValueError(f"{name} must be {dtype} with {n} elements")


def _rows_of(t, name: str, rows: int, cols: int):
    """(argument, row stride) of rows x cols values: a contiguous tensor, or a 2-D one whose
    rows are contiguous.  The first cols values of the tensor's rows where it has that many rows of
    more, as of a slice of it; else its values in order."""
    if t.is_contiguous():
        if t.dim() > 1 and (width := t.shape[-1]) > cols and t.numel() >= rows * width:
            return t, width
        _room(name, t, rows * cols)
        return t, cols
    if t.dim() != 2 or t.stride(1) != 1 or t.shape[0] < rows or t.shape[1] < cols or (rows > 1 and t.stride(0) < cols):
        raise ValueError(f"{name} must be contiguous, or [rows, cols] with contiguous rows that do not overlap")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a device tensor")
    if t.get_device() != _current_device():
        raise ValueError(f"{name} is on device {t.get_device()}, the current device is {_current_device()}")
    return t.data_ptr(), t.stride(0)


def mxfp4_bytes(rows: int, cols: int) -> int:
    """Bytes of a [rows, cols] MXFP4 matrix; -1 if invalid."""
    return int(lib().mxfp4_bytes(rows, cols))


def quantize_mxfp4(x, out, rows: int, cols: int, stream=None) -> None:
    """out = MXFP4 of x [rows, cols] (float32, float16 or bfloat16; rows may be strided or longer)."""
    d = _dtype(x, "x")
    p, row_stride = _rows_of(x, "x", rows, cols)
    _mx_room("out", out, rows, cols)
    _entry(_QUANTIZE, "quantize_mxfp4_device", stream, p, d, row_stride, out, rows, cols)


def dequantize_mxfp4(q, y, rows: int, cols: int, stream=None) -> None:
    """y [rows, cols] (float32, float16 or bfloat16; rows may be strided or longer) = the values of q."""
    d = _dtype(y, "y")
    p, row_stride = _rows_of(y, "y", rows, cols)
    _mx_room("q", q, rows, cols)
    _entry(_DEQUANTIZE, "dequantize_mxfp4_device", stream, q, p, d, row_stride, rows, cols)


def mat_mul_mxfp4(w, xq, y, K: int, N: int, M: int, stream=None) -> None:
    """y[M, N] = MXFP4 xq [M, K] . MXFP4 w [N, K]^T."""
    d = _dtype(y, "y")
    _room("y", y, M * N)
    _mx_room("w", w, N, K)
    _mx_room("xq", xq, M, K)
    _entry(_MAT_MUL, "mat_mul_mxfp4_device", stream, w, xq, y, d, K, N, M)


def linear_mxfp4_workspace_bytes(in_features: int, num_tokens: int) -> int:
    return int(lib().linear_mxfp4_workspace_bytes(in_features, num_tokens))


def linear_mxfp4(x, w, y, in_features: int, out_features: int, num_tokens: int, ws=None, stream=None) -> None:
    """linear_mxfp4_forward_device: y [T, out] = MXFP4(x [T, in]) . w [out, in]^T; x and y in
    float32, float16 or bfloat16, ws of linear_mxfp4_workspace_bytes."""
    dx, dy = _dtype(x, "x"), _dtype(y, "y")
    _room("x", x, num_tokens * in_features)
    _room("y", y, num_tokens * out_features)
    _mx_room("w", w, out_features, in_features)
    if ws is not None and ws.numel() * ws.element_size() < lib().linear_mxfp4_workspace_bytes(in_features, num_tokens):
        raise ValueError("ws is smaller than linear_mxfp4_workspace_bytes")
    _entry(_LINEAR, "linear_mxfp4_forward_device", stream, ws, x, dx, w, y, dy, in_features, out_features, num_tokens)


def grouped_mat_mul_mxfp4(w, xq, expert_offsets, y, K: int, N: int, n_routes: int, route_dst=None,
                          stream=None) -> None:
    """mat_mul_mxfp4_grouped_device: rows sorted by expert times their experts' weights.  route_dst, where
    given, names rows of y; they are the caller's to keep inside it."""
    d = _dtype(y, "y")
    n_experts = expert_offsets.numel() - 1
    _typed("expert_offsets", expert_offsets, _torch.int32, 2)
    if route_dst is not None:
        _typed("route_dst", route_dst, _torch.int32, n_routes)
    _room("y", y, N if route_dst is not None else n_routes * N)
    _mx_room("w", w, n_experts * N, K)
    _mx_room("xq", xq, n_routes, K)
    _entry(_GROUPED, "mat_mul_mxfp4_grouped_device", stream, w, xq, expert_offsets, n_experts, route_dst, y, d, K, N,
           n_routes)


def moe_gate_up_swiglu_mxfp4(w_gate, w_up, xq_perm, offsets, num_experts: int, mid_q, hidden: int, inter: int,
                             n_routes: int, stream=None) -> None:
    """mid_q [n_routes, inter] = MXFP4 of silu(x . w_gate) * (x . w_up) of rows sorted by expert."""
    _mx_room("w_gate", w_gate, num_experts * inter, hidden)
    _mx_room("w_up", w_up, num_experts * inter, hidden)
    _mx_room("xq_perm", xq_perm, n_routes, hidden)
    _mx_room("mid_q", mid_q, n_routes, inter)
    if _dtypes is None:
        _load_torch()
    _typed("offsets", offsets, _torch.int32, num_experts + 1)
    _entry(_GATE_UP, "moe_mxfp4_gate_up_swiglu_device", stream, w_gate, w_up, xq_perm, offsets, num_experts, mid_q,
           hidden, inter, n_routes)


def moe_ffn_mxfp4_workspace_bytes(num_tokens: int, hidden: int, inter: int, num_experts: int, top_k: int) -> int:
    return int(lib().moe_mxfp4_ffn_workspace_bytes(num_tokens, hidden, inter, num_experts, top_k))


def moe_ffn_mxfp4(x, logits, w_gate, w_up, w_down, y, num_tokens: int, hidden: int, inter: int, num_experts: int,
                  top_k: int, ws, stream=None) -> None:
    """The MoE FFN with MXFP4 experts: x and y [T, hidden] of one dtype, logits float32 [T, E]."""
    d = _dtype(x, "x")
    _same_dtype("y", d, y)
    _room("x", x, num_tokens * hidden)
    _room("y", y, num_tokens * hidden)
    _typed("logits", logits, _torch.float32, num_tokens * num_experts)
    _mx_room("w_gate", w_gate, num_experts * inter, hidden)
    _mx_room("w_up", w_up, num_experts * inter, hidden)
    _mx_room("w_down", w_down, num_experts * hidden, inter)
    _entry(_FFN, "moe_mxfp4_ffn_forward_device", stream, x, logits, w_gate, w_up, w_down, y, d, num_tokens, hidden,
           inter, num_experts, top_k, ws, ws.numel() * ws.element_size())


def moe_dispatch_rows(ids, x, x_sorted, offsets, src_route, dst_of_route, num_tokens: int, top_k: int, hidden: int,
                      num_experts: int, stream=None) -> None:
    """Rows of x [T, hidden] to their experts: x_sorted[p] = x[src_route[p] // top_k], and the
    tables; a route with an id outside [0, num_experts) is dropped (dst_of_route -1)."""
    d = _dtype(x, "x")
    _same_dtype("x_sorted", d, x_sorted)
    r = num_tokens * top_k
    i32 = _torch.int32
    _typed("ids", ids, i32, r)
    _typed("offsets", offsets, i32, num_experts + 1)
    _typed("src_route", src_route, i32, r)
    _typed("dst_of_route", dst_of_route, i32, r)
    _room("x", x, num_tokens * hidden)
    _room("x_sorted", x_sorted, r * hidden)
    _entry(_DISPATCH, "moe_dispatch_rows_device", stream, ids, x, d, num_tokens, top_k, hidden, num_experts, offsets,
           src_route, dst_of_route, x_sorted)


def moe_dispatch_rows_backward(grad_sorted, dst_of_route, grad_x, num_tokens: int, hidden: int, top_k: int,
                               stream=None) -> None:
    """grad_x [T, hidden] = the sum of each token's sorted rows of grad_sorted."""
    d = _dtype(grad_sorted, "grad_sorted")
    _same_dtype("grad_x", d, grad_x)
    _typed("dst_of_route", dst_of_route, _torch.int32, num_tokens * top_k)
    _room("grad_sorted", grad_sorted, num_tokens * top_k * hidden)
    _room("grad_x", grad_x, num_tokens * hidden)
    _entry(_DISPATCH_BACKWARD, "moe_dispatch_rows_backward_device", stream, grad_sorted, d, dst_of_route, grad_x,
           num_tokens, hidden, top_k)


def moe_combine_rows(expert_out, dst_of_route, weights, y, num_tokens: int, hidden: int, top_k: int,
                     stream=None) -> None:
    """y [T, hidden] = sum over k of weights[t, k] * expert_out[dst_of_route[t, k]]."""
    d = _dtype(expert_out, "expert_out")
    _same_dtype("y", d, y)
    _typed("dst_of_route", dst_of_route, _torch.int32, num_tokens * top_k)
    _typed("weights", weights, _torch.float32, num_tokens * top_k)
    _room("expert_out", expert_out, num_tokens * top_k * hidden)
    _room("y", y, num_tokens * hidden)
    _entry(_COMBINE, "moe_combine_rows_device", stream, expert_out, d, dst_of_route, weights, y, num_tokens, hidden,
           top_k)


def moe_combine_rows_backward(grad_y, expert_out, dst_of_route, weights, grad_expert_out, grad_weights,
                              num_tokens: int, hidden: int, top_k: int, stream=None) -> None:
    """The combine's gradients: grad_expert_out[dst] = weight * grad_y[t], grad_weights[t, k] = <grad_y[t], row>."""
    d = _dtype(grad_y, "grad_y")
    _same_dtype("expert_out", d, expert_out)
    _same_dtype("grad_expert_out", d, grad_expert_out)
    r = num_tokens * top_k
    _typed("dst_of_route", dst_of_route, _torch.int32, r)
    _typed("weights", weights, _torch.float32, r)
    _typed("grad_weights", grad_weights, _torch.float32, r)
    _room("grad_y", grad_y, num_tokens * hidden)
    _room("expert_out", expert_out, r * hidden)
    _room("grad_expert_out", grad_expert_out, r * hidden)
    _entry(_COMBINE_BACKWARD, "moe_combine_rows_backward_device", stream, grad_y, expert_out, d, dst_of_route, weights,
           grad_expert_out, grad_weights, num_tokens, hidden, top_k)


# ---------------------------------------------------------------- products of float matrices
def _optional(t, name: str, d: int, n: int) -> None:
    """None, or a tensor of the dtype d with at least n elements."""
    if t is not None:
        _same_dtype(name, d, t)
        _room(name, t, n)


def _strided(t, name: str, rows: int, cols: int):
    """(argument, row stride) of rows x cols values, (None, 0) of None."""
    return (None, 0) if t is None else _rows_of(t, name, rows, cols)


def _grad_dtype(d: int, *grads) -> int:
    """The dtype of the weights' gradients that are given: d or float32."""
    found = {_dtype(g, "a weight's gradient") for g in grads if g is not None} or {d}
    if len(found) != 1 or not found <= {d, DTYPE_F32}:
        raise ValueError("gradients of weights must have one dtype, the weights' or float32")
    return found.pop()


def _bytes_of(ws) -> int:
    return 0 if ws is None else ws.numel() * ws.element_size()


def linear_rows_workspace_bytes(dtype: int, in_features: int, out_features: int, num_tokens: int) -> int:
    return int(lib().linear_rows_workspace_bytes(dtype, in_features, out_features, num_tokens))


def linear_rows(x, w, y, in_features: int, out_features: int, num_tokens: int, bias=None, residual=None,
                activation: int = ACT_NONE, pre=None, ws=None, stream=None) -> None:
    """y [T, out] = act(x [T, in] . w [out, in]^T + bias) + residual, all of one dtype (float32, float16 or
    bfloat16).  Rows of x, residual and y may be strided; residual may be y.  pre [T, out], where given,
    receives x . w^T + bias for the backward pass; ws of linear_rows_workspace_bytes (None where that is 0)."""
    d = _dtype(x, "x")
    for name, t in (("w", w), ("y", y)):
        _same_dtype(name, d, t)
    _room("w", w, out_features * in_features)
    _optional(bias, "bias", d, out_features)
    _optional(residual, "residual", d, 0)
    _optional(pre, "pre", d, num_tokens * out_features)
    px, x_stride = _rows_of(x, "x", num_tokens, in_features)
    pr, r_stride = _strided(residual, "residual", num_tokens, out_features)
    py, y_stride = _rows_of(y, "y", num_tokens, out_features)
    _entry(_LINEAR_ROWS, "linear_rows_forward_device", stream, px, x_stride, w, bias, pr, r_stride, py, y_stride, pre, d,
           activation, in_features, out_features, num_tokens, ws, _bytes_of(ws))


def linear_rows_backward_workspace_bytes(dtype: int, in_features: int, out_features: int, num_tokens: int,
                                         activation: int | None = None, grad_dtype: int | None = None) -> int:
    """Enough for any backward pass of these sizes; with an activation and the dtype of the weights' gradients (the
    rows' where it is None) for those."""
    if activation is None and grad_dtype is None:
        return int(lib().linear_rows_backward_workspace_bytes(dtype, in_features, out_features, num_tokens))
    return int(lib().linear_rows_backward_workspace_bytes_for(
        dtype, dtype if grad_dtype is None else grad_dtype, ACT_SILU if activation is None else activation, in_features,
        out_features, num_tokens))


def linear_rows_backward(grad_y, x, w, grad_x, grad_w, grad_b, in_features: int, out_features: int, num_tokens: int,
                         activation: int = ACT_NONE, pre=None, ws=None, stream=None) -> None:
    """The gradients of linear_rows (None: not wanted) from that of y: grad_x of x's dtype, grad_w and grad_b
    of x's or float32.  pre is what the forward pass kept (needed with an activation).  The residual's
    gradient is grad_y."""
    d = _dtype(grad_y, "grad_y")
    gd = _grad_dtype(d, grad_w, grad_b)
    _optional(x, "x", d, 0)
    _optional(w, "w", d, out_features * in_features)
    _optional(pre, "pre", d, num_tokens * out_features)
    _optional(grad_x, "grad_x", d, 0)
    _optional(grad_w, "grad_w", gd, out_features * in_features)
    _optional(grad_b, "grad_b", gd, out_features)
    pg, g_stride = _rows_of(grad_y, "grad_y", num_tokens, out_features)
    px, x_stride = _strided(x, "x", num_tokens, in_features)
    pgx, gx_stride = _strided(grad_x, "grad_x", num_tokens, in_features)
    _entry(_LINEAR_ROWS_BACKWARD, "linear_rows_backward_device", stream, pg, g_stride, px, x_stride, w, pre, pgx,
           gx_stride, grad_w, grad_b, d, gd, activation, in_features, out_features, num_tokens, ws, _bytes_of(ws))


def grouped_mat_mul_rows_workspace_bytes(dtype: int, K: int, N: int, n_routes: int, num_experts: int) -> int:
    return int(lib().mat_mul_rows_grouped_workspace_bytes(dtype, K, N, n_routes, num_experts))


def grouped_mat_mul_rows(x, w, expert_offsets, y, K: int, N: int, n_routes: int, ws=None, stream=None) -> None:
    """mat_mul_rows_grouped_device: rows of x [n_routes, K] sorted by expert times their experts' weights w
    [E, N, K]; E is one less than expert_offsets' (int32) length."""
    d = _dtype(x, "x")
    n_experts = expert_offsets.numel() - 1
    for name, t, n in (("x", x, n_routes * K), ("w", w, n_experts * N * K), ("y", y, n_routes * N)):
        _optional(t, name, d, n)
    _typed("expert_offsets", expert_offsets, _torch.int32, 2)
    _entry(_ROWS_GROUPED, "mat_mul_rows_grouped_device", stream, x, w, expert_offsets, n_experts, y, d, K, N, n_routes,
           ws, _bytes_of(ws))


def grouped_mat_mul_rows_backward_workspace_bytes(dtype: int, K: int, N: int, n_routes: int, num_experts: int) -> int:
    return int(lib().mat_mul_rows_grouped_backward_workspace_bytes(dtype, K, N, n_routes, num_experts))


def grouped_mat_mul_rows_backward(grad_y, x, w, expert_offsets, grad_x, grad_w, K: int, N: int, n_routes: int,
                                  ws=None, stream=None) -> None:
    """The gradients of grouped_mat_mul_rows (None: not wanted): grad_x [n_routes, K] of grad_y's dtype, grad_w
    [E, N, K] of that or float32."""
    d = _dtype(grad_y, "grad_y")
    gd = _grad_dtype(d, grad_w)
    n_experts = expert_offsets.numel() - 1
    for name, t, n in (("grad_y", grad_y, n_routes * N), ("x", x, n_routes * K), ("w", w, n_experts * N * K),
                       ("grad_x", grad_x, n_routes * K)):
        _optional(t, name, d, n)
    _optional(grad_w, "grad_w", gd, n_experts * N * K)
    _typed("expert_offsets", expert_offsets, _torch.int32, 2)
    _entry(_ROWS_GROUPED_BACKWARD, "mat_mul_rows_grouped_backward_device", stream, grad_y, x, w, expert_offsets,
           n_experts, grad_x, grad_w, d, gd, K, N, n_routes, ws, _bytes_of(ws))


def moe_gate_up_swiglu_rows_workspace_bytes(dtype: int, hidden: int, inter: int, n_routes: int, num_experts: int) -> int:
    return int(lib().moe_rows_gate_up_swiglu_workspace_bytes(dtype, hidden, inter, n_routes, num_experts))


def moe_gate_up_swiglu_rows(x, w_gate, w_up, expert_offsets, num_experts: int, mid, hidden: int, inter: int,
                            n_routes: int, gate_up=None, ws=None, stream=None) -> None:
    """mid [n_routes, inter] = silu(x . w_gate^T) * (x . w_up^T) of rows sorted by expert, w_gate and w_up
    [E, inter, hidden]; gate_up [n_routes, 2 * inter], where given, receives both products."""
    d = _dtype(x, "x")
    for name, t, n in (("x", x, n_routes * hidden), ("w_gate", w_gate, num_experts * inter * hidden),
                       ("w_up", w_up, num_experts * inter * hidden), ("mid", mid, n_routes * inter),
                       ("gate_up", gate_up, n_routes * 2 * inter)):
        _optional(t, name, d, n)
    _typed("expert_offsets", expert_offsets, _torch.int32, num_experts + 1)
    _entry(_ROWS_GATE_UP, "moe_rows_gate_up_swiglu_device", stream, x, w_gate, w_up, expert_offsets, num_experts,
           gate_up, mid, d, hidden, inter, n_routes, ws, _bytes_of(ws))


def moe_gate_up_swiglu_rows_backward_workspace_bytes(dtype: int, hidden: int, inter: int, n_routes: int,
                                                     num_experts: int, grad_dtype: int | None = None) -> int:
    """Enough for any backward pass of these sizes; with the dtype of the weights' gradients for those."""
    if grad_dtype is None:
        return int(lib().moe_rows_gate_up_swiglu_backward_workspace_bytes(dtype, hidden, inter, n_routes, num_experts))
    return int(lib().moe_rows_gate_up_swiglu_backward_workspace_bytes_for(dtype, grad_dtype, hidden, inter, n_routes,
                                                                          num_experts))


def moe_gate_up_swiglu_rows_backward(grad_mid, gate_up, x, w_gate, w_up, expert_offsets, num_experts: int, grad_x,
                                     grad_w_gate, grad_w_up, hidden: int, inter: int, n_routes: int, ws=None,
                                     stream=None) -> None:
    """The gradients of moe_gate_up_swiglu_rows (None: not wanted) from that of mid and the saved gate_up:
    grad_x of their dtype, grad_w_gate and grad_w_up of that or float32."""
    d = _dtype(grad_mid, "grad_mid")
    gd = _grad_dtype(d, grad_w_gate, grad_w_up)
    weights = num_experts * inter * hidden
    for name, t, n in (("grad_mid", grad_mid, n_routes * inter), ("gate_up", gate_up, n_routes * 2 * inter),
                       ("x", x, n_routes * hidden), ("w_gate", w_gate, weights), ("w_up", w_up, weights),
                       ("grad_x", grad_x, n_routes * hidden)):
        _optional(t, name, d, n)
    _optional(grad_w_gate, "grad_w_gate", gd, weights)
    _optional(grad_w_up, "grad_w_up", gd, weights)
    _typed("expert_offsets", expert_offsets, _torch.int32, num_experts + 1)
    _entry(_ROWS_GATE_UP_BACKWARD, "moe_rows_gate_up_swiglu_backward_device", stream, grad_mid, gate_up, x, w_gate,
           w_up, expert_offsets, num_experts, grad_x, grad_w_gate, grad_w_up, d, gd, hidden, inter, n_routes, ws,
           _bytes_of(ws))


ROWS_FORWARD, ROWS_SWIGLU, ROWS_INPUT, ROWS_WEIGHT = range(4)
ROWS_TILE_64, ROWS_TILE_128, ROWS_TILE_160, ROWS_TILE_256 = range(4)
ROWS_DIRECT = 64  # + waves


def rows_kernel(form: int, kernel: int, p, q, y, cols: int, rows: int, sums: int, p2=None, y2=None, offsets=None,
                slices: int = 1, ws=None, stream=None) -> None:
    """jjo_rows_kernel_device: one product of float matrices on a given kernel (measurements and tests)."""
    d = _dtype(p, "p")
    halves = 2 if (p2 if form == ROWS_INPUT else y2) is not None else 1
    E = 1 if offsets is None else offsets.numel() - 1
    weights = 1 if form == ROWS_WEIGHT else E
    for name, t, n in (("p", p, weights * cols * sums), ("p2", p2, weights * cols * sums), ("q", q, halves * rows * sums),
                       ("y", y, (E if form == ROWS_WEIGHT else 1) * rows * cols),
                       ("y2", y2, (E if form == ROWS_WEIGHT else 1) * rows * cols)):
        _optional(t, name, d, n)
    _check(lib().jjo_rows_kernel_device(
        _stream(stream), form, kernel, slices, d, *(None if t is None else _dev(t, "an operand") for t in (p, p2, q, offsets)),
        E, *(None if t is None else _dev(t, "an output") for t in (y, y2)), cols, rows, sums,
        None if ws is None else _dev(ws, "ws"), _bytes_of(ws)), "jjo_rows_kernel_device")
