"""The MXFP4 format and the operators on it in fp64 (NumPy), and the error bounds of fp32 sums."""
import numpy as np

E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
BOUNDS = (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)  # between neighbours; a tie goes to the even code


def scale_byte(amax):
    """The scale byte of fp64 block maxima (NaN or infinity: 255)."""
    amax = np.asarray(amax, np.float64)
    bad = ~np.isfinite(amax)
    _, e = np.frexp(np.where(bad | (amax == 0), 1.0, amax))  # amax = m * 2^e, m in [0.5, 1)
    s = np.where(amax == 0, 0, np.maximum(e - 1 - 2 + 127, 0))
    return np.where(bad, 255, s).astype(np.uint8)


def round_codes(v):
    """e2m1 codes of fp64 values that are already divided by their scale."""
    a = np.abs(v)
    code = np.zeros(v.shape, np.uint8)
    for i, b in enumerate(BOUNDS):
        code += (a >= b) if i % 2 else (a > b)  # the tie's even neighbour is above an odd-numbered bound
    return code | (np.signbit(v).astype(np.uint8) << 3)


def values(code):
    return np.where(code & 8, -1.0, 1.0) * E2M1[code & 7]


def scale_value(s):
    return np.where(s == 255, np.nan, np.ldexp(1.0, s.astype(np.int64) - 127))


def quantize(x):
    """(codes [rows, cols], scale bytes [rows, cols/32]) of a 2-D array."""
    g = np.asarray(x, np.float64).reshape(x.shape[0], -1, 32)
    with np.errstate(invalid="ignore"):
        s = scale_byte(np.where(np.isnan(g).any(2), np.nan, np.abs(g).max(2)))
        v = np.where((s == 255)[..., None], 0.0, g / np.ldexp(1.0, s.astype(np.int64) - 127)[..., None])
    return round_codes(v).reshape(x.shape), s


def pack(code, s):
    return np.concatenate([(code[:, 0::2] | (code[:, 1::2] << 4)).reshape(-1), s.reshape(-1)])


def unpack(q, rows, cols):
    b = q[:rows * cols // 2].reshape(rows, cols // 2)
    code = np.stack([b & 15, b >> 4], 2).reshape(rows, cols)
    return code, q[rows * cols // 2:rows * cols // 32 * 17].reshape(rows, cols // 32)


def dequantize(q, rows, cols):
    code, s = unpack(q, rows, cols)
    return (values(code).reshape(rows, -1, 32) * scale_value(s)[..., None]).reshape(rows, cols)


def sum_bound(a, b):
    """The error of a . b^T summed in fp32: a block's 32 products have at most 13 significant
    bits together, so a block is exact; at most K/32 blocks and eight slices are added, each
    addition off by at most one step (2^-23) of the running magnitude, which the sum of the
    absolute products bounds."""
    k = a.shape[1]
    return (k // 32 + 8) * 2.0 ** -23 * (np.abs(a) @ np.abs(b).T)


HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}  # half the smallest subnormal


def rounding(y, dtype):
    """How far one rounding of fp64 values to dtype can be off."""
    return HALF_STEP[dtype] * np.abs(y) + TINY[dtype]
