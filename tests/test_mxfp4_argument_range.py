"""The MXFP4 and sorted-row entries on the extremes of their integer arguments: no signed overflow
before they are refused.  The entries' own file is compiled for the host with the compiler's
overflow checks, with stand-ins for what it calls."""
if __name__ == "__main__":  # `python tests/<file>.py`, as the reference runs its tests
    import sys as _sys

    import pytest as _pytest
    _sys.exit(_pytest.main([__file__, "-q"]))
import subprocess
import sys
from pathlib import Path

import pytest

from jjjetson_ops_amd import build

STAND_INS = """
#include "mxfp4_common.hpp"
namespace jjo {
void clear_error() {}
int set_error(int code, const char *, ...) { return code; }
int hip_fail(hipError_t, const char *) { abort(); }
int require_device() { return JJO_ERR_NO_DEVICE; }  // what is not refused ends here
int mxfp4_down_slices(int, int, int, int) { return 2; }
typedef const void *P;
typedef const int32_t *Ids;
typedef hipStream_t S;
hipError_t launch_quantize_mxfp4(P, int, int64_t, void *, int64_t, int64_t, S) { abort(); }
hipError_t launch_dequantize_mxfp4(P, void *, int, int64_t, int64_t, int64_t, S) { abort(); }
hipError_t launch_mxfp4_gemv(P, P, int, void *, int, int, int, S) { abort(); }
hipError_t launch_mxfp4_mm(P, P, void *, int, int, int, int, const MxGroups &, S, int) { abort(); }
hipError_t launch_mxfp4_swiglu(P, P, P, void *, int, int, int, const MxGroups &, S) { abort(); }
hipError_t launch_mxfp4_route(P, int, const float *, int, int, int, int, float *, int32_t *, int32_t *, int32_t *,
                              int32_t *, void *, S) { abort(); }
hipError_t launch_moe_dispatch_rows(Ids, P, int, int, int, int, int, int32_t *, int32_t *, int32_t *, void *, S) {
    abort();
}
hipError_t launch_moe_join_rows(P, int, Ids, const float *, void *, int, int, int, int, S, int) { abort(); }
hipError_t launch_moe_combine_rows_backward(P, P, int, Ids, const float *, void *, float *, int, int, int, S) { abort(); }
}
"""
CALLS = """
import ctypes, itertools, sys
L = ctypes.CDLL(sys.argv[1])
A = ctypes.c_void_p(256)
I, Q = [1, 32, 1 << 23, 2**31 - 1, -1, -2**31], [1, 32, 1 << 40, 2**63 - 1, -1, -2**63]
i, q = ctypes.c_int, ctypes.c_int64
def every(name, n, call, values=I, kind=i):
    f = getattr(L, name)
    for v in itertools.product(values, repeat=n):
        print(name, v, file=sys.stderr)
        call(f, *map(kind, v))
every("mxfp4_bytes", 2, lambda f, a, b: f(a, b), Q, q)
every("quantize_mxfp4_device", 3, lambda f, s, r, c: f(None, A, 0, s, A, r, c), Q, q)
every("dequantize_mxfp4_device", 3, lambda f, s, r, c: f(None, A, A, 2, s, r, c), Q, q)
every("mat_mul_mxfp4_device", 3, lambda f, a, b, c: f(A, A, A, 0, a, b, c, None))
every("linear_mxfp4_workspace_bytes", 2, lambda f, a, b: f(a, b))
every("linear_mxfp4_forward_device", 3, lambda f, a, b, c: f(None, A, A, 0, A, A, 0, a, b, c))
every("mat_mul_mxfp4_grouped_device", 4, lambda f, e, a, b, c: f(A, A, A, e, A, A, 0, a, b, c, None))
every("moe_mxfp4_gate_up_swiglu_device", 4, lambda f, e, a, b, c: f(None, A, A, A, A, e, A, a, b, c))
every("moe_mxfp4_ffn_workspace_bytes", 5, lambda f, *v: f(*v))
every("moe_mxfp4_ffn_forward_device", 5, lambda f, *v: f(None, A, A, A, A, A, A, 0, *v, A, q(1 << 62)))
every("moe_dispatch_rows_device", 4, lambda f, *v: f(None, A, A, 0, *v, A, A, A, A))
every("moe_dispatch_rows_backward_device", 3, lambda f, *v: f(None, A, 0, A, A, *v))
every("moe_combine_rows_device", 3, lambda f, *v: f(None, A, 0, A, A, A, *v))
every("moe_combine_rows_backward_device", 3, lambda f, *v: f(None, A, A, 0, A, A, A, A, *v))
print("done")
"""


def test_no_overflow_on_refused_arguments(tmp_path):
    if not Path(build.HIPCC).exists():
        pytest.skip("no hipcc")
    (tmp_path / "stand_ins.hip").write_text(STAND_INS)
    lib = tmp_path / "entries.so"
    subprocess.run([build.HIPCC, *build.HIP_FLAGS, "--offload-host-only", "-O1", "-shared",
                    "-Xarch_host", "-fsanitize=signed-integer-overflow",
                    "-Xarch_host", "-fsanitize-trap=signed-integer-overflow",
                    str(build.CSRC / "capi_mxfp4.hip"), str(tmp_path / "stand_ins.hip"), "-o", str(lib)], check=True)
    r = subprocess.run([sys.executable, "-c", CALLS, str(lib)], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout.strip() == "done", (r.returncode, r.stderr.splitlines()[-1:])
