"""The float products' entries on the extremes of their integer arguments: no signed overflow before they are
refused.  The entries' own file and the choice of a kernel are compiled for the host with the compiler's overflow
checks, with stand-ins for what they call."""
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
#include "rows_mm.hpp"
namespace jjo {
void clear_error() {}
int set_error(int code, const char *, ...) { return code; }
int hip_fail(hipError_t, const char *) { abort(); }
int require_device() { return JJO_ERR_NO_DEVICE; }  // what is not refused ends here
hipError_t launch_rows_mm(RowsMode, int, const RowsMm &, hipStream_t, const RowsChoice *) { abort(); }
hipError_t launch_rows_act_backward(const void *, int64_t, const void *, void *, int, int64_t, int, int, void *, bool,
                                    float *, int, int, hipStream_t) { abort(); }
hipError_t launch_rows_swiglu_backward(const void *, const void *, void *, int, int64_t, int, const int32_t *, int, int,
                                       int, hipStream_t) { abort(); }
}
"""
CALLS = """
import ctypes, itertools, sys
L = ctypes.CDLL(sys.argv[1])
A = ctypes.c_void_p(256)
I, S = [1, 64, 4095, 1 << 20, 1 << 28, 2**31 - 1, -1, -2**31], [64, 1 << 40, 2**63 - 1, -1, -2**63]
i, q = ctypes.c_int, ctypes.c_int64
B = q(2**63 - 1)
def every(name, n, call, values=I, kind=i):
    f = getattr(L, name)
    f.restype = ctypes.c_int64
    for v in itertools.product(values, repeat=n):
        print(name, v, file=sys.stderr)
        call(f, *map(kind, v))
for d in (0, 1, 2):
    for n in ("linear_rows", "linear_rows_backward"):
        every(n + "_workspace_bytes", 3, lambda f, *v: f(d, *v))
    for n in ("mat_mul_rows_grouped", "mat_mul_rows_grouped_backward", "moe_rows_gate_up_swiglu",
              "moe_rows_gate_up_swiglu_backward"):
        every(n + "_workspace_bytes", 4, lambda f, *v: f(d, *v))
every("linear_rows_forward_device", 3, lambda f, *v: f(None, A, q(1 << 28), A, A, A, q(1 << 28), A, q(1 << 28), A, 2, 4, *v, A, B))
every("linear_rows_forward_device", 3, lambda f, a, b, c: f(None, A, a, A, A, A, b, A, c, A, 2, 4, 64, 64, 1 << 28, A, B), S, q)
every("linear_rows_backward_device", 3, lambda f, *v: f(None, A, q(1 << 28), A, q(1 << 28), A, A, A, q(1 << 28), A, A, 2, 0, 4, *v, A, B))
every("linear_rows_backward_device", 3, lambda f, a, b, c: f(None, A, a, A, b, A, A, A, c, A, A, 2, 0, 4, 64, 64, 1 << 28, A, B), S, q)
every("mat_mul_rows_grouped_device", 4, lambda f, e, *v: f(None, A, A, A, e, A, 2, *v, A, B))
every("mat_mul_rows_grouped_backward_device", 4, lambda f, e, *v: f(None, A, A, A, A, e, A, A, 2, 0, *v, A, B))
every("moe_rows_gate_up_swiglu_device", 4, lambda f, e, *v: f(None, A, A, A, A, e, A, A, 1, *v, A, B))
every("moe_rows_gate_up_swiglu_backward_device", 4, lambda f, e, *v: f(None, A, A, A, A, A, A, e, A, A, A, 1, 0, *v, A, B))
every("jjo_rows_kernel_device", 3, lambda f, *v: f(None, 3, 1, 64, 0, A, None, A, A, 4096, A, A, *v, A, B))
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
                    str(build.CSRC / "capi_rows.hip"), str(build.CSRC / "rows_choose.hip"),
                    str(tmp_path / "stand_ins.hip"), "-o", str(lib)], check=True)
    r = subprocess.run([sys.executable, "-c", CALLS, str(lib)], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout.strip() == "done", (r.returncode, r.stderr.splitlines()[-1:])
