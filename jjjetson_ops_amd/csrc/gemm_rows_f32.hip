// The kernels of the float products, fp32 operands.
#include "rows_mm_run.hpp"

namespace jjo {
template hipError_t rows_mm_run<MxF32>(RowsMode, const RowsMm &, const RowsChoice &, hipStream_t);
}
