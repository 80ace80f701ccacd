// The kernels of the float products, fp16 operands.
#include "rows_mm_run.hpp"

namespace jjo {
template hipError_t rows_mm_run<MxF16>(RowsMode, const RowsMm &, const RowsChoice &, hipStream_t);
}
