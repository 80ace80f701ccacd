// The kernels of the float products, bf16 operands.
#include "rows_mm_run.hpp"

namespace jjo {
template hipError_t rows_mm_run<MxBF16>(RowsMode, const RowsMm &, const RowsChoice &, hipStream_t);
}
