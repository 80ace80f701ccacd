// Tiles of the float products, fp16 operands.
#include "rows_mm_tile.hpp"

namespace jjo {
template hipError_t rows_mm_tiles<MxF16>(RowsMode, const RowsMm &, int, hipStream_t);
}
