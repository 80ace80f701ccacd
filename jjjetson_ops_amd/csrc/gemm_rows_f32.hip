// Tiles of the float products, fp32 operands.
#include "rows_mm_tile.hpp"

namespace jjo {
template hipError_t rows_mm_tiles<MxF32>(RowsMode, const RowsMm &, int, hipStream_t);
}
