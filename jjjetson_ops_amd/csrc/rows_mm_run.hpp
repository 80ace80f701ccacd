// The kernel of a float product, by the choice made for its sizes (rows_mm_choose).
#pragma once

#include "rows_mm_direct.hpp"

namespace jjo {

template <class E>
hipError_t rows_mm_run(RowsMode mode, const RowsMm &p, const RowsChoice &c, hipStream_t stream) {
    if (c.tile == kRowsDirect) {
        if (mode == kRowsForward) return run_rows_direct<E, false>(p, c.waves, stream);
        if (mode == kRowsSwiglu) return run_rows_direct<E, true>(p, c.waves, stream);
        return hipErrorInvalidValue;
    }
    switch (mode) {
        case kRowsForward: return rows_by_tile<E, kRowsForward>(p, c.tile, stream);
        case kRowsSwiglu: return rows_by_tile<E, kRowsSwiglu>(p, c.tile, stream);
        case kRowsInput: return rows_by_tile<E, kRowsInput>(p, c.tile, stream);
        case kRowsWeight: return rows_by_tile<E, kRowsWeight>(p, c.tile, stream);
    }
    return hipErrorInvalidValue;
}

}  // namespace jjo
