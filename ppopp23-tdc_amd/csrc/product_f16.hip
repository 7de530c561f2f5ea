// Products of half-precision matrices (see product_tile.hpp).
#include "product_tile.hpp"

namespace tdc {

int launch_product_f16(TileArgs a, const TilePlan &p, int layout, void *stream) {
    const hipStream_t s = (hipStream_t)stream;
    if (layout == kAlong) return launch_product_of<TDC_F16, false, false, TDC_F16>(a, p, s);
    if (layout == kWAcross) return launch_product_of<TDC_F16, false, true, TDC_F16>(a, p, s);
    return launch_product_of<TDC_F16, true, true, TDC_F16>(a, p, s);
}

}  // namespace tdc
