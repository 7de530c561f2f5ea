// Product of matrices in microscaled 8-bit floating point (see product_tile.hpp).
#include "product_tile.hpp"

namespace tdc {

int launch_product_mx8(TileArgs a, const TilePlan &p, int y_dtype, void *stream) {
    const hipStream_t s = (hipStream_t)stream;
    if (y_dtype == TDC_F16) return launch_product_of<TDC_MX8, false, false, TDC_F16>(a, p, s);
    return launch_product_of<TDC_MX8, false, false, TDC_BF16>(a, p, s);
}

}  // namespace tdc
