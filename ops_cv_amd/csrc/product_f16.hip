// Matrix products of FLOAT16 operands (product_tile.hpp).
#include "gated.hpp"
#include "product_launch.hpp"

namespace opscv {
namespace prod {

hipError_t launch_products_f16(const ProductArgs& a, int tile, hipStream_t stream)
{
    return launch_gated_typed<_Float16>(a, tile, stream);
}

hipError_t launch_gradients_f16(const ProductArgs* x, const ProductArgs* weights, int tile, hipStream_t stream)
{
    return launch_gradients_typed<_Float16>(x, weights, tile, stream);
}

}  // namespace prod
}  // namespace opscv
