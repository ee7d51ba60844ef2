// Matrix products of FLOAT operands (product_tile.hpp).
#include "gated.hpp"
#include "product_launch.hpp"

namespace opscv {
namespace prod {

hipError_t launch_products_f32(const ProductArgs& a, int tile, hipStream_t stream)
{
    return launch_gated_typed<float>(a, tile, stream);
}

hipError_t launch_gradients_f32(const ProductArgs* x, const ProductArgs* weights, int tile, hipStream_t stream)
{
    return launch_gradients_typed<float>(x, weights, tile, stream);
}

}  // namespace prod
}  // namespace opscv
