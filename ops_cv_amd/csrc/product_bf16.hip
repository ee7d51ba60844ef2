// Matrix products of BF16 operands (product_tile.hpp).
#include "gated.hpp"
#include "product_launch.hpp"

namespace opscv {
namespace prod {

hipError_t launch_products_bf16(const ProductArgs& a, int tile, hipStream_t stream)
{
    return launch_gated_typed<__bf16>(a, tile, stream);
}

hipError_t launch_gradients_bf16(const ProductArgs* x, const ProductArgs* weights, int tile, hipStream_t stream)
{
    return launch_gradients_typed<__bf16>(x, weights, tile, stream);
}

}  // namespace prod
}  // namespace opscv
