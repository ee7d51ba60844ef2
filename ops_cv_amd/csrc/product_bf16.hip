// Matrix products of BF16 operands (product_tile.hpp).
#include "gated.hpp"
#include "product_launch.hpp"

namespace opscv {
namespace prod {

hipError_t launch_product_bf16(const ProductArgs& a, int kind, int tile, hipStream_t stream)
{
    return launch_typed<__bf16>(a, kind, tile, stream);
}

}  // namespace prod
}  // namespace opscv
