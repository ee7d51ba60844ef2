#include <hip/hip_runtime.h>

#include "attention_backward_kernel.hpp"

namespace opscv {

hipError_t run_attention_grad_f32(const AttentionArgs& a, bool vectors, hipStream_t stream)
{
    return vectors ? att::run_backward<float, true>(a, stream) : att::run_backward<float, false>(a, stream);
}

}  // namespace opscv
