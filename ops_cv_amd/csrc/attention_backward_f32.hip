#include <hip/hip_runtime.h>

#include "attention_backward_kernel.hpp"

namespace opscv {

hipError_t run_attention_grad_f32(const AttentionArgs& a, const att::GradPlan& plan, bool vectors, hipStream_t stream)
{
    return vectors ? att::run_backward<float, true>(a, plan, stream) : att::run_backward<float, false>(a, plan, stream);
}

}  // namespace opscv
