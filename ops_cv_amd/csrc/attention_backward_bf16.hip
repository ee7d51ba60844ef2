#include <hip/hip_runtime.h>

#include "attention_backward_kernel.hpp"

namespace opscv {

hipError_t run_attention_grad_bf16(const AttentionArgs& a, const att::GradPlan& plan, bool vectors, hipStream_t stream)
{
    return vectors ? att::run_backward<__bf16, true>(a, plan, stream) : att::run_backward<__bf16, false>(a, plan, stream);
}

}  // namespace opscv
