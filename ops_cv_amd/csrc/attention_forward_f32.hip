#include <hip/hip_runtime.h>

#include "attention_forward_kernel.hpp"

namespace opscv {

hipError_t run_attention_f32(const AttentionArgs& a, const att::ForwardPlan& plan, bool vectors, hipStream_t stream)
{
    return vectors ? att::run_forward<float, true>(a, plan, stream) : att::run_forward<float, false>(a, plan, stream);
}

}  // namespace opscv
