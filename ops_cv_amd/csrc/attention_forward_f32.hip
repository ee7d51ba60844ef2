#include <hip/hip_runtime.h>

#include "attention_forward_kernel.hpp"

namespace opscv {

hipError_t run_attention_f32(const AttentionArgs& a, bool vectors, hipStream_t stream)
{
    return vectors ? att::run_forward<float, true>(a, stream) : att::run_forward<float, false>(a, stream);
}

}  // namespace opscv
