// Launch interface of the operators on token sequences.  Each launcher checks what its kernels assume and returns
// hipErrorInvalidValue instead of launching where it does not hold.
#pragma once

#include <hip/hip_runtime_api.h>

#include "acl_types.hpp"

namespace opscv {

hipError_t launch_residual_norm(const NormArgs& a, hipStream_t stream);
hipError_t launch_residual_norm_grad(const NormGradArgs& a, hipStream_t stream);
// rows of NormGradArgs::partial
int64_t norm_grad_partials(const NormGradArgs& a);
hipError_t launch_rotary_table(const RotaryTableArgs& a, hipStream_t stream);
hipError_t launch_rotary(const RotaryArgs& a, hipStream_t stream);
hipError_t launch_window_attention(const AttentionArgs& a, hipStream_t stream);
// 32-bit words of AttentionArgs::scratch: partial results where the keys of a query are split, 0 where they are not.  A call
// makes as many launches as its sequences take; -1, here and for the gradients, where one sequence does not fit a launch.
int64_t attention_scratch_floats(const AttentionArgs& a);
hipError_t launch_window_attention_grad(const AttentionArgs& a, hipStream_t stream);
int64_t attention_grad_scratch_floats(const AttentionArgs& a);
// names for opscvExecutorVariant
const char* attention_variant(const AttentionArgs& a);

}  // namespace opscv
