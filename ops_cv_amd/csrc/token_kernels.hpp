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
hipError_t launch_layer_norm(const LayerNormArgs& a, hipStream_t stream);
hipError_t launch_layer_norm_grad(const LayerNormGradArgs& a, hipStream_t stream);
// rows of each half of LayerNormGradArgs::partial
int64_t layer_norm_grad_partials(const LayerNormGradArgs& a);
hipError_t launch_dropout(const DropoutArgs& a, hipStream_t stream);
hipError_t launch_gated(const GatedArgs& a, hipStream_t stream);
hipError_t launch_gated_grad(const GatedArgs& a, hipStream_t stream);
// bytes of GatedArgs::scratch.  The addresses of the operands that are used in place have to be set; those of packed ones are
// on 256 bytes (null stands for one).
int64_t gated_scratch_bytes(const GatedArgs& a);
int64_t gated_grad_scratch_bytes(const GatedArgs& a);
// the operators of opscv_blocks.cpp, whose operands have been checked (execute_token_plan)
hipError_t launch_block_plan(void* workspace, const aclOpExecutor* ex, hipStream_t stream);
// names for opscvExecutorVariant
const char* attention_variant(const AttentionArgs& a);

}  // namespace opscv
