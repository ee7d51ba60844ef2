#include <hip/hip_runtime.h>
#include "token_kernels.hpp"
namespace opscv {
hipError_t launch_window_attention_grad(const AttentionArgs&, hipStream_t) { return hipErrorNotSupported; }
int64_t attention_grad_scratch_floats(const AttentionArgs&) { return 0; }
}
