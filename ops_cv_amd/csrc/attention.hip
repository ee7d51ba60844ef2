// Attention to a window around each token and to the first tokens: which kernels a call runs.
#include <hip/hip_runtime.h>

#include "attention_backward_kernel.hpp"
#include "attention_forward_kernel.hpp"
#include "token_elem.hpp"
#include "token_kernels.hpp"

namespace opscv {

namespace {

// whether every row of the operands can be read in 16-byte vectors
template <typename... S>
bool vectors(const AttentionArgs& a, const S&... operands)
{
    const int e = a.elem == (int)Elem::F32 ? 4 : 2;
    bool fits = a.d * e % 16 == 0;
    for (const Strided* s : {&operands...}) {
        for (int i = 0; i < 3; i++) {
            fits = fits && tok::aligned(s->ptr, s->stride[i], e, 16);
        }
    }
    return fits;
}

}  // namespace

hipError_t launch_window_attention(const AttentionArgs& a, hipStream_t stream)
{
    if (a.batch < 1 || a.tokens < 1 || a.kv_heads < 1 || a.heads % a.kv_heads != 0 || a.d < 1 || a.d > 256) {
        return hipErrorInvalidValue;
    }
    const bool fits = vectors(a, a.q, a.k, a.v, a.out);
    switch ((Elem)a.elem) {
        case Elem::F32: return run_attention_f32(a, fits, stream);
        case Elem::F16: return run_attention_f16(a, fits, stream);
        default: return run_attention_bf16(a, fits, stream);
    }
}

int64_t attention_scratch_floats(const AttentionArgs& a)
{
    const att::ForwardPlan p = att::plan_forward(a);
    return p.splits > 1 ? a.batch * a.kv_heads * p.splits * p.rows * att::partial_floats(a.d) : 0;
}

hipError_t launch_window_attention_grad(const AttentionArgs& a, hipStream_t stream)
{
    if (a.batch < 1 || a.kv_heads < 1 || a.heads % a.kv_heads != 0 || a.d < 1 || a.d > 256) {
        return hipErrorInvalidValue;
    }
    const bool fits = vectors(a, a.q, a.k, a.v, a.out, a.grad_out, a.grad_q, a.grad_k, a.grad_v);
    switch ((Elem)a.elem) {
        case Elem::F32: return run_attention_grad_f32(a, fits, stream);
        case Elem::F16: return run_attention_grad_f16(a, fits, stream);
        default: return run_attention_grad_bf16(a, fits, stream);
    }
}

int64_t attention_grad_scratch_floats(const AttentionArgs& a)
{
    const att::GradPlan p = att::plan_grad(a);
    return p.stats + p.sink_partials + p.partials;
}

const char* attention_variant(const AttentionArgs& a)
{
    const att::ForwardPlan p = att::plan_forward(a);
    return p.few_rows ? (p.splits > 1 ? "attention_few_rows_split" : "attention_few_rows")
                      : (p.splits > 1 ? "attention_rows_split" : "attention_rows");
}

}  // namespace opscv
