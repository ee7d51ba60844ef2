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

// run(a, plan, vectors, stream) for every launch of the call
template <typename Plan, typename Run>
hipError_t run_launches(const AttentionArgs& a, Plan&& plan_of, bool fits, Run&& run, hipStream_t stream)
{
    hipError_t e = hipSuccess;
    int64_t done = 0;
    att::by_launches(a, plan_of, [&](const AttentionArgs& s, const auto& plan) {
        e = e == hipSuccess ? run(s, plan, fits, stream) : e;
        done += s.batch;
    });
    return done == a.batch ? e : hipErrorInvalidValue;
}

// the most that floats(a, plan) is over the launches of the call; -1 where not one sequence fits a launch
template <typename Plan, typename Floats>
int64_t most_scratch(const AttentionArgs& a, Plan&& plan_of, Floats&& floats)
{
    int64_t most = -1;
    att::by_launches(a, plan_of, [&](const AttentionArgs& s, const auto& plan) {
        const int64_t n = plan.fits ? floats(s, plan) : -1;
        most = n > most ? n : most;
    });
    return most;
}

}  // namespace

hipError_t launch_window_attention(const AttentionArgs& a, hipStream_t stream)
{
    if (a.batch < 1 || a.tokens < 1 || a.kv_heads < 1 || a.heads % a.kv_heads != 0 || a.d < 1 || a.d > 256) {
        return hipErrorInvalidValue;
    }
    const auto run = a.elem == (int)Elem::F32   ? run_attention_f32
                     : a.elem == (int)Elem::F16 ? run_attention_f16
                                                : run_attention_bf16;
    return run_launches(a, att::plan_forward, vectors(a, a.q, a.k, a.v, a.out), run, stream);
}

int64_t attention_scratch_floats(const AttentionArgs& a)
{
    return most_scratch(a, att::plan_forward, [](const AttentionArgs& s, const att::ForwardPlan& p) {
        return p.splits > 1 ? s.batch * s.kv_heads * p.splits * p.rows * att::partial_floats(s.d) : 0;
    });
}

hipError_t launch_window_attention_grad(const AttentionArgs& a, hipStream_t stream)
{
    if (a.batch < 1 || a.kv_heads < 1 || a.heads % a.kv_heads != 0 || a.d < 1 || a.d > 256) {
        return hipErrorInvalidValue;
    }
    const auto run = a.elem == (int)Elem::F32   ? run_attention_grad_f32
                     : a.elem == (int)Elem::F16 ? run_attention_grad_f16
                                                : run_attention_grad_bf16;
    return run_launches(a, att::plan_grad, vectors(a, a.q, a.k, a.v, a.out, a.grad_out, a.grad_q, a.grad_k, a.grad_v), run,
                        stream);
}

int64_t attention_grad_scratch_floats(const AttentionArgs& a)
{
    return most_scratch(a, att::plan_grad, [](const AttentionArgs&, const att::GradPlan& p) {
        return p.stats + p.sink_partials + p.partials;
    });
}

const char* attention_variant(const AttentionArgs& a)
{
    const att::ForwardPlan p = att::plan_forward(a);
    return p.few_rows ? (p.splits > 1 ? "attention_few_rows_split" : "attention_few_rows")
                      : (p.splits > 1 ? "attention_rows_split" : "attention_rows");
}

}  // namespace opscv
