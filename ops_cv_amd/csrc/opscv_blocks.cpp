// Layer norm, dropout and gated projections: parameter validation, planning and the second-phase entries
// (include/opscv_tokens.h).
#include "opscv_tokens.h"
#include "product_plan.hpp"
#include "token_kernels.hpp"
#include "token_plan.hpp"

using namespace opscv;
using namespace opscv::tokplan;

namespace {

constexpr int64_t kMostGated = (int64_t)1 << 19;      // width, inner
constexpr int64_t kMostGatedRows = (int64_t)1 << 20;  // backward

// slots of aclOpExecutor::operands
enum LayerNormSlot { kLnX, kLnResidual, kLnWeight, kLnBias, kLnY, kLnSum, kLnMean, kLnRstd };
enum LayerNormGradSlot { kLgY, kLgSumGrad, kLgSum, kLgWeight, kLgMean, kLgRstd, kLgX, kLgWeightGrad, kLgBiasGrad, kLgScratch };
enum DropoutSlot { kDrX, kDrResidual, kDrState, kDrY };
enum GatedSlot { kGaX, kGaGateWeight, kGaUpWeight, kGaGateBias, kGaUpBias, kGaY, kGaGate, kGaUp, kGaScratch };
enum GatedGradSlot { kGgY, kGgX, kGgGateWeight, kGgUpWeight, kGgGate, kGgUp, kGgGradX, kGgGradGateWeight, kGgGradUpWeight,
                     kGgGradGateBias, kGgGradUpBias, kGgScratch };

// A vector of the norm's columns: (width), of the activations' type or FLOAT, and of the same type as those before it.
aclnnStatus check_columns(const char* api, const char* name, const aclTensor* w, const aclTensor* x, aclDataType* dtype)
{
    if (w == nullptr) {
        return ACLNN_SUCCESS;
    }
    OPSCV_CHECK(check_weight(api, name, w, x));
    if (*dtype != ACL_DT_UNDEFINED && w->dtype != *dtype) {
        return invalid("%s: %s has another type than the other vectors of the width", api, name);
    }
    *dtype = w->dtype;
    return ACLNN_SUCCESS;
}

int columns_bytes(const aclTensor* w, int bytes) { return w->dtype == ACL_FLOAT ? 4 : bytes; }

// `t` is rows like `like`, with another width.
aclnnStatus check_rows_of(const char* api, const char* name, const aclTensor* t, const aclTensor* like, int64_t width)
{
    if (t->ndim != like->ndim || memcmp(t->dims, like->dims, sizeof(int64_t) * (size_t)(like->ndim - 1)) != 0 ||
        t->dims[t->ndim - 1] != width) {
        return invalid("%s: %s must be the rows of x with %lld elements each", api, name, (long long)width);
    }
    if (t->dtype != like->dtype) {
        return invalid("%s: %s has another type than x", api, name);
    }
    return ACLNN_SUCCESS;
}

aclnnStatus check_matrix(const char* api, const char* name, const aclTensor* t, const GatedArgs& a, aclDataType dtype)
{
    if (t->ndim != 2 || t->dims[0] != a.inner || t->dims[1] != a.width || t->dtype != dtype) {
        return invalid("%s: %s must be (inner, width) of x's type", api, name);
    }
    return ACLNN_SUCCESS;
}

aclnnStatus check_vector(const char* api, const char* name, const aclTensor* t, const GatedArgs& a, aclDataType dtype)
{
    if (t->ndim != 1 || t->dims[0] != a.inner || t->dtype != dtype) {
        return invalid("%s: %s must be (inner) of x's type", api, name);
    }
    return ACLNN_SUCCESS;
}

// What both directions of the gated projections share.
aclnnStatus check_gated(const char* api, const aclTensor* x, const aclTensor* gate_weight, const aclTensor* up_weight,
                        int64_t activation, int64_t most_rows, GatedArgs* a)
{
    Elem e;
    OPSCV_CHECK(norm_rows(api, x, &e, &a->rows, &a->width));
    a->elem = (int)e;
    if (gate_weight->ndim != 2) {
        return invalid("%s: gateWeight must have two dimensions", api);
    }
    a->inner = gate_weight->dims[0];
    OPSCV_CHECK(check_matrix(api, "gateWeight", gate_weight, *a, x->dtype));
    OPSCV_CHECK(check_matrix(api, "upWeight", up_weight, *a, x->dtype));
    if (a->inner < 1 || a->inner > kMostGated || a->width > kMostGated || a->rows > most_rows) {
        return invalid("%s: width and inner of 1 to 2^19 and up to %lld rows, got %lld, %lld and %lld", api,
                       (long long)most_rows, (long long)a->width, (long long)a->inner, (long long)a->rows);
    }
    if (activation < OPSCV_GATE_SILU || activation > OPSCV_GATE_GELU_TANH) {
        return invalid("%s: unknown activation %lld", api, (long long)activation);
    }
    a->activation = (int)activation;
    a->compute_units = compute_unit_count();
    return ACLNN_SUCCESS;
}

// How the products are made, planned before their scratch memory.
aclnnStatus check_plan(const char* api, const ProductPlan& plan, GatedArgs* a)
{
    if (plan.us == 0.0) {
        return invalid("%s: %lld rows of %lld and %lld features are more workgroups than a launch holds", api, (long long)a->rows,
                       (long long)a->width, (long long)a->inner);
    }
    a->plan = plan;
    return ACLNN_SUCCESS;
}

// Scratch memory, the last of the workspace's slices: it needs the operands' places to be planned.
void plan_bytes(aclOpExecutor* ex, int slot, int64_t bytes) { plan_scratch(ex, slot, (bytes + 3) / 4); }

// Operand `slot` as rows whose address, where they are packed, is that of a workspace slice on 256 bytes: what the layout of
// the scratch memory goes by in both phases.
void plan_operand(aclOpExecutor* ex, int slot, const aclTensor* t, int bytes, bool output, Rows* r)
{
    plan_rows(ex, slot, t, bytes, output, r);
    const PlannedPtr& p = ex->operands[slot];
    r->ptr = p.in_workspace ? nullptr : p.direct;
}

}  // namespace

namespace opscv {

hipError_t launch_block_plan(void* workspace, const aclOpExecutor* ex, hipStream_t stream)
{
    const auto at = [&](int slot) { return resolve(ex->operands[slot], workspace); };
    switch (ex->kind) {
        case OpKind::LayerNorm: {
            LayerNormArgs a = ex->layer_norm;
            a.x.ptr = at(kLnX);
            a.residual.ptr = at(kLnResidual);
            a.weight = at(kLnWeight);
            a.bias = at(kLnBias);
            a.y.ptr = at(kLnY);
            a.sum.ptr = at(kLnSum);
            a.mean = (float*)at(kLnMean);
            a.rstd = (float*)at(kLnRstd);
            return launch_layer_norm(a, stream);
        }
        case OpKind::LayerNormGrad: {
            LayerNormGradArgs a = ex->layer_norm_grad;
            a.grad_y.ptr = at(kLgY);
            a.grad_sum.ptr = at(kLgSumGrad);
            a.sum.ptr = at(kLgSum);
            a.weight = at(kLgWeight);
            a.mean = (const float*)at(kLgMean);
            a.rstd = (const float*)at(kLgRstd);
            a.grad_x.ptr = at(kLgX);
            a.grad_weight = at(kLgWeightGrad);
            a.grad_bias = at(kLgBiasGrad);
            a.partial = (float*)at(kLgScratch);
            return launch_layer_norm_grad(a, stream);
        }
        case OpKind::Dropout: {
            DropoutArgs a = ex->dropout;
            a.x.ptr = at(kDrX);
            a.residual.ptr = at(kDrResidual);
            a.state = (const int64_t*)at(kDrState);
            a.y.ptr = at(kDrY);
            return launch_dropout(a, stream);
        }
        case OpKind::Gated: {
            GatedArgs a = ex->gated;
            a.x.ptr = at(kGaX);
            a.gate_weight.ptr = at(kGaGateWeight);
            a.up_weight.ptr = at(kGaUpWeight);
            a.gate_bias = at(kGaGateBias);
            a.up_bias = at(kGaUpBias);
            a.y.ptr = at(kGaY);
            a.gate.ptr = at(kGaGate);
            a.up.ptr = at(kGaUp);
            a.scratch = (char*)at(kGaScratch);
            return launch_gated(a, stream);
        }
        case OpKind::GatedGrad: {
            GatedArgs a = ex->gated;
            a.grad_y.ptr = at(kGgY);
            a.x.ptr = at(kGgX);
            a.gate_weight.ptr = at(kGgGateWeight);
            a.up_weight.ptr = at(kGgUpWeight);
            a.gate.ptr = at(kGgGate);
            a.up.ptr = at(kGgUp);
            a.grad_x.ptr = at(kGgGradX);
            a.grad_gate_weight.ptr = at(kGgGradGateWeight);
            a.grad_up_weight.ptr = at(kGgGradUpWeight);
            a.grad_gate_bias = at(kGgGradGateBias);
            a.grad_up_bias = at(kGgGradUpBias);
            a.scratch = (char*)at(kGgScratch);
            return launch_gated_grad(a, stream);
        }
        default: return hipErrorInvalidValue;
    }
}

}  // namespace opscv

extern "C" {

aclnnStatus opscvLayerNormGetWorkspaceSize(const aclTensor* x, const aclTensor* residual, const aclTensor* weight,
                                           const aclTensor* bias, double eps, aclTensor* y, aclTensor* sum, aclTensor* mean,
                                           aclTensor* rstd, uint64_t* workspaceSize, aclOpExecutor** executor)
{
    const char* const api = "opscvLayerNorm";
    Executor ex;
    OPSCV_CHECK(begin(api, workspaceSize, executor, &ex));
    if (x == nullptr || y == nullptr) {
        return missing(api, "x and y");
    }
    LayerNormArgs& a = ex->layer_norm;
    Elem e;
    OPSCV_CHECK(norm_rows(api, x, &e, &a.rows, &a.width));
    a.elem = (int)e;
    aclDataType columns = ACL_DT_UNDEFINED;
    OPSCV_CHECK(check_columns(api, "weight", weight, x, &columns));
    OPSCV_CHECK(check_columns(api, "bias", bias, x, &columns));
    OPSCV_CHECK(check_rows(api, "y", y, x));
    if (residual != nullptr) {
        OPSCV_CHECK(check_rows(api, "residual", residual, x));
    }
    if (sum != nullptr) {
        OPSCV_CHECK(check_rows(api, "sum", sum, x));
    }
    if (mean != nullptr) {
        OPSCV_CHECK(check_row_values(api, "mean", mean, x));
    }
    if (rstd != nullptr) {
        OPSCV_CHECK(check_row_values(api, "rstd", rstd, x));
    }
    a.eps = (float)eps;
    if (!(eps >= 0.0) || !std::isfinite(a.eps)) {
        return invalid("%s: eps must be finite and not negative", api);
    }
    if (a.rows == 0) {
        return finish(api, ex, workspaceSize, executor);
    }
    ex->kind = OpKind::LayerNorm;
    a.weight_float = (e != Elem::F32 && columns == ACL_FLOAT) ? 1 : 0;
    const int bytes = elem_size(e);
    plan_rows(ex.get(), kLnX, x, bytes, false, &a.x);
    if (residual != nullptr) {
        plan_rows(ex.get(), kLnResidual, residual, bytes, false, &a.residual);
    }
    if (weight != nullptr) {
        plan_dense(ex.get(), kLnWeight, weight, columns_bytes(weight, bytes), false);
    }
    if (bias != nullptr) {
        plan_dense(ex.get(), kLnBias, bias, columns_bytes(bias, bytes), false);
    }
    plan_rows(ex.get(), kLnY, y, bytes, true, &a.y);
    if (sum != nullptr) {
        plan_rows(ex.get(), kLnSum, sum, bytes, true, &a.sum);
    }
    if (mean != nullptr) {
        plan_dense(ex.get(), kLnMean, mean, 4, true);
    }
    if (rstd != nullptr) {
        plan_dense(ex.get(), kLnRstd, rstd, 4, true);
    }
    return finish(api, ex, workspaceSize, executor);
}

aclnnStatus opscvLayerNorm(void* workspace, uint64_t workspaceSize, aclOpExecutor* executor, aclrtStream stream)
{
    return run_executor(workspace, workspaceSize, executor, stream, OpKind::LayerNorm, "opscvLayerNorm");
}

aclnnStatus opscvLayerNormBackwardGetWorkspaceSize(const aclTensor* gradY, const aclTensor* gradSum, const aclTensor* sum,
                                                   const aclTensor* weight, const aclTensor* mean, const aclTensor* rstd,
                                                   aclTensor* gradX, aclTensor* gradWeight, aclTensor* gradBias,
                                                   uint64_t* workspaceSize, aclOpExecutor** executor)
{
    const char* const api = "opscvLayerNormBackward";
    Executor ex;
    OPSCV_CHECK(begin(api, workspaceSize, executor, &ex));
    if (gradY == nullptr || sum == nullptr || mean == nullptr || rstd == nullptr || gradX == nullptr) {
        return missing(api, "gradY, sum, mean, rstd and gradX");
    }
    LayerNormGradArgs& a = ex->layer_norm_grad;
    Elem e;
    OPSCV_CHECK(norm_rows(api, sum, &e, &a.rows, &a.width));
    a.elem = (int)e;
    OPSCV_CHECK(check_rows(api, "gradY", gradY, sum));
    OPSCV_CHECK(check_rows(api, "gradX", gradX, sum));
    if (gradSum != nullptr) {
        OPSCV_CHECK(check_rows(api, "gradSum", gradSum, sum));
    }
    aclDataType columns = ACL_DT_UNDEFINED;
    OPSCV_CHECK(check_columns(api, "weight", weight, sum, &columns));
    OPSCV_CHECK(check_columns(api, "gradWeight", gradWeight, sum, &columns));
    OPSCV_CHECK(check_columns(api, "gradBias", gradBias, sum, &columns));
    OPSCV_CHECK(check_row_values(api, "mean", mean, sum));
    OPSCV_CHECK(check_row_values(api, "rstd", rstd, sum));
    if (a.rows == 0 && gradWeight == nullptr && gradBias == nullptr) {
        return finish(api, ex, workspaceSize, executor);
    }
    ex->kind = OpKind::LayerNormGrad;
    a.weight_float = (e != Elem::F32 && columns == ACL_FLOAT) ? 1 : 0;
    const int bytes = elem_size(e);
    plan_rows(ex.get(), kLgY, gradY, bytes, false, &a.grad_y);
    if (gradSum != nullptr) {
        plan_rows(ex.get(), kLgSumGrad, gradSum, bytes, false, &a.grad_sum);
    }
    plan_rows(ex.get(), kLgSum, sum, bytes, false, &a.sum);
    if (weight != nullptr) {
        plan_dense(ex.get(), kLgWeight, weight, columns_bytes(weight, bytes), false);
    }
    plan_dense(ex.get(), kLgMean, mean, 4, false);
    plan_dense(ex.get(), kLgRstd, rstd, 4, false);
    plan_rows(ex.get(), kLgX, gradX, bytes, true, &a.grad_x);
    if (gradWeight != nullptr) {
        plan_dense(ex.get(), kLgWeightGrad, gradWeight, columns_bytes(gradWeight, bytes), true);
    }
    if (gradBias != nullptr) {
        plan_dense(ex.get(), kLgBiasGrad, gradBias, columns_bytes(gradBias, bytes), true);
    }
    if (gradWeight != nullptr || gradBias != nullptr) {
        plan_scratch(ex.get(), kLgScratch, 2 * layer_norm_grad_partials(a) * a.width);
    }
    return finish(api, ex, workspaceSize, executor);
}

aclnnStatus opscvLayerNormBackward(void* workspace, uint64_t workspaceSize, aclOpExecutor* executor, aclrtStream stream)
{
    return run_executor(workspace, workspaceSize, executor, stream, OpKind::LayerNormGrad, "opscvLayerNormBackward");
}

aclnnStatus opscvDropoutGetWorkspaceSize(const aclTensor* x, const aclTensor* residual, const aclTensor* state, double p,
                                         aclTensor* y, uint64_t* workspaceSize, aclOpExecutor** executor)
{
    const char* const api = "opscvDropout";
    Executor ex;
    OPSCV_CHECK(begin(api, workspaceSize, executor, &ex));
    if (x == nullptr || state == nullptr || y == nullptr) {
        return missing(api, "x, state and y");
    }
    DropoutArgs& a = ex->dropout;
    Elem e;
    OPSCV_CHECK(norm_rows(api, x, &e, &a.rows, &a.width));
    a.elem = (int)e;
    OPSCV_CHECK(check_rows(api, "y", y, x));
    if (residual != nullptr) {
        OPSCV_CHECK(check_rows(api, "residual", residual, x));
    }
    if (state->ndim != 1 || state->dims[0] != 2 || state->dtype != ACL_INT64) {
        return invalid("%s: state must be two INT64, seed and offset", api);
    }
    if (!(p >= 0.0) || !(p <= 1.0)) {
        return invalid("%s: p must be 0 to 1", api);
    }
    if (a.rows == 0) {
        return finish(api, ex, workspaceSize, executor);
    }
    ex->kind = OpKind::Dropout;
    a.threshold = (uint32_t)std::nearbyint(p * 65536.0);
    a.scale = a.threshold < 65536 ? (float)(65536.0 / (65536.0 - (double)a.threshold)) : 0.0f;
    const int bytes = elem_size(e);
    plan_rows(ex.get(), kDrX, x, bytes, false, &a.x);
    if (residual != nullptr) {
        plan_rows(ex.get(), kDrResidual, residual, bytes, false, &a.residual);
    }
    Whole w;
    plan_whole(ex.get(), kDrState, state, &w);
    a.state_stride = w.stride[0];
    plan_rows(ex.get(), kDrY, y, bytes, true, &a.y);
    return finish(api, ex, workspaceSize, executor);
}

aclnnStatus opscvDropout(void* workspace, uint64_t workspaceSize, aclOpExecutor* executor, aclrtStream stream)
{
    return run_executor(workspace, workspaceSize, executor, stream, OpKind::Dropout, "opscvDropout");
}

aclnnStatus opscvGatedProjectionGetWorkspaceSize(const aclTensor* x, const aclTensor* gateWeight, const aclTensor* upWeight,
                                                 const aclTensor* gateBias, const aclTensor* upBias, int64_t activation,
                                                 aclTensor* y, aclTensor* gate, aclTensor* up, uint64_t* workspaceSize,
                                                 aclOpExecutor** executor)
{
    const char* const api = "opscvGatedProjection";
    Executor ex;
    OPSCV_CHECK(begin(api, workspaceSize, executor, &ex));
    if (x == nullptr || gateWeight == nullptr || upWeight == nullptr || y == nullptr ||
        (gateBias == nullptr) != (upBias == nullptr) || (gate == nullptr) != (up == nullptr)) {
        return missing(api, "x, both weights and y, and one bias or sum beside the other,");
    }
    GatedArgs& a = ex->gated;
    OPSCV_CHECK(check_gated(api, x, gateWeight, upWeight, activation, kMostExtent, &a));
    OPSCV_CHECK(check_rows_of(api, "y", y, x, a.inner));
    if (gate != nullptr) {
        OPSCV_CHECK(check_rows_of(api, "gate", gate, x, a.inner));
        OPSCV_CHECK(check_rows_of(api, "up", up, x, a.inner));
    }
    if (gateBias != nullptr) {
        OPSCV_CHECK(check_vector(api, "gateBias", gateBias, a, x->dtype));
        OPSCV_CHECK(check_vector(api, "upBias", upBias, a, x->dtype));
    }
    if (a.rows == 0) {
        return finish(api, ex, workspaceSize, executor);
    }
    ex->kind = OpKind::Gated;
    OPSCV_CHECK(check_plan(api, prod::gated_plan(a), &a));
    const int bytes = elem_size((Elem)a.elem);
    plan_operand(ex.get(), kGaX, x, bytes, false, &a.x);
    plan_operand(ex.get(), kGaGateWeight, gateWeight, bytes, false, &a.gate_weight);
    plan_operand(ex.get(), kGaUpWeight, upWeight, bytes, false, &a.up_weight);
    if (gateBias != nullptr) {
        plan_dense(ex.get(), kGaGateBias, gateBias, bytes, false);
        plan_dense(ex.get(), kGaUpBias, upBias, bytes, false);
    }
    plan_rows(ex.get(), kGaY, y, bytes, true, &a.y);
    if (gate != nullptr) {
        plan_rows(ex.get(), kGaGate, gate, bytes, true, &a.gate);
        plan_rows(ex.get(), kGaUp, up, bytes, true, &a.up);
    }
    plan_bytes(ex.get(), kGaScratch, gated_scratch_bytes(a));
    return finish(api, ex, workspaceSize, executor);
}

aclnnStatus opscvGatedProjection(void* workspace, uint64_t workspaceSize, aclOpExecutor* executor, aclrtStream stream)
{
    return run_executor(workspace, workspaceSize, executor, stream, OpKind::Gated, "opscvGatedProjection");
}

aclnnStatus opscvGatedProjectionBackwardGetWorkspaceSize(const aclTensor* gradY, const aclTensor* x,
                                                         const aclTensor* gateWeight, const aclTensor* upWeight,
                                                         const aclTensor* gate, const aclTensor* up, int64_t activation,
                                                         aclTensor* gradX, aclTensor* gradGateWeight,
                                                         aclTensor* gradUpWeight, aclTensor* gradGateBias,
                                                         aclTensor* gradUpBias, uint64_t* workspaceSize,
                                                         aclOpExecutor** executor)
{
    const char* const api = "opscvGatedProjectionBackward";
    Executor ex;
    OPSCV_CHECK(begin(api, workspaceSize, executor, &ex));
    if (gradY == nullptr || x == nullptr || gateWeight == nullptr || upWeight == nullptr || gate == nullptr ||
        up == nullptr || (gradGateWeight == nullptr) != (gradUpWeight == nullptr) ||
        (gradGateBias == nullptr) != (gradUpBias == nullptr) ||
        (gradX == nullptr && gradGateWeight == nullptr && gradGateBias == nullptr)) {
        return missing(api, "gradY, x, both weights and both sums, a gradient, and one weight's or bias's beside the other,");
    }
    GatedArgs& a = ex->gated;
    OPSCV_CHECK(check_gated(api, x, gateWeight, upWeight, activation, kMostGatedRows, &a));
    OPSCV_CHECK(check_rows_of(api, "gradY", gradY, x, a.inner));
    OPSCV_CHECK(check_rows_of(api, "gate", gate, x, a.inner));
    OPSCV_CHECK(check_rows_of(api, "up", up, x, a.inner));
    if (gradX != nullptr) {
        OPSCV_CHECK(check_rows(api, "gradX", gradX, x));
    }
    if (gradGateWeight != nullptr) {
        OPSCV_CHECK(check_matrix(api, "gradGateWeight", gradGateWeight, a, x->dtype));
        OPSCV_CHECK(check_matrix(api, "gradUpWeight", gradUpWeight, a, x->dtype));
    }
    if (gradGateBias != nullptr) {
        OPSCV_CHECK(check_vector(api, "gradGateBias", gradGateBias, a, x->dtype));
        OPSCV_CHECK(check_vector(api, "gradUpBias", gradUpBias, a, x->dtype));
    }
    if (a.rows == 0 && gradGateWeight == nullptr && gradGateBias == nullptr) {
        return finish(api, ex, workspaceSize, executor);
    }
    ex->kind = OpKind::GatedGrad;
    a.want_x = gradX != nullptr && a.rows > 0 ? 1 : 0;
    a.want_weights = gradGateWeight != nullptr ? 1 : 0;
    a.want_biases = gradGateBias != nullptr ? 1 : 0;
    if (a.want_x != 0 || a.want_weights != 0) {
        OPSCV_CHECK(check_plan(api, prod::gated_grad_plan(a), &a));
    }
    const int bytes = elem_size((Elem)a.elem);
    plan_rows(ex.get(), kGgY, gradY, bytes, false, &a.grad_y);
    if (a.want_weights != 0) {
        plan_operand(ex.get(), kGgX, x, bytes, false, &a.x);
    }
    if (a.want_x != 0) {
        plan_operand(ex.get(), kGgGateWeight, gateWeight, bytes, false, &a.gate_weight);
        plan_operand(ex.get(), kGgUpWeight, upWeight, bytes, false, &a.up_weight);
    }
    plan_rows(ex.get(), kGgGate, gate, bytes, false, &a.gate);
    plan_rows(ex.get(), kGgUp, up, bytes, false, &a.up);
    if (a.want_x != 0) {
        plan_rows(ex.get(), kGgGradX, gradX, bytes, true, &a.grad_x);
    }
    if (a.want_weights != 0) {
        plan_rows(ex.get(), kGgGradGateWeight, gradGateWeight, bytes, true, &a.grad_gate_weight);
        plan_rows(ex.get(), kGgGradUpWeight, gradUpWeight, bytes, true, &a.grad_up_weight);
    }
    if (a.want_biases != 0) {
        plan_dense(ex.get(), kGgGradGateBias, gradGateBias, bytes, true);
        plan_dense(ex.get(), kGgGradUpBias, gradUpBias, bytes, true);
    }
    plan_bytes(ex.get(), kGgScratch, gated_grad_scratch_bytes(a));
    return finish(api, ex, workspaceSize, executor);
}

aclnnStatus opscvGatedProjectionBackward(void* workspace, uint64_t workspaceSize, aclOpExecutor* executor,
                                         aclrtStream stream)
{
    return run_executor(workspace, workspaceSize, executor, stream, OpKind::GatedGrad, "opscvGatedProjectionBackward");
}

}  // extern "C"
