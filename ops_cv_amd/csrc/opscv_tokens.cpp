// Operators on token sequences: parameter validation, planning and the second-phase entries (include/opscv_tokens.h).
#include <cmath>
#include <cstring>
#include <memory>
#include <new>

#include "executor.hpp"
#include "kernels.hpp"
#include "opscv_tokens.h"
#include "token_kernels.hpp"

using namespace opscv;

namespace {

constexpr int64_t kMostExtent = (int64_t)1 << 30;
constexpr int64_t kMostTokenStride = (int64_t)1 << 22;  // elements
// tokens of a sequence and reaches of a window: sums of any three fit 32 bits
constexpr int64_t kMostTokens = (int64_t)1 << 28;
constexpr int64_t kMostHeadDim = 256;
constexpr int64_t kMostRotaryDim = 1024;

typedef std::unique_ptr<aclOpExecutor> Executor;

// What both arguments that return something are checked for, and the executor of the call.
aclnnStatus begin(const char* api, uint64_t* workspaceSize, aclOpExecutor** executor, Executor* ex)
{
    if (workspaceSize == nullptr || executor == nullptr) {
        set_error("%s: workspaceSize and executor must not be NULL", api);
        return ACLNN_ERR_PARAM_NULLPTR;
    }
    ex->reset(new (std::nothrow) aclOpExecutor());
    if (!*ex) {
        set_error("%s: cannot allocate the executor", api);
        return ACLNN_ERR_INNER_CREATE_EXECUTOR;
    }
    return ACLNN_SUCCESS;
}

aclnnStatus finish(const char* api, Executor& ex, uint64_t* workspaceSize, aclOpExecutor** executor)
{
    if (const aclnnStatus ps = plan_status(ex.get(), api); ps != ACLNN_SUCCESS) {
        return ps;
    }
    *workspaceSize = ex->workspace_bytes;
    *executor = ex.release();
    return ACLNN_SUCCESS;
}

aclnnStatus missing(const char* api, const char* names)
{
    set_error("%s: %s must not be NULL", api, names);
    return ACLNN_ERR_PARAM_NULLPTR;
}

template <typename... A>
aclnnStatus invalid(const char* format, A... a)
{
    set_error(format, a...);
    return ACLNN_ERR_PARAM_INVALID;
}

bool same_dims(const aclTensor* a, const aclTensor* b)
{
    return a->ndim == b->ndim && memcmp(a->dims, b->dims, sizeof(int64_t) * (size_t)a->ndim) == 0;
}

// the leading dimensions of `t`, one value per row
bool per_row(const aclTensor* r, const aclTensor* t)
{
    return r->ndim == t->ndim - 1 && memcmp(r->dims, t->dims, sizeof(int64_t) * (size_t)r->ndim) == 0;
}

bool extents_fit(const aclTensor* t)
{
    for (int64_t i = 0; i < t->ndim; i++) {
        if (t->dims[i] > kMostExtent) {
            return false;
        }
    }
    return true;
}

// Operand `slot` of the executor: the tensor packed dense.
void plan_dense(aclOpExecutor* ex, int slot, const aclTensor* t, int elem_bytes, bool output)
{
    ex->operands[slot] = plan_view(ex, t, elem_bytes, output);
    ex->required |= t->empty() ? 0u : 1u << slot;
}

// Operand `slot`, used in place where its last dimension is dense, packed otherwise; the strides that the kernel walks.
void plan_strided(aclOpExecutor* ex, int slot, const aclTensor* t, int elem_bytes, bool output, Strided* s)
{
    const int last = (int)t->ndim - 1;
    bool in_place = t->dims[last] == 1 || t->strides[last] == 1;
    // kernels walk up to 64 tokens, of which none begins inside another, from a 64-bit address with 32-bit offsets in bytes
    for (int i = 0; i < last; i++) {
        in_place = in_place && (t->dims[i] <= 1 || (t->strides[i] >= 0 && (i != 1 || (t->strides[i] >= t->dims[last] &&
                                                                                       t->strides[i] <= kMostTokenStride))));
    }
    if (in_place) {
        PlannedPtr p;
        p.direct = (t->data == nullptr) ? nullptr : (char*)t->data + t->offset * (int64_t)elem_bytes;
        ex->operands[slot] = p;
        ex->required |= t->empty() ? 0u : 1u << slot;
        for (int i = 0; i < last; i++) {
            s->stride[i] = t->dims[i] > 1 ? t->strides[i] : (i == 1 ? t->dims[last] : 0);
        }
        return;
    }
    plan_dense(ex, slot, t, elem_bytes, output);
    int64_t stride = t->dims[last];
    for (int i = last - 1; i >= 0; i--) {
        s->stride[i] = stride;
        stride *= t->dims[i];
    }
}

// Operand `slot` as rows of its last dimension: in place where the leading dimensions are evenly spaced rows.
void plan_rows(aclOpExecutor* ex, int slot, const aclTensor* t, int elem_bytes, bool output, Rows* r)
{
    const int last = (int)t->ndim - 1;
    bool even = t->dims[last] == 1 || t->strides[last] == 1;
    int64_t stride = 0, expect = 0;  // of the innermost dimension of more than one row; of the next one outwards
    for (int i = last - 1; i >= 0 && even; i--) {
        if (t->dims[i] == 1) {
            continue;
        }
        if (expect == 0) {
            stride = t->strides[i];
            expect = stride * t->dims[i];
            even = stride > 0 || !output;
        } else {
            even = t->strides[i] == expect;
            expect *= t->dims[i];
        }
        even = even && expect != 0;
    }
    if (even) {
        PlannedPtr p;
        p.direct = (t->data == nullptr) ? nullptr : (char*)t->data + t->offset * (int64_t)elem_bytes;
        ex->operands[slot] = p;
        ex->required |= t->empty() ? 0u : 1u << slot;
        r->row_stride = stride;
        return;
    }
    plan_dense(ex, slot, t, elem_bytes, output);
    r->row_stride = t->dims[last];
}

// A vector or matrix of whole numbers, always read in place.
void plan_whole(aclOpExecutor* ex, int slot, const aclTensor* t, Whole* w)
{
    w->wide = t->dtype == ACL_INT64 ? 1 : 0;
    for (int i = 0; i < t->ndim; i++) {
        w->stride[i] = t->strides[i];
    }
    ex->operands[slot].direct = (t->data == nullptr) ? nullptr : (char*)t->data + t->offset * (w->wide ? 8 : 4);
    ex->required |= t->empty() ? 0u : 1u << slot;
}

void plan_scratch(aclOpExecutor* ex, int slot, int64_t floats)
{
    if (floats > 0) {
        PlannedPtr p;
        p.in_workspace = true;
        p.ws_offset = (ex->workspace_bytes + 255) / 256 * 256;
        ex->workspace_bytes = p.ws_offset + (uint64_t)floats * 4;
        ex->operands[slot] = p;
    }
}

bool whole_type(const aclTensor* t) { return t->dtype == ACL_INT32 || t->dtype == ACL_INT64; }

// Weight of a norm: (width), of the activations' type or FLOAT.
aclnnStatus check_weight(const char* api, const char* name, const aclTensor* w, const aclTensor* x)
{
    if (w->ndim != 1 || w->dims[0] != x->dims[x->ndim - 1]) {
        return invalid("%s: %s must have one dimension, the width of the rows", api, name);
    }
    if (w->dtype != x->dtype && w->dtype != ACL_FLOAT) {
        return invalid("%s: %s must have the type of the rows or FLOAT", api, name);
    }
    return ACLNN_SUCCESS;
}

// Rows of one type and shape
aclnnStatus check_rows(const char* api, const char* name, const aclTensor* t, const aclTensor* like, bool dtype = true)
{
    if (!same_dims(t, like)) {
        return invalid("%s: %s has another shape than the other rows", api, name);
    }
    if (dtype && t->dtype != like->dtype) {
        return invalid("%s: %s has another type than the other rows", api, name);
    }
    return ACLNN_SUCCESS;
}

aclnnStatus check_row_values(const char* api, const char* name, const aclTensor* t, const aclTensor* like)
{
    if (!per_row(t, like) || t->dtype != ACL_FLOAT) {
        return invalid("%s: %s must hold one FLOAT per row", api, name);
    }
    return ACLNN_SUCCESS;
}

#define OPSCV_CHECK(call)                                    \
    if (const aclnnStatus st_ = (call); st_ != ACLNN_SUCCESS) { \
        return st_;                                          \
    }

// What the rows of a norm must be; their number and width.
aclnnStatus norm_rows(const char* api, const aclTensor* x, Elem* e, int64_t* rows, int64_t* width)
{
    if (x->ndim < 1 || x->ndim > kViewDims) {
        return invalid("%s: rows have one to %d dimensions, got %lld", api, kViewDims, (long long)x->ndim);
    }
    if (!elem_of(x->dtype, e)) {
        return invalid("%s: dtype %d is not in {FLOAT, FLOAT16, BF16}", api, (int)x->dtype);
    }
    *width = x->dims[x->ndim - 1];
    *rows = 1;
    for (int i = 0; i + 1 < x->ndim; i++) {
        *rows *= x->dims[i];
    }
    if (*width < 1 || *width > kMostExtent || *rows > INT32_MAX) {
        return invalid("%s: rows of 1 to 2^30 elements and fewer than 2^31 rows, got %lld by %lld", api, (long long)*rows,
                       (long long)*width);
    }
    return ACLNN_SUCCESS;
}

// The operands that attention's two directions share.
aclnnStatus check_attention(const char* api, const aclTensor* q, const aclTensor* k, const aclTensor* v,
                            const aclTensor* q_lengths, const aclTensor* kv_lengths, double scale, int64_t left,
                            int64_t right, int64_t sinks, AttentionArgs* a)
{
    Elem e;
    if (q->ndim != 4 || k->ndim != 4 || !same_dims(k, v)) {
        return invalid("%s: query, key and value have four dimensions, key and value the same", api);
    }
    if (!elem_of(q->dtype, &e) || k->dtype != q->dtype || v->dtype != q->dtype) {
        return invalid("%s: query, key and value must have one type of {FLOAT, FLOAT16, BF16}", api);
    }
    a->elem = (int)e;
    a->batch = q->dims[0];
    a->tokens = q->dims[1];
    a->heads = q->dims[2];
    a->d = q->dims[3];
    a->kv_tokens = k->dims[1];
    a->kv_heads = k->dims[2];
    if (k->dims[0] != a->batch || k->dims[3] != a->d) {
        return invalid("%s: key and value must have the batch and the head size of query", api);
    }
    if (a->d < 1 || a->d > kMostHeadDim) {
        return invalid("%s: heads of 1 to %lld features, got %lld", api, (long long)kMostHeadDim, (long long)a->d);
    }
    if (a->kv_heads < 1 || a->heads < 1 || a->heads % a->kv_heads != 0) {
        return invalid("%s: %lld heads cannot share %lld key heads", api, (long long)a->heads, (long long)a->kv_heads);
    }
    if (!extents_fit(q) || !extents_fit(k) || a->batch * a->heads > INT32_MAX || a->tokens > kMostTokens ||
        a->kv_tokens > kMostTokens || a->tokens * a->heads > kMostExtent) {
        return invalid("%s: extents too large", api);
    }
    for (const aclTensor* n : {q_lengths, kv_lengths}) {
        if (n != nullptr && (n->ndim != 1 || n->dims[0] != a->batch || !whole_type(n))) {
            return invalid("%s: lengths must be one INT32 or INT64 per sequence", api);
        }
    }
    if (left < 0 || right < 0 || sinks < 0) {
        return invalid("%s: left, right and sinks must not be negative", api);
    }
    a->scale = (float)scale;
    if (!std::isfinite(a->scale) || !(a->scale > 0.0f)) {
        return invalid("%s: scale must be positive and finite", api);
    }
    a->left = left < kMostTokens ? left : kMostTokens;
    a->right = right < kMostTokens ? right : kMostTokens;
    a->sinks = sinks < kMostTokens ? sinks : kMostTokens;
    a->compute_units = compute_unit_count();
    return ACLNN_SUCCESS;
}

aclnnStatus check_lse(const char* api, const aclTensor* lse, const AttentionArgs& a)
{
    if (lse->ndim != 3 || lse->dims[0] != a.batch || lse->dims[1] != a.heads || lse->dims[2] != a.tokens ||
        lse->dtype != ACL_FLOAT) {
        return invalid("%s: lse must be FLOAT (batch, heads, tokens)", api);
    }
    return ACLNN_SUCCESS;
}

void plan_lse(aclOpExecutor* ex, int slot, const aclTensor* lse, Strided* s)
{
    for (int i = 0; i < 3; i++) {
        s->stride[i] = lse->strides[i];
    }
    ex->operands[slot].direct = (lse->data == nullptr) ? nullptr : (char*)lse->data + lse->offset * 4;
    ex->required |= lse->empty() ? 0u : 1u << slot;
}

// slots of aclOpExecutor::operands
enum NormSlot { kNormX, kNormResidual, kNormWeight, kNormY, kNormScale, kNormSum, kNormRstd };
enum NormGradSlot { kNgY, kNgSumGrad, kNgSum, kNgWeight, kNgRstd, kNgX, kNgWeightGrad, kNgScratch };
enum RotarySlot { kRoQuery, kRoKey, kRoPositions, kRoTable, kRoQueryOut, kRoKeyOut };
enum AttentionSlot { kAtQ, kAtK, kAtV, kAtQLengths, kAtKvLengths, kAtOut, kAtLse, kAtGradOut, kAtGradQ, kAtGradK, kAtGradV,
                     kAtScratch };

}  // namespace

namespace opscv {

aclnnStatus execute_token_plan(void* workspace, const aclOpExecutor* ex, hipStream_t stream, const char* api,
                               hipError_t* e)
{
    for (int i = 0; i < aclOpExecutor::kOperands; i++) {
        if ((ex->required >> i & 1u) != 0 && resolve(ex->operands[i], workspace) == nullptr) {
            set_error("%s: tensor data pointer is NULL", api);
            return ACLNN_ERR_PARAM_NULLPTR;
        }
    }
    const auto at = [&](int slot) { return resolve(ex->operands[slot], workspace); };
    switch (ex->kind) {
        case OpKind::ResidualNorm: {
            NormArgs a = ex->norm;
            a.x.ptr = at(kNormX);
            a.residual.ptr = at(kNormResidual);
            a.weight = at(kNormWeight);
            a.y.ptr = at(kNormY);
            a.scale = (float*)at(kNormScale);
            a.sum.ptr = at(kNormSum);
            a.rstd = (float*)at(kNormRstd);
            *e = launch_residual_norm(a, stream);
            break;
        }
        case OpKind::ResidualNormGrad: {
            NormGradArgs a = ex->norm_grad;
            a.grad_y.ptr = at(kNgY);
            a.grad_sum.ptr = at(kNgSumGrad);
            a.sum.ptr = at(kNgSum);
            a.weight = at(kNgWeight);
            a.rstd = (const float*)at(kNgRstd);
            a.grad_x.ptr = at(kNgX);
            a.grad_weight = at(kNgWeightGrad);
            a.partial = (float*)at(kNgScratch);
            *e = launch_residual_norm_grad(a, stream);
            break;
        }
        case OpKind::RotaryTable: {
            RotaryTableArgs a = ex->rotary_table;
            a.table = (float*)at(kRoTable);
            *e = launch_rotary_table(a, stream);
            break;
        }
        case OpKind::Rotary: {
            RotaryArgs a = ex->rotary;
            a.query.ptr = at(kRoQuery);
            a.key.ptr = at(kRoKey);
            a.position.ptr = at(kRoPositions);
            a.table = (const float*)at(kRoTable);
            a.query_out.ptr = at(kRoQueryOut);
            a.key_out.ptr = at(kRoKeyOut);
            *e = launch_rotary(a, stream);
            break;
        }
        default: {
            AttentionArgs a = ex->attention;
            a.q.ptr = at(kAtQ);
            a.k.ptr = at(kAtK);
            a.v.ptr = at(kAtV);
            a.q_lengths.ptr = at(kAtQLengths);
            a.kv_lengths.ptr = at(kAtKvLengths);
            a.out.ptr = at(kAtOut);
            a.lse.ptr = at(kAtLse);
            a.grad_out.ptr = at(kAtGradOut);
            a.grad_q.ptr = at(kAtGradQ);
            a.grad_k.ptr = at(kAtGradK);
            a.grad_v.ptr = at(kAtGradV);
            a.scratch = (float*)at(kAtScratch);
            *e = ex->kind == OpKind::WindowAttention ? launch_window_attention(a, stream)
                                                     : launch_window_attention_grad(a, stream);
            break;
        }
    }
    return ACLNN_SUCCESS;
}

}  // namespace opscv

extern "C" {

aclnnStatus opscvResidualNormGetWorkspaceSize(const aclTensor* x, const aclTensor* residual, const aclTensor* weight,
                                              double eps, aclTensor* y, aclTensor* scale, aclTensor* sum,
                                              aclTensor* rstd, uint64_t* workspaceSize, aclOpExecutor** executor)
{
    const char* const api = "opscvResidualNorm";
    Executor ex;
    OPSCV_CHECK(begin(api, workspaceSize, executor, &ex));
    if (x == nullptr || weight == nullptr || y == nullptr) {
        return missing(api, "x, weight and y");
    }
    NormArgs& a = ex->norm;
    Elem e;
    OPSCV_CHECK(norm_rows(api, x, &e, &a.rows, &a.width));
    a.elem = (int)e;
    a.int8 = y->dtype == ACL_INT8 ? 1 : 0;
    OPSCV_CHECK(check_weight(api, "weight", weight, x));
    OPSCV_CHECK(check_rows(api, "y", y, x, a.int8 == 0));
    if (residual != nullptr) {
        OPSCV_CHECK(check_rows(api, "residual", residual, x));
    }
    if (sum != nullptr) {
        OPSCV_CHECK(check_rows(api, "sum", sum, x));
    }
    if (a.int8 != 0 && scale == nullptr) {
        return missing(api, "scale of an INT8 y");
    }
    if (scale != nullptr) {
        if (a.int8 == 0) {
            return invalid("%s: scale goes with an INT8 y only", api);
        }
        OPSCV_CHECK(check_row_values(api, "scale", scale, x));
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
    ex->kind = OpKind::ResidualNorm;
    a.weight_float = (e != Elem::F32 && weight->dtype == ACL_FLOAT) ? 1 : 0;
    const int bytes = elem_size(e);
    plan_rows(ex.get(), kNormX, x, bytes, false, &a.x);
    if (residual != nullptr) {
        plan_rows(ex.get(), kNormResidual, residual, bytes, false, &a.residual);
    }
    plan_dense(ex.get(), kNormWeight, weight, weight->dtype == ACL_FLOAT ? 4 : bytes, false);
    plan_rows(ex.get(), kNormY, y, a.int8 != 0 ? 1 : bytes, true, &a.y);
    if (scale != nullptr) {
        plan_dense(ex.get(), kNormScale, scale, 4, true);
    }
    if (sum != nullptr) {
        plan_rows(ex.get(), kNormSum, sum, bytes, true, &a.sum);
    }
    if (rstd != nullptr) {
        plan_dense(ex.get(), kNormRstd, rstd, 4, true);
    }
    return finish(api, ex, workspaceSize, executor);
}

aclnnStatus opscvResidualNorm(void* workspace, uint64_t workspaceSize, aclOpExecutor* executor, aclrtStream stream)
{
    return run_executor(workspace, workspaceSize, executor, stream, OpKind::ResidualNorm, "opscvResidualNorm");
}

aclnnStatus opscvResidualNormBackwardGetWorkspaceSize(const aclTensor* gradY, const aclTensor* gradSum,
                                                      const aclTensor* sum, const aclTensor* weight,
                                                      const aclTensor* rstd, aclTensor* gradX, aclTensor* gradWeight,
                                                      uint64_t* workspaceSize, aclOpExecutor** executor)
{
    const char* const api = "opscvResidualNormBackward";
    Executor ex;
    OPSCV_CHECK(begin(api, workspaceSize, executor, &ex));
    if (gradY == nullptr || sum == nullptr || weight == nullptr || rstd == nullptr || gradX == nullptr) {
        return missing(api, "gradY, sum, weight, rstd and gradX");
    }
    NormGradArgs& a = ex->norm_grad;
    Elem e;
    OPSCV_CHECK(norm_rows(api, sum, &e, &a.rows, &a.width));
    a.elem = (int)e;
    OPSCV_CHECK(check_rows(api, "gradY", gradY, sum));
    OPSCV_CHECK(check_rows(api, "gradX", gradX, sum));
    if (gradSum != nullptr) {
        OPSCV_CHECK(check_rows(api, "gradSum", gradSum, sum));
    }
    OPSCV_CHECK(check_weight(api, "weight", weight, sum));
    OPSCV_CHECK(check_row_values(api, "rstd", rstd, sum));
    if (gradWeight != nullptr) {
        OPSCV_CHECK(check_weight(api, "gradWeight", gradWeight, sum));
        if (gradWeight->dtype != weight->dtype) {
            return invalid("%s: gradWeight must have the type of weight", api);
        }
    }
    if (a.rows == 0 && gradWeight == nullptr) {
        return finish(api, ex, workspaceSize, executor);
    }
    ex->kind = OpKind::ResidualNormGrad;
    a.weight_float = (e != Elem::F32 && weight->dtype == ACL_FLOAT) ? 1 : 0;
    const int bytes = elem_size(e), weight_bytes = weight->dtype == ACL_FLOAT ? 4 : bytes;
    plan_rows(ex.get(), kNgY, gradY, bytes, false, &a.grad_y);
    if (gradSum != nullptr) {
        plan_rows(ex.get(), kNgSumGrad, gradSum, bytes, false, &a.grad_sum);
    }
    plan_rows(ex.get(), kNgSum, sum, bytes, false, &a.sum);
    plan_dense(ex.get(), kNgWeight, weight, weight_bytes, false);
    plan_dense(ex.get(), kNgRstd, rstd, 4, false);
    plan_rows(ex.get(), kNgX, gradX, bytes, true, &a.grad_x);
    if (gradWeight != nullptr) {
        plan_dense(ex.get(), kNgWeightGrad, gradWeight, weight_bytes, true);
        plan_scratch(ex.get(), kNgScratch, norm_grad_partials(a) * a.width);
    }
    return finish(api, ex, workspaceSize, executor);
}

aclnnStatus opscvResidualNormBackward(void* workspace, uint64_t workspaceSize, aclOpExecutor* executor,
                                      aclrtStream stream)
{
    return run_executor(workspace, workspaceSize, executor, stream, OpKind::ResidualNormGrad,
                        "opscvResidualNormBackward");
}

aclnnStatus opscvRotaryTableGetWorkspaceSize(double base, int64_t scaling, double factor, int64_t originalLength,
                                             double magnitude, aclTensor* table, uint64_t* workspaceSize,
                                             aclOpExecutor** executor)
{
    const char* const api = "opscvRotaryTable";
    Executor ex;
    OPSCV_CHECK(begin(api, workspaceSize, executor, &ex));
    if (table == nullptr) {
        return missing(api, "table");
    }
    if (table->ndim != 2 || table->dtype != ACL_FLOAT || table->dims[1] < 2 || table->dims[1] % 2 != 0 ||
        table->dims[1] > kMostRotaryDim || table->dims[0] > kMostExtent) {
        return invalid("%s: table must be FLOAT (positions, rot) with an even rot of 2 to %lld", api,
                       (long long)kMostRotaryDim);
    }
    if (!(base > 1.0) || !std::isfinite(base) || !std::isfinite(magnitude)) {
        return invalid("%s: base must be finite and over 1, magnitude finite", api);
    }
    if (scaling < OPSCV_ROTARY_PLAIN || scaling > OPSCV_ROTARY_BY_PARTS) {
        return invalid("%s: unknown scaling %lld", api, (long long)scaling);
    }
    if (scaling != OPSCV_ROTARY_PLAIN && (!(factor >= 1.0) || !std::isfinite(factor))) {
        return invalid("%s: factor must be finite and 1 or more", api);
    }
    if (scaling == OPSCV_ROTARY_BASE && table->dims[1] <= 2) {
        return invalid("%s: a stretched base needs more than two rotated features", api);
    }
    if (scaling == OPSCV_ROTARY_BY_PARTS && originalLength < 1) {
        return invalid("%s: originalLength must be positive", api);
    }
    if (table->empty()) {
        return finish(api, ex, workspaceSize, executor);
    }
    ex->kind = OpKind::RotaryTable;
    RotaryTableArgs& a = ex->rotary_table;
    a.positions = table->dims[0];
    a.rot = table->dims[1];
    a.base = base;
    a.scaling = scaling;
    a.factor = scaling == OPSCV_ROTARY_PLAIN ? 1.0 : factor;
    a.original_length = originalLength;
    a.magnitude = magnitude;
    Rows r;
    plan_rows(ex.get(), kRoTable, table, 4, true, &r);
    a.row_stride = r.row_stride;
    return finish(api, ex, workspaceSize, executor);
}

aclnnStatus opscvRotaryTable(void* workspace, uint64_t workspaceSize, aclOpExecutor* executor, aclrtStream stream)
{
    return run_executor(workspace, workspaceSize, executor, stream, OpKind::RotaryTable, "opscvRotaryTable");
}

aclnnStatus opscvRotaryGetWorkspaceSize(const aclTensor* query, const aclTensor* key, const aclTensor* positions,
                                        const aclTensor* table, bool interleaved, bool inverse, aclTensor* queryOut,
                                        aclTensor* keyOut, uint64_t* workspaceSize, aclOpExecutor** executor)
{
    const char* const api = "opscvRotary";
    Executor ex;
    OPSCV_CHECK(begin(api, workspaceSize, executor, &ex));
    if (query == nullptr || table == nullptr || queryOut == nullptr || (key == nullptr) != (keyOut == nullptr)) {
        return missing(api, "query, table and queryOut, and one of key and keyOut beside the other,");
    }
    Elem e;
    if (query->ndim != 4 || !elem_of(query->dtype, &e)) {
        return invalid("%s: query must be (batch, tokens, heads, d) of {FLOAT, FLOAT16, BF16}", api);
    }
    OPSCV_CHECK(check_rows(api, "queryOut", queryOut, query));
    RotaryArgs& a = ex->rotary;
    a.elem = (int)e;
    a.batch = query->dims[0];
    a.tokens = query->dims[1];
    a.heads = query->dims[2];
    a.d = query->dims[3];
    if (key != nullptr) {
        if (key->ndim != 4 || key->dtype != query->dtype || key->dims[0] != a.batch || key->dims[1] != a.tokens ||
            key->dims[3] != a.d) {
            return invalid("%s: key must have query's type, batch, tokens and head size", api);
        }
        OPSCV_CHECK(check_rows(api, "keyOut", keyOut, key));
        a.kv_heads = key->dims[2];
    }
    if (table->ndim != 2 || table->dtype != ACL_FLOAT) {
        return invalid("%s: table must be FLOAT (positions, rot)", api);
    }
    a.positions = table->dims[0];
    a.rot = table->dims[1];
    if (a.d < 1 || a.d > kMostRotaryDim || a.rot % 2 != 0 || a.rot < 2 || a.rot > a.d) {
        return invalid("%s: an even number of rotated features out of 2 to %lld, got %lld of %lld", api,
                       (long long)kMostRotaryDim, (long long)a.rot, (long long)a.d);
    }
    if (positions != nullptr && (positions->ndim != 2 || positions->dims[0] != a.batch || positions->dims[1] != a.tokens ||
                                 !whole_type(positions))) {
        return invalid("%s: positions must be INT32 or INT64 (batch, tokens)", api);
    }
    if (!extents_fit(query) || !extents_fit(table) || a.kv_heads > kMostExtent || a.batch * a.tokens > INT32_MAX) {
        return invalid("%s: extents too large", api);
    }
    if (a.batch == 0 || a.tokens == 0 || a.heads + a.kv_heads == 0) {
        return finish(api, ex, workspaceSize, executor);
    }
    ex->kind = OpKind::Rotary;
    a.interleaved = interleaved ? 1 : 0;
    a.inverse = inverse ? 1 : 0;
    const int bytes = elem_size(e);
    plan_strided(ex.get(), kRoQuery, query, bytes, false, &a.query);
    plan_strided(ex.get(), kRoQueryOut, queryOut, bytes, true, &a.query_out);
    if (key != nullptr) {
        plan_strided(ex.get(), kRoKey, key, bytes, false, &a.key);
        plan_strided(ex.get(), kRoKeyOut, keyOut, bytes, true, &a.key_out);
    }
    if (positions != nullptr) {
        plan_whole(ex.get(), kRoPositions, positions, &a.position);
    }
    Rows r;
    plan_rows(ex.get(), kRoTable, table, 4, false, &r);
    a.table_stride = r.row_stride;
    return finish(api, ex, workspaceSize, executor);
}

aclnnStatus opscvRotary(void* workspace, uint64_t workspaceSize, aclOpExecutor* executor, aclrtStream stream)
{
    return run_executor(workspace, workspaceSize, executor, stream, OpKind::Rotary, "opscvRotary");
}

aclnnStatus opscvWindowAttentionGetWorkspaceSize(const aclTensor* query, const aclTensor* key, const aclTensor* value,
                                                 const aclTensor* qLengths, const aclTensor* kvLengths, double scale,
                                                 int64_t left, int64_t right, int64_t sinks, aclTensor* out,
                                                 aclTensor* lse, uint64_t* workspaceSize, aclOpExecutor** executor)
{
    const char* const api = "opscvWindowAttention";
    Executor ex;
    OPSCV_CHECK(begin(api, workspaceSize, executor, &ex));
    if (query == nullptr || key == nullptr || value == nullptr || out == nullptr) {
        return missing(api, "query, key, value and out");
    }
    AttentionArgs& a = ex->attention;
    OPSCV_CHECK(check_attention(api, query, key, value, qLengths, kvLengths, scale, left, right, sinks, &a));
    OPSCV_CHECK(check_rows(api, "out", out, query));
    if (lse != nullptr) {
        OPSCV_CHECK(check_lse(api, lse, a));
    }
    if (a.batch == 0 || a.tokens == 0) {
        return finish(api, ex, workspaceSize, executor);
    }
    const int64_t scratch = attention_scratch_floats(a);
    if (scratch < 0) {
        return invalid("%s: more rows of a sequence than a launch holds", api);
    }
    ex->kind = OpKind::WindowAttention;
    const int bytes = elem_size((Elem)a.elem);
    plan_strided(ex.get(), kAtQ, query, bytes, false, &a.q);
    plan_strided(ex.get(), kAtK, key, bytes, false, &a.k);
    plan_strided(ex.get(), kAtV, value, bytes, false, &a.v);
    plan_strided(ex.get(), kAtOut, out, bytes, true, &a.out);
    if (qLengths != nullptr) {
        plan_whole(ex.get(), kAtQLengths, qLengths, &a.q_lengths);
    }
    if (kvLengths != nullptr) {
        plan_whole(ex.get(), kAtKvLengths, kvLengths, &a.kv_lengths);
    }
    if (lse != nullptr) {
        plan_lse(ex.get(), kAtLse, lse, &a.lse);
    }
    plan_scratch(ex.get(), kAtScratch, scratch);
    return finish(api, ex, workspaceSize, executor);
}

aclnnStatus opscvWindowAttention(void* workspace, uint64_t workspaceSize, aclOpExecutor* executor, aclrtStream stream)
{
    return run_executor(workspace, workspaceSize, executor, stream, OpKind::WindowAttention, "opscvWindowAttention");
}

aclnnStatus opscvWindowAttentionBackwardGetWorkspaceSize(
    const aclTensor* gradOut, const aclTensor* query, const aclTensor* key, const aclTensor* value, const aclTensor* out,
    const aclTensor* lse, const aclTensor* qLengths, const aclTensor* kvLengths, double scale, int64_t left,
    int64_t right, int64_t sinks, aclTensor* gradQuery, aclTensor* gradKey, aclTensor* gradValue,
    uint64_t* workspaceSize, aclOpExecutor** executor)
{
    const char* const api = "opscvWindowAttentionBackward";
    Executor ex;
    OPSCV_CHECK(begin(api, workspaceSize, executor, &ex));
    if (gradOut == nullptr || query == nullptr || key == nullptr || value == nullptr || out == nullptr ||
        lse == nullptr || gradQuery == nullptr || gradKey == nullptr || gradValue == nullptr) {
        return missing(api, "every operand but the lengths");
    }
    AttentionArgs& a = ex->attention;
    OPSCV_CHECK(check_attention(api, query, key, value, qLengths, kvLengths, scale, left, right, sinks, &a));
    OPSCV_CHECK(check_rows(api, "gradOut", gradOut, query));
    OPSCV_CHECK(check_rows(api, "out", out, query));
    OPSCV_CHECK(check_rows(api, "gradQuery", gradQuery, query));
    OPSCV_CHECK(check_rows(api, "gradKey", gradKey, key));
    OPSCV_CHECK(check_rows(api, "gradValue", gradValue, key));
    OPSCV_CHECK(check_lse(api, lse, a));
    if (query->empty() && key->empty()) {
        return finish(api, ex, workspaceSize, executor);
    }
    const int64_t scratch = attention_grad_scratch_floats(a);
    if (scratch < 0) {
        return invalid("%s: more rows or keys of a sequence than a launch holds", api);
    }
    ex->kind = OpKind::WindowAttentionGrad;
    const int bytes = elem_size((Elem)a.elem);
    plan_strided(ex.get(), kAtQ, query, bytes, false, &a.q);
    plan_strided(ex.get(), kAtK, key, bytes, false, &a.k);
    plan_strided(ex.get(), kAtV, value, bytes, false, &a.v);
    plan_strided(ex.get(), kAtOut, out, bytes, false, &a.out);
    plan_strided(ex.get(), kAtGradOut, gradOut, bytes, false, &a.grad_out);
    plan_strided(ex.get(), kAtGradQ, gradQuery, bytes, true, &a.grad_q);
    plan_strided(ex.get(), kAtGradK, gradKey, bytes, true, &a.grad_k);
    plan_strided(ex.get(), kAtGradV, gradValue, bytes, true, &a.grad_v);
    if (qLengths != nullptr) {
        plan_whole(ex.get(), kAtQLengths, qLengths, &a.q_lengths);
    }
    if (kvLengths != nullptr) {
        plan_whole(ex.get(), kAtKvLengths, kvLengths, &a.kv_lengths);
    }
    plan_lse(ex.get(), kAtLse, lse, &a.lse);
    plan_scratch(ex.get(), kAtScratch, scratch);
    return finish(api, ex, workspaceSize, executor);
}

aclnnStatus opscvWindowAttentionBackward(void* workspace, uint64_t workspaceSize, aclOpExecutor* executor,
                                         aclrtStream stream)
{
    return run_executor(workspace, workspaceSize, executor, stream, OpKind::WindowAttentionGrad,
                        "opscvWindowAttentionBackward");
}

}  // extern "C"
