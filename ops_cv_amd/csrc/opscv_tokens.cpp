// Operators on token sequences: parameter validation, planning and the second-phase entries (include/opscv_tokens.h).
#include "opscv_tokens.h"
#include "token_kernels.hpp"
#include "token_plan.hpp"

using namespace opscv;
using namespace opscv::tokplan;

namespace {

// tokens of a sequence and reaches of a window: sums of any three fit 32 bits
constexpr int64_t kMostTokens = (int64_t)1 << 28;
constexpr int64_t kMostHeadDim = 256;

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

// Sections and layout of opscvRotaryAxes, and the columns of its table.
aclnnStatus rotary_axes(const char* api, const aclIntArray* sections, int64_t layout, const aclTensor* table, RotaryArgs* a)
{
    if (sections->v.empty() || sections->v.size() > 4) {
        return invalid("%s: one to four axes, got %lld sections", api, (long long)sections->v.size());
    }
    if (layout < OPSCV_AXES_CONSECUTIVE || layout > OPSCV_AXES_DEALT) {
        return invalid("%s: unknown layout %lld", api, (long long)layout);
    }
    a->axes = (int)sections->v.size();
    a->layout = (int)layout;
    int64_t pairs = 0, most = 0;
    for (int i = 0; i < a->axes; i++) {
        const int64_t n = sections->v[(size_t)i];
        if (n < 0 || n > kMostRotaryDim / 2) {
            return invalid("%s: sections of 0 to %lld pairs, got %lld", api, (long long)(kMostRotaryDim / 2), (long long)n);
        }
        a->sections[i] = n;
        pairs += n;
        most = n > most ? n : most;
    }
    a->rot = 2 * pairs;
    a->columns = layout == OPSCV_AXES_RESTART ? most : pairs;
    if (table->dims[1] != 2 * a->columns) {
        return invalid("%s: table must have %lld columns, got %lld", api, (long long)(2 * a->columns),
                       (long long)table->dims[1]);
    }
    return ACLNN_SUCCESS;
}

// First phase of opscvRotary, and with `sections` of opscvRotaryAxes.
aclnnStatus rotary_plan(const char* api, OpKind kind, const aclTensor* query, const aclTensor* key,
                        const aclTensor* positions, const aclTensor* table, const aclIntArray* sections, int64_t layout,
                        bool interleaved, bool inverse, aclTensor* queryOut, aclTensor* keyOut, uint64_t* workspaceSize,
                        aclOpExecutor** executor)
{
    Executor ex;
    OPSCV_CHECK(begin(api, workspaceSize, executor, &ex));
    if (query == nullptr || table == nullptr || queryOut == nullptr || (key == nullptr) != (keyOut == nullptr)) {
        return missing(api, "query, table and queryOut, and one of key and keyOut beside the other,");
    }
    if (kind == OpKind::RotaryAxes && (sections == nullptr || positions == nullptr)) {
        return missing(api, "positions and sections");
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
    a.columns = a.rot / 2;
    if (kind == OpKind::RotaryAxes) {
        OPSCV_CHECK(rotary_axes(api, sections, layout, table, &a));
    }
    if (a.d < 1 || a.d > kMostRotaryDim || a.rot % 2 != 0 || a.rot < 2 || a.rot > a.d) {
        return invalid("%s: an even number of rotated features out of 2 to %lld, got %lld of %lld", api,
                       (long long)kMostRotaryDim, (long long)a.rot, (long long)a.d);
    }
    const int lead = kind == OpKind::RotaryAxes ? 1 : 0;
    if (positions != nullptr &&
        (positions->ndim != 2 + lead || (lead != 0 && positions->dims[0] != a.axes) ||
         positions->dims[lead] != a.batch || positions->dims[lead + 1] != a.tokens || !whole_type(positions))) {
        return invalid("%s: positions must be INT32 or INT64 (%sbatch, tokens)", api, lead != 0 ? "axes, " : "");
    }
    if (!extents_fit(query) || !extents_fit(table) || a.kv_heads > kMostExtent || a.batch * a.tokens > INT32_MAX) {
        return invalid("%s: extents too large", api);
    }
    if (a.batch == 0 || a.tokens == 0 || a.heads + a.kv_heads == 0) {
        return finish(api, ex, workspaceSize, executor);
    }
    ex->kind = kind;
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
        if (lead != 0) {
            a.position.axis_stride = positions->strides[0];
            a.position.stride[0] = positions->strides[1];
            a.position.stride[1] = positions->strides[2];
        }
    }
    Rows r;
    plan_rows(ex.get(), kRoTable, table, 4, false, &r);
    a.table_stride = r.row_stride;
    return finish(api, ex, workspaceSize, executor);
}

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
        case OpKind::Rotary:
        case OpKind::RotaryAxes: {
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
        case OpKind::LayerNorm:
        case OpKind::LayerNormGrad:
        case OpKind::Dropout:
        case OpKind::Gated:
        case OpKind::GatedGrad: *e = launch_block_plan(workspace, ex, stream); break;
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
    return rotary_plan("opscvRotary", OpKind::Rotary, query, key, positions, table, nullptr, 0, interleaved, inverse,
                       queryOut, keyOut, workspaceSize, executor);
}

aclnnStatus opscvRotary(void* workspace, uint64_t workspaceSize, aclOpExecutor* executor, aclrtStream stream)
{
    return run_executor(workspace, workspaceSize, executor, stream, OpKind::Rotary, "opscvRotary");
}

aclnnStatus opscvRotaryAxesGetWorkspaceSize(const aclTensor* query, const aclTensor* key, const aclTensor* positions,
                                            const aclTensor* table, const aclIntArray* sections, int64_t layout,
                                            bool interleaved, bool inverse, aclTensor* queryOut, aclTensor* keyOut,
                                            uint64_t* workspaceSize, aclOpExecutor** executor)
{
    return rotary_plan("opscvRotaryAxes", OpKind::RotaryAxes, query, key, positions, table, sections, layout, interleaved,
                       inverse, queryOut, keyOut, workspaceSize, executor);
}

aclnnStatus opscvRotaryAxes(void* workspace, uint64_t workspaceSize, aclOpExecutor* executor, aclrtStream stream)
{
    return run_executor(workspace, workspaceSize, executor, stream, OpKind::RotaryAxes, "opscvRotaryAxes");
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
