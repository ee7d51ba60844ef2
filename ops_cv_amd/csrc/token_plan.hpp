// First phases of the operators on token sequences: argument checks and the planning of operands (opscv_tokens.cpp,
// opscv_blocks.cpp).
#pragma once

#include <cmath>
#include <cstring>
#include <memory>
#include <new>

#include "executor.hpp"
#include "kernels.hpp"

namespace opscv {
namespace tokplan {

constexpr int64_t kMostExtent = (int64_t)1 << 30;
constexpr int64_t kMostTokenStride = (int64_t)1 << 22;  // elements
constexpr int64_t kMostRotaryDim = 1024;

typedef std::unique_ptr<aclOpExecutor> Executor;

// What both arguments that return something are checked for, and the executor of the call.
inline aclnnStatus begin(const char* api, uint64_t* workspaceSize, aclOpExecutor** executor, Executor* ex)
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

inline aclnnStatus finish(const char* api, Executor& ex, uint64_t* workspaceSize, aclOpExecutor** executor)
{
    if (const aclnnStatus ps = plan_status(ex.get(), api); ps != ACLNN_SUCCESS) {
        return ps;
    }
    *workspaceSize = ex->workspace_bytes;
    *executor = ex.release();
    return ACLNN_SUCCESS;
}

inline aclnnStatus missing(const char* api, const char* names)
{
    set_error("%s: %s must not be NULL", api, names);
    return ACLNN_ERR_PARAM_NULLPTR;
}

template <typename... A>
inline aclnnStatus invalid(const char* format, A... a)
{
    set_error(format, a...);
    return ACLNN_ERR_PARAM_INVALID;
}

inline bool same_dims(const aclTensor* a, const aclTensor* b)
{
    return a->ndim == b->ndim && memcmp(a->dims, b->dims, sizeof(int64_t) * (size_t)a->ndim) == 0;
}

// the leading dimensions of `t`, one value per row
inline bool per_row(const aclTensor* r, const aclTensor* t)
{
    return r->ndim == t->ndim - 1 && memcmp(r->dims, t->dims, sizeof(int64_t) * (size_t)r->ndim) == 0;
}

inline bool extents_fit(const aclTensor* t)
{
    for (int64_t i = 0; i < t->ndim; i++) {
        if (t->dims[i] > kMostExtent) {
            return false;
        }
    }
    return true;
}

// Operand `slot` of the executor: the tensor packed dense.
inline void plan_dense(aclOpExecutor* ex, int slot, const aclTensor* t, int elem_bytes, bool output)
{
    ex->operands[slot] = plan_view(ex, t, elem_bytes, output);
    ex->required |= t->empty() ? 0u : 1u << slot;
}

// Operand `slot`, used in place where its last dimension is dense, packed otherwise; the strides that the kernel walks.
inline void plan_strided(aclOpExecutor* ex, int slot, const aclTensor* t, int elem_bytes, bool output, Strided* s)
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
inline void plan_rows(aclOpExecutor* ex, int slot, const aclTensor* t, int elem_bytes, bool output, Rows* r)
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
inline void plan_whole(aclOpExecutor* ex, int slot, const aclTensor* t, Whole* w)
{
    w->wide = t->dtype == ACL_INT64 ? 1 : 0;
    for (int i = 0; i < t->ndim; i++) {
        w->stride[i] = t->strides[i];
    }
    ex->operands[slot].direct = (t->data == nullptr) ? nullptr : (char*)t->data + t->offset * (w->wide ? 8 : 4);
    ex->required |= t->empty() ? 0u : 1u << slot;
}

inline void plan_scratch(aclOpExecutor* ex, int slot, int64_t floats)
{
    if (floats > 0) {
        PlannedPtr p;
        p.in_workspace = true;
        p.ws_offset = (ex->workspace_bytes + 255) / 256 * 256;
        ex->workspace_bytes = p.ws_offset + (uint64_t)floats * 4;
        ex->operands[slot] = p;
    }
}

inline bool whole_type(const aclTensor* t) { return t->dtype == ACL_INT32 || t->dtype == ACL_INT64; }

// Weight of a norm: (width), of the activations' type or FLOAT.
inline aclnnStatus check_weight(const char* api, const char* name, const aclTensor* w, const aclTensor* x)
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
inline aclnnStatus check_rows(const char* api, const char* name, const aclTensor* t, const aclTensor* like, bool dtype = true)
{
    if (!same_dims(t, like)) {
        return invalid("%s: %s has another shape than the other rows", api, name);
    }
    if (dtype && t->dtype != like->dtype) {
        return invalid("%s: %s has another type than the other rows", api, name);
    }
    return ACLNN_SUCCESS;
}

inline aclnnStatus check_row_values(const char* api, const char* name, const aclTensor* t, const aclTensor* like)
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
inline aclnnStatus norm_rows(const char* api, const aclTensor* x, Elem* e, int64_t* rows, int64_t* width)
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
        // what is too many stays so, unless another dimension is 0
        *rows = x->dims[i] == 0 ? 0 : *rows > INT32_MAX / x->dims[i] ? (int64_t)INT32_MAX + 1 : *rows * x->dims[i];
    }
    if (*width < 1 || *width > kMostExtent || *rows > INT32_MAX) {
        return invalid("%s: rows of 1 to 2^30 elements and fewer than 2^31 rows, got %lld by %lld", api, (long long)*rows,
                       (long long)*width);
    }
    return ACLNN_SUCCESS;
}

}  // namespace tokplan
}  // namespace opscv
