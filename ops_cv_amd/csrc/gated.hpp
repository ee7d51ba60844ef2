// What the parts of the gated projections call of each other.
#pragma once

#include <hip/hip_runtime_api.h>

#include "acl_types.hpp"

namespace opscv {
namespace prod {

struct ProductArgs;

hipError_t launch_product_f32(const ProductArgs& a, int kind, int tile, hipStream_t stream);
hipError_t launch_product_f16(const ProductArgs& a, int kind, int tile, hipStream_t stream);
hipError_t launch_product_bf16(const ProductArgs& a, int kind, int tile, hipStream_t stream);

// Rows of `width` elements, copied to rows of `to_stride`, zeros from `width` to `padded` on.
hipError_t launch_pad_rows(Elem e, const void* from, int64_t from_stride, int64_t rows, int64_t width, void* to,
                           int64_t to_stride, int64_t padded, hipStream_t stream);

// to[c][r] = from[r][c], zeros for r from `rows` to `padded` on.
hipError_t launch_transpose(Elem e, const void* from, int64_t from_stride, int64_t rows, int64_t width, void* to,
                            int64_t to_stride, int64_t padded, hipStream_t stream);

// Gradients of gate and up, as the products want them (gated_layout.hip).
struct GateGradArgs {
    int elem = 0, activation = 0;
    int64_t rows = 0, inner = 0;
    const void *grad_y = nullptr, *gate = nullptr, *up = nullptr;
    int64_t grad_y_stride = 0, gate_stride = 0, up_stride = 0;
    // (rows, 2 padded_inner): dGate, zeros, dUp, zeros; may be null
    void* by_rows = nullptr;
    int64_t padded_inner = 0;
    // (2 inner, padded_rows): the transposed dGate and dUp, zeros behind; may be null
    void* by_columns = nullptr;
    int64_t padded_rows = 0;
    // sums over the rows of each tile of kGateTile rows: (tiles, 2 inner); may be null
    float* sums = nullptr;
    // FLOAT16: largest absolute values as bits, by rows and by columns (2 inner), and the factors that undo the scales
    uint32_t *row_most = nullptr, *column_most = nullptr;
    float *row_factor = nullptr, *column_factor = nullptr;
};
constexpr int kGateTile = 64;

hipError_t launch_gate_grad(const GateGradArgs& a, hipStream_t stream);

// out[t][f] = factor[t] * sum of the parts
struct JoinArgs {
    const float* parts = nullptr;
    int64_t count = 0, tokens = 0, features = 0;
    void* out[2] = {nullptr, nullptr};
    int64_t out_stride[2] = {0, 0};
    int64_t turn = 0;
    const float* token_scale = nullptr;
};
hipError_t launch_join(Elem e, const JoinArgs& a, hipStream_t stream);

// Sums of the rows of (rows, 2 inner): the first inner to `gate`, the others to `up`.
hipError_t launch_bias_sums(Elem e, const float* sums, int64_t rows, int64_t inner, void* gate, void* up, hipStream_t stream);

}  // namespace prod
}  // namespace opscv
