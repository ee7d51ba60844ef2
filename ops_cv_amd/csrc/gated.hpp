// What the parts of the gated projections call of each other.
#pragma once

#include <hip/hip_runtime_api.h>

#include "acl_types.hpp"

namespace opscv {
namespace prod {

struct ProductArgs;

// the gated forward product, and both products of the gradients (one may be null)
hipError_t launch_products_f32(const ProductArgs& a, int tile, hipStream_t stream);
hipError_t launch_products_f16(const ProductArgs& a, int tile, hipStream_t stream);
hipError_t launch_products_bf16(const ProductArgs& a, int tile, hipStream_t stream);
hipError_t launch_gradients_f32(const ProductArgs* x, const ProductArgs* weights, int tile, hipStream_t stream);
hipError_t launch_gradients_f16(const ProductArgs* x, const ProductArgs* weights, int tile, hipStream_t stream);
hipError_t launch_gradients_bf16(const ProductArgs* x, const ProductArgs* weights, int tile, hipStream_t stream);

// Rows of `width` elements, copied to rows of `padded` with zeros behind them.
struct PadArgs {
    struct Copy {
        const void* from = nullptr;
        int64_t from_stride = 0, rows = 0;
        void* to = nullptr;
    };
    Copy copy[3];
    int count = 0;
    int64_t width = 0, padded = 0;
};
hipError_t launch_pad_rows(Elem e, const PadArgs& a, hipStream_t stream);

// Gradients of gate and up, as the products want them (gated_layout.hip).
struct GateGradArgs {
    int elem = 0, activation = 0;
    int64_t rows = 0, inner = 0;
    const void *grad_y = nullptr, *gate = nullptr, *up = nullptr;
    int64_t grad_y_stride = 0, gate_stride = 0, up_stride = 0;
    // (rows, 2 padded): dGate, zeros, dUp, zeros; FLOAT16: in the scale of each row.  May be null.
    void* by_rows = nullptr;
    // FLOAT16: the same in the scale of each column.  May be null.
    void* by_columns = nullptr;
    int64_t padded = 0;
    int64_t rows_each = 0;  // of a workgroup: gate_rows()
    // sums over the rows of each workgroup: (rows / rows_each, 2 inner); may be null
    float* sums = nullptr;
    // FLOAT16: largest absolute values as bits, by rows and by columns (2 inner), and the factors that undo the scales; null
    // for the direction that is not written
    uint32_t *row_most = nullptr, *column_most = nullptr;
    float *row_factor = nullptr, *column_factor = nullptr;
};
constexpr int kGateRows = 64;

// Rows of a workgroup of them: kGateRows, or fewer while that leaves less than four workgroups to a CU (1355 rows of 1792 bf16: 18
// us with 64, their arithmetic done by one wavefront a SIMD).
inline int64_t gate_rows(int64_t rows, int64_t padded, int elem_bytes, int compute_units)
{
    const int64_t columns = (padded * elem_bytes + 511) / 512;  // workgroups of a row: 32 vectors each
    int64_t each = kGateRows;
    while (each > 8 && columns * ((rows + each - 1) / each) < (int64_t)4 * compute_units) {
        each /= 2;
    }
    return each;
}

hipError_t launch_gate_grad(const GateGradArgs& a, hipStream_t stream);

// The sums of the gated product's parts, in the places of its results (product_tile.hpp).
hipError_t launch_join_gated(Elem e, const ProductArgs& a, hipStream_t stream);

// What is left of the gradients after their products, in one launch: sums of parts, where there are any (`partial`), and of the
// biases' rows, (rows, 2 inner), the first inner to `gate`, the others to `up`.
struct FinishArgs {
    const ProductArgs *x = nullptr, *weights = nullptr;
    const float* sums = nullptr;
    int64_t sum_rows = 0, inner = 0;
    void *gate = nullptr, *up = nullptr;  // both or neither
};
hipError_t launch_finish(Elem e, const FinishArgs& a, hipStream_t stream);

}  // namespace prod
}  // namespace opscv
