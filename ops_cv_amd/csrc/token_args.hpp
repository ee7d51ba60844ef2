// Operands and parameters of the operators on token sequences, as planned by their first phases.
#pragma once

#include <cstdint>

namespace opscv {

// An operand used in place: element strides of its leading dimensions, the last one dense.
struct Strided {
    void* ptr = nullptr;
    int64_t stride[3] = {0, 0, 0};
};

// A vector of whole numbers (lengths), or a matrix of them (positions).
struct Whole {
    const void* ptr = nullptr;
    int64_t stride[2] = {0, 0};
    int wide = 0;  // 1: 64 bits, 0: 32 bits
};

// Rows `row_stride` elements apart, dense inside.
struct Rows {
    void* ptr = nullptr;
    int64_t row_stride = 0;
};

struct NormArgs {
    int elem = 0;         // Elem of x, residual, sum and y
    int weight_float = 0;  // weight (and its gradient) in FLOAT where elem is another type
    int int8 = 0;         // y in 8 bits, with scale
    int streaming = 0;    // set by the launcher
    int64_t rows = 0, width = 0;
    float eps = 0.0f;
    Rows x, residual, y, sum;  // residual and sum: ptr may be null
    const void* weight = nullptr;
    float* scale = nullptr;
    float* rstd = nullptr;
};

struct NormGradArgs {
    int elem = 0;
    int weight_float = 0;
    int64_t rows = 0, width = 0;
    Rows grad_y, grad_sum, sum, grad_x;  // grad_sum: ptr may be null
    const void* weight = nullptr;
    const float* rstd = nullptr;
    void* grad_weight = nullptr;  // may be null
    float* partial = nullptr;     // norm_grad_partials() rows of `width` sums, with grad_weight only
};

struct RotaryTableArgs {
    int64_t positions = 0, rot = 0, row_stride = 0;
    int64_t scaling = 0, original_length = 0;
    double base = 0.0, factor = 1.0, magnitude = 1.0;
    float* table = nullptr;
};

struct RotaryArgs {
    int elem = 0;
    int interleaved = 0, inverse = 0;
    int64_t batch = 0, tokens = 0, heads = 0, kv_heads = 0, d = 0, rot = 0, positions = 0;
    Strided query, key, query_out, key_out;  // strides of batch, token, head
    Whole position;
    const float* table = nullptr;
    int64_t table_stride = 0;
};

struct AttentionArgs {
    int elem = 0;
    int64_t batch = 0, tokens = 0, kv_tokens = 0, heads = 0, kv_heads = 0, d = 0;
    int64_t left = 0, right = 0, sinks = 0;  // clamped to 2^28 by the first phase
    float scale = 0.0f;
    int compute_units = 0;  // of the device that was current in the first phase: how far the keys are split
    Strided q, k, v, out;   // strides of batch, token, head
    Strided lse;            // strides of batch, head, token; ptr may be null in the forward pass
    Whole q_lengths, kv_lengths;
    // backward
    Strided grad_out, grad_q, grad_k, grad_v;
    float* scratch = nullptr;  // attention_scratch_floats() / attention_grad_scratch_floats()
};

}  // namespace opscv
