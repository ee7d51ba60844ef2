// Gated projections and their gradients: which products they are made of, and where their operands lie.
//
//   gate = x Wg^T + bg, up = x Wu^T + bu, y = act(gate) up                              4 M F D operations, one launch
//   dGate = gy up act'(gate), dUp = gy act(gate)
//   gx = [dGate dUp] [Wg; Wu]                                                           4 M F D
//   [gWg; gWu] = [dGate dUp]^T x                                                        4 M F D
//
// Forward, both operands are rows of their terms as they stand.  Backward, the sums run over the inner features and over the
// rows: the weights, x, dGate and dUp are read turned (product_tile.hpp), and both products go out in one launch.  Operands
// whose rows do not start on 16 bytes, or are not made of whole vectors, are copied with zeros behind them.
#include "gated.hpp"

#include "product_plan.hpp"
#include "product_tile.hpp"
#include "token_elem.hpp"
#include "token_kernels.hpp"

namespace opscv {

using namespace prod;

namespace {

int64_t rounded(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

// Slices of the scratch memory, one behind the other on 256 bytes.
struct Slices {
    int64_t bytes = 0;
    int64_t take(int64_t n)
    {
        const int64_t at = bytes;
        bytes += rounded(n, 256);
        return at;
    }
};

// Whether rows of `width` elements can be copied to LDS as they stand: whole vectors, on 16 bytes, near enough together for
// 32-bit offsets within a tile.
bool in_place(const Rows& r, int64_t rows, int64_t width, int e)
{
    return width * e % 16 == 0 && tok::aligned(r.ptr, r.row_stride, e, 16) && r.row_stride >= 0 &&
           (rows == 1 || r.row_stride <= (int64_t)1 << 20);
}

// ------------------------------------------------------------------------------------------------------------ forward

struct ForwardLayout {
    int64_t terms = 0;                       // width in whole vectors
    int64_t x = -1, gate = -1, up = -1;      // offsets of padded copies; -1: in place
    int64_t parts = -1;
    int64_t bytes = 0;
};

ForwardLayout forward_layout(const GatedArgs& a)
{
    const int e = elem_size((Elem)a.elem);
    ForwardLayout l;
    Slices s;
    l.terms = rounded(a.width, 16 / e);
    if (!in_place(a.x, a.rows, a.width, e)) {
        l.x = s.take(a.rows * l.terms * e);
    }
    if (!in_place(a.gate_weight, a.inner, a.width, e)) {
        l.gate = s.take(a.inner * l.terms * e);
    }
    if (!in_place(a.up_weight, a.inner, a.width, e)) {
        l.up = s.take(a.inner * l.terms * e);
    }
    if (a.plan.parts[0] > 1) {
        l.parts = s.take(a.plan.parts[0] * a.rows * 2 * a.inner * 4);
    }
    l.bytes = s.bytes;
    return l;
}

// An operand where it lies, or its place among the copies that are to be made.
void lay_out(const Rows& r, int64_t rows, char* copy, const void** ptr, int64_t* stride, PadArgs* pads)
{
    *ptr = copy == nullptr ? r.ptr : copy;
    *stride = copy == nullptr ? r.row_stride : pads->padded;
    if (copy != nullptr) {
        PadArgs::Copy& c = pads->copy[pads->count++];
        c.from = r.ptr;
        c.from_stride = r.row_stride;
        c.rows = rows;
        c.to = copy;
    }
}

// ----------------------------------------------------------------------------------------------------------- backward

struct BackwardLayout {
    int64_t padded = 0;  // inner in whole stages: a stage is of one weight
    int64_t width = 0;   // in whole vectors
    int64_t gate = -1, up = -1, x = -1;  // padded copies; -1: in place
    int64_t by_rows = -1, by_columns = -1;
    int64_t most = -1, factors = -1, sums = -1, parts_x = -1, parts_weights = -1;
    int64_t bytes = 0;
};

int64_t gate_rows_of(const GatedArgs& a, int64_t padded)
{
    return gate_rows(a.rows, padded, elem_size((Elem)a.elem), a.compute_units);
}

// rows of the biases' partial sums
int64_t sum_rows(const GatedArgs& a, int64_t padded)
{
    const int64_t each = gate_rows_of(a, padded);
    return (a.rows + each - 1) / each;
}

// FLOAT16: rows and columns that have a scale, of the gradients that are wanted
int64_t scales(const GatedArgs& a) { return (a.want_x != 0 ? a.rows : 0) + (a.want_weights != 0 ? 2 * a.inner : 0); }

BackwardLayout backward_layout(const GatedArgs& a)
{
    const int e = elem_size((Elem)a.elem);
    BackwardLayout l;
    Slices s;
    l.padded = rounded(a.inner, kRowBytes / e);
    l.width = rounded(a.width, 16 / e);
    const bool want_x = a.want_x != 0, want_weights = a.want_weights != 0;
    if (want_x) {
        if (!in_place(a.gate_weight, a.inner, a.width, e)) {
            l.gate = s.take(a.inner * l.width * e);
        }
        if (!in_place(a.up_weight, a.inner, a.width, e)) {
            l.up = s.take(a.inner * l.width * e);
        }
    }
    if (want_weights) {
        if (!in_place(a.x, a.rows, a.width, e)) {
            l.x = s.take(a.rows * l.width * e);
        }
    }
    const bool scaled = a.elem == (int)Elem::F16;
    if (want_x || (want_weights && !scaled)) {
        l.by_rows = s.take(a.rows * 2 * l.padded * e);
    }
    if (want_weights && scaled) {
        l.by_columns = s.take(a.rows * 2 * l.padded * e);
    }
    if (scaled && (want_x || want_weights)) {
        l.most = s.take(scales(a) * 4);
        l.factors = s.take(scales(a) * 4);
    }
    if (a.want_biases != 0) {
        l.sums = s.take(sum_rows(a, l.padded) * 2 * a.inner * 4);
    }
    const int64_t parts_x = a.plan.parts[0], parts_weights = a.plan.parts[want_x ? 1 : 0];
    if (want_x && parts_x > 1) {
        l.parts_x = s.take(parts_x * a.rows * l.width * 4);
    }
    if (want_weights && parts_weights > 1) {
        l.parts_weights = s.take(parts_weights * 2 * l.padded * l.width * 4);
    }
    l.bytes = s.bytes;
    return l;
}

#define OPSCV_LAUNCH(call)                                   \
    if (const hipError_t e_ = (call); e_ != hipSuccess) {    \
        return e_;                                           \
    }

}  // namespace

int64_t gated_scratch_bytes(const GatedArgs& a) { return forward_layout(a).bytes; }

int64_t gated_grad_scratch_bytes(const GatedArgs& a) { return backward_layout(a).bytes; }

hipError_t launch_gated(const GatedArgs& a, hipStream_t stream)
{
    const Elem elem = (Elem)a.elem;
    const ForwardLayout l = forward_layout(a);
    if (a.rows < 1 || a.width < 1 || a.inner < 1 || (l.bytes > 0 && a.scratch == nullptr)) {
        return hipErrorInvalidValue;
    }
    const auto at = [&](int64_t offset) { return offset < 0 ? nullptr : a.scratch + offset; };
    ProductArgs p;
    PadArgs pads;
    pads.width = a.width;
    pads.padded = l.terms;
    lay_out(a.x, a.rows, at(l.x), &p.q, &p.q_stride, &pads);
    lay_out(a.gate_weight, a.inner, at(l.gate), &p.p[0], &p.p_stride[0], &pads);
    lay_out(a.up_weight, a.inner, at(l.up), &p.p[1], &p.p_stride[1], &pads);
    OPSCV_LAUNCH(launch_pad_rows(elem, pads, stream));
    p.tokens = p.rows = a.rows;
    p.features = p.columns = a.inner;
    p.terms = l.terms;
    const Rows* const out[3] = {&a.y, &a.gate, &a.up};
    for (int i = 0; i < 3; i++) {
        p.out[i] = out[i]->ptr;
        p.out_stride[i] = out[i]->row_stride;
    }
    p.bias[0] = a.gate_bias;
    p.bias[1] = a.up_bias;
    p.activation = a.activation;
    p.partial = (float*)at(l.parts);
    p.parts = (uint32_t)a.plan.parts[0];
    p.part_stages = (uint32_t)a.plan.part_stages[0];
    switch (elem) {
        case Elem::F32: OPSCV_LAUNCH(launch_products_f32(p, a.plan.tile, stream)); break;
        case Elem::F16: OPSCV_LAUNCH(launch_products_f16(p, a.plan.tile, stream)); break;
        default: OPSCV_LAUNCH(launch_products_bf16(p, a.plan.tile, stream)); break;
    }
    return p.partial != nullptr ? launch_join_gated(elem, p, stream) : hipSuccess;
}

hipError_t launch_gated_grad(const GatedArgs& a, hipStream_t stream)
{
    const Elem elem = (Elem)a.elem;
    const BackwardLayout l = backward_layout(a);
    if (a.rows < 0 || a.width < 1 || a.inner < 1 || (l.bytes > 0 && a.scratch == nullptr)) {
        return hipErrorInvalidValue;
    }
    const auto at = [&](int64_t offset) { return offset < 0 ? nullptr : a.scratch + offset; };
    GateGradArgs g;
    g.elem = a.elem;
    g.activation = a.activation;
    g.rows = a.rows;
    g.inner = a.inner;
    g.grad_y = a.grad_y.ptr;
    g.gate = a.gate.ptr;
    g.up = a.up.ptr;
    g.grad_y_stride = a.grad_y.row_stride;
    g.gate_stride = a.gate.row_stride;
    g.up_stride = a.up.row_stride;
    g.by_rows = at(l.by_rows);
    g.by_columns = at(l.by_columns);
    g.padded = l.padded;
    g.rows_each = gate_rows_of(a, l.padded);
    g.sums = (float*)at(l.sums);
    if (l.most >= 0) {
        const int64_t rows = a.want_x != 0 ? a.rows : 0;
        uint32_t* const most = (uint32_t*)at(l.most);
        float* const factors = (float*)at(l.factors);
        g.row_most = a.want_x != 0 ? most : nullptr;
        g.row_factor = a.want_x != 0 ? factors : nullptr;
        g.column_most = a.want_weights != 0 ? most + rows : nullptr;
        g.column_factor = a.want_weights != 0 ? factors + rows : nullptr;
    }
    OPSCV_LAUNCH(launch_gate_grad(g, stream));
    PadArgs pads;
    pads.width = a.width;
    pads.padded = l.width;
    ProductArgs x, weights;
    if (a.want_x != 0) {
        lay_out(a.gate_weight, a.inner, at(l.gate), &x.p[0], &x.p_stride[0], &pads);
        lay_out(a.up_weight, a.inner, at(l.up), &x.p[1], &x.p_stride[1], &pads);
        x.p_turn = l.padded;
        x.p_terms = a.inner;
        x.q = g.by_rows;
        x.q_stride = 2 * l.padded;
        x.tokens = x.rows = a.rows;
        x.features = l.width;
        x.columns = a.width;
        x.terms = 2 * l.padded;
        x.out[0] = a.grad_x.ptr;
        x.out_stride[0] = a.grad_x.row_stride;
        x.token_scale = g.row_factor;
        x.partial = (float*)at(l.parts_x);
        x.parts = (uint32_t)a.plan.parts[0];
        x.part_stages = (uint32_t)a.plan.part_stages[0];
    }
    if (a.want_weights != 0) {
        const int own = a.want_x != 0 ? 1 : 0;
        lay_out(a.x, a.rows, at(l.x), &weights.p[0], &weights.p_stride[0], &pads);
        weights.p[1] = weights.p[0];
        weights.p_stride[1] = weights.p_stride[0];
        weights.p_turn = rounded(a.rows, kRowBytes);  // all terms are of the first
        weights.p_terms = a.rows;
        weights.q = g.by_columns != nullptr ? g.by_columns : g.by_rows;
        weights.q_stride = 2 * l.padded;
        weights.tokens = 2 * l.padded;
        weights.turn = l.padded;
        weights.rows = a.inner;
        weights.features = l.width;
        weights.columns = a.width;
        weights.terms = a.rows;
        weights.out[0] = a.grad_gate_weight.ptr;
        weights.out[1] = a.grad_up_weight.ptr;
        weights.out_stride[0] = a.grad_gate_weight.row_stride;
        weights.out_stride[1] = a.grad_up_weight.row_stride;
        weights.token_scale = a.rows > 0 ? g.column_factor : nullptr;
        weights.partial = (float*)at(l.parts_weights);
        weights.parts = (uint32_t)a.plan.parts[own];
        weights.part_stages = (uint32_t)a.plan.part_stages[own];
    }
    OPSCV_LAUNCH(launch_pad_rows(elem, pads, stream));
    if (a.want_x != 0 || a.want_weights != 0) {
        const ProductArgs* const px = a.want_x != 0 ? &x : nullptr;
        const ProductArgs* const pw = a.want_weights != 0 ? &weights : nullptr;
        switch (elem) {
            case Elem::F32: OPSCV_LAUNCH(launch_gradients_f32(px, pw, a.plan.tile, stream)); break;
            case Elem::F16: OPSCV_LAUNCH(launch_gradients_f16(px, pw, a.plan.tile, stream)); break;
            default: OPSCV_LAUNCH(launch_gradients_bf16(px, pw, a.plan.tile, stream)); break;
        }
    }
    FinishArgs f;
    f.x = &x;
    f.weights = &weights;
    if (a.want_biases != 0) {
        f.sums = g.sums;
        f.sum_rows = sum_rows(a, l.padded);
        f.inner = a.inner;
        f.gate = a.grad_gate_bias;
        f.up = a.grad_up_bias;
    }
    return launch_finish(elem, f, stream);
}

}  // namespace opscv
