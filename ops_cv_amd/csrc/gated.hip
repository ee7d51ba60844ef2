// Gated projections and their gradients: which products they are made of, and where their operands lie.
//
//   gate = x Wg^T + bg, up = x Wu^T + bu, y = act(gate) up                              4 M F D operations, one launch
//   dGate = gy up act'(gate), dUp = gy act(gate)
//   gx = [dGate dUp] [Wg; Wu]                                                           4 M F D
//   [gWg; gWu] = [dGate dUp]^T x                                                        4 M F D
//
// Forward, both operands are rows of their terms as they stand; rows that do not start on 16 bytes, or are not made of whole
// vectors, are copied with zeros behind them.  Backward, the sums run over the inner features and over the rows: x and the
// weights are laid out transposed, dGate and dUp computed both ways (gated_layout.hip), and both gradients are one plain
// product each over 2 F or M terms.
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

hipError_t launch_product(Elem e, const ProductArgs& a, int kind, int tile, hipStream_t stream)
{
    switch (e) {
        case Elem::F32: return launch_product_f32(a, kind, tile, stream);
        case Elem::F16: return launch_product_f16(a, kind, tile, stream);
        default: return launch_product_bf16(a, kind, tile, stream);
    }
}

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
    l.bytes = s.bytes;
    return l;
}

// ----------------------------------------------------------------------------------------------------------- backward

struct BackwardLayout {
    int64_t inner = 0, rows = 0;  // in whole vectors
    int64_t by_rows = -1, weights = -1, by_columns = -1, x = -1;
    int64_t most = -1, factors = -1, sums = -1, parts = -1;
    ProductPlan for_x, for_weights;
    int64_t bytes = 0;
};

BackwardLayout backward_layout(const GatedArgs& a)
{
    const int e = elem_size((Elem)a.elem);
    BackwardLayout l;
    Slices s;
    l.inner = rounded(a.inner, 16 / e);
    l.rows = rounded(a.rows, 16 / e);
    int64_t parts = 0;
    if (a.want_x != 0 && a.rows > 0) {
        l.for_x = plan_product(a.rows, a.width, 2 * l.inner * e, false, a.compute_units);
        l.by_rows = s.take(a.rows * 2 * l.inner * e);
        l.weights = s.take(a.width * 2 * l.inner * e);
        parts = l.for_x.parts > 1 ? l.for_x.parts * a.rows * a.width : 0;
    }
    if (a.want_weights != 0) {
        l.for_weights = plan_product(2 * a.inner, a.width, l.rows * e, false, a.compute_units);
        l.by_columns = s.take(2 * a.inner * l.rows * e);
        l.x = s.take(a.width * l.rows * e);
        const int64_t own = l.for_weights.parts > 1 ? l.for_weights.parts * 2 * a.inner * a.width : 0;
        parts = parts > own ? parts : own;
    }
    if (a.elem == (int)Elem::F16) {
        l.most = s.take((a.rows + 2 * a.inner) * 4);
        l.factors = s.take((a.rows + 2 * a.inner) * 4);
    }
    if (a.want_biases != 0) {
        l.sums = s.take((a.rows + kGateTile - 1) / kGateTile * 2 * a.inner * 4);
    }
    if (parts > 0) {
        l.parts = s.take(parts * 4);  // one product after the other
    }
    l.bytes = s.bytes;
    return l;
}

// A plain product, in parts where that is planned.
hipError_t run_plain(Elem e, ProductArgs p, const ProductPlan& plan, float* parts, hipStream_t stream)
{
    for (int i = 0; i < 2; i++) {
        p.wide[i] = tok::aligned(p.out[i], p.out_stride[i], elem_size(e), 16) ? 1 : 0;
    }
    if (plan.parts <= 1) {
        return launch_product(e, p, kPlain, plan.tile, stream);
    }
    JoinArgs j;
    j.parts = parts;
    j.count = plan.parts;
    j.tokens = p.tokens;
    j.features = p.features;
    for (int i = 0; i < 2; i++) {
        j.out[i] = p.out[i];
        j.out_stride[i] = p.out_stride[i];
    }
    j.turn = p.turn;
    j.token_scale = p.token_scale;
    p.out[0] = parts;
    p.parts = (uint32_t)plan.parts;
    p.part_stages = plan.part_stages;
    const hipError_t status = launch_product(e, p, kPartial, plan.tile, stream);
    return status != hipSuccess ? status : launch_join(e, j, stream);
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
    const int e = elem_size(elem);
    const ForwardLayout l = forward_layout(a);
    if (a.rows < 1 || a.width < 1 || a.inner < 1 || (l.bytes > 0 && a.scratch == nullptr)) {
        return hipErrorInvalidValue;
    }
    const auto laid_out = [&](const Rows& r, int64_t rows, int64_t copy, const void** ptr, int64_t* stride) {
        *ptr = copy < 0 ? r.ptr : a.scratch + copy;
        *stride = copy < 0 ? r.row_stride : l.terms;
        return copy < 0 ? hipSuccess
                        : launch_pad_rows(elem, r.ptr, r.row_stride, rows, a.width, a.scratch + copy, l.terms, l.terms, stream);
    };
    ProductArgs p;
    OPSCV_LAUNCH(laid_out(a.x, a.rows, l.x, &p.q, &p.q_stride));
    OPSCV_LAUNCH(laid_out(a.gate_weight, a.inner, l.gate, &p.p[0], &p.p_stride[0]));
    OPSCV_LAUNCH(laid_out(a.up_weight, a.inner, l.up, &p.p[1], &p.p_stride[1]));
    p.tokens = a.rows;
    p.features = a.inner;
    p.terms = l.terms;
    const Rows* const out[3] = {&a.y, &a.gate, &a.up};
    for (int i = 0; i < 3; i++) {
        p.out[i] = out[i]->ptr;
        p.out_stride[i] = out[i]->row_stride;
        p.wide[i] = tok::aligned(p.out[i], p.out_stride[i], e, 16) ? 1 : 0;
    }
    p.bias[0] = a.gate_bias;
    p.bias[1] = a.up_bias;
    p.activation = a.activation;
    const ProductPlan plan = plan_product(a.rows, 2 * a.inner, l.terms * e, true, a.compute_units);
    return launch_product(elem, p, kGated, plan.tile, stream);
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
    g.padded_inner = l.inner;
    g.by_columns = at(l.by_columns);
    g.padded_rows = l.rows;
    g.sums = (float*)at(l.sums);
    if (l.most >= 0) {
        g.row_most = (uint32_t*)at(l.most);
        g.column_most = g.row_most + a.rows;
        g.row_factor = (float*)at(l.factors);
        g.column_factor = g.row_factor + a.rows;
    }
    OPSCV_LAUNCH(launch_gate_grad(g, stream));
    if (l.by_rows >= 0) {
        char* const weights = at(l.weights);
        const int64_t e = elem_size(elem);
        OPSCV_LAUNCH(launch_transpose(elem, a.gate_weight.ptr, a.gate_weight.row_stride, a.inner, a.width, weights, 2 * l.inner,
                                      l.inner, stream));
        OPSCV_LAUNCH(launch_transpose(elem, a.up_weight.ptr, a.up_weight.row_stride, a.inner, a.width, weights + l.inner * e,
                                      2 * l.inner, l.inner, stream));
        ProductArgs p;
        p.p[0] = p.p[1] = weights;
        p.p_stride[0] = p.p_stride[1] = 2 * l.inner;
        p.q = g.by_rows;
        p.q_stride = 2 * l.inner;
        p.tokens = a.rows;
        p.features = a.width;
        p.terms = 2 * l.inner;
        p.out[0] = p.out[1] = a.grad_x.ptr;
        p.out_stride[0] = p.out_stride[1] = a.grad_x.row_stride;
        p.turn = a.rows;
        p.token_scale = g.row_factor;
        OPSCV_LAUNCH(run_plain(elem, p, l.for_x, (float*)at(l.parts), stream));
    }
    if (a.want_weights != 0) {
        OPSCV_LAUNCH(launch_transpose(elem, a.x.ptr, a.x.row_stride, a.rows, a.width, at(l.x), l.rows, l.rows, stream));
        ProductArgs p;
        p.p[0] = p.p[1] = at(l.x);
        p.p_stride[0] = p.p_stride[1] = l.rows;
        p.q = g.by_columns;
        p.q_stride = l.rows;
        p.tokens = 2 * a.inner;
        p.features = a.width;
        p.terms = l.rows;
        p.out[0] = a.grad_gate_weight.ptr;
        p.out[1] = a.grad_up_weight.ptr;
        p.out_stride[0] = a.grad_gate_weight.row_stride;
        p.out_stride[1] = a.grad_up_weight.row_stride;
        p.turn = a.inner;
        p.token_scale = a.rows > 0 ? g.column_factor : nullptr;
        OPSCV_LAUNCH(run_plain(elem, p, l.for_weights, (float*)at(l.parts), stream));
    }
    if (a.want_biases != 0) {
        OPSCV_LAUNCH(launch_bias_sums(elem, g.sums, (a.rows + kGateTile - 1) / kGateTile, a.inner, a.grad_gate_bias,
                                      a.grad_up_bias, stream));
    }
    return hipSuccess;
}

}  // namespace opscv
