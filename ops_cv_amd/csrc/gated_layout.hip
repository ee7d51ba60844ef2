// Around the matrix products of the gated projections: operands copied to whole vectors, the gradients of gate and up, sums of
// partial products and of the biases' gradients.  All bound by memory.
//
//   dGate = gy up act'(gate),  dUp = gy act(gate)
//
// They are written once, rounded to the type, and both products read them: the matrix cores take 16-bit numbers on both sides,
// and a second product of what the rounding leaves would double the time (4096 rows of 2048 to 8192 bf16: 474 us).  It makes the
// gradients 1.4 times as far off as the rounding of their own results does (0.0024 for 0.0017 bf16, 0.0003 for 0.0002 FLOAT16).
//
// FLOAT16 has a range of 2^5 over and 2^14 under the values that gradients have when they are well scaled, and products of gy,
// up and a slope leave it on both sides: there every row is multiplied by the power of two that takes its largest value to
// 2^14..2^15, found by a first pass, and its results of the product, the gradient of x, are divided by it.  The weights'
// gradients sum over the rows, so they read the same numbers in a scale of every column.
//
// 4096 rows of 8192 bf16: 55 us, 6.1 TB/s; FLOAT16 48 for the largest values and 84 for the numbers
// in both scales.
#include <hip/hip_runtime.h>

#include "gated.hpp"
#include "launch_limits.hpp"
#include "product_tile.hpp"
#include "token_elem.hpp"
#include "token_rows.hpp"

namespace opscv {
namespace prod {

using namespace tok;

namespace {

constexpr int kThreads = 256;
constexpr int kRows = kGateRows;

template <typename T>
constexpr int kVec = 16 / (int)sizeof(T);

// One copy for every blockIdx.y.
template <typename T>
__global__ __launch_bounds__(kThreads) void pad_rows_kernel(PadArgs a)
{
    const PadArgs::Copy& copy = a.copy[blockIdx.y];
    const int64_t vectors = a.padded / kVec<T>, total = copy.rows * vectors;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < total; i += (int64_t)gridDim.x * kThreads) {
        const int64_t r = i / vectors, c = (i - r * vectors) * kVec<T>;
        const T* const from = (const T*)copy.from + r * copy.from_stride + c;
        Loose<T> k;
        if (c + kVec<T> <= a.width) {
            k = *reinterpret_cast<const Loose<T>*>(from);
        } else {
#pragma unroll
            for (int e = 0; e < kVec<T>; e++) {
                k.v[e] = c + e < a.width ? from[e] : (T)0.0f;
            }
        }
        *reinterpret_cast<Pack16*>((T*)copy.to + r * a.padded + c) = __builtin_bit_cast(Pack16, k);
    }
}

// ------------------------------------------------------------------------------------------- gradients of gate and up

// What a thread reads of a row: kVec columns.
struct GateRead {
    Pack16 grad_y, gate, up;
};

template <typename T>
__device__ __forceinline__ Pack16 read_columns(const T* row, int64_t c, int64_t width)
{
    if (c + kVec<T> <= width) {
        return __builtin_bit_cast(Pack16, *reinterpret_cast<const Loose<T>*>(row + c));
    }
    Loose<T> k;
#pragma unroll
    for (int e = 0; e < kVec<T>; e++) {
        k.v[e] = c + e < width ? row[c + e] : (T)0.0f;
    }
    return __builtin_bit_cast(Pack16, k);
}

// Rows from `end` on are read as the last one, columns past the end are zeros.
template <typename T>
__device__ __forceinline__ GateRead gate_read(const GateGradArgs& a, int64_t row, int64_t end, int64_t c)
{
    const int64_t r = row < end ? row : end - 1;
    return {read_columns((const T*)a.grad_y + r * a.grad_y_stride, c, a.inner),
            read_columns((const T*)a.gate + r * a.gate_stride, c, a.inner),
            read_columns((const T*)a.up + r * a.up_stride, c, a.inner)};
}

// dGate and dUp of what was read; zeros where `live` is false.
template <typename T, int KIND>
__device__ __forceinline__ void gate_values(const GateRead& x, bool live, float (&dg)[kVec<T>], float (&du)[kVec<T>])
{
    const Loose<T> grad_y = __builtin_bit_cast(Loose<T>, x.grad_y), gate = __builtin_bit_cast(Loose<T>, x.gate),
                   up = __builtin_bit_cast(Loose<T>, x.up);
#pragma unroll
    for (int e = 0; e < kVec<T>; e++) {
        float value, slope;
        activate_both((float)gate.v[e], KIND, &value, &slope);
        const float gy = (float)grad_y.v[e];
        dg[e] = live ? gy * (float)up.v[e] * slope : 0.0f;
        du[e] = live ? gy * value : 0.0f;
    }
}

constexpr int kAhead = 4;  // rows of a thread that are read together

// The power of two that takes `most` (bits of an absolute value) to 2^14..2^15, at most 2^100.
__device__ __forceinline__ float lift(uint32_t most)
{
    if (most == 0) {
        return 1.0f;
    }
    int e = (int)(most >> 23);  // of 2^(e - 127) and more; 0: less than 2^-126
    e = 127 + 14 - (e - 127);
    return __uint_as_float((uint32_t)(e < 227 ? e : 227) << 23);
}

__global__ __launch_bounds__(kThreads) void clear_kernel(uint32_t* at, int64_t words)
{
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < words; i += (int64_t)gridDim.x * kThreads) {
        at[i] = 0;
    }
}

// Bits of |x|, 0 where it is not finite: what no scale can help.
__device__ __forceinline__ uint32_t size_of(float x)
{
    const uint32_t u = __float_as_uint(x) & 0x7FFFFFFFu;
    return u < 0x7F800000u ? u : 0u;
}

// A workgroup's part: rows_each rows (kRows at most) of kThreads / 8 vectors; a thread's vectors are those of every eighth row.
// SHORT: rows_each is less than kRows, or there are no more rows, and the loops end where the rows do.  Those ends keep the
// compiler from moving the loads of the next rows up: 4096 rows of 8192 bf16, 56 us without them and 62 with.
template <typename T>
constexpr int kColumns = kThreads / 8 * kVec<T>;

// Largest values of rows and columns.  The order of the atomic maxima does not matter.
template <typename T, int KIND, bool SHORT>
__global__ __launch_bounds__(kThreads) void gate_most_kernel(GateGradArgs a)
{
    constexpr int N = kVec<T>;
    __shared__ uint32_t rows[kRows], columns[2][kColumns<T>];
    for (int i = (int)threadIdx.x; i < kRows + 2 * kColumns<T>; i += kThreads) {
        (i < kRows ? rows[i] : columns[(i - kRows) / kColumns<T>][(i - kRows) % kColumns<T>]) = 0;
    }
    __syncthreads();
    const int64_t row0 = (int64_t)blockIdx.y * a.rows_each, column0 = (int64_t)blockIdx.x * kColumns<T>;
    const int64_t end = row0 + a.rows_each < a.rows ? row0 + a.rows_each : a.rows;
    const int c = (int)threadIdx.x % 32 * N;
    uint32_t most[2][N] = {{0}};
    GateRead x[kAhead];
#pragma unroll
    for (int i = 0; i < kRows / 8; i++) {
        if (SHORT && row0 + i * 8 >= end) {
            break;
        }
        if (i % kAhead == 0) {
#pragma unroll
            for (int k = 0; k < kAhead; k++) {
                if (!SHORT || row0 + (i + k) * 8 < end) {
                    x[k] = gate_read<T>(a, row0 + (i + k) * 8 + (int)threadIdx.x / 32, end, column0 + c);
                }
            }
        }
        const int r = i * 8 + (int)threadIdx.x / 32;
        float dg[N], du[N];
        gate_values<T, KIND>(x[i % kAhead], row0 + r < end, dg, du);
        uint32_t row = 0;
#pragma unroll
        for (int e = 0; e < N; e++) {
            const uint32_t g = size_of(dg[e]), u = size_of(du[e]);
            most[0][e] = most[0][e] > g ? most[0][e] : g;
            most[1][e] = most[1][e] > u ? most[1][e] : u;
            row = row > g ? row : g;
            row = row > u ? row : u;
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) {
            const uint32_t other = (uint32_t)__shfl_xor((int)row, d, 64);
            row = row > other ? row : other;
        }
        if (c == 0) {
            rows[r] = row;
        }
    }
    if (a.column_most != nullptr) {
#pragma unroll
        for (int e = 0; e < N; e++) {
            atomicMax(&columns[0][c + e], most[0][e]);
            atomicMax(&columns[1][c + e], most[1][e]);
        }
    }
    __syncthreads();
    for (int i = (int)threadIdx.x; i < kRows + 2 * kColumns<T>; i += kThreads) {
        if (i < kRows) {
            if (a.row_most != nullptr && row0 + i < end) {
                atomicMax(&a.row_most[row0 + i], rows[i]);
            }
        } else if (a.column_most != nullptr) {
            const int half = (i - kRows) / kColumns<T>, at = (i - kRows) % kColumns<T>;
            if (column0 + at < a.inner) {
                atomicMax(&a.column_most[half * a.inner + column0 + at], columns[half][at]);
            }
        }
    }
}

template <typename T, int KIND, bool SHORT>
__global__ __launch_bounds__(kThreads) void gate_grad_kernel(GateGradArgs a)
{
    constexpr int N = kVec<T>;
    constexpr bool kScaled = std::is_same_v<T, _Float16>;
    __shared__ float sums[2][8][kColumns<T>];
    const int64_t row0 = (int64_t)blockIdx.y * a.rows_each, column0 = (int64_t)blockIdx.x * kColumns<T>;
    const int64_t end = row0 + a.rows_each < a.rows ? row0 + a.rows_each : a.rows;
    const int c = (int)threadIdx.x % 32 * N, part = (int)threadIdx.x / 32;
    float by_column[2][kScaled ? N : 1], total[2][N];
#pragma unroll
    for (int e = 0; e < N; e++) {
        total[0][e] = total[1][e] = 0.0f;
        if constexpr (kScaled) {
#pragma unroll
            for (int half = 0; half < 2; half++) {
                by_column[half][e] = 1.0f;
                if (a.column_most != nullptr && column0 + c + e < a.inner) {
                    by_column[half][e] = lift(a.column_most[half * a.inner + column0 + c + e]);
                    if (blockIdx.y == 0 && part == 0) {
                        a.column_factor[half * a.inner + column0 + c + e] = 1.0f / by_column[half][e];
                    }
                }
            }
        }
    }
    GateRead read[kAhead];
#pragma unroll
    for (int i = 0; i < kRows / 8; i++) {
        if (SHORT && row0 + i * 8 >= end) {
            break;
        }
        if (i % kAhead == 0) {
#pragma unroll
            for (int k = 0; k < kAhead; k++) {
                if (!SHORT || row0 + (i + k) * 8 < end) {
                    read[k] = gate_read<T>(a, row0 + (i + k) * 8 + part, end, column0 + c);
                }
            }
        }
        const int64_t row = row0 + i * 8 + part;
        float dg[N], du[N], x[N];
        gate_values<T, KIND>(read[i % kAhead], row < end, dg, du);
        float by_row = 1.0f;
        if (kScaled && a.row_most != nullptr && row < end) {
            by_row = lift(a.row_most[row]);
            if (blockIdx.x == 0 && c == 0) {
                a.row_factor[row] = 1.0f / by_row;
            }
        }
#pragma unroll
        for (int e = 0; e < N; e++) {
            total[0][e] += dg[e];
            total[1][e] += du[e];
        }
        if (row < end && column0 + c < a.padded) {
            const int64_t at = row * 2 * a.padded + column0 + c;
#pragma unroll
            for (int half = 0; half < 2; half++) {
                const float(&d)[N] = half == 0 ? dg : du;
                if (a.by_rows != nullptr) {
#pragma unroll
                    for (int e = 0; e < N; e++) {
                        x[e] = d[e] * by_row;
                    }
                    store<T, N>((T*)a.by_rows + at + half * a.padded, x, false);
                }
                if constexpr (kScaled) {
                    if (a.by_columns != nullptr) {
#pragma unroll
                        for (int e = 0; e < N; e++) {
                            x[e] = d[e] * by_column[half][e];
                        }
                        store<T, N>((T*)a.by_columns + at + half * a.padded, x, false);
                    }
                }
            }
        }
    }
    if (a.sums != nullptr) {
#pragma unroll
        for (int e = 0; e < N; e++) {
            sums[0][part][c + e] = total[0][e];
            sums[1][part][c + e] = total[1][e];
        }
        __syncthreads();
        for (int i = (int)threadIdx.x; i < 2 * kColumns<T>; i += kThreads) {
            const int half = i / kColumns<T>, at = i % kColumns<T>;
            float sum = 0.0f;
#pragma unroll
            for (int k = 0; k < 8; k++) {
                sum += sums[half][k][at];
            }
            if (column0 + at < a.inner) {
                a.sums[(int64_t)blockIdx.y * 2 * a.inner + half * a.inner + column0 + at] = sum;
            }
        }
    }
}

template <typename T, int KIND, bool SHORT>
hipError_t run_gate_grad(const GateGradArgs& a, hipStream_t stream)
{
    if (a.rows_each < 8 || a.rows_each > kRows || a.rows_each % 8 != 0 || a.padded % kVec<T> != 0 || a.padded < a.inner) {
        return hipErrorInvalidValue;
    }
    const int64_t columns = (a.padded + kColumns<T> - 1) / kColumns<T>, rows = (a.rows + a.rows_each - 1) / a.rows_each;
    if (columns > 65535 || rows > 65535) {
        return hipErrorInvalidValue;
    }
    const dim3 grid((unsigned)columns, (unsigned)rows);
    if constexpr (std::is_same_v<T, _Float16>) {
        // the columns' follow the rows'; the biases' sums are of unscaled numbers and need neither
        const int64_t words = (a.row_most != nullptr ? a.rows : 0) + (a.column_most != nullptr ? 2 * a.inner : 0);
        const int64_t blocks = (words + kThreads - 1) / kThreads;
        if ((a.by_rows != nullptr) != (a.row_most != nullptr) || (a.by_columns != nullptr) != (a.column_most != nullptr)) {
            return hipErrorInvalidValue;
        }
        if (words > 0) {
            hipLaunchKernelGGL(clear_kernel, dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(kThreads), 0, stream,
                               a.row_most != nullptr ? a.row_most : a.column_most, words);
            hipLaunchKernelGGL((gate_most_kernel<T, KIND, SHORT>), grid, dim3(kThreads), 0, stream, a);
        }
    }
    hipLaunchKernelGGL((gate_grad_kernel<T, KIND, SHORT>), grid, dim3(kThreads), 0, stream, a);
    return hipGetLastError();
}

// Sums of a vector's parts, in order; four are read together (7 rows of 1191, 15 parts: 6.5 us one by one).
template <int N>
__device__ __forceinline__ void join_parts(const float* from, int64_t part, uint32_t parts, int64_t c, int64_t width, float (&x)[N])
{
    constexpr uint32_t kTogether = 4;
    load_part<float, N, false>(from, c, width, x);
    for (uint32_t k = 1; k < parts; k += kTogether) {
        float y[kTogether][N];
#pragma unroll
        for (uint32_t j = 0; j < kTogether; j++) {
            // parts past the last one are read as it, and left out
            load_part<float, N, false>(from + (k + j < parts ? k + j : parts - 1) * part, c, width, y[j]);
        }
#pragma unroll
        for (uint32_t j = 0; j < kTogether; j++) {
            if (k + j < parts) {
#pragma unroll
                for (int e = 0; e < N; e++) {
                    x[e] += y[j][e];
                }
            }
        }
    }
}

constexpr int kJoin = 4;  // features of a thread

template <typename T>
__device__ __forceinline__ void join(const ProductArgs& a, uint32_t block, uint32_t blocks)
{
    const int64_t vectors = (a.columns + kJoin - 1) / kJoin, total = a.tokens * vectors;
    for (int64_t i = (int64_t)block * kThreads + threadIdx.x; i < total; i += (int64_t)blocks * kThreads) {
        const int64_t t = i / vectors, f = (i - t * vectors) * kJoin;
        const bool second = t >= a.turn;
        const int64_t row = second ? t - a.turn : t;
        if (row >= a.rows) {
            continue;
        }
        float x[kJoin];
        join_parts<kJoin>(a.partial + t * a.features, a.tokens * a.features, a.parts, f, a.features, x);
        if (a.token_scale != nullptr) {
            const float scale = a.token_scale[second ? a.rows + row : row];
#pragma unroll
            for (int e = 0; e < kJoin; e++) {
                x[e] *= scale;
            }
        }
        store_part<T, kJoin, false>((T*)a.out[second] + row * a.out_stride[second], f, a.columns, x, false);
    }
}

// The first workgroups join x's parts, the next ones the weights', the others sum up the biases' rows: launches of their own
// would each take 4 to 5 us (512 rows of 512 to 2048 bf16, all gradients: 25 us).
template <typename T>
__global__ __launch_bounds__(kThreads) void finish_kernel(ProductArgs x, ProductArgs weights, uint32_t x_blocks,
                                                          uint32_t weight_blocks, const float* sums, int64_t sum_rows,
                                                          int64_t inner, T* gate, T* up)
{
    uint32_t block = blockIdx.x;
    if (block < x_blocks) {
        join<T>(x, block, x_blocks);
        return;
    }
    block -= x_blocks;
    if (block < weight_blocks) {
        join<T>(weights, block, weight_blocks);
        return;
    }
    block -= weight_blocks;
    const uint32_t blocks = (uint32_t)((inner + 31) / 32);
    const bool second = block >= blocks;
    column_sums<T>(second ? sums + inner : sums, second ? block - blocks : block, sum_rows, inner, 2 * inner, second ? up : gate);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void join_gated_kernel(ProductArgs a)
{
    const int64_t vectors = (a.columns + kJoin - 1) / kJoin, total = a.tokens * vectors;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < total; i += (int64_t)gridDim.x * kThreads) {
        const int64_t t = i / vectors, f = (i - t * vectors) * kJoin;
        float x[2][kJoin], y[kJoin];
#pragma unroll
        for (int half = 0; half < 2; half++) {
            join_parts<kJoin>(a.partial + (2 * t + half) * a.features, a.tokens * 2 * a.features, a.parts, f, a.features, x[half]);
            if (a.bias[half] != nullptr) {
                load_part<T, kJoin, false>((const T*)a.bias[half], f, a.features, y);
#pragma unroll
                for (int e = 0; e < kJoin; e++) {
                    x[half][e] += y[e];
                }
            }
        }
#pragma unroll
        for (int e = 0; e < kJoin; e++) {
            y[e] = activate(x[0][e], a.activation) * x[1][e];
        }
        store_part<T, kJoin, false>((T*)a.out[0] + t * a.out_stride[0], f, a.columns, y, false);
        if (a.out[1] != nullptr) {
            store_part<T, kJoin, false>((T*)a.out[1] + t * a.out_stride[1], f, a.columns, x[0], false);
            store_part<T, kJoin, false>((T*)a.out[2] + t * a.out_stride[2], f, a.columns, x[1], false);
        }
    }
}

// f(T) by the operands' type
template <typename F>
hipError_t typed(Elem e, F&& f)
{
    return by_type((int)e, 0, [&](auto* t, auto*) { return f(t); });
}

unsigned blocks_of(int64_t items)
{
    const int64_t blocks = (items + kThreads - 1) / kThreads;
    return (unsigned)(blocks < 1 << 16 ? blocks : 1 << 16);
}

}  // namespace

hipError_t launch_pad_rows(Elem e, const PadArgs& a, hipStream_t stream)
{
    int64_t rows = 0;
    for (int i = 0; i < a.count; i++) {
        rows = a.copy[i].rows > rows ? a.copy[i].rows : rows;
    }
    if (rows < 1) {
        return hipSuccess;
    }
    return typed(e, [&](auto* t) {
        typedef std::remove_pointer_t<decltype(t)> T;
        if (a.padded % kVec<T> != 0 || a.padded < a.width) {
            return hipErrorInvalidValue;
        }
        hipLaunchKernelGGL((pad_rows_kernel<T>), dim3(blocks_of(rows * (a.padded / kVec<T>)), (unsigned)a.count), dim3(kThreads),
                           0, stream, a);
        return hipGetLastError();
    });
}

hipError_t launch_gate_grad(const GateGradArgs& a, hipStream_t stream)
{
    if (a.rows < 1) {
        return hipSuccess;
    }
    return typed((Elem)a.elem, [&](auto* t) {
        typedef std::remove_pointer_t<decltype(t)> T;
        const bool few = a.rows_each < kRows || a.rows < kRows;
        switch (a.activation) {
            case 0: return few ? run_gate_grad<T, 0, true>(a, stream) : run_gate_grad<T, 0, false>(a, stream);
            case 1: return few ? run_gate_grad<T, 1, true>(a, stream) : run_gate_grad<T, 1, false>(a, stream);
            default: return few ? run_gate_grad<T, 2, true>(a, stream) : run_gate_grad<T, 2, false>(a, stream);
        }
    });
}

hipError_t launch_join_gated(Elem e, const ProductArgs& a, hipStream_t stream)
{
    return typed(e, [&](auto* t) {
        typedef std::remove_pointer_t<decltype(t)> T;
        hipLaunchKernelGGL((join_gated_kernel<T>), dim3(blocks_of(a.tokens * ((a.columns + kJoin - 1) / kJoin))), dim3(kThreads), 0,
                           stream, a);
        return hipGetLastError();
    });
}

hipError_t launch_finish(Elem e, const FinishArgs& a, hipStream_t stream)
{
    const auto blocks = [](const ProductArgs& p) {
        return p.partial == nullptr ? 0u : blocks_of(p.tokens * ((p.columns + kJoin - 1) / kJoin));
    };
    const uint32_t x = blocks(*a.x), weights = blocks(*a.weights);
    const uint32_t biases = a.gate == nullptr ? 0u : 2u * (uint32_t)((a.inner + 31) / 32);
    if (x + weights + biases == 0) {
        return hipSuccess;
    }
    if (a.inner < 0 || a.inner > (int64_t)1 << 24) {
        return hipErrorInvalidValue;
    }
    return typed(e, [&](auto* t) {
        typedef std::remove_pointer_t<decltype(t)> T;
        hipLaunchKernelGGL((finish_kernel<T>), dim3(x + weights + biases), dim3(kThreads), 0, stream, *a.x, *a.weights, x, weights,
                           a.sums, a.sum_rows, a.inner, (T*)a.gate, (T*)a.up);
        return hipGetLastError();
    });
}

}  // namespace prod
}  // namespace opscv
