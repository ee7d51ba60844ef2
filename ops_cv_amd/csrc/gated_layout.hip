// Around the matrix products of the gated projections: operands laid out as rows of their terms, the gradients of gate and up,
// sums of partial products and of the biases' gradients.  All bound by memory.
//
//   dGate = gy up act'(gate),  dUp = gy act(gate)
//
// Both are needed by rows (gradient of x: sums over the inner features) and by columns (gradients of the weights: sums over
// the rows), so a tile of 64 x 64 is computed once and written both ways, through LDS.  FLOAT16 has a range of 2^5 over and
// 2^14 under the values that gradients have when they are well scaled, and sums of products of gy, up and a slope leave it on
// both sides: there every row and column is multiplied by the power of two that takes its largest value to 2^14..2^15, found
// by a first pass, and the products' results are divided by it.
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
constexpr int kTile = kGateTile;

template <typename T>
constexpr int kVec = 16 / (int)sizeof(T);

template <typename T>
__global__ __launch_bounds__(kThreads) void pad_rows_kernel(const T* from, int64_t from_stride, int64_t rows, int64_t width,
                                                            T* to, int64_t to_stride, int64_t padded)
{
    const int64_t vectors = padded / kVec<T>, total = rows * vectors;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < total; i += (int64_t)gridDim.x * kThreads) {
        const int64_t r = i / vectors, c = (i - r * vectors) * kVec<T>;
        Pack<T, kVec<T>> k;
#pragma unroll
        for (int e = 0; e < kVec<T>; e++) {
            k.v[e] = c + e < width ? from[r * from_stride + c + e] : (T)0.0f;
        }
        *reinterpret_cast<Pack<T, kVec<T>>*>(to + r * to_stride + c) = k;
    }
}

// A tile of 64 x 64 in LDS, written by rows and read by columns; four bytes more a row keep a column off one bank.
template <typename T>
struct Turn {
    T v[kTile][kTile + 4 / (int)sizeof(T)];
};

// Column c of the tile, rows r..: one vector of the transposed rows.
template <typename T>
__device__ __forceinline__ void put_turned(const Turn<T>& tile, T* to, int64_t to_stride, int64_t column0, int64_t columns,
                                           int64_t row0, int64_t padded)
{
    constexpr int kParts = kTile / kVec<T>;  // vectors of a column
    for (int i = (int)threadIdx.x; i < kTile * kParts; i += kThreads) {
        const int c = i / kParts, r = i % kParts * kVec<T>;
        if (column0 + c < columns && row0 + r < padded) {
            Pack<T, kVec<T>> k;
#pragma unroll
            for (int e = 0; e < kVec<T>; e++) {
                k.v[e] = tile.v[r + e][c];
            }
            *reinterpret_cast<Pack<T, kVec<T>>*>(to + (column0 + c) * to_stride + row0 + r) = k;
        }
    }
}

template <typename T, bool WIDE>
__global__ __launch_bounds__(kThreads) void transpose_kernel(const T* from, int64_t from_stride, int64_t rows, int64_t width,
                                                             T* to, int64_t to_stride, int64_t padded)
{
    __shared__ Turn<T> tile;
    constexpr int kParts = kTile / kVec<T>, kRows = kThreads / kParts;
    const int64_t row0 = (int64_t)blockIdx.y * kTile, column0 = (int64_t)blockIdx.x * kTile;
    const int c = (int)threadIdx.x % kParts * kVec<T>;
#pragma unroll
    for (int i = 0; i < kTile / kRows; i++) {
        const int r = i * kRows + (int)threadIdx.x / kParts;
        const T* const row = from + (row0 + r) * from_stride + column0 + c;
        Pack<T, kVec<T>> k;
#pragma unroll
        for (int e = 0; e < kVec<T>; e++) {
            k.v[e] = (T)0.0f;
        }
        if (row0 + r < rows) {
            if (WIDE && column0 + c + kVec<T> <= width) {
                k = *reinterpret_cast<const Pack<T, kVec<T>>*>(row);
            } else {
#pragma unroll
                for (int e = 0; e < kVec<T>; e++) {
                    if (column0 + c + e < width) {
                        k.v[e] = row[e];
                    }
                }
            }
        }
#pragma unroll
        for (int e = 0; e < kVec<T>; e++) {
            tile.v[r][c + e] = k.v[e];
        }
    }
    __syncthreads();
    put_turned<T>(tile, to, to_stride, column0, width, row0, padded);
}

// ------------------------------------------------------------------------------------------- gradients of gate and up

// Values of a thread: kVec columns of one row; zeros outside.
template <typename T, bool WIDE>
__device__ __forceinline__ void gate_values(const GateGradArgs& a, int64_t row, int64_t c, float (&dg)[kVec<T>],
                                            float (&du)[kVec<T>])
{
    constexpr int N = kVec<T>;
    if (row >= a.rows || c >= a.inner) {
#pragma unroll
        for (int e = 0; e < N; e++) {
            dg[e] = du[e] = 0.0f;
        }
        return;
    }
    float gy[N], gate[N], up[N];
    const auto get = [&](const void* from, int64_t stride, float (&x)[N]) {
        const T* const at = (const T*)from + row * stride;
        if (WIDE && c + N <= a.inner) {
            load<T, N>(at + c, x);
        } else {
            load_part<T, N, false>(at, c, a.inner, x);
        }
    };
    get(a.grad_y, a.grad_y_stride, gy);
    get(a.gate, a.gate_stride, gate);
    get(a.up, a.up_stride, up);
#pragma unroll
    for (int e = 0; e < N; e++) {
        float value, slope;
        activate_both(gate[e], a.activation, &value, &slope);
        dg[e] = c + e < a.inner ? gy[e] * up[e] * slope : 0.0f;
        du[e] = c + e < a.inner ? gy[e] * value : 0.0f;
    }
}

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

// Largest values of rows and columns.  The order of the atomic maxima does not matter.
template <typename T, bool WIDE>
__global__ __launch_bounds__(kThreads) void gate_most_kernel(GateGradArgs a)
{
    constexpr int N = kVec<T>, kParts = kTile / N, kRows = kThreads / kParts;
    __shared__ uint32_t rows[kTile], columns[2][kTile];
    for (int i = (int)threadIdx.x; i < 3 * kTile; i += kThreads) {
        (i < kTile ? rows[i] : columns[i / kTile - 1][i % kTile]) = 0;
    }
    __syncthreads();
    const int64_t row0 = (int64_t)blockIdx.y * kTile, column0 = (int64_t)blockIdx.x * kTile;
    const int c = (int)threadIdx.x % kParts * N;
    uint32_t most[2][N] = {{0}};
#pragma unroll
    for (int i = 0; i < kTile / kRows; i++) {
        const int r = i * kRows + (int)threadIdx.x / kParts;
        float dg[N], du[N];
        gate_values<T, WIDE>(a, row0 + r, column0 + c, dg, du);
        uint32_t row = 0;
#pragma unroll
        for (int e = 0; e < N; e++) {
            const uint32_t g = size_of(dg[e]), u = size_of(du[e]);
            most[0][e] = most[0][e] > g ? most[0][e] : g;
            most[1][e] = most[1][e] > u ? most[1][e] : u;
            row = row > g ? row : g;
            row = row > u ? row : u;
        }
        atomicMax(&rows[r], row);
    }
#pragma unroll
    for (int e = 0; e < N; e++) {
        atomicMax(&columns[0][c + e], most[0][e]);
        atomicMax(&columns[1][c + e], most[1][e]);
    }
    __syncthreads();
    for (int i = (int)threadIdx.x; i < 3 * kTile; i += kThreads) {
        const int at = i % kTile;
        if (i < kTile) {
            if (row0 + at < a.rows) {
                atomicMax(&a.row_most[row0 + at], rows[at]);
            }
        } else if (column0 + at < a.inner) {
            atomicMax(&a.column_most[(i / kTile - 1) * a.inner + column0 + at], columns[i / kTile - 1][at]);
        }
    }
}

template <typename T, bool WIDE, bool SCALED>
__global__ __launch_bounds__(kThreads) void gate_grad_kernel(GateGradArgs a)
{
    constexpr int N = kVec<T>, kParts = kTile / N, kRows = kThreads / kParts;
    __shared__ Turn<T> tile[2];
    __shared__ float sums[2][kRows][kTile];
    const int64_t row0 = (int64_t)blockIdx.y * kTile, column0 = (int64_t)blockIdx.x * kTile;
    const int c = (int)threadIdx.x % kParts * N, thread_row = (int)threadIdx.x / kParts;
    float by_column[2][N], total[2][N];
#pragma unroll
    for (int e = 0; e < N; e++) {
        by_column[0][e] = by_column[1][e] = 1.0f;
        total[0][e] = total[1][e] = 0.0f;
        if (SCALED && column0 + c + e < a.inner) {
            by_column[0][e] = lift(a.column_most[column0 + c + e]);
            by_column[1][e] = lift(a.column_most[a.inner + column0 + c + e]);
            if (blockIdx.y == 0 && thread_row == 0) {
                a.column_factor[column0 + c + e] = 1.0f / by_column[0][e];
                a.column_factor[a.inner + column0 + c + e] = 1.0f / by_column[1][e];
            }
        }
    }
#pragma unroll
    for (int i = 0; i < kTile / kRows; i++) {
        const int r = i * kRows + thread_row;
        const int64_t row = row0 + r;
        float dg[N], du[N];
        gate_values<T, WIDE>(a, row, column0 + c, dg, du);
        float by_row = 1.0f;
        if (SCALED && row < a.rows) {
            by_row = lift(a.row_most[row]);
            if (blockIdx.x == 0 && c == 0) {
                a.row_factor[row] = 1.0f / by_row;
            }
        }
        if (a.by_rows != nullptr && row < a.rows && column0 + c < a.padded_inner) {
            float x[N];
            T* const to = (T*)a.by_rows + row * 2 * a.padded_inner + column0 + c;
#pragma unroll
            for (int e = 0; e < N; e++) {
                x[e] = dg[e] * by_row;
            }
            store<T, N>(to, x, false);
#pragma unroll
            for (int e = 0; e < N; e++) {
                x[e] = du[e] * by_row;
            }
            store<T, N>(to + a.padded_inner, x, false);
        }
#pragma unroll
        for (int e = 0; e < N; e++) {
            total[0][e] += dg[e];
            total[1][e] += du[e];
            tile[0].v[r][c + e] = (T)(dg[e] * by_column[0][e]);
            tile[1].v[r][c + e] = (T)(du[e] * by_column[1][e]);
        }
    }
    if (a.sums != nullptr) {
#pragma unroll
        for (int e = 0; e < N; e++) {
            sums[0][thread_row][c + e] = total[0][e];
            sums[1][thread_row][c + e] = total[1][e];
        }
    }
    __syncthreads();
    if (a.by_columns != nullptr) {
        put_turned<T>(tile[0], (T*)a.by_columns, a.padded_rows, column0, a.inner, row0, a.padded_rows);
        put_turned<T>(tile[1], (T*)a.by_columns + a.inner * a.padded_rows, a.padded_rows, column0, a.inner, row0, a.padded_rows);
    }
    if (a.sums != nullptr && threadIdx.x < 2 * kTile) {
        const int half = (int)threadIdx.x / kTile, at = (int)threadIdx.x % kTile;
        float sum = 0.0f;
        for (int r = 0; r < kRows; r++) {
            sum += sums[half][r][at];
        }
        if (column0 + at < a.inner) {
            a.sums[(int64_t)blockIdx.y * 2 * a.inner + half * a.inner + column0 + at] = sum;
        }
    }
}

template <typename T>
hipError_t run_gate_grad(const GateGradArgs& a, hipStream_t stream)
{
    const int64_t columns = (a.inner + kTile - 1) / kTile, rows = (a.rows + kTile - 1) / kTile;
    if (columns > 65535 || rows > 65535) {
        return hipErrorInvalidValue;
    }
    const int e = (int)sizeof(T);
    const bool wide = aligned(a.grad_y, a.grad_y_stride, e, 16) && aligned(a.gate, a.gate_stride, e, 16) &&
                      aligned(a.up, a.up_stride, e, 16);
    const dim3 grid((unsigned)columns, (unsigned)rows);
    constexpr bool kScaled = std::is_same_v<T, _Float16>;
    if (kScaled) {
        const int64_t words = a.rows + 2 * a.inner, blocks = (words + kThreads - 1) / kThreads;
        hipLaunchKernelGGL(clear_kernel, dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(kThreads), 0, stream, a.row_most,
                           words);  // the columns' follow the rows'
        if (wide) {
            hipLaunchKernelGGL((gate_most_kernel<T, true>), grid, dim3(kThreads), 0, stream, a);
        } else {
            hipLaunchKernelGGL((gate_most_kernel<T, false>), grid, dim3(kThreads), 0, stream, a);
        }
    }
    if (wide) {
        hipLaunchKernelGGL((gate_grad_kernel<T, true, kScaled>), grid, dim3(kThreads), 0, stream, a);
    } else {
        hipLaunchKernelGGL((gate_grad_kernel<T, false, kScaled>), grid, dim3(kThreads), 0, stream, a);
    }
    return hipGetLastError();
}

template <typename T>
__global__ __launch_bounds__(kThreads) void join_kernel(JoinArgs a)
{
    const int64_t total = a.tokens * a.features;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < total; i += (int64_t)gridDim.x * kThreads) {
        const int64_t t = i / a.features, f = i - t * a.features;
        float sum = 0.0f;
        for (int64_t k = 0; k < a.count; k++) {
            sum += a.parts[k * total + i];
        }
        if (a.token_scale != nullptr) {
            sum *= a.token_scale[t];
        }
        const bool second = t >= a.turn;
        ((T*)a.out[second])[(second ? t - a.turn : t) * a.out_stride[second] + f] = (T)sum;
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

hipError_t launch_pad_rows(Elem e, const void* from, int64_t from_stride, int64_t rows, int64_t width, void* to,
                           int64_t to_stride, int64_t padded, hipStream_t stream)
{
    if (rows < 1) {
        return hipSuccess;
    }
    return typed(e, [&](auto* t) {
        typedef std::remove_pointer_t<decltype(t)> T;
        if (padded % kVec<T> != 0 || to_stride % kVec<T> != 0) {
            return hipErrorInvalidValue;
        }
        hipLaunchKernelGGL((pad_rows_kernel<T>), dim3(blocks_of(rows * (padded / kVec<T>))), dim3(kThreads), 0, stream,
                           (const T*)from, from_stride, rows, width, (T*)to, to_stride, padded);
        return hipGetLastError();
    });
}

hipError_t launch_transpose(Elem e, const void* from, int64_t from_stride, int64_t rows, int64_t width, void* to,
                            int64_t to_stride, int64_t padded, hipStream_t stream)
{
    return typed(e, [&](auto* t) {
        typedef std::remove_pointer_t<decltype(t)> T;
        const int64_t columns = (width + kTile - 1) / kTile, row_tiles = (rows + kTile - 1) / kTile;
        if (rows < 1) {
            return hipSuccess;
        }
        if (padded % kVec<T> != 0 || to_stride % kVec<T> != 0 || columns > 65535 || row_tiles > 65535) {
            return hipErrorInvalidValue;
        }
        const dim3 grid((unsigned)columns, (unsigned)row_tiles);
        if (aligned(from, from_stride, (int)sizeof(T), 16)) {
            hipLaunchKernelGGL((transpose_kernel<T, true>), grid, dim3(kThreads), 0, stream, (const T*)from, from_stride, rows,
                               width, (T*)to, to_stride, padded);
        } else {
            hipLaunchKernelGGL((transpose_kernel<T, false>), grid, dim3(kThreads), 0, stream, (const T*)from, from_stride, rows,
                               width, (T*)to, to_stride, padded);
        }
        return hipGetLastError();
    });
}

hipError_t launch_gate_grad(const GateGradArgs& a, hipStream_t stream)
{
    if (a.rows < 1) {
        return hipSuccess;
    }
    return typed((Elem)a.elem, [&](auto* t) { return run_gate_grad<std::remove_pointer_t<decltype(t)>>(a, stream); });
}

hipError_t launch_join(Elem e, const JoinArgs& a, hipStream_t stream)
{
    return typed(e, [&](auto* t) {
        typedef std::remove_pointer_t<decltype(t)> T;
        hipLaunchKernelGGL((join_kernel<T>), dim3(blocks_of(a.tokens * a.features)), dim3(kThreads), 0, stream, a);
        return hipGetLastError();
    });
}

hipError_t launch_bias_sums(Elem e, const float* sums, int64_t rows, int64_t inner, void* gate, void* up, hipStream_t stream)
{
    return typed(e, [&](auto* t) {
        typedef std::remove_pointer_t<decltype(t)> T;
        launch_column_sums<T>(sums, rows, inner, (T*)gate, stream, 2 * inner);
        launch_column_sums<T>(sums + inner, rows, inner, (T*)up, stream, 2 * inner);
        return hipGetLastError();
    });
}

}  // namespace prod
}  // namespace opscv
