// Rows of the norms: reductions over the threads of a row, and sums of partial sums over rows.
#pragma once

#include <hip/hip_runtime.h>

#include <type_traits>

#include "acl_types.hpp"
#include "token_elem.hpp"

namespace opscv {
namespace tok {

constexpr int kMostPerLane = 32;          // elements of a row that a thread keeps in registers
constexpr int64_t kMostBlocks = 1 << 20;  // more rows than these take are walked

inline dim3 grid(int64_t blocks) { return dim3((unsigned)(blocks < kMostBlocks ? blocks : kMostBlocks)); }

// Sums over the threads of `R` rows at once, as row_reduce.
template <int THREADS, int R>
static __device__ __forceinline__ void rows_reduce(float (&sum)[R], float (*shared)[R][16], int slot)
{
#pragma unroll
    for (int k = 0; k < R; k++) {
        sum[k] = wave_sum(sum[k]);
    }
    if constexpr (THREADS > 64) {
        const int wave = (int)threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
            for (int k = 0; k < R; k++) {
                shared[slot][k][wave] = sum[k];
            }
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < R; k++) {
            sum[k] = 0.0f;
#pragma unroll
            for (int i = 0; i < THREADS / 64; i++) {
                sum[k] += shared[slot][k][i];
            }
        }
    }
}

// Sums of the rows of partial sums: 32 columns a workgroup of 256 threads, every eighth row a thread, joined in order.
template <typename W>
static __device__ __forceinline__ void column_sums(const float* partial, int64_t block, int64_t rows, int64_t width, int64_t stride,
                                                   W* out)
{
    __shared__ float shared[8][32];
    const int column = (int)threadIdx.x & 31, part = (int)threadIdx.x >> 5;
    const int64_t c = block * 32 + column;
    float total = 0.0f;
    if (c < width) {
#pragma unroll 8
        for (int64_t r = part; r < rows; r += 8) {
            total += partial[r * stride + c];
        }
    }
    shared[part][column] = total;
    __syncthreads();
    if (part == 0 && c < width) {
#pragma unroll
        for (int i = 1; i < 8; i++) {
            total += shared[i][column];
        }
        out[c] = (W)total;
    }
}

// Of one or two gradients (blockIdx.z).
template <typename W>
static __global__ __launch_bounds__(256) void column_sums_kernel(const float* first, const float* second, int64_t rows,
                                                                 int64_t width, int64_t stride, W* first_out, W* second_out)
{
    column_sums<W>(blockIdx.z == 0 ? first : second, (int64_t)blockIdx.y * gridDim.x + blockIdx.x, rows, width, stride,
                   blockIdx.z == 0 ? first_out : second_out);
}

// Either output may be null.
template <typename W>
void launch_column_sums(const float* first, const float* second, int64_t rows, int64_t width, W* first_out, W* second_out,
                        hipStream_t stream)
{
    if (first_out == nullptr) {
        first = second;
        first_out = second_out;
        second_out = nullptr;
    }
    // rows of more than 2^25 columns take more than one row of workgroups: 2^24 of 256 threads are more than a launch holds
    // in one
    const int64_t blocks = (width + 31) / 32;
    const dim3 columns((unsigned)(blocks < kMostBlocks ? blocks : kMostBlocks), (unsigned)((blocks + kMostBlocks - 1) / kMostBlocks),
                       second_out != nullptr ? 2 : 1);
    hipLaunchKernelGGL((column_sums_kernel<W>), columns, dim3(256), 0, stream, first, second, rows, width, width,
                       first_out, second_out);
}

// f(T, W) by the operands' types
template <typename F>
hipError_t by_type(int elem, int weight_float, F&& f)
{
    switch ((Elem)elem) {
        case Elem::F32: return f((float*)nullptr, (float*)nullptr);
        case Elem::F16: return weight_float != 0 ? f((_Float16*)nullptr, (float*)nullptr) : f((_Float16*)nullptr, (_Float16*)nullptr);
        default: return weight_float != 0 ? f((__bf16*)nullptr, (float*)nullptr) : f((__bf16*)nullptr, (__bf16*)nullptr);
    }
}

}  // namespace tok
}  // namespace opscv
