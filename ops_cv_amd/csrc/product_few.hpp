// The gated projections of few rows: single tokens of some sequences.
//
// Bound by memory, that is by reading both weights once: what counts is how many of their bytes are under way.  A workgroup
// makes 16 features of y for all rows, so that there are many workgroups; its eight wavefronts take the terms in turn, 128
// bytes of every feature's row each, straight from memory into the operands of 16 x 16 products (four neighbouring lanes read
// 64 bytes of a row), and their sums are joined in LDS, in order.  The rows of x come from L2 once for every workgroup.
// bf16, one row of 4096 to 14336: 46.5 us, 5.1 TB/s; 8 of 4096 to 4096 14.6, 4.6 TB/s.
#pragma once

#include <hip/hip_runtime.h>

#include <type_traits>

#include "product_tile.hpp"

namespace opscv {
namespace prod {

constexpr int kFewWaves = 8, kFewFeatures = 16;

typedef float f32x4_acc __attribute__((ext_vector_type(4)));

// 16 bytes of terms of a row a lane: lane l holds row l % 16 and vector l / 16 of four.
template <typename T>
struct Step16;

template <>
struct Step16<__bf16> {
    static __device__ __forceinline__ f32x4_acc mul(Pack16 a, Pack16 b, f32x4_acc c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(att::bf16x8, a), __builtin_bit_cast(att::bf16x8, b), c,
                                                       0, 0, 0);
    }
};

template <>
struct Step16<_Float16> {
    static __device__ __forceinline__ f32x4_acc mul(Pack16 a, Pack16 b, f32x4_acc c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(att::f16x8, a), __builtin_bit_cast(att::f16x8, b), c, 0,
                                                      0, 0);
    }
};

template <>
struct Step16<float> {
    static __device__ __forceinline__ f32x4_acc mul(Pack16 a, Pack16 b, f32x4_acc c)
    {
        const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], y[e], c, 0, 0, 0);
        }
        return c;
    }
};

// TB blocks of 16 rows of x; AHEAD stages of 128 bytes of terms are read at a time.
template <typename T, int TB, int AHEAD>
__global__ __launch_bounds__(64 * kFewWaves) __attribute__((amdgpu_waves_per_eu(4, 4))) void gated_few_kernel(ProductArgs a)
{
    constexpr int kE = (int)sizeof(T);
    __shared__ float sums[kFewWaves][2][TB][kFewFeatures * 16];
    const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
    const int64_t f0 = (int64_t)blockIdx.x * kFewFeatures;
    const int row = lane & 15, quarter = lane >> 4;
    // rows past the end are read as the last one, and their results left
    const int64_t f = f0 + row < a.features ? f0 + row : a.features - 1;
    const char* const gate = (const char*)a.p[0] + f * a.p_stride[0] * kE + quarter * 16;
    const char* const up = (const char*)a.p[1] + f * a.p_stride[1] * kE + quarter * 16;
    const char* x[TB];
#pragma unroll
    for (int b = 0; b < TB; b++) {
        const int64_t t = b * 16 + row < a.tokens ? b * 16 + row : a.tokens - 1;
        x[b] = (const char*)a.q + t * a.q_stride * kE + quarter * 16;
    }
    const int64_t bytes = a.terms * kE;
    f32x4_acc acc[2][TB];
#pragma unroll
    for (int b = 0; b < TB; b++) {
        acc[0][b] = acc[1][b] = f32x4_acc{0.0f, 0.0f, 0.0f, 0.0f};
    }
    const Pack16 zero = {{0, 0, 0, 0}};
    // one stage of AHEAD: two vectors a lane of each operand, 64 bytes apart
    const auto run = [&](int64_t first, auto whole) {
        Pack16 g[AHEAD][2], u[AHEAD][2], v[AHEAD][2][TB];
#pragma unroll
        for (int s = 0; s < AHEAD; s++) {
            const int64_t at = first + (int64_t)s * kFewWaves * kRowBytes;
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int64_t here = at + i * 64;
                // terms past the end: zeros on both sides
                const bool there = whole.value || here + quarter * 16 < bytes;
                g[s][i] = there ? *reinterpret_cast<const Pack16*>(gate + here) : zero;
                u[s][i] = there ? *reinterpret_cast<const Pack16*>(up + here) : zero;
#pragma unroll
                for (int b = 0; b < TB; b++) {
                    v[s][i][b] = there ? *reinterpret_cast<const Pack16*>(x[b] + here) : zero;
                }
            }
        }
#pragma unroll
        for (int s = 0; s < AHEAD; s++) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
#pragma unroll
                for (int b = 0; b < TB; b++) {
                    acc[0][b] = Step16<T>::mul(g[s][i], v[s][i][b], acc[0][b]);
                    acc[1][b] = Step16<T>::mul(u[s][i], v[s][i][b], acc[1][b]);
                }
            }
        }
    };
    int64_t at = (int64_t)wave * kRowBytes;
    for (; at + ((int64_t)(AHEAD - 1) * kFewWaves + 1) * kRowBytes <= bytes; at += (int64_t)AHEAD * kFewWaves * kRowBytes) {
        run(at, std::true_type());
    }
    if (at < bytes) {
        run(at, std::false_type());
    }
    // lane l's registers are features 4 (l / 16) .. + 3 of row l % 16
#pragma unroll
    for (int b = 0; b < TB; b++) {
#pragma unroll
        for (int r = 0; r < 4; r++) {
            sums[wave][0][b][row * kFewFeatures + 4 * quarter + r] = acc[0][b][r];
            sums[wave][1][b][row * kFewFeatures + 4 * quarter + r] = acc[1][b][r];
        }
    }
    __syncthreads();
    for (int i = (int)threadIdx.x; i < TB * 16 * kFewFeatures; i += 64 * kFewWaves) {
        const int64_t t = i / kFewFeatures, own = f0 + i % kFewFeatures;
        if (t >= a.tokens || own >= a.columns) {
            continue;
        }
        float both[2] = {0.0f, 0.0f};
#pragma unroll
        for (int half = 0; half < 2; half++) {
#pragma unroll
            for (int w = 0; w < kFewWaves; w++) {
                both[half] += sums[w][half][i / (16 * kFewFeatures)][i % (16 * kFewFeatures)];
            }
            if (a.bias[0] != nullptr) {
                both[half] += (float)((const T*)a.bias[half])[own];
            }
        }
        ((T*)a.out[0])[t * a.out_stride[0] + own] = (T)(activate(both[0], a.activation) * both[1]);
        if (a.out[1] != nullptr) {
            ((T*)a.out[1])[t * a.out_stride[1] + own] = (T)both[0];
            ((T*)a.out[2])[t * a.out_stride[2] + own] = (T)both[1];
        }
    }
}

}  // namespace prod
}  // namespace opscv
