// Root-mean-square norm of rows with the residual's addition, its result also in 8 bits, and its gradients.
//
//   h = x + r,  rstd = 1 / sqrt(mean(h^2) + eps),  y = h rstd w
//   8 bits: t = h w, m = max|t|, y = round(t (127 / m)), scale = m rstd / 127
//
// rstd cancels in the 8-bit numbers, so they do not depend on the order of the sum of squares; h stays in 32 bits between
// the addition and the norm (only the `sum` that is handed on is rounded to its type).
//
// Bound by memory: every element is read once and written once, so a row stays in registers between its sum and its
// scaling.  A row belongs to one wavefront (up to 32 elements a lane), to 256 threads, or to 1024; longer rows are read
// twice.  Statistics are 32-bit sums over a lane's elements, then over lanes, then over wavefronts.  8192 rows of 4096 bf16
// with a residual: 48.9 us, 5.5 TB/s; into 8 bits (FLOAT16, 4099 rows of 5120): 35; gradients of 16384 rows of 2048: 67.9.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "token_elem.hpp"
#include "token_kernels.hpp"

namespace opscv {

using namespace tok;

namespace {

constexpr int kMostPerLane = 32;   // elements of a row that a thread keeps in registers
constexpr int64_t kMostBlocks = 1 << 20;  // more rows than these take are walked
constexpr int kPartialRows = 512;  // rows of partial sums of the weight's gradient: two workgroups per CU

dim3 grid(int64_t blocks) { return dim3((unsigned)(blocks < kMostBlocks ? blocks : kMostBlocks)); }

// Sum (and, with `most`, largest value) over the threads of a row: THREADS of them, 64 or a whole workgroup.  `slot`
// alternates between calls, so that one barrier a call is enough.
template <int THREADS>
__device__ __forceinline__ void row_reduce(float& sum, float* most, float (*shared)[2][16], int slot)
{
    sum = wave_sum(sum);
    if (most != nullptr) {
        *most = wave_larger(*most);
    }
    if constexpr (THREADS > 64) {
        const int wave = (int)threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) {
            shared[slot][0][wave] = sum;
            if (most != nullptr) {
                shared[slot][1][wave] = *most;
            }
        }
        __syncthreads();
        sum = 0.0f;
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < THREADS / 64; i++) {
            sum += shared[slot][0][i];
            if (most != nullptr) {
                m = larger(m, shared[slot][1][i]);
            }
        }
        if (most != nullptr) {
            *most = m;
        }
    }
}

// How a row's products become 8-bit numbers: q = round((t * lift) * step).
struct Int8Steps {
    float lift, step;
};

// 127 / m is no number of 32 bits where m is less than 3.7e-37; there both are taken 2^64 times as large, which rounds nothing.
// step 0 for a row of zeros, whose scale is 0 also where eps is and rstd infinite, and, with scale NaN, where the row holds a
// NaN or an infinity.
__device__ __forceinline__ Int8Steps int8_steps(float most, float rstd, float* scale)
{
    const bool finite = most < INFINITY;  // false for NaN too
    *scale = !finite ? NAN : most > 0.0f ? most * rstd / 127.0f : 0.0f;
    const float lift = most < 0x1p-100f ? 0x1p64f : 1.0f;
    return {lift, (finite && most > 0.0f) ? 127.0f / (most * lift) : 0.0f};
}

template <typename T, typename W, bool INT8, int VEC, bool WIDE>
__device__ __forceinline__ void put_row_part(const NormArgs& a, int64_t row, int64_t c, const float (&h)[VEC], float rstd,
                                             Int8Steps steps)
{
    float w[VEC], y[VEC];
    load_part<W, VEC, WIDE>((const W*)a.weight, c, a.width, w);
    if constexpr (INT8) {
        Pack<int8_t, VEC> k;
#pragma unroll
        for (int i = 0; i < VEC; i++) {
            // step is 0 for rows without a finite range; |t * step| is at most 127 and a rounding
            const float q = rintf(h[i] * w[i] * steps.lift * steps.step);
            k.v[i] = steps.step == 0.0f ? (int8_t)0 : (int8_t)(int)fminf(fmaxf(q, -127.0f), 127.0f);
        }
        int8_t* const to = (int8_t*)a.y.ptr + row * a.y.row_stride + c;
        if constexpr (WIDE) {
            *reinterpret_cast<Pack<int8_t, VEC>*>(to) = k;
        } else {
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                if (c + i < a.width) {
                    to[i] = k.v[i];
                }
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < VEC; i++) {
            y[i] = h[i] * w[i] * rstd;
        }
        store_part<T, VEC, WIDE>((T*)a.y.ptr + row * a.y.row_stride, c, a.width, y, a.streaming != 0);
    }
}

template <typename T, int VEC, bool WIDE>
__device__ __forceinline__ void get_row_part(const NormArgs& a, int64_t row, int64_t c, float (&h)[VEC])
{
    load_part<T, VEC, WIDE>((const T*)a.x.ptr + row * a.x.row_stride, c, a.width, h);
    if (a.residual.ptr != nullptr) {
        float r[VEC];
        load_part<T, VEC, WIDE>((const T*)a.residual.ptr + row * a.residual.row_stride, c, a.width, r);
#pragma unroll
        for (int i = 0; i < VEC; i++) {
            h[i] += r[i];
        }
    }
}

// THREADS per row; a workgroup is 256 threads, or THREADS where that is more.  NV vectors of VEC elements a thread.
template <typename T, typename W, bool INT8, int THREADS, int NV, int VEC, bool WIDE>
__global__ __launch_bounds__(THREADS > 256 ? THREADS : 256) void norm_kernel(NormArgs a)
{
    constexpr int kRows = THREADS >= 256 ? 1 : 256 / THREADS;
    __shared__ float shared[2][2][16];
    const int lane = (int)threadIdx.x % THREADS;
    int slot = 0;
    // where a barrier follows (THREADS >= 256), a workgroup has one row and all its threads make as many turns
    for (int64_t row = (int64_t)blockIdx.x * kRows + (int)threadIdx.x / THREADS; row < a.rows;
         row += (int64_t)gridDim.x * kRows) {
        float h[NV][VEC], sum = 0.0f, most = 0.0f;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const int64_t c = ((int64_t)j * THREADS + lane) * VEC;
            if (c < a.width) {
                get_row_part<T, VEC, WIDE>(a, row, c, h[j]);
            } else {
#pragma unroll
                for (int i = 0; i < VEC; i++) {
                    h[j][i] = 0.0f;
                }
            }
        }
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const int64_t c = ((int64_t)j * THREADS + lane) * VEC;
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                sum += h[j][i] * h[j][i];
            }
            if (c < a.width) {
                if (a.sum.ptr != nullptr) {
                    store_part<T, VEC, WIDE>((T*)a.sum.ptr + row * a.sum.row_stride, c, a.width, h[j], a.streaming != 0);
                }
                if constexpr (INT8) {
                    float w[VEC];
                    load_part<W, VEC, WIDE>((const W*)a.weight, c, a.width, w);
#pragma unroll
                    for (int i = 0; i < VEC; i++) {
                        most = larger(most, fabsf(h[j][i] * w[i]));
                    }
                }
            }
        }
        row_reduce<THREADS>(sum, INT8 ? &most : nullptr, shared, slot);
        slot ^= 1;
        const float rstd = 1.0f / sqrtf(sum / (float)a.width + a.eps);
        float scale = 0.0f;
        const Int8Steps steps = INT8 ? int8_steps(most, rstd, &scale) : Int8Steps{};
        if (lane == 0) {
            if (a.rstd != nullptr) {
                a.rstd[row] = rstd;
            }
            if (INT8) {
                a.scale[row] = scale;
            }
        }
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const int64_t c = ((int64_t)j * THREADS + lane) * VEC;
            if (c < a.width) {
                put_row_part<T, W, INT8, VEC, WIDE>(a, row, c, h[j], rstd, steps);
            }
        }
    }
}

// Rows longer than 1024 threads hold: read once for the statistics and once more for the result (`sum` is written in the
// second pass, since it may be x).
template <typename T, typename W, bool INT8, int VEC, bool WIDE>
__global__ __launch_bounds__(1024) void norm_long_kernel(NormArgs a)
{
    __shared__ float shared[2][2][16];
    int slot = 0;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        float sum = 0.0f, most = 0.0f;
        for (int64_t c = (int64_t)threadIdx.x * VEC; c < a.width; c += 1024 * VEC) {
            float h[VEC], w[VEC];
            get_row_part<T, VEC, WIDE>(a, row, c, h);
            load_part<W, VEC, WIDE>((const W*)a.weight, c, a.width, w);
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                sum += h[i] * h[i];
                most = larger(most, fabsf(h[i] * w[i]));
            }
        }
        row_reduce<1024>(sum, INT8 ? &most : nullptr, shared, slot);
        slot ^= 1;
        const float rstd = 1.0f / sqrtf(sum / (float)a.width + a.eps);
        float scale = 0.0f;
        const Int8Steps steps = INT8 ? int8_steps(most, rstd, &scale) : Int8Steps{};
        if (threadIdx.x == 0) {
            if (a.rstd != nullptr) {
                a.rstd[row] = rstd;
            }
            if (INT8) {
                a.scale[row] = scale;
            }
        }
        for (int64_t c = (int64_t)threadIdx.x * VEC; c < a.width; c += 1024 * VEC) {
            float h[VEC];
            get_row_part<T, VEC, WIDE>(a, row, c, h);
            if (a.sum.ptr != nullptr) {
                store_part<T, VEC, WIDE>((T*)a.sum.ptr + row * a.sum.row_stride, c, a.width, h, a.streaming != 0);
            }
            put_row_part<T, W, INT8, VEC, WIDE>(a, row, c, h, rstd, steps);
        }
    }
}

template <typename T, typename W, bool INT8, int VEC, bool WIDE>
hipError_t run_norm(const NormArgs& a, hipStream_t stream)
{
    constexpr int kVectors = kMostPerLane / VEC;
    const int64_t vectors = (a.width + VEC - 1) / VEC;
    if (vectors <= 64 * kVectors / 2) {
        hipLaunchKernelGGL((norm_kernel<T, W, INT8, 64, kVectors / 2, VEC, WIDE>), grid((a.rows + 3) / 4), dim3(256),
                           0, stream, a);
    } else if (vectors <= 256 * kVectors / 2) {
        hipLaunchKernelGGL((norm_kernel<T, W, INT8, 256, kVectors / 2, VEC, WIDE>), grid(a.rows), dim3(256), 0, stream,
                           a);
    } else if (vectors <= 256 * kVectors) {
        hipLaunchKernelGGL((norm_kernel<T, W, INT8, 256, kVectors, VEC, WIDE>), grid(a.rows), dim3(256), 0, stream, a);
    } else if (vectors <= 1024 * kVectors) {
        hipLaunchKernelGGL((norm_kernel<T, W, INT8, 1024, kVectors, VEC, WIDE>), grid(a.rows), dim3(1024), 0, stream,
                           a);
    } else {
        hipLaunchKernelGGL((norm_long_kernel<T, W, INT8, VEC, WIDE>), grid(a.rows), dim3(1024), 0, stream, a);
    }
    return hipGetLastError();
}

template <typename T, typename W>
hipError_t run_norm_type(const NormArgs& a, hipStream_t stream)
{
    constexpr int kVec = 16 / (int)sizeof(T);
    const int e = (int)sizeof(T), ye = a.int8 != 0 ? 1 : e;
    // whole vectors where every row starts on one, their elements one by one otherwise
    const bool vectors = a.width % kVec == 0 && aligned(a.x.ptr, a.x.row_stride, e, 16) &&
                         aligned(a.residual.ptr, a.residual.row_stride, e, 16) &&
                         aligned(a.sum.ptr, a.sum.row_stride, e, 16) &&
                         aligned(a.y.ptr, a.y.row_stride, ye, kVec * ye) &&
                         aligned(a.weight, 0, 1, kVec * (int)sizeof(W));
    if (a.int8 != 0) {
        return vectors ? run_norm<T, W, true, kVec, true>(a, stream) : run_norm<T, W, true, kVec, false>(a, stream);
    }
    return vectors ? run_norm<T, W, false, kVec, true>(a, stream) : run_norm<T, W, false, kVec, false>(a, stream);
}

// ------------------------------------------------------------------------------------------------------ gradients

// Sums over the threads of `R` rows at once, as row_reduce.
template <int THREADS, int R>
__device__ __forceinline__ void rows_reduce(float (&sum)[R], float (*shared)[R][16], int slot)
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

// Gradient of the rows, and of the weight's columns over the rows of one workgroup, which it adds up in registers and
// leaves in its row of `partial`.  THREADS per row; wavefronts of 64-thread rows join their sums through LDS.  R rows at a
// time, as many as a thread's registers hold, so that enough loads are under way with two workgroups a CU (more of them
// would write more partial sums): 16384 rows of 2048 bf16 74 us with one row, 68 with four.
template <typename T, typename W, int THREADS, int NV, int VEC, bool WIDE, bool WEIGHT, int R>
__global__ __launch_bounds__(THREADS > 256 ? THREADS : 256) void norm_grad_kernel(NormGradArgs a)
{
    constexpr int kGroups = THREADS >= 256 ? 1 : 256 / THREADS;
    __shared__ float shared[2][R][16];
    const int lane = (int)threadIdx.x % THREADS;
    float w[NV][VEC], total[NV][VEC];
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const int64_t c = ((int64_t)j * THREADS + lane) * VEC;
#pragma unroll
        for (int i = 0; i < VEC; i++) {
            total[j][i] = w[j][i] = 0.0f;
        }
        if (c < a.width) {
            load_part<W, VEC, WIDE>((const W*)a.weight, c, a.width, w[j]);
        }
    }
    int slot = 0;
    // every thread of a workgroup makes as many turns: the barrier of rows_reduce is met by all (THREADS >= 256: the same
    // rows; 64: no barrier)
    for (int64_t row0 = ((int64_t)blockIdx.x * kGroups + (int)threadIdx.x / THREADS) * R; row0 < a.rows;
         row0 += (int64_t)gridDim.x * kGroups * R) {
        float n[R][NV][VEC], g[R][NV][VEC], rstd[R], along[R];
#pragma unroll
        for (int k = 0; k < R; k++) {
            const int64_t row = row0 + k;
            const bool live = row < a.rows;
            rstd[k] = live ? a.rstd[row] : 0.0f;
#pragma unroll
            for (int j = 0; j < NV; j++) {
                const int64_t c = ((int64_t)j * THREADS + lane) * VEC;
                if (live && c < a.width) {
                    load_part<T, VEC, WIDE>((const T*)a.sum.ptr + row * a.sum.row_stride, c, a.width, n[k][j]);
                    load_part<T, VEC, WIDE>((const T*)a.grad_y.ptr + row * a.grad_y.row_stride, c, a.width, g[k][j]);
                } else {
#pragma unroll
                    for (int i = 0; i < VEC; i++) {
                        n[k][j][i] = g[k][j][i] = 0.0f;
                    }
                }
            }
        }
#pragma unroll
        for (int k = 0; k < R; k++) {
            along[k] = 0.0f;
#pragma unroll
            for (int j = 0; j < NV; j++) {
#pragma unroll
                for (int i = 0; i < VEC; i++) {
                    n[k][j][i] *= rstd[k];
                    if (WEIGHT) {
                        total[j][i] += g[k][j][i] * n[k][j][i];
                    }
                    g[k][j][i] *= w[j][i];
                    along[k] += g[k][j][i] * n[k][j][i];
                }
            }
        }
        rows_reduce<THREADS, R>(along, shared, slot);
        slot ^= 1;
#pragma unroll
        for (int k = 0; k < R; k++) {
            const int64_t row = row0 + k;
            if (row >= a.rows) {
                break;
            }
            const float mean = along[k] / (float)a.width;
#pragma unroll
            for (int j = 0; j < NV; j++) {
                const int64_t c = ((int64_t)j * THREADS + lane) * VEC;
                if (c < a.width) {
                    float s[VEC] = {0.0f};
                    if (a.grad_sum.ptr != nullptr) {
                        load_part<T, VEC, WIDE>((const T*)a.grad_sum.ptr + row * a.grad_sum.row_stride, c, a.width, s);
                    }
#pragma unroll
                    for (int i = 0; i < VEC; i++) {
                        s[i] += (g[k][j][i] - n[k][j][i] * mean) * rstd[k];
                    }
                    store_part<T, VEC, WIDE>((T*)a.grad_x.ptr + row * a.grad_x.row_stride, c, a.width, s, false);
                }
            }
        }
    }
    if constexpr (WEIGHT) {
        // the one workgroup of few rows writes the gradient itself
        __shared__ float joined[kGroups > 1 ? THREADS * VEC : 1];
        const auto put = [&](int64_t c, float x) {
            if (gridDim.x == 1) {
                ((W*)a.grad_weight)[c] = (W)x;
            } else {
                a.partial[(int64_t)blockIdx.x * a.width + c] = x;
            }
        };
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const int64_t c = ((int64_t)j * THREADS + lane) * VEC;
            if constexpr (kGroups > 1) {
                for (int turn = 0; turn < kGroups; turn++) {  // the wavefronts add in order
                    if ((int)threadIdx.x / THREADS == turn) {
#pragma unroll
                        for (int i = 0; i < VEC; i++) {
                            float& slot_sum = joined[i * THREADS + lane];
                            slot_sum = turn == 0 ? total[j][i] : slot_sum + total[j][i];
                            if (turn == kGroups - 1 && c + i < a.width) {
                                put(c + i, slot_sum);
                            }
                        }
                    }
                    __syncthreads();
                }
            } else {
#pragma unroll
                for (int i = 0; i < VEC; i++) {
                    if (c + i < a.width) {
                        put(c + i, total[j][i]);
                    }
                }
            }
        }
    }
}

// Rows longer than 1024 threads hold, read twice: the sum along the row, then the gradient.  The weight's gradient comes
// from norm_weight_long_kernel.
template <typename T, typename W, int VEC, bool WIDE>
__global__ __launch_bounds__(1024) void norm_grad_long_kernel(NormGradArgs a)
{
    __shared__ float shared[2][2][16];
    int slot = 0;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const float rstd = a.rstd[row];
        const T* const sum = (const T*)a.sum.ptr + row * a.sum.row_stride;
        const T* const gy = (const T*)a.grad_y.ptr + row * a.grad_y.row_stride;
        float along = 0.0f;
        for (int64_t c = (int64_t)threadIdx.x * VEC; c < a.width; c += 1024 * VEC) {
            float n[VEC], g[VEC], w[VEC];
            load_part<T, VEC, WIDE>(sum, c, a.width, n);
            load_part<T, VEC, WIDE>(gy, c, a.width, g);
            load_part<W, VEC, WIDE>((const W*)a.weight, c, a.width, w);
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                along += g[i] * w[i] * (n[i] * rstd);
            }
        }
        row_reduce<1024>(along, nullptr, shared, slot);
        slot ^= 1;
        along /= (float)a.width;
        for (int64_t c = (int64_t)threadIdx.x * VEC; c < a.width; c += 1024 * VEC) {
            float n[VEC], g[VEC], w[VEC], s[VEC] = {0.0f};
            load_part<T, VEC, WIDE>(sum, c, a.width, n);
            load_part<T, VEC, WIDE>(gy, c, a.width, g);
            load_part<W, VEC, WIDE>((const W*)a.weight, c, a.width, w);
            if (a.grad_sum.ptr != nullptr) {
                load_part<T, VEC, WIDE>((const T*)a.grad_sum.ptr + row * a.grad_sum.row_stride, c, a.width, s);
            }
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                s[i] += (g[i] * w[i] - n[i] * rstd * along) * rstd;
            }
            store_part<T, VEC, WIDE>((T*)a.grad_x.ptr + row * a.grad_x.row_stride, c, a.width, s, false);
        }
    }
}

// One column a thread, every gridDim.y-th row: before the rows' gradient is written, since that may be gradY itself.
template <typename T>
__global__ __launch_bounds__(256) void norm_weight_long_kernel(NormGradArgs a)
{
    const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (c >= a.width) {
        return;
    }
    float total = 0.0f;
    for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
        total += (float)((const T*)a.grad_y.ptr)[row * a.grad_y.row_stride + c] *
                 ((float)((const T*)a.sum.ptr)[row * a.sum.row_stride + c] * a.rstd[row]);
    }
    a.partial[(int64_t)blockIdx.y * a.width + c] = total;
}

// Sum of the rows of `partial`: 32 columns a workgroup, every eighth row a thread, joined in order.
template <typename W>
__global__ __launch_bounds__(256) void norm_weight_kernel(const float* __restrict__ partial, int64_t rows, int64_t width,
                                                          W* __restrict__ out)
{
    __shared__ float shared[8][32];
    const int column = (int)threadIdx.x & 31, part = (int)threadIdx.x >> 5;
    const int64_t c = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 32 + column;
    float total = 0.0f;
    if (c < width) {
#pragma unroll 8
        for (int64_t r = part; r < rows; r += 8) {
            total += partial[r * width + c];
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

template <typename T, typename W, int THREADS, int NV, int VEC, bool WIDE>
void launch_norm_grad(const NormGradArgs& a, hipStream_t stream)
{
    constexpr int kThreads = THREADS > 256 ? THREADS : 256;
    constexpr int kRowsATime = THREADS > 256 ? 1 : kMostPerLane / (NV * VEC);
    constexpr int64_t kRowsABlock = (THREADS >= 256 ? 1 : 256 / THREADS) * kRowsATime;
    if (a.grad_weight != nullptr) {
        hipLaunchKernelGGL((norm_grad_kernel<T, W, THREADS, NV, VEC, WIDE, true, kRowsATime>),
                           dim3((unsigned)norm_grad_partials(a)), dim3(kThreads), 0, stream, a);
    } else {
        hipLaunchKernelGGL((norm_grad_kernel<T, W, THREADS, NV, VEC, WIDE, false, kRowsATime>),
                           grid((a.rows + kRowsABlock - 1) / kRowsABlock), dim3(kThreads), 0, stream, a);
    }
}

template <typename T, typename W, int VEC, bool WIDE>
hipError_t run_norm_grad(const NormGradArgs& a, hipStream_t stream)
{
    constexpr int kVectors = kMostPerLane / VEC;
    const int64_t vectors = (a.width + VEC - 1) / VEC, partials = norm_grad_partials(a);
    bool joined = partials == 1;  // the kernel of short rows writes a single partial sum where it belongs
    if (vectors <= 64 * kVectors / 2) {
        launch_norm_grad<T, W, 64, kVectors / 2, VEC, WIDE>(a, stream);
    } else if (vectors <= 256 * kVectors / 4) {
        launch_norm_grad<T, W, 256, kVectors / 4, VEC, WIDE>(a, stream);
    } else if (vectors <= 256 * kVectors / 2) {
        launch_norm_grad<T, W, 256, kVectors / 2, VEC, WIDE>(a, stream);
    } else if (vectors <= 256 * kVectors) {
        launch_norm_grad<T, W, 256, kVectors, VEC, WIDE>(a, stream);
    } else if (vectors <= 1024 * kVectors) {
        launch_norm_grad<T, W, 1024, kVectors, VEC, WIDE>(a, stream);
    } else {
        joined = false;
        if (a.grad_weight != nullptr) {
            hipLaunchKernelGGL((norm_weight_long_kernel<T>), dim3((unsigned)((a.width + 255) / 256), (unsigned)partials),
                               dim3(256), 0, stream, a);
        }
        if (a.rows > 0) {
            hipLaunchKernelGGL((norm_grad_long_kernel<T, W, VEC, WIDE>), grid(a.rows), dim3(1024), 0, stream, a);
        }
    }
    if (a.grad_weight != nullptr && !joined) {
        // rows of more than 2^25 columns take more than one row of workgroups: 2^24 of 256 threads are more than a launch holds
        // in one
        const int64_t blocks = (a.width + 31) / 32;
        const dim3 columns((unsigned)(blocks < kMostBlocks ? blocks : kMostBlocks), (unsigned)((blocks + kMostBlocks - 1) / kMostBlocks));
        hipLaunchKernelGGL((norm_weight_kernel<W>), columns, dim3(256), 0, stream, a.partial, partials, a.width,
                           (W*)a.grad_weight);
    }
    return hipGetLastError();
}

template <typename T, typename W>
hipError_t run_norm_grad_type(const NormGradArgs& a, hipStream_t stream)
{
    constexpr int kVec = 16 / (int)sizeof(T);
    const int e = (int)sizeof(T);
    const bool vectors = a.width % kVec == 0 && aligned(a.grad_y.ptr, a.grad_y.row_stride, e, 16) &&
                         aligned(a.grad_sum.ptr, a.grad_sum.row_stride, e, 16) &&
                         aligned(a.sum.ptr, a.sum.row_stride, e, 16) &&
                         aligned(a.grad_x.ptr, a.grad_x.row_stride, e, 16) &&
                         aligned(a.weight, 0, 1, kVec * (int)sizeof(W));
    return vectors ? run_norm_grad<T, W, kVec, true>(a, stream) : run_norm_grad<T, W, kVec, false>(a, stream);
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

}  // namespace

int64_t norm_grad_partials(const NormGradArgs& a)
{
    // A workgroup takes up to eight rows at a time; one row of partial sums even where there are no rows.  Of wide rows it
    // takes one or two, and few of them go to as many workgroups as there are CUs (64 rows of 5120 FLOAT: 10.8 us, eight rows
    // a workgroup 25.8; 419: 16.6 and 28.7), unless one workgroup, which needs no second kernel, is as fast (four rows of
    // 2048: 6.6 us, of 5120: 14.5).
    constexpr int64_t kWide = 1024, kWidest = 4096;
    const int64_t groups = (a.rows + 7) / 8;
    if (a.rows <= 1 || (groups == 1 && a.width <= kWidest)) {
        return 1;
    }
    const int64_t spread = a.width <= kWide ? groups : (a.rows < 256 ? a.rows : 256);
    return groups < spread ? spread : (groups < kPartialRows ? groups : kPartialRows);
}

hipError_t launch_residual_norm(const NormArgs& args, hipStream_t stream)
{
    if (args.rows < 1 || args.width < 1) {
        return hipErrorInvalidValue;
    }
    NormArgs a = args;
    a.streaming = a.rows * a.width * elem_size((Elem)a.elem) >= kStreamBytes ? 1 : 0;
    return by_type(a.elem, a.weight_float, [&](auto* t, auto* w) {
        return run_norm_type<std::remove_pointer_t<decltype(t)>, std::remove_pointer_t<decltype(w)>>(a, stream);
    });
}

hipError_t launch_residual_norm_grad(const NormGradArgs& a, hipStream_t stream)
{
    if (a.width < 1 || (a.grad_weight != nullptr && a.partial == nullptr)) {
        return hipErrorInvalidValue;
    }
    return by_type(a.elem, a.weight_float, [&](auto* t, auto* w) {
        return run_norm_grad_type<std::remove_pointer_t<decltype(t)>, std::remove_pointer_t<decltype(w)>>(a, stream);
    });
}

}  // namespace opscv
