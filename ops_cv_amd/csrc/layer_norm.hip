// Layer norm of rows with the residual's addition, and its gradients.
//
//   h = x + r,  m = mean(h),  rstd = 1 / sqrt(mean((h - m)^2) + eps),  y = (h - m) rstd w + b
//   n = (h - m) rstd, g = gy w:  gx = (g - mean(g) - n mean(g n)) rstd + gs,  gw = sum gy n,  gb = sum gy
//
// The squares are taken of h - m0 in a second round over the registers, not as mean(h^2) - m^2, which loses the variance of
// rows whose mean is large beside their spread; h stays in 32 bits between the addition and the norm.  m0 is the mean as
// summed up in 32 bits, off by some 2^-24 of the values, which is much of a small spread; the mean of h - m0, from the same
// round, corrects it:
//   m = m0 + mean(h - m0),  variance = mean((h - m0)^2) - mean(h - m0)^2
//
// Bound by memory: every element is read once and written once, so a row stays in registers between its sums and its
// result.  A row belongs to one wavefront (up to 16 elements a lane, or 24), to 256 threads, or to 1024; longer rows are read three
// times.  Sums are 32-bit, over a thread's elements, then over lanes, then over wavefronts, in a fixed order.  10952 rows of 1280
// fp16, x, residual, sum and y: 23.3 us, 4.8 TB/s (22.7 without the mean's correction); gradients of 16384 rows of 2048 bf16 with their other gradient 60.4, 4.5 TB/s,
// of which the join of the columns' partial sums is 4.5; eight rows of 4096: 6.3, the launch.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "token_elem.hpp"
#include "token_kernels.hpp"
#include "token_rows.hpp"

namespace opscv {

using namespace tok;

namespace {

constexpr int kPartialRows = 512;  // rows of partial sums of the columns' gradients: two workgroups per CU

template <typename W, int VEC, bool WIDE>
__device__ __forceinline__ void get_columns(const void* from, int64_t c, int64_t width, float otherwise, float (&w)[VEC])
{
    if (from != nullptr) {
        load_part<W, VEC, WIDE>((const W*)from, c, width, w);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; i++) {
            w[i] = otherwise;
        }
    }
}

template <typename T, int VEC, bool WIDE>
__device__ __forceinline__ void get_row_part(const LayerNormArgs& a, int64_t row, int64_t c, float (&h)[VEC])
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

template <typename T, typename W, int VEC, bool WIDE>
__device__ __forceinline__ void put_row_part(const LayerNormArgs& a, int64_t row, int64_t c, const float (&h)[VEC], float mean,
                                             float rstd)
{
    float w[VEC], b[VEC], y[VEC];
    get_columns<W, VEC, WIDE>(a.weight, c, a.width, 1.0f, w);
    get_columns<W, VEC, WIDE>(a.bias, c, a.width, 0.0f, b);
#pragma unroll
    for (int i = 0; i < VEC; i++) {
        y[i] = (h[i] - mean) * rstd * w[i] + b[i];
    }
    store_part<T, VEC, WIDE>((T*)a.y.ptr + row * a.y.row_stride, c, a.width, y, a.streaming != 0);
}

__device__ __forceinline__ void put_statistics(const LayerNormArgs& a, int64_t row, float mean, float rstd)
{
    if (a.mean != nullptr) {
        a.mean[row] = mean;
    }
    if (a.rstd != nullptr) {
        a.rstd[row] = rstd;
    }
}

// Mean and rstd from the first mean and the sums of what it leaves of the elements, and of its squares.
__device__ __forceinline__ void statistics(const LayerNormArgs& a, float first, const float (&left)[2], float* mean, float* rstd)
{
    const float more = left[0] / (float)a.width, variance = left[1] / (float)a.width - more * more;
    *mean = more == more ? first + more : first;  // an infinite mean leaves NaN
    *rstd = 1.0f / sqrtf((variance < 0.0f ? 0.0f : variance) + a.eps);
}

// THREADS per row; a workgroup is 256 threads, or THREADS where that is more.  NV vectors of VEC elements a thread.
template <typename T, typename W, int THREADS, int NV, int VEC, bool WIDE>
__global__ __launch_bounds__(THREADS > 256 ? THREADS : 256) void layer_norm_kernel(LayerNormArgs a)
{
    constexpr int kRows = THREADS >= 256 ? 1 : 256 / THREADS;
    __shared__ float shared[1][1][16], shared_left[1][2][16];
    const int lane = (int)threadIdx.x % THREADS;
    // where a barrier follows (THREADS >= 256), a workgroup has one row and all its threads make as many turns
    for (int64_t row = (int64_t)blockIdx.x * kRows + (int)threadIdx.x / THREADS; row < a.rows;
         row += (int64_t)gridDim.x * kRows) {
        float h[NV][VEC], sum[1] = {0.0f};
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
                sum[0] += h[j][i];
            }
            if (c < a.width && a.sum.ptr != nullptr) {
                store_part<T, VEC, WIDE>((T*)a.sum.ptr + row * a.sum.row_stride, c, a.width, h[j], a.streaming != 0);
            }
        }
        // two reductions a row, each with places of its own: one barrier a reduction is enough
        rows_reduce<THREADS, 1>(sum, shared, 0);
        const float first = sum[0] / (float)a.width;
        float left[2] = {0.0f, 0.0f}, mean, rstd;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const int64_t c = ((int64_t)j * THREADS + lane) * VEC;
            if (c < a.width) {
#pragma unroll
                for (int i = 0; i < VEC; i++) {
                    const float d = WIDE || c + i < a.width ? h[j][i] - first : 0.0f;
                    left[0] += d;
                    left[1] += d * d;
                }
            }
        }
        rows_reduce<THREADS, 2>(left, shared_left, 0);
        statistics(a, first, left, &mean, &rstd);
        if (lane == 0) {
            put_statistics(a, row, mean, rstd);
        }
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const int64_t c = ((int64_t)j * THREADS + lane) * VEC;
            if (c < a.width) {
                put_row_part<T, W, VEC, WIDE>(a, row, c, h[j], mean, rstd);
            }
        }
    }
}

// Rows longer than 1024 threads hold: read for the mean, for the squares and for the result (`sum` is written in the last
// round, since it may be x).  A thread adds up thousands of numbers here, and the correction of the mean is as good as the
// first mean is near: its sum is compensated (Kahan, "Further remarks on reducing truncation errors", 1965), a vector at a time.
template <typename T, typename W, int VEC, bool WIDE>
__global__ __launch_bounds__(1024) void layer_norm_long_kernel(LayerNormArgs a)
{
    __shared__ float shared[1][1][16], shared_left[1][2][16];
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        float sum[1] = {0.0f}, lost = 0.0f;
        for (int64_t c = (int64_t)threadIdx.x * VEC; c < a.width; c += 1024 * VEC) {
            float h[VEC], part = 0.0f;
            get_row_part<T, VEC, WIDE>(a, row, c, h);
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                part += h[i];
            }
            part -= lost;
            const float total = sum[0] + part;
            lost = (total - sum[0]) - part;
            lost = lost == lost ? lost : 0.0f;  // an infinite sum stays one
            sum[0] = total;
        }
        rows_reduce<1024, 1>(sum, shared, 0);
        const float first = sum[0] / (float)a.width;
        float left[2] = {0.0f, 0.0f}, mean, rstd;
        for (int64_t c = (int64_t)threadIdx.x * VEC; c < a.width; c += 1024 * VEC) {
            float h[VEC];
            get_row_part<T, VEC, WIDE>(a, row, c, h);
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                const float d = WIDE || c + i < a.width ? h[i] - first : 0.0f;
                left[0] += d;
                left[1] += d * d;
            }
        }
        rows_reduce<1024, 2>(left, shared_left, 0);
        statistics(a, first, left, &mean, &rstd);
        if (threadIdx.x == 0) {
            put_statistics(a, row, mean, rstd);
        }
        for (int64_t c = (int64_t)threadIdx.x * VEC; c < a.width; c += 1024 * VEC) {
            float h[VEC];
            get_row_part<T, VEC, WIDE>(a, row, c, h);
            if (a.sum.ptr != nullptr) {
                store_part<T, VEC, WIDE>((T*)a.sum.ptr + row * a.sum.row_stride, c, a.width, h, a.streaming != 0);
            }
            put_row_part<T, W, VEC, WIDE>(a, row, c, h, mean, rstd);
        }
    }
}

template <typename T, typename W, int VEC, bool WIDE>
hipError_t run_layer_norm(const LayerNormArgs& a, hipStream_t stream)
{
    constexpr int kVectors = kMostPerLane / VEC;
    const int64_t vectors = (a.width + VEC - 1) / VEC;
    if (vectors <= 64 * kVectors / 2) {
        hipLaunchKernelGGL((layer_norm_kernel<T, W, 64, kVectors / 2, VEC, WIDE>), grid((a.rows + 3) / 4), dim3(256), 0,
                           stream, a);
    } else if (sizeof(T) == 2 && vectors <= 64 * 3 && a.rows >= 4096) {
        // Little more than 1024 elements leave many of 256 threads without any: 10952 rows of 1280 bf16 23 us here and 27
        // with 256 threads, of 1025 26 and 41.  Rows of 2048, and of floats, are slower here (35 us and 34; 45 and 42), and
        // 2048 rows of 1280 want the threads (8 us and 11).
        hipLaunchKernelGGL((layer_norm_kernel<T, W, 64, 3, VEC, WIDE>), grid((a.rows + 3) / 4), dim3(256), 0, stream, a);
    } else if (vectors <= 256 * kVectors / 2) {
        hipLaunchKernelGGL((layer_norm_kernel<T, W, 256, kVectors / 2, VEC, WIDE>), grid(a.rows), dim3(256), 0, stream, a);
    } else if (vectors <= 256 * kVectors) {
        hipLaunchKernelGGL((layer_norm_kernel<T, W, 256, kVectors, VEC, WIDE>), grid(a.rows), dim3(256), 0, stream, a);
    } else if (vectors <= 1024 * kVectors) {
        hipLaunchKernelGGL((layer_norm_kernel<T, W, 1024, kVectors, VEC, WIDE>), grid(a.rows), dim3(1024), 0, stream, a);
    } else {
        hipLaunchKernelGGL((layer_norm_long_kernel<T, W, VEC, WIDE>), grid(a.rows), dim3(1024), 0, stream, a);
    }
    return hipGetLastError();
}

template <typename T, typename W>
hipError_t run_layer_norm_type(const LayerNormArgs& a, hipStream_t stream)
{
    constexpr int kVec = 16 / (int)sizeof(T);
    const int e = (int)sizeof(T);
    // whole vectors where every row starts on one, their elements one by one otherwise
    const bool vectors = a.width % kVec == 0 && aligned(a.x.ptr, a.x.row_stride, e, 16) &&
                         aligned(a.residual.ptr, a.residual.row_stride, e, 16) &&
                         aligned(a.sum.ptr, a.sum.row_stride, e, 16) && aligned(a.y.ptr, a.y.row_stride, e, 16) &&
                         aligned(a.weight, 0, 1, kVec * (int)sizeof(W)) && aligned(a.bias, 0, 1, kVec * (int)sizeof(W));
    return vectors ? run_layer_norm<T, W, kVec, true>(a, stream) : run_layer_norm<T, W, kVec, false>(a, stream);
}

// ------------------------------------------------------------------------------------------------------ gradients

// What a thread reads of R rows, in the tensors' type.
template <typename T, int NV, int VEC, int R>
struct RowsRead {
    Pack<T, VEC> sum[R][NV], grad_y[R][NV], grad_sum[R][NV];
    float rstd[R], mean[R];
};

template <typename T, int N, bool WIDE>
__device__ __forceinline__ Pack<T, N> read_part(const T* row, int64_t c, int64_t width)
{
    if constexpr (WIDE) {
        return *reinterpret_cast<const Pack<T, N>*>(row + c);
    } else {
        Pack<T, N> k;
        if (c + N <= width) {
            const Loose<T, N> l = *reinterpret_cast<const Loose<T, N>*>(row + c);
#pragma unroll
            for (int i = 0; i < N; i++) {
                k.v[i] = l.v[i];
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; i++) {
                k.v[i] = c + i < width ? row[c + i] : (T)0.0f;
            }
        }
        return k;
    }
}

template <typename T, int THREADS, int NV, int VEC, bool WIDE, int R>
__device__ __forceinline__ void read_rows(const LayerNormGradArgs& a, int64_t row0, int lane, RowsRead<T, NV, VEC, R>& x)
{
#pragma unroll
    for (int k = 0; k < R; k++) {
        // rows past the end are read as the last one, and left out
        const int64_t row = row0 + k < a.rows ? row0 + k : a.rows - 1;
        x.rstd[k] = a.rstd[row];
        x.mean[k] = a.mean[row];
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const int64_t c = ((int64_t)j * THREADS + lane) * VEC;
            if (c < a.width) {
                x.sum[k][j] = read_part<T, VEC, WIDE>((const T*)a.sum.ptr + row * a.sum.row_stride, c, a.width);
                x.grad_y[k][j] = read_part<T, VEC, WIDE>((const T*)a.grad_y.ptr + row * a.grad_y.row_stride, c, a.width);
                if (a.grad_sum.ptr != nullptr) {
                    x.grad_sum[k][j] = read_part<T, VEC, WIDE>((const T*)a.grad_sum.ptr + row * a.grad_sum.row_stride, c, a.width);
                }
            }
        }
    }
}

// Gradient of the rows, and of the weight's and bias's columns over the rows of one workgroup, which it adds up in registers
// and leaves in its rows of `partial`.  THREADS per row; wavefronts of 64-thread rows join their sums through LDS.  R rows at
// a time, and with AHEAD the next ones' loads go out before these are worked on, so that enough of them are under way with two
// workgroups a CU (more of them would write more partial sums): 16384 rows of 2048 bf16 with their other gradient 79 us
// without.
template <typename T, typename W, int THREADS, int NV, int VEC, bool WIDE, bool COLUMNS, int R, bool AHEAD>
__global__ __launch_bounds__(THREADS > 256 ? THREADS : 256) void layer_norm_grad_kernel(LayerNormGradArgs a)
{
    constexpr int kGroups = THREADS >= 256 ? 1 : 256 / THREADS;
    __shared__ float shared[2][2 * R][16];
    const int lane = (int)threadIdx.x % THREADS;
    float w[NV][VEC], total_n[NV][VEC], total[NV][VEC];
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const int64_t c = ((int64_t)j * THREADS + lane) * VEC;
#pragma unroll
        for (int i = 0; i < VEC; i++) {
            total_n[j][i] = total[j][i] = w[j][i] = 0.0f;
        }
        if (c < a.width) {
            get_columns<W, VEC, WIDE>(a.weight, c, a.width, 1.0f, w[j]);
        }
    }
    int slot = 0;
    // every thread of a workgroup makes as many turns: the barrier of rows_reduce is met by all (THREADS >= 256: the same
    // rows; 64: no barrier)
    const int64_t step = (int64_t)gridDim.x * kGroups * R;
    int64_t row0 = ((int64_t)blockIdx.x * kGroups + (int)threadIdx.x / THREADS) * R;
    RowsRead<T, NV, VEC, R> next;
    if (AHEAD && row0 < a.rows) {
        read_rows<T, THREADS, NV, VEC, WIDE, R>(a, row0, lane, next);
    }
    for (; row0 < a.rows; row0 += step) {
        RowsRead<T, NV, VEC, R> x;
        if constexpr (AHEAD) {
            x = next;
            if (row0 + step < a.rows) {
                read_rows<T, THREADS, NV, VEC, WIDE, R>(a, row0 + step, lane, next);
            }
        } else {
            read_rows<T, THREADS, NV, VEC, WIDE, R>(a, row0, lane, x);
        }
        float along[2 * R];
        const auto values = [&](int k, int j, int i, float* n, float* g) {
            *n = ((float)x.sum[k][j].v[i] - x.mean[k]) * x.rstd[k];
            *g = (float)x.grad_y[k][j].v[i];
        };
#pragma unroll
        for (int k = 0; k < R; k++) {
            along[2 * k] = along[2 * k + 1] = 0.0f;
            const bool live = row0 + k < a.rows;
#pragma unroll
            for (int j = 0; j < NV; j++) {
                if (((int64_t)j * THREADS + lane) * VEC < a.width && live) {
#pragma unroll
                    for (int i = 0; i < VEC; i++) {
                        float n, g;  // past the row's end g is 0
                        values(k, j, i, &n, &g);
                        if (COLUMNS) {
                            total_n[j][i] += g * n;
                            total[j][i] += g;
                        }
                        g *= w[j][i];
                        along[2 * k] += g;
                        along[2 * k + 1] += g * n;
                    }
                }
            }
        }
        rows_reduce<THREADS, 2 * R>(along, shared, slot);
        slot ^= 1;
#pragma unroll
        for (int k = 0; k < R; k++) {
            const int64_t row = row0 + k;
            if (row >= a.rows) {
                break;
            }
            const float mean_g = along[2 * k] / (float)a.width, mean_gn = along[2 * k + 1] / (float)a.width;
#pragma unroll
            for (int j = 0; j < NV; j++) {
                const int64_t c = ((int64_t)j * THREADS + lane) * VEC;
                if (c < a.width) {
                    float s[VEC];
#pragma unroll
                    for (int i = 0; i < VEC; i++) {
                        float n, g;
                        values(k, j, i, &n, &g);
                        s[i] = (g * w[j][i] - mean_g - n * mean_gn) * x.rstd[k];
                        if (a.grad_sum.ptr != nullptr) {
                            s[i] += (float)x.grad_sum[k][j].v[i];
                        }
                    }
                    store_part<T, VEC, WIDE>((T*)a.grad_x.ptr + row * a.grad_x.row_stride, c, a.width, s, false);
                }
            }
        }
    }
    if constexpr (COLUMNS) {
        // the one workgroup of few rows writes the gradients itself
        __shared__ float joined[kGroups > 1 ? THREADS * VEC : 1];
        const auto put = [&](void* out, int part, int64_t c, float x) {
            if (out == nullptr) {
                return;
            }
            if (gridDim.x == 1) {
                ((W*)out)[c] = (W)x;
            } else {
                a.partial[((int64_t)part * gridDim.x + blockIdx.x) * a.width + c] = x;
            }
        };
#pragma unroll
        for (int part = 0; part < 2; part++) {
            void* const out = part == 0 ? a.grad_weight : a.grad_bias;
#pragma unroll
            for (int j = 0; j < NV; j++) {
                const int64_t c = ((int64_t)j * THREADS + lane) * VEC;
                const float(&own)[VEC] = part == 0 ? total_n[j] : total[j];
                if constexpr (kGroups > 1) {
                    for (int turn = 0; turn < kGroups; turn++) {  // the wavefronts add in order
                        if ((int)threadIdx.x / THREADS == turn) {
#pragma unroll
                            for (int i = 0; i < VEC; i++) {
                                float& slot_sum = joined[i * THREADS + lane];
                                slot_sum = turn == 0 ? own[i] : slot_sum + own[i];
                                if (turn == kGroups - 1 && c + i < a.width) {
                                    put(out, part, c + i, slot_sum);
                                }
                            }
                        }
                        __syncthreads();
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < VEC; i++) {
                        if (c + i < a.width) {
                            put(out, part, c + i, own[i]);
                        }
                    }
                }
            }
        }
    }
}

// Rows longer than 1024 threads hold, read twice: the sums along the row, then the gradient.  The columns' gradients come
// from layer_norm_columns_long_kernel.
template <typename T, typename W, int VEC, bool WIDE>
__global__ __launch_bounds__(1024) void layer_norm_grad_long_kernel(LayerNormGradArgs a)
{
    __shared__ float shared[2][2][16];
    int slot = 0;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const float rstd = a.rstd[row], mean = a.mean[row];
        const T* const sum = (const T*)a.sum.ptr + row * a.sum.row_stride;
        const T* const gy = (const T*)a.grad_y.ptr + row * a.grad_y.row_stride;
        float along[2] = {0.0f, 0.0f};
        for (int64_t c = (int64_t)threadIdx.x * VEC; c < a.width; c += 1024 * VEC) {
            float n[VEC], g[VEC], w[VEC];
            load_part<T, VEC, WIDE>(sum, c, a.width, n);
            load_part<T, VEC, WIDE>(gy, c, a.width, g);
            get_columns<W, VEC, WIDE>(a.weight, c, a.width, 1.0f, w);
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                const float gw = g[i] * w[i];
                along[0] += gw;
                along[1] += gw * ((n[i] - mean) * rstd);
            }
        }
        rows_reduce<1024, 2>(along, shared, slot);
        slot ^= 1;
        const float mean_g = along[0] / (float)a.width, mean_gn = along[1] / (float)a.width;
        for (int64_t c = (int64_t)threadIdx.x * VEC; c < a.width; c += 1024 * VEC) {
            float n[VEC], g[VEC], w[VEC], s[VEC] = {0.0f};
            load_part<T, VEC, WIDE>(sum, c, a.width, n);
            load_part<T, VEC, WIDE>(gy, c, a.width, g);
            get_columns<W, VEC, WIDE>(a.weight, c, a.width, 1.0f, w);
            if (a.grad_sum.ptr != nullptr) {
                load_part<T, VEC, WIDE>((const T*)a.grad_sum.ptr + row * a.grad_sum.row_stride, c, a.width, s);
            }
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                s[i] += (g[i] * w[i] - mean_g - (n[i] - mean) * rstd * mean_gn) * rstd;
            }
            store_part<T, VEC, WIDE>((T*)a.grad_x.ptr + row * a.grad_x.row_stride, c, a.width, s, false);
        }
    }
}

// One column a thread, every gridDim.y-th row: before the rows' gradient is written, since that may be gradY itself.
template <typename T>
__global__ __launch_bounds__(256) void layer_norm_columns_long_kernel(LayerNormGradArgs a)
{
    const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (c >= a.width) {
        return;
    }
    float total_n = 0.0f, total = 0.0f;
    for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
        const float g = (float)((const T*)a.grad_y.ptr)[row * a.grad_y.row_stride + c];
        total_n += g * (((float)((const T*)a.sum.ptr)[row * a.sum.row_stride + c] - a.mean[row]) * a.rstd[row]);
        total += g;
    }
    a.partial[(int64_t)blockIdx.y * a.width + c] = total_n;
    a.partial[((int64_t)gridDim.y + blockIdx.y) * a.width + c] = total;
}

template <typename T, typename W, int THREADS, int NV, int VEC, bool WIDE>
void launch_grad(const LayerNormGradArgs& a, hipStream_t stream)
{
    constexpr int kThreads = THREADS > 256 ? THREADS : 256;
    // as many rows as 64 bytes of each tensor a thread hold, whatever the alignment: the columns' sums depend on it; the
    // registers of a second set are there for whole vectors only
    constexpr int kMost = 64 / (int)sizeof(T);
    constexpr int kRowsATime = THREADS > 256 || kMost < NV * VEC ? 1 : kMost / (NV * VEC);
    constexpr bool kAhead = WIDE && THREADS <= 256 && NV * VEC <= kMost;
    constexpr int64_t kRowsABlock = (THREADS >= 256 ? 1 : 256 / THREADS) * kRowsATime;
    if (a.grad_weight != nullptr || a.grad_bias != nullptr) {
        hipLaunchKernelGGL((layer_norm_grad_kernel<T, W, THREADS, NV, VEC, WIDE, true, kRowsATime, kAhead>),
                           dim3((unsigned)layer_norm_grad_partials(a)), dim3(kThreads), 0, stream, a);
    } else {
        hipLaunchKernelGGL((layer_norm_grad_kernel<T, W, THREADS, NV, VEC, WIDE, false, kRowsATime, kAhead>),
                           grid((a.rows + kRowsABlock - 1) / kRowsABlock), dim3(kThreads), 0, stream, a);
    }
}

template <typename T, typename W, int VEC, bool WIDE>
hipError_t run_grad(const LayerNormGradArgs& a, hipStream_t stream)
{
    constexpr int kVectors = kMostPerLane / VEC;
    const int64_t vectors = (a.width + VEC - 1) / VEC, partials = layer_norm_grad_partials(a);
    const bool columns = a.grad_weight != nullptr || a.grad_bias != nullptr;
    bool joined = partials == 1;  // the kernel of short rows writes single partial sums where they belong
    if (vectors <= 64 * kVectors / 2) {
        launch_grad<T, W, 64, kVectors / 2, VEC, WIDE>(a, stream);
    } else if (vectors <= 256 * kVectors / 4) {
        launch_grad<T, W, 256, kVectors / 4, VEC, WIDE>(a, stream);
    } else if (vectors <= 256 * kVectors / 2) {
        launch_grad<T, W, 256, kVectors / 2, VEC, WIDE>(a, stream);
    } else if (vectors <= 256 * kVectors) {
        launch_grad<T, W, 256, kVectors, VEC, WIDE>(a, stream);
    } else if (vectors <= 1024 * kVectors / 2) {  // more would not fit the registers of 1024 threads
        launch_grad<T, W, 1024, kVectors / 2, VEC, WIDE>(a, stream);
    } else {
        joined = false;
        if (columns) {
            hipLaunchKernelGGL((layer_norm_columns_long_kernel<T>), dim3((unsigned)((a.width + 255) / 256), (unsigned)partials),
                               dim3(256), 0, stream, a);
        }
        if (a.rows > 0) {
            hipLaunchKernelGGL((layer_norm_grad_long_kernel<T, W, VEC, WIDE>), grid(a.rows), dim3(1024), 0, stream, a);
        }
    }
    if (columns && !joined) {
        launch_column_sums<W>(a.partial, a.partial + partials * a.width, partials, a.width, (W*)a.grad_weight, (W*)a.grad_bias,
                              stream);
    }
    return hipGetLastError();
}

template <typename T, typename W>
hipError_t run_grad_type(const LayerNormGradArgs& a, hipStream_t stream)
{
    constexpr int kVec = 16 / (int)sizeof(T);
    const int e = (int)sizeof(T);
    const bool vectors = a.width % kVec == 0 && aligned(a.grad_y.ptr, a.grad_y.row_stride, e, 16) &&
                         aligned(a.grad_sum.ptr, a.grad_sum.row_stride, e, 16) &&
                         aligned(a.sum.ptr, a.sum.row_stride, e, 16) &&
                         aligned(a.grad_x.ptr, a.grad_x.row_stride, e, 16) &&
                         aligned(a.weight, 0, 1, kVec * (int)sizeof(W));
    return vectors ? run_grad<T, W, kVec, true>(a, stream) : run_grad<T, W, kVec, false>(a, stream);
}

}  // namespace

int64_t layer_norm_grad_partials(const LayerNormGradArgs& a)
{
    // as of the other norm's gradients, whose kernels have the same shape: up to eight rows of a workgroup at a time, few wide
    // rows spread over as many workgroups as there are CUs, one workgroup where it needs no second kernel
    constexpr int64_t kWide = 1024, kWidest = 4096;
    const int64_t groups = (a.rows + 7) / 8;
    if (a.rows <= 1 || (groups == 1 && a.width <= kWidest)) {
        return 1;
    }
    const int64_t spread = a.width <= kWide ? groups : (a.rows < 256 ? a.rows : 256);
    return groups < spread ? spread : (groups < kPartialRows ? groups : kPartialRows);
}

hipError_t launch_layer_norm(const LayerNormArgs& args, hipStream_t stream)
{
    if (args.rows < 1 || args.width < 1) {
        return hipErrorInvalidValue;
    }
    LayerNormArgs a = args;
    a.streaming = a.rows * a.width * elem_size((Elem)a.elem) >= kStreamBytes ? 1 : 0;
    return by_type(a.elem, a.weight_float, [&](auto* t, auto* w) {
        return run_layer_norm_type<std::remove_pointer_t<decltype(t)>, std::remove_pointer_t<decltype(w)>>(a, stream);
    });
}

hipError_t launch_layer_norm_grad(const LayerNormGradArgs& a, hipStream_t stream)
{
    if (a.width < 1 || ((a.grad_weight != nullptr || a.grad_bias != nullptr) && a.partial == nullptr)) {
        return hipErrorInvalidValue;
    }
    return by_type(a.elem, a.weight_float, [&](auto* t, auto* w) {
        return run_grad_type<std::remove_pointer_t<decltype(t)>, std::remove_pointer_t<decltype(w)>>(a, stream);
    });
}

}  // namespace opscv
