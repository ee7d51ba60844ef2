// Dropout with the residual's addition; its mask is computed from a counter.
//
//   y = r + keep(e) x s,  keep(e) = number(e) >= threshold,  s = 65536 / (65536 - threshold)
//
// number(e) is a 16-bit half of a word of Philox 4x32-10 (Salmon, Moraes, Dror, Shaw, 2011) on the counter (e / 8, offset), so
// that any element's number can be made alone, and the gradient makes the same ones again.  Sixteen bits a number: a word
// each would be twice as much arithmetic (20 products of 32 by 32 bits for four elements, at a quarter of the rate of other
// instructions), and a step of 2^-16 in p is exact in the mean, since s belongs to the threshold and not to p.
//
// Bound by memory: each element is read once and written once.  A thread owns the eight elements of one counter, whose
// arithmetic hides behind its loads.  16384 rows of 4096 bf16 with a residual 70 us, 5.8 TB/s (part of it stays in the 256 MB
// cache); 5477 rows of 1283 FLOAT 11.7, 4.8 TB/s.
#include <hip/hip_runtime.h>

#include "token_elem.hpp"
#include "token_kernels.hpp"

namespace opscv {

using namespace tok;

namespace {

constexpr int kThreads = 256;
constexpr int kGroup = 8;  // elements of a counter

struct Words {
    uint32_t v[4];
};

__device__ __forceinline__ Words philox(uint64_t counter, uint64_t offset, uint64_t seed)
{
    uint32_t c0 = (uint32_t)counter, c1 = (uint32_t)(counter >> 32), c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
    uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
    for (int i = 0; i < 10; i++) {
        const uint64_t p = (uint64_t)c0 * 0xD2511F53u, q = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(q >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)q;
        c2 = (uint32_t)(p >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)p;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return {{c0, c1, c2, c3}};
}

// Bit i: whether element i of the group is kept.
__device__ __forceinline__ uint32_t kept(const Words& w, uint32_t threshold)
{
    uint32_t bits = 0;
#pragma unroll
    for (int i = 0; i < kGroup; i++) {
        const uint32_t number = (i & 1) != 0 ? w.v[i / 2] >> 16 : w.v[i / 2] & 0xFFFFu;
        bits |= number >= threshold ? 1u << i : 0u;
    }
    return bits;
}

// WIDE: rows are whole groups on 16-byte boundaries (a dense tensor is one row, whose last group may be a part), and a thread
// reads its group as vectors.
template <typename T, bool WIDE>
__global__ __launch_bounds__(kThreads) void dropout_kernel(DropoutArgs a, int streaming)
{
    constexpr int kVec = 16 / (int)sizeof(T);
    const int64_t total = a.rows * a.width, groups = (total + kGroup - 1) / kGroup;
    const uint64_t seed = (uint64_t)a.state[0], offset = (uint64_t)a.state[a.state_stride];
    for (int64_t g = (int64_t)blockIdx.x * kThreads + threadIdx.x; g < groups; g += (int64_t)gridDim.x * kThreads) {
        int64_t row = 0, c = g * kGroup;
        if (a.rows > 1) {
            row = c / a.width;
            c -= row * a.width;
        }
        if (WIDE && g * kGroup + kGroup <= total) {
            float x[kGroup], r[kGroup];
#pragma unroll
            for (int i = 0; i < kGroup; i += kVec) {
                load<T, kVec>((const T*)a.x.ptr + row * a.x.row_stride + c + i, *reinterpret_cast<float(*)[kVec]>(x + i));
                if (a.residual.ptr != nullptr) {
                    load<T, kVec>((const T*)a.residual.ptr + row * a.residual.row_stride + c + i,
                                  *reinterpret_cast<float(*)[kVec]>(r + i));
                }
            }
            const uint32_t keep = kept(philox((uint64_t)g, offset, seed), a.threshold);
#pragma unroll
            for (int i = 0; i < kGroup; i++) {
                x[i] = (keep >> i & 1u) != 0 ? x[i] * a.scale : 0.0f;
                if (a.residual.ptr != nullptr) {
                    x[i] += r[i];
                }
            }
#pragma unroll
            for (int i = 0; i < kGroup; i += kVec) {
                store<T, kVec>((T*)a.y.ptr + row * a.y.row_stride + c + i, *reinterpret_cast<float(*)[kVec]>(x + i),
                               streaming != 0);
            }
        } else {
            const uint32_t keep = kept(philox((uint64_t)g, offset, seed), a.threshold);
            for (int i = 0; i < kGroup && g * kGroup + i < total; i++) {
                const float x = (float)((const T*)a.x.ptr)[row * a.x.row_stride + c];
                float y = (keep >> i & 1u) != 0 ? x * a.scale : 0.0f;
                if (a.residual.ptr != nullptr) {
                    y += (float)((const T*)a.residual.ptr)[row * a.residual.row_stride + c];
                }
                ((T*)a.y.ptr)[row * a.y.row_stride + c] = (T)y;
                if (++c == a.width) {
                    c = 0;
                    row++;
                }
            }
        }
    }
}

template <typename T>
hipError_t run(const DropoutArgs& args, hipStream_t stream)
{
    DropoutArgs a = args;
    const int e = (int)sizeof(T);
    if (a.rows == 1 || (a.x.row_stride == a.width && a.y.row_stride == a.width &&
                        (a.residual.ptr == nullptr || a.residual.row_stride == a.width))) {
        a.width *= a.rows;  // one row
        a.rows = 1;
        a.x.row_stride = a.y.row_stride = a.residual.row_stride = 0;
    }
    const bool wide = (a.width % kGroup == 0 || a.rows == 1) && aligned(a.x.ptr, a.x.row_stride, e, 16) &&
                      aligned(a.y.ptr, a.y.row_stride, e, 16) && aligned(a.residual.ptr, a.residual.row_stride, e, 16);
    const int64_t total = a.rows * a.width, blocks = ((total + kGroup - 1) / kGroup + kThreads - 1) / kThreads;
    const dim3 grid((unsigned)(blocks < 1 << 20 ? blocks : 1 << 20));
    const int streaming = total * e >= kStreamBytes ? 1 : 0;
    if (wide) {
        hipLaunchKernelGGL((dropout_kernel<T, true>), grid, dim3(kThreads), 0, stream, a, streaming);
    } else {
        hipLaunchKernelGGL((dropout_kernel<T, false>), grid, dim3(kThreads), 0, stream, a, streaming);
    }
    return hipGetLastError();
}

}  // namespace

hipError_t launch_dropout(const DropoutArgs& a, hipStream_t stream)
{
    if (a.rows < 1 || a.width < 1 || a.state == nullptr || a.threshold > 65536) {
        return hipErrorInvalidValue;
    }
    switch ((Elem)a.elem) {
        case Elem::F32: return run<float>(a, stream);
        case Elem::F16: return run<_Float16>(a, stream);
        default: return run<__bf16>(a, stream);
    }
}

}  // namespace opscv
