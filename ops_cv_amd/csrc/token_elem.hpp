// Elements of the operators on token sequences: vectors of up to 16 bytes, read and written whole, computed in 32 bits.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace opscv {
namespace tok {

template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
    T v[N];
};

template <typename T, int N>
static __device__ __forceinline__ void load(const T* p, float (&x)[N])
{
    const Pack<T, N> k = *reinterpret_cast<const Pack<T, N>*>(p);
#pragma unroll
    for (int i = 0; i < N; i++) {
        x[i] = (float)k.v[i];
    }
}

// `streaming`: written past the caches, for outputs that they would not hold until they are read (kStreamBytes)
template <typename T, int N>
static __device__ __forceinline__ void store(T* p, const float (&x)[N], bool streaming)
{
    Pack<T, N> k;
#pragma unroll
    for (int i = 0; i < N; i++) {
        k.v[i] = (T)x[i];
    }
    if constexpr (sizeof(k) == 16) {
        if (streaming) {
            typedef float f32x4 __attribute__((ext_vector_type(4)));
            // between the two: or the compiler makes one store of both ways, and that an ordinary one
            __asm__ volatile("; streaming");
            __builtin_nontemporal_store(__builtin_bit_cast(f32x4, k), reinterpret_cast<f32x4*>(p));
            __asm__ volatile("; streaming");
            return;
        }
    }
    *reinterpret_cast<Pack<T, N>*>(p) = k;
}

// Outputs from the L2 caches' size on (8 x 4 MB) are written with streaming stores.  8192 rows of 4096 bf16 through the norm:
// 52.7 us without, 48.8 with; two prompts of 4096 tokens through the rotation: 42.2 and 34.2.  (The gradients of the norm
// get slower by it.)
constexpr int64_t kStreamBytes = (int64_t)32 << 20;

// Elements c .. c + N - 1 of a row of `width`: whole vectors (WIDE; c + N <= width), or one by one, zeros from the row's
// end on.  Both ways a lane owns the same elements, so sums over lanes do not depend on a row's alignment.
template <typename T, int N, bool WIDE>
static __device__ __forceinline__ void load_part(const T* row, int64_t c, int64_t width, float (&x)[N])
{
    if constexpr (WIDE) {
        load<T, N>(row + c, x);
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) {
            x[i] = c + i < width ? (float)row[c + i] : 0.0f;
        }
    }
}

template <typename T, int N, bool WIDE>
static __device__ __forceinline__ void store_part(T* row, int64_t c, int64_t width, const float (&x)[N], bool streaming)
{
    if constexpr (WIDE) {
        store<T, N>(row + c, x, streaming);
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) {
            if (c + i < width) {
                row[c + i] = (T)x[i];
            }
        }
    }
}

static __device__ __forceinline__ float wave_sum(float v)
{
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
        v += __shfl_xor(v, d, 64);
    }
    return v;
}

// the larger one; NaN where either is
static __device__ __forceinline__ float larger(float a, float b) { return (a > b || a != a) ? a : b; }

static __device__ __forceinline__ float wave_larger(float v)
{
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
        v = larger(v, __shfl_xor(v, d, 64));
    }
    return v;
}

// whether `p` and a step of `stride` elements keep vectors of `bytes` aligned
inline bool aligned(const void* p, int64_t stride, int elem_bytes, int bytes)
{
    return reinterpret_cast<uintptr_t>(p) % (uintptr_t)bytes == 0 && stride * elem_bytes % bytes == 0;
}

}  // namespace tok
}  // namespace opscv
