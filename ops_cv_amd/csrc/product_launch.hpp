// Launches of the matrix products (product_tile.hpp), by type; product_f32.hip, product_f16.hip, product_bf16.hip.
#pragma once

#include <hip/hip_runtime.h>

#include <atomic>

#include "kernels.hpp"
#include "launch_limits.hpp"
#include "product_plan.hpp"
#include "product_tile.hpp"

namespace opscv {
namespace prod {

template <typename T, int KIND, int FB, int TB, int WF, int WT>
hipError_t launch_shape(ProductArgs a, hipStream_t stream)
{
    typedef Shape<T, KIND, FB, TB, WF, WT> S;
    const int64_t token_tiles = (a.tokens + S::kTokens - 1) / S::kTokens;
    const int64_t feature_tiles = (a.features + S::kResults - 1) / S::kResults;
    const int64_t blocks = token_tiles * feature_tiles * a.parts;
    const int64_t e = (int64_t)sizeof(T), furthest = kInside - kRowBytes - a.terms * e;
    const int64_t p_rows = KIND == kGated ? S::kFeatures / 2 : S::kFeatures;
    if (a.tokens < 1 || a.features < 1 || a.terms < 0 || a.terms * e % 16 != 0 || !fits_launch(blocks, S::kThreads) ||
        S::kTokens * a.q_stride * e > furthest || p_rows * a.p_stride[0] * e > furthest ||
        p_rows * a.p_stride[1] * e > furthest || a.q_stride < 0 || a.p_stride[0] < 0 || a.p_stride[1] < 0) {
        return hipErrorInvalidValue;
    }
    a.token_tiles = (uint32_t)token_tiles;
    a.feature_tiles = (uint32_t)feature_tiles;
    static std::atomic<uint32_t> allowed{0};
    if (S::kLds > 65536) {
        const hipError_t e = allow_dynamic_lds((const void*)product_kernel<T, KIND, FB, TB, WF, WT>, S::kLds, allowed);
        if (e != hipSuccess) {
            return e;
        }
    }
    hipLaunchKernelGGL((product_kernel<T, KIND, FB, TB, WF, WT>), dim3((unsigned)blocks), dim3(S::kThreads), S::kLds, stream,
                       a);
    return hipGetLastError();
}

template <typename T>
hipError_t launch_typed(const ProductArgs& a, int kind, int tile, hipStream_t stream)
{
    if (kind == kGated) {
        return tile == kTile256 ? launch_shape<T, kGated, 2, 4, 4, 2>(a, stream) : launch_shape<T, kGated, 2, 2, 2, 2>(a, stream);
    }
    if (kind == kPlain) {
        return tile == kTile256 ? launch_shape<T, kPlain, 2, 4, 4, 2>(a, stream) : launch_shape<T, kPlain, 2, 2, 2, 2>(a, stream);
    }
    return launch_shape<T, kPartial, 2, 2, 2, 2>(a, stream);
}

}  // namespace prod
}  // namespace opscv
