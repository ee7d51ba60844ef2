// Launches of the matrix products (product_tile.hpp), by type; product_f32.hip, product_f16.hip, product_bf16.hip.
#pragma once

#include <hip/hip_runtime.h>

#include <atomic>

#include "kernels.hpp"
#include "launch_limits.hpp"
#include "product_few.hpp"
#include "product_plan.hpp"

namespace opscv {
namespace prod {

// Workgroups of a product, 0 where it does not fit what the kernels assume.
template <typename T, bool GATED, bool P_TURNED, bool Q_TURNED, typename S>
int64_t prepare(ProductArgs* a)
{
    constexpr int64_t kE = (int64_t)sizeof(T), kVec = 16 / kE, kTerms = kRowBytes / kE;
    const int64_t results = GATED ? S::kFeatures / 2 : S::kFeatures;
    const int64_t furthest = (int64_t)kInside - 2 * kRowBytes - (P_TURNED && Q_TURNED ? 0 : a->terms * kE);
    const int64_t p_rows = P_TURNED ? kTerms : results, q_rows = Q_TURNED ? kTerms : S::kTokens;
    bool fits = a->tokens >= 1 && a->features >= 1 && a->terms >= 0 && a->parts >= 1;
    // vectors of 16 bytes are whole: of terms, or of turned features and tokens, which a row has room for
    fits = fits && ((P_TURNED && Q_TURNED) || a->terms % kVec == 0);
    fits = fits && (!P_TURNED || (a->features % kVec == 0 && a->p_turn % kTerms == 0));
    fits = fits && (!Q_TURNED || a->tokens % kVec == 0) && (a->turn % 32 == 0 || a->turn > a->tokens);
    for (const int64_t stride : {a->p_stride[0], a->p_stride[1], a->q_stride}) {
        fits = fits && stride >= 0 && stride * kE % 16 == 0;
    }
    fits = fits && p_rows * a->p_stride[0] * kE <= furthest && p_rows * a->p_stride[1] * kE <= furthest &&
           q_rows * a->q_stride * kE <= furthest;
    const int64_t token_tiles = (a->tokens + S::kTokens - 1) / S::kTokens;
    const int64_t feature_tiles = (a->features + results - 1) / results, blocks = token_tiles * feature_tiles * a->parts;
    if (!fits || !fits_launch(blocks, S::kThreads)) {
        return 0;
    }
    a->token_tiles = (uint32_t)token_tiles;
    a->feature_tiles = (uint32_t)feature_tiles;
    return blocks;
}

template <typename... A>
hipError_t launch_kernel(void (*kernel)(A...), int64_t blocks, int threads, int lds, hipStream_t stream,
                         std::atomic<uint32_t>& allowed, A... args)
{
    if (!fits_launch(blocks, threads)) {
        return hipErrorInvalidValue;
    }
    if (lds > 65536) {
        const hipError_t e = allow_dynamic_lds((const void*)kernel, lds, allowed);
        if (e != hipSuccess) {
            return e;
        }
    }
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3((unsigned)threads), (unsigned)lds, stream, args...);
    return hipGetLastError();
}

template <typename T, typename S>
hipError_t launch_gated_shape(ProductArgs a, hipStream_t stream)
{
    static std::atomic<uint32_t> allowed{0};
    const int64_t blocks = prepare<T, true, false, false, S>(&a);
    return blocks < 1 ? hipErrorInvalidValue : launch_kernel(gated_kernel<T, S>, blocks, S::kThreads, S::kLds, stream, allowed, a);
}

// `x` or `weights` may be null: one product alone
template <typename T, typename SX, typename SW>
hipError_t launch_gradients_shape(const ProductArgs* x, const ProductArgs* weights, hipStream_t stream)
{
    static_assert(SX::kThreads == SW::kThreads, "one launch");
    static std::atomic<uint32_t> allowed{0};
    ProductArgs ax, aw;
    int64_t first = 0, others = 0;
    if (x != nullptr) {
        ax = *x;
        first = prepare<T, false, true, false, SX>(&ax);
    }
    if (weights != nullptr) {
        aw = *weights;
        others = prepare<T, false, true, true, SW>(&aw);
    }
    if ((x != nullptr && first < 1) || (weights != nullptr && others < 1)) {
        return hipErrorInvalidValue;
    }
    if (first + others == 0) {
        return hipSuccess;
    }
    constexpr int kLds = SX::kLds > SW::kLds ? SX::kLds : SW::kLds;
    return launch_kernel(gradients_kernel<T, SX, SW>, first + others, SX::kThreads, kLds, stream, allowed, ax, aw, (uint32_t)first);
}

template <typename T, int TB, int AHEAD>
hipError_t launch_few(const ProductArgs& a, hipStream_t stream)
{
    const int64_t e = (int64_t)sizeof(T), blocks = (a.features + kFewFeatures - 1) / kFewFeatures;
    if (a.tokens < 1 || a.tokens > TB * 16 || a.features < 1 || a.terms < 1 || a.terms * e % 16 != 0 ||
        !fits_launch(blocks, 64 * kFewWaves)) {
        return hipErrorInvalidValue;
    }
    hipLaunchKernelGGL((gated_few_kernel<T, TB, AHEAD>), dim3((unsigned)blocks), dim3(64 * kFewWaves), 0, stream, a);
    return hipGetLastError();
}

template <typename T>
hipError_t launch_gated_typed(const ProductArgs& a, int tile, hipStream_t stream)
{
    if (tile == kTileFew) {
        return a.tokens <= 16   ? launch_few<T, 1, 4>(a, stream)
               : a.tokens <= 32 ? launch_few<T, 2, 2>(a, stream)
                                : launch_few<T, 4, 1>(a, stream);
    }
    if constexpr (sizeof(T) == 2) {
        if (tile == kTileDeep) {
            return launch_gated_shape<T, Deep>(a, stream);
        }
    } else {
        if (tile == kTileSlim) {
            return launch_gated_shape<T, Slim>(a, stream);
        }
    }
    return tile == kTile256 ? launch_gated_shape<T, LargeGated>(a, stream) : launch_gated_shape<T, Small>(a, stream);
}

template <typename T>
hipError_t launch_gradients_typed(const ProductArgs* x, const ProductArgs* weights, int tile, hipStream_t stream)
{
    if constexpr (sizeof(T) == 4) {
        if (tile == kTileSlim) {
            return launch_gradients_shape<T, Slim, Small>(x, weights, stream);
        }
    }
    return tile == kTile256 ? launch_gradients_shape<T, Large, Large>(x, weights, stream)
                            : launch_gradients_shape<T, Small, Small>(x, weights, stream);
}

}  // namespace prod
}  // namespace opscv
