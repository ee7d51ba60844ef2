// Which tiles a matrix product is made of, and into how many parts its sums are split (host only).
#pragma once

#include <cstdint>

namespace opscv {
namespace prod {

constexpr int kTile128 = 0;  // 128 x 128 rows of the operands, four wavefronts, two workgroups a CU
constexpr int kTile256 = 1;  // 256 x 256, eight wavefronts

struct ProductPlan {
    int tile = kTile128;
    int64_t parts = 1;        // of the terms; more than one: partial sums that a second kernel joins
    int64_t part_stages = 0;  // stages of 128 bytes of terms
};

// `features`: rows of the features' operand (gated: of both together).
inline ProductPlan plan_product(int64_t tokens, int64_t features, int64_t term_bytes, bool gated, int units)
{
    ProductPlan p;
    const int64_t big = ((tokens + 255) / 256) * ((features + 255) / 256);
    if (big >= units) {
        p.tile = kTile256;
        return p;
    }
    const int64_t small = ((tokens + 127) / 128) * ((features + 127) / 128), stages = (term_bytes + 127) / 128;
    // results that do not give every CU a workgroup: their sums are split, 16 stages a part at least
    if (!gated && small < units && stages >= 32) {
        int64_t parts = units / small;
        parts = parts < stages / 16 ? parts : stages / 16;
        p.part_stages = (stages + parts - 1) / parts;
        p.parts = (stages + p.part_stages - 1) / p.part_stages;
    }
    return p;
}

}  // namespace prod
}  // namespace opscv
