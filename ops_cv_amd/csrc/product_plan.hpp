// Which tiles the matrix products are made of, and into how many parts their sums are split (host only).
#pragma once

#include <cstdint>

namespace opscv {
namespace prod {

// One product: rows of its operands in tiles (gated: features of both weights together), stages of 128 bytes of terms.
struct ProductSize {
    int64_t tokens = 0, features = 0, stages = 0;
    int64_t tiles(int64_t side) const { return (tokens + side - 1) / side * ((features + side - 1) / side); }
};

struct ProductPlan {
    bool large = false;                           // tiles of 256 x 256, else of 128 x 128
    int64_t parts[2] = {1, 1}, part_stages[2] = {0, 0};  // of the terms; more than one part: a second kernel joins their sums
};

// Time of up to two products in one launch, in stages of a large tile on one CU (about a microsecond).  A CU takes one large
// tile, or two small ones, of a quarter of the work each, at 0.85 of the rate (8192 terms squared bf16: 877 us in large tiles,
// 1035 in small ones).  Parts: as many as let the longest workgroup end with the others, 16 stages each at least; their sums
// are written and read again, 4 MB a microsecond.
inline ProductPlan plan_products(const ProductSize* size, int count, bool split, int units)
{
    ProductPlan best;
    double best_cost = 0.0;
    for (const bool large : {false, true}) {
        const int64_t side = large ? 256 : 128, slots = large ? units : 2 * units;
        const double each = large ? 1.0 : 0.5 / 0.85;  // of a stage, where all slots are taken
        ProductPlan p;
        p.large = large;
        int64_t total = 0;
        for (int i = 0; i < count; i++) {
            total += size[i].tiles(side) * size[i].stages;
        }
        const int64_t even = (total + slots - 1) / slots, shortest = even > 16 ? even : 16;
        double joined = 0.0, longest = 0.0, shared = 0.0;
        for (int i = 0; i < count; i++) {
            const int64_t stages = size[i].stages;
            p.part_stages[i] = stages;
            if (split && stages > shortest + shortest / 4) {
                const int64_t parts = (stages + shortest - 1) / shortest;
                p.part_stages[i] = (stages + parts - 1) / parts;
                p.parts[i] = (stages + p.part_stages[i] - 1) / p.part_stages[i];
                joined += 5.0 + (double)(2 * p.parts[i] * size[i].tokens * size[i].features * 4) / 4e6;
            }
            longest = longest > (double)p.part_stages[i] ? longest : (double)p.part_stages[i];
            shared += (double)(size[i].tiles(side) * p.parts[i] * p.part_stages[i]) / (double)slots;
        }
        if (count == 1) {  // workgroups of one length: whole rounds
            const int64_t groups = size[0].tiles(side) * p.parts[0];
            shared = (double)((groups + slots - 1) / slots * p.part_stages[0]);
        }
        const double cost = (longest > shared ? longest : shared) * each + joined;
        if (best_cost == 0.0 || cost < best_cost) {
            best = p;
            best_cost = cost;
        }
    }
    return best;
}

}  // namespace prod
}  // namespace opscv
