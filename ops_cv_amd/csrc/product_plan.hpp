// Which tiles the matrix products are made of, and into how many parts their sums are split (host only).
#pragma once

#include <cstdint>

#include "token_args.hpp"

namespace opscv {
namespace prod {

constexpr int64_t kFewRows = 64;  // up to these, gated projections are product_few.hpp's

// One product: rows of its operands in tiles (gated: features of both weights together), stages of 128 bytes of terms.
struct ProductSize {
    int64_t tokens = 0, features = 0, stages = 0;
    int64_t tiles(int64_t side) const { return (tokens + side - 1) / side * ((features + side - 1) / side); }
};

// When the last workgroup ends, in its own stages, if each of `slots` takes the next workgroup as soon as it is free:
// count[0] workgroups of length[0] first, then count[1] of length[1].
inline int64_t last_end(const int64_t* count, const int64_t* length, int64_t slots)
{
    // slots by the time at which they are free: a length adds one time at most, and the start's slots are another
    constexpr int kTimes = 8;
    int64_t time[kTimes] = {0}, free[kTimes] = {slots};
    int n = 1;
    int64_t last = 0;
    for (int i = 0; i < 2; i++) {
        int64_t left = length[i] > 0 ? count[i] : 0;
        while (left > 0) {
            int first = 0;
            for (int k = 1; k < n; k++) {
                first = time[k] < time[first] ? k : first;
            }
            const int64_t take = left < free[first] ? left : free[first], end = time[first] + length[i];
            left -= take;
            free[first] -= take;
            if (free[first] == 0) {
                time[first] = time[n - 1];
                free[first] = free[n - 1];
                n--;
            }
            last = last > end ? last : end;
            int same = 0;
            while (same < n && time[same] != end) {
                same++;
            }
            if (same < n) {
                free[same] += take;
            } else if (n < kTimes) {
                time[n] = end;
                free[n++] = take;
            }
        }
    }
    return last;
}

// Time of up to two products in one launch, in stages of a large tile on one CU (about a microsecond of 16-bit numbers).  A CU
// takes one large tile, or two small ones, of a quarter of the work each, at 0.85 of the rate (8192 terms squared bf16: 877 us
// in large tiles, 1035 in small ones).  Parts, of eight stages at least, so that the workgroups end together: their sums are
// written and read again, 4 MB a microsecond.  777 rows, 1001 to 2731 FLOAT, both gradients: 247 us with parts of the longer
// sum alone, sized by the total.
inline ProductPlan plan_products(const ProductSize* size, int count, bool split, double stage_us, int units)
{
    ProductPlan best;
    double best_cost = 0.0;
    for (int large = 0; large < 2; large++) {
        const int64_t side = large != 0 ? 256 : 128, slots = large != 0 ? units : 2 * units;
        const double each = (large != 0 ? 1.0 : 0.5 / 0.85) * stage_us;
        int64_t tiles[2] = {0, 0}, most[2] = {1, 1};
        for (int i = 0; i < count; i++) {
            tiles[i] = size[i].tiles(side);
            // four rounds of workgroups at most: after that, parts have nothing to even out
            most[i] = !split ? 1 : size[i].stages / 8 < 16 ? size[i].stages / 8 : 16;
            most[i] = most[i] * tiles[i] <= 4 * slots ? most[i] : 4 * slots / tiles[i];
            most[i] = most[i] > 1 ? most[i] : 1;
        }
        for (int64_t first = 1; first <= most[0]; first++) {
            for (int64_t second = 1; second <= most[1]; second++) {
                ProductPlan p;
                p.large = large != 0;
                const int64_t wanted[2] = {first, second};
                int64_t groups[2] = {0, 0};
                double joined = 0.0;
                for (int i = 0; i < count; i++) {
                    const int64_t stages = size[i].stages > 0 ? size[i].stages : 1;
                    p.part_stages[i] = (stages + wanted[i] - 1) / wanted[i];
                    p.parts[i] = (stages + p.part_stages[i] - 1) / p.part_stages[i];
                    groups[i] = tiles[i] * p.parts[i];
                    if (p.parts[i] > 1) {
                        joined += 4.0 + (double)(2 * p.parts[i] * size[i].tokens * size[i].features * 4) / 4e6;
                    }
                }
                const double cost = (double)last_end(groups, p.part_stages, slots) * each + joined;
                if (best_cost == 0.0 || cost < best_cost) {
                    best = p;
                    best_cost = cost;
                }
            }
        }
    }
    return best;
}

}  // namespace prod
}  // namespace opscv
