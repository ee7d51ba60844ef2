// Which tiles the matrix products are made of, and into how many parts their sums are split (host only).
#pragma once

#include <cstdint>
#include <initializer_list>

#include "acl_types.hpp"
#include "launch_limits.hpp"
#include "token_args.hpp"

namespace opscv {
namespace prod {

constexpr int kTile128 = 0;  // four wavefronts, two workgroups a CU
constexpr int kTile256 = 1;  // eight wavefronts, one workgroup a CU
constexpr int kTileFew = 2;  // product_few.hpp: the gated projections of few rows
constexpr int kTileSlim = 3;  // kTile128, but 32 rows by 256 features for the forward product or the gradient of x, FLOAT
constexpr int kTileDeep = 4;  // kTile128 with more stages under way, eight wavefronts and one workgroup a CU, forward, 16 bits

constexpr int64_t kFewRows = 64;

constexpr int kRowBytes = 128;  // of a row in a stage: eight vectors of 16 bytes

// One product: rows of its operands in tiles (gated: features of both weights together), stages of 128 bytes of terms.
struct ProductSize {
    int64_t tokens = 0, features = 0, stages = 0;
    int64_t tiles(int64_t high, int64_t wide) const { return (tokens + high - 1) / high * ((features + wide - 1) / wide); }
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

// Up to two products in one launch, by the time that each way would take:
//   - a CU makes a stage of a 256 tile in 1.7 us (8.4 MFLOP of 16 bits at 5 TFLOP/s; FLOAT 8.0), one of a 128 tile in a quarter of
//     that, 16 bits at 0.85 of the rate (8192 terms squared bf16: 877 us in large tiles, 1035 in small ones; FLOAT 139 and 132
//     TFLOP/s); alone on a CU not under 1 us, what a stage takes to come from memory, which gives 5 TB/s to all, or 0.8 where
//     three more are under way (128 rows of 4096 to 14336 bf16 71 us and 56, 512 of 4096 to 4096 55 and 44; with more tiles than CUs,
//     768 rows, 64 and 82; FLOAT and the gradients, whose operands take longer out of LDS, gain nothing);
//   - the terms in parts, of four stages at least, so that there is a workgroup for every CU and they end together: the parts'
//     sums are written and read again, 4 MB a microsecond, and 8 us are charged for every product in parts, for the kernel that
//     joins them and the start and end of workgroups.  That is what a product alone takes; both of the gradients' are joined by
//     one kernel, of 4 to 6.6 us, and charged for twice.
// 256 rows, 1024 to 4096 FLOAT: 71 us in one part.  777 rows, 1001 to 2731 FLOAT, both gradients: 247 us where parts were sized
// by the total alone.
// `us` is 0 where no way fits a launch.
// `slim`: the first product may be made of slim tiles.  Rows that end inside a tile leave a part of it empty, and FLOAT is slow
// enough that it shows: 2048 to 7168, both gradients of 8, 64, 160 and 777 rows, 98, 118, 224 and 794 us in tiles of 128 and 63, 95,
// 196 and 841 with slim ones, whose stage takes 7 / 12 of the time for half of the products; forward 389 rows of 1280 to 4480 126
// and 96, 128 rows 43 and 54.  16 bits read memory all the time either way (gradients of 8 rows 38 and 35, of 160 54 and 54).
// `deep`: the one product may be made of deep ones.
inline ProductPlan plan_products(const ProductSize* size, int count, int elem_bytes, int units, bool slim, bool deep)
{
    ProductPlan best;
    for (const int tile : {kTileDeep, kTile128, kTile256, kTileSlim}) {
        if ((tile == kTileSlim && !slim) || (tile == kTileDeep && !deep)) {
            continue;
        }
        const int64_t side = tile == kTile256 ? 256 : 128;
        // a stage of a slim tile takes 7 / 12 of what one of 128 does
        const int64_t weight[2] = {tile == kTileSlim ? 7 : 1, tile == kTileSlim ? 12 : 1};
        const double full = elem_bytes == 4 ? 8.0 : 1.7, small = full / 4.0 / (elem_bytes == 4 ? 1.0 : 0.85);
        const bool single = tile == kTile256 || tile == kTileDeep;  // one workgroup a CU, of eight wavefronts
        const double alone = tile == kTile256 ? full : (tile == kTileSlim ? small / 12.0 : small);
        int64_t tiles[2] = {0, 0}, most[2] = {1, 1};
        double from_memory = 0.0;
        for (int i = 0; i < count; i++) {
            tiles[i] = tile == kTileSlim && i == 0 ? size[i].tiles(32, 256) : size[i].tiles(side, side);
            from_memory += (double)((size[i].tokens + size[i].features) * size[i].stages * 128) / 5e6;
            // eight rounds of workgroups at most: after that, parts have nothing to even out
            most[i] = size[i].stages / 4 < 16 ? size[i].stages / 4 : 16;
            most[i] = most[i] * tiles[i] <= 8 * units ? most[i] : 8 * units / tiles[i];
            most[i] = most[i] > 1 ? most[i] : 1;
        }
        for (int64_t first = 1; first <= most[0]; first++) {
            for (int64_t second = 1; second <= most[1]; second++) {
                ProductPlan p;
                p.tile = tile;
                const int64_t wanted[2] = {first, second};
                int64_t groups[2] = {0, 0};
                for (int i = 0; i < count; i++) {
                    const int64_t stages = size[i].stages > 0 ? size[i].stages : 1;
                    p.part_stages[i] = (stages + wanted[i] - 1) / wanted[i];
                    p.parts[i] = (stages + p.part_stages[i] - 1) / p.part_stages[i];
                    groups[i] = tiles[i] * p.parts[i];
                    if (p.parts[i] > 1) {
                        p.us += 8.0 + (double)(2 * p.parts[i] * size[i].tokens * size[i].features * 4) / 4e6;
                    }
                }
                if (tile == kTileDeep && (groups[0] > units || p.parts[0] > 1)) {
                    continue;
                }
                if (!fits_launch(groups[0] + groups[1], single ? 512 : 256)) {
                    continue;
                }
                const int64_t share = !single && groups[0] + groups[1] > units ? 2 : 1;  // workgroups of a CU
                const double least = tile == kTileDeep ? 0.8 : (tile == kTileSlim ? 1.2 / 7.0 : 1.0);
                const double stage = (double)share * alone > least ? (double)share * alone : least;
                const int64_t length[2] = {p.part_stages[0] * weight[0], p.part_stages[1] * weight[1]};
                // not before all slots have had an equal share: most ways are ruled out by that
                const double equal = (double)(groups[0] * length[0] + groups[1] * length[1]) / (double)(share * units) * stage;
                if (best.us != 0.0 && p.us + (equal > from_memory ? equal : from_memory) >= best.us) {
                    continue;
                }
                const double last = (double)last_end(groups, length, share * units) * stage;
                p.us += last > from_memory ? last : from_memory;
                if (best.us == 0.0 || p.us < best.us) {
                    best = p;
                }
            }
        }
    }
    return best;
}

// Time of the kernel of few rows: the weights at 5 TB/s, and more for more rows (4096 to 14336 bf16, 1, 8, 16, 32 and 64 rows: 47,
// 51, 61, 71 and 94 us, where tiles in two parts take 58 with 8 and 62 with 64; FLOAT 96, 105, 118, 129 and 245).
inline double few_us(int64_t rows, int64_t weight_bytes, int elem_bytes)
{
    const double more = elem_bytes == 4 && rows > 32 ? 2.5 : 1.0 + (double)rows / 64.0;
    return (double)weight_bytes / 5e6 * more;
}

// The forward product of the gated projections, y's features in both weights; `us` is 0 where none fits a launch.
inline ProductPlan gated_plan(const GatedArgs& a)
{
    const int e = elem_size((Elem)a.elem);
    const ProductSize size{a.rows, 2 * a.inner, (a.width * e + kRowBytes - 1) / kRowBytes};
    ProductPlan p = plan_products(&size, 1, e, a.compute_units, e == 4, e == 2);
    const double few = few_us(a.rows, 2 * a.inner * a.width * e, e);
    if (a.rows <= kFewRows && (p.us == 0.0 || few <= p.us)) {
        p = ProductPlan();
        p.tile = kTileFew;
        p.us = few;
    }
    return p;
}

// The products of their gradients that are wanted, one at least: x's, then the weights'.
inline ProductPlan gated_grad_plan(const GatedArgs& a)
{
    const int e = elem_size((Elem)a.elem);
    const auto rounded = [](int64_t n, int64_t to) { return (n + to - 1) / to * to; };
    const int64_t padded = rounded(a.inner, kRowBytes / e), width = rounded(a.width, 16 / e);
    ProductSize size[2];
    int count = 0;
    if (a.want_x != 0) {
        size[count++] = {a.rows, width, 2 * padded * e / kRowBytes};
    }
    if (a.want_weights != 0) {
        size[count++] = {2 * padded, width, (a.rows * e + kRowBytes - 1) / kRowBytes};
    }
    return plan_products(size, count, e, a.compute_units, a.want_x != 0 && e == 4, false);
}

}  // namespace prod
}  // namespace opscv
