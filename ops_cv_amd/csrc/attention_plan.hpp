// How attention's work is cut: the numbers that the host and the kernels agree on.
#pragma once

#include <cstdint>

#include "acl_types.hpp"

namespace opscv {
namespace att {

// A product's result is 32 x 32; heads are cut into blocks of 32 features, and a tile's row has room for PITCH.
constexpr int kBlock = 32;

constexpr int blocks_of(int64_t d) { return d <= 64 ? 2 : d <= 96 ? 3 : d <= 128 ? 4 : 8; }
constexpr int pitch_of(int blocks) { return blocks <= 2 ? 64 : blocks <= 4 ? 128 : 256; }

// Shape of a forward workgroup: kRowWaves wavefronts with 32 rows each (a row is a query of one of the heads that share
// a key head) that read the same tiles, or one row wavefront's worth of rows with kKeyWaves wavefronts that take tiles of
// their own in turn.
struct ForwardShape {
    int row_waves, key_waves, keys, stages;
    constexpr int threads() const { return 64 * row_waves * key_waves; }
    constexpr int rows() const { return kBlock * row_waves; }
};

// LDS decides: a tile of keys and one of values per stage and group of wavefronts, of at most 160 KB in all, so that two
// workgroups fit a CU where rows are shared.
constexpr ForwardShape forward_shape(int elem_bytes, int pitch, bool few_rows)
{
    const int row = elem_bytes * pitch;  // bytes
    if (!few_rows) {
        return ForwardShape{4, 1, row <= 256 ? 64 : 32, row <= 512 ? 2 : 1};
    }
    return row <= 256 ? ForwardShape{1, 4, 32, 2} : row <= 512 ? ForwardShape{1, 4, 32, 1} : ForwardShape{1, 2, 32, 1};
}

struct ForwardPlan {
    bool few_rows = false;
    int64_t rows = 0;   // of a key head: queries times heads that share it
    int64_t tiles = 0;  // workgroups' worth of rows
    int64_t splits = 1; // parts that the keys of a tile are cut into
    int64_t blocks = 0; // workgroups
};

// Partial results of a split: per row the largest score, the sum, and the weighted values.
constexpr int64_t partial_floats(int64_t d) { return 2 + (d + 3) / 4 * 4; }

inline ForwardPlan plan_forward(const AttentionArgs& a)
{
    ForwardPlan p;
    const int64_t group = a.heads / a.kv_heads;
    p.rows = a.tokens * group;
    p.few_rows = p.rows <= kBlock;
    const ForwardShape s = forward_shape(a.elem == 0 ? 4 : 2, pitch_of(blocks_of(a.d)), p.few_rows);
    p.tiles = (p.rows + s.rows() - 1) / s.rows();
    const int64_t whole = a.batch * a.kv_heads * p.tiles;
    // keys that the rows of one tile see at most, in tiles of keys
    const int64_t window = a.left + a.right + s.rows() / group + 2;
    const int64_t keys = a.kv_tokens < window + a.sinks ? a.kv_tokens : window + a.sinks;
    const int64_t key_tiles = (keys + s.keys - 1) / s.keys;
    // two workgroups for every CU where that many parts leave each wavefront four tiles or more
    const int64_t want = (2 * (int64_t)a.compute_units + whole - 1) / whole, most = key_tiles / (4 * s.key_waves);
    p.splits = want < most ? want : most;
    p.splits = p.splits < 1 ? 1 : (p.splits > 64 ? 64 : p.splits);
    p.blocks = whole * p.splits;
    return p;
}

}  // namespace att
}  // namespace opscv
