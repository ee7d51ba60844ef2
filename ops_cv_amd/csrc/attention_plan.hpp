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

// ---------------------------------------------------------------------------------------------------------- gradients

// The keys' gradients: a workgroup has four wavefronts with 32 keys each and walks tiles of 32 queries of one head.
constexpr int kKeyWaves = 4;
constexpr int kGradKeys = kKeyWaves * kBlock;

struct GradPlan {
    int64_t rows = 0, tiles = 0;       // of the queries' gradients, as in the forward pass
    int64_t key_tiles = 0;             // of a key head
    int64_t sink_tiles = 0;            // the first of them, seen by queries of any position
    int64_t sink_parts = 1, parts = 1; // parts that the queries of such a tile, and of the others, are cut into
    // 32-bit words of the scratch: statistics of the rows, partial gradients of the sinks' tiles and of the others
    int64_t stats = 0, sink_partials = 0, partials = 0;
};

inline GradPlan plan_grad(const AttentionArgs& a)
{
    GradPlan p;
    const int64_t group = a.heads / a.kv_heads, bh = a.batch * a.kv_heads;
    p.rows = a.tokens * group;
    p.tiles = (p.rows + 4 * kBlock - 1) / (4 * kBlock);
    p.key_tiles = (a.kv_tokens + kGradKeys - 1) / kGradKeys;
    const int64_t sinks = a.sinks < a.kv_tokens ? a.sinks : a.kv_tokens;
    p.sink_tiles = (sinks + kGradKeys - 1) / kGradKeys;
    // steps (tiles of 32 queries, of every head of the group) of a tile of keys, at most
    const int64_t all = (a.tokens + kBlock - 1) / kBlock;
    const int64_t window = (a.left + a.right + kGradKeys + kBlock - 1) / kBlock + 1;
    const int64_t steps = group * (window < all ? window : all);
    // two workgroups for every CU where that leaves a part eight steps or more
    const int64_t whole = bh * p.key_tiles > 0 ? bh * p.key_tiles : 1;
    int64_t each = (steps * whole + 2 * a.compute_units - 1) / (2 * a.compute_units);
    each = each < 8 ? 8 : each;
    each = each < steps ? each : (steps > 0 ? steps : 1);
    p.parts = (steps + each - 1) / each;
    p.sink_parts = (group * all + each - 1) / each;
    p.parts = p.parts < 1 ? 1 : p.parts;
    p.sink_parts = p.sink_parts < 1 ? 1 : p.sink_parts;
    p.stats = 3 * a.batch * a.heads * a.tokens;
    const int64_t tile_floats = 2 * kGradKeys * ((a.d + 3) / 4 * 4);
    p.sink_partials = p.sink_parts > 1 ? bh * p.sink_tiles * p.sink_parts * tile_floats : 0;
    p.partials = p.parts > 1 ? bh * (p.key_tiles - p.sink_tiles) * p.parts * tile_floats : 0;
    return p;
}

}  // namespace att
}  // namespace opscv
