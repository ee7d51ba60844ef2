// How attention's work is cut: the numbers that the host and the kernels agree on.
#pragma once

#include <cstdint>

#include "acl_types.hpp"
#include "launch_limits.hpp"

namespace opscv {
namespace att {

// A product's result is 32 x 32; heads are cut into blocks of 32 features, and a tile's row has room for PITCH.
constexpr int kBlock = 32;

constexpr int blocks_of(int64_t d) { return d <= 32 ? 1 : d <= 64 ? 2 : d <= 96 ? 3 : d <= 128 ? 4 : 8; }
constexpr int pitch_of(int blocks) { return blocks <= 2 ? 64 : blocks <= 4 ? 128 : 256; }

// Shape of a workgroup that walks keys: row_waves wavefronts with 32 rows each (a row is a query of one of the heads that
// share a key head) that read the same tiles, or few rows: 32 of them, and key_waves wavefronts that take tiles of their own
// in turn.
struct ForwardShape {
    int row_waves, key_waves, keys, stages;
    constexpr int threads() const { return 64 * row_waves * key_waves; }
    constexpr int rows() const { return kBlock * row_waves; }
};

// LDS decides: a tile of keys and one of values per stage and group of wavefronts.  Two workgroups of shared rows fit a CU's
// 160 KB; of few rows, one of four wavefronts with two tiles each under way, or, where a tile is larger, five of one
// wavefront and one tile.
constexpr ForwardShape forward_shape(int elem_bytes, int pitch, bool few_rows)
{
    const int row = elem_bytes * pitch;  // bytes
    if (few_rows) {
        return row <= 256 ? ForwardShape{1, 4, 32, 2} : ForwardShape{1, 1, 32, 1};
    }
    return ForwardShape{4, 1, row <= 256 ? 64 : 32, row <= 512 ? 2 : 1};
}

struct ForwardPlan {
    bool few_rows = false;
    int64_t rows = 0;   // of a key head: queries times heads that share it
    int64_t tiles = 0;  // workgroups' worth of rows
    int64_t splits = 1; // parts that the keys of a tile are cut into
    int64_t blocks = 0; // workgroups
    int64_t joins = 0;  // threads that join the parts, one for four features of a row
    bool fits = false;  // one launch
};

// Workgroups with work, as they are launched: as many for every XCD.
constexpr int64_t launched(int64_t blocks) { return (blocks + 7) / 8 * 8; }

// Partial results of a split: per row the largest score, the sum, and the weighted values.
constexpr int64_t partial_floats(int64_t d) { return 2 + (d + 3) / 4 * 4; }

// Tiles of 32 rows instead of tiles of 128: where those would leave CUs without work, where there are no more rows, and for
// FLOAT.  On both sides of the line, us with tiles of 32 and of 128 (tiles of 128 in brackets), forward and gradients:
//   8 heads of 128 on 8, window 1024, bf16    [128] 30 and 35, 80 and 89   [224] 54 and 52, 124 and 106
//                                             [256] 56 and 45, 135 and 112   [512] 112 and 52, 253 and 185
//   pictures of 1369 tokens, heads of 64      [176] 18 and 26, 58 and 58   [264] 23 and 29, 68 and 65
//                                             [352] 28 and 33, 76 and 73
//   2048 tokens, 8 heads of 256 on 8, fp16    [128] 98 and 104, 323 and 282   [256] 155 and 163, 389 and 342
// FLOAT, forward: pictures of 1369 tokens, 16 heads of 64, one 56 and 67, four 197 and 173; 4096 tokens, 32 heads of 128 on 8
// 672 and 692; 2 x 4096, 16 of 96 on 4 550 and 541.  Tiles of 128 would be the faster ones of many tiles of narrow heads
// (8192 tokens, 16 heads of 64 on 4: 481 and 310; 5 x 911, 16 of 32 on 2: 129 and 78) and of heads of 256 (2048 tokens, 8
// heads: 748 and 620); there is no such kernel.
inline bool few_rows(const AttentionArgs& a)
{
    const int64_t rows = a.tokens * (a.heads / a.kv_heads);
    return a.elem == 0 || rows <= kBlock ||
           a.batch * a.kv_heads * ((rows + 4 * kBlock - 1) / (4 * kBlock)) < a.compute_units;
}

inline ForwardPlan plan_forward(const AttentionArgs& a)
{
    ForwardPlan p;
    const int64_t group = a.heads / a.kv_heads;
    p.rows = a.tokens * group;
    p.few_rows = few_rows(a);
    const ForwardShape s = forward_shape(a.elem == 0 ? 4 : 2, pitch_of(blocks_of(a.d)), p.few_rows);
    p.tiles = (p.rows + s.rows() - 1) / s.rows();
    const int64_t whole = a.batch * a.kv_heads * p.tiles;
    // keys that the rows of one tile see at most, in tiles of keys
    const int64_t window = a.left + a.right + s.rows() / group + 2;
    const int64_t keys = a.kv_tokens < window + a.sinks ? a.kv_tokens : window + a.sinks;
    const int64_t key_tiles = (keys + s.keys - 1) / s.keys;
    // Eight wavefronts for every CU where that many parts leave each four tiles or more; single wavefronts of FLOAT, whose
    // products take sixteen times as many cycles, one tile (one token on a window of 129, 8 heads of 96 on 1: 13 us, 25 with
    // four; five sequences of 256 tokens, a head of 128, window 86: 16 and 26).
    const int64_t waves = s.row_waves * s.key_waves, least = waves == 1 && a.elem == 0 ? 1 : 4 * s.key_waves;
    const int64_t want = (8 * (int64_t)a.compute_units / waves + whole - 1) / whole, most = key_tiles / least;
    p.splits = want < most ? want : most;
    p.splits = p.splits < 1 ? 1 : (p.splits > 64 ? 64 : p.splits);
    p.blocks = whole * p.splits;
    p.joins = p.splits > 1 ? a.batch * a.kv_heads * p.rows * ((a.d + 3) / 4) : 0;
    p.fits = fits_launch(launched(p.blocks), s.threads()) && p.joins <= INT32_MAX;
    return p;
}

// ---------------------------------------------------------------------------------------------------------- gradients

// The queries' gradients: as the forward pass, but for FLOAT of more than 64 features, whose tiles fill LDS: 32 rows and one
// wavefront, or, where there are at most two tiles of 32 rows for every CU, four that share the keys.  That line on both
// sides, the whole backward call with one wavefront and with four: 4 x 1024 tokens, heads of 128, causal, 2 on 1 (256 tiles)
// 311 and 177, 4 on 2 (512) 388 and 289, 8 on 8 (1024) 554 and 548; 2048 tokens, 8 heads of 96 on 2, window 512 (512) 208 and
// 186, two such (1024) 317 and 365; 2 x 777, 12 of 72 on 4, window 101 (584) 92 and 107.
//  There, and for heads of more than 128 features, the values come
// straight from memory: FLOAT's products take long enough for that (4 x 1024 tokens, 2 heads of 128, causal: four wavefronts
// 81 us, one 217; 16 x 512, 2 heads of 256 on 1: 205 and 334), and yet from LDS they come sooner (one wavefront: 2 x 777
// tokens, 12 heads of 72 on 4, window 101: 38 us, with values from memory 42, with four wavefronts 53).
constexpr bool grad_values_direct(int elem_bytes, int pitch, bool few_rows)
{
    return elem_bytes == 4 && (pitch > 128 || (pitch > 64 && few_rows));
}
constexpr ForwardShape grad_query_shape(int elem_bytes, int pitch, bool few_rows)
{
    return elem_bytes == 2 || pitch <= 64 ? forward_shape(elem_bytes, pitch, few_rows)
           : few_rows                     ? ForwardShape{1, 4, 32, 1}
                                          : ForwardShape{1, 1, 32, 1};
}

// The keys' gradients: a wavefront has 32 keys and walks tiles of 32 queries of one head.  16-bit types: four wavefronts walk
// together, so that a tile of queries is loaded once for 128 keys.  FLOAT: each by itself, for the same reason as above.
constexpr int grad_key_waves(bool is_float, int nb) { return is_float && nb <= 4 ? 1 : 4; }

struct GradPlan {
    bool few_rows = false;
    int64_t rows = 0, tiles = 0;       // of the queries' gradients, as in the forward pass
    int64_t keys = 0;                  // of a tile
    int64_t key_tiles = 0;             // of a key head
    int64_t sink_tiles = 0;            // the first of them, seen by queries of any position
    int64_t sink_parts = 1, parts = 1; // parts that the queries of such a tile, and of the others, are cut into at most
    // 32-bit words of the scratch: statistics of the rows, partial gradients of the sinks' tiles and of the others
    int64_t stat_pitch = 0, stats = 0, sink_partials = 0, partials = 0;
    // workgroups of the two kernels, and threads of the join, for the sinks' tiles and for the others
    int64_t query_blocks = 0, key_blocks = 0, sink_joins = 0, joins = 0;
    bool fits = false;  // one launch each
};

inline GradPlan plan_grad(const AttentionArgs& a)
{
    GradPlan p;
    const int64_t group = a.heads / a.kv_heads, bh = a.batch * a.kv_heads;
    p.rows = a.tokens * group;
    p.few_rows = few_rows(a);
    const int64_t tile_rows = p.few_rows ? kBlock : 4 * kBlock;
    p.tiles = (p.rows + tile_rows - 1) / tile_rows;
    if (a.elem == 0 && a.d > 64) {
        p.few_rows = bh * p.tiles <= 2 * a.compute_units;
    }
    p.keys = kBlock * grad_key_waves(a.elem == 0, blocks_of(a.d));
    p.key_tiles = (a.kv_tokens + p.keys - 1) / p.keys;
    const int64_t sinks = a.sinks < a.kv_tokens ? a.sinks : a.kv_tokens;
    p.sink_tiles = (sinks + p.keys - 1) / p.keys;
    // steps (tiles of 32 queries, of every head of the group) of a tile of keys, at most
    const int64_t all = (a.tokens + kBlock - 1) / kBlock;
    const int64_t window = (a.left + a.right + p.keys + kBlock - 1) / kBlock + 1;
    const int64_t steps = group * (window < all ? window : all);
    // As few parts as fill the card with one round of workgroups, every tile's steps in equal parts: ten wavefronts for every
    // CU, of which eight run at a time, where a part has eight steps or more.  The whole backward call with 8, 10 and 16:
    // 4096 tokens, 32 heads of 128 on 8, window 1024, bf16 317, 284 and 299 us (parts of as many steps each, whose last is
    // what is left: 325 at the time, for 294); 8 pictures of 1369 tokens, 16 heads of 64 174, 174, 174; 2 x 2048, 16 heads of
    // 64, causal 143, 143, 134; 4 x 1024, 8 of 128 on 2 83, 89, 101; 8192 tokens, 8 of 128 on 1, window 512 128, 150, 152.
    // FLOAT: one step or more, and as many wavefronts as its registers leave room for: four from three blocks of features on,
    // eight of two, and of one block many short parts.  With 4, 8 and 32: 4 x 1024, 2 heads of 128 on 1 177, 178, 262; 2 x
    // 2048, 8 of 96 on 2, window 512 319, 301, 344; 2 x 777, 12 of 72 on 4 93, 92, 108; 16 x 512, 2 of 256 on 1 468, 432, 768;
    // 4 x 512, 8 of 64 128, 98, 120; 3 x 1024, 64 of 32 on 8, window 256 610, 469, 456; 5 x 911, 16 of 32 on 2 504, 346, 305.
    const int64_t sink_steps = group * all;
    const int64_t waves = a.elem != 0 ? 10 : blocks_of(a.d) > 2 ? 4 : blocks_of(a.d) == 2 ? 8 : 32;
    const int64_t room = a.compute_units * waves * kBlock / p.keys;
    const auto items = [&](int64_t each) {
        return bh * (p.sink_tiles * ((sink_steps + each - 1) / each) +
                     (p.key_tiles - p.sink_tiles) * ((steps + each - 1) / each));
    };
    int64_t low = a.elem == 0 ? 1 : 8, high = steps > low ? steps : low;  // the fewest steps whose parts fit, or all
    while (low < high) {
        const int64_t middle = (low + high) / 2;
        if (items(middle) <= room) {
            high = middle;
        } else {
            low = middle + 1;
        }
    }
    p.parts = (steps + low - 1) / low;
    p.sink_parts = (sink_steps + low - 1) / low;
    p.parts = p.parts < 1 ? 1 : p.parts;
    p.sink_parts = p.sink_parts < 1 ? 1 : p.sink_parts;
    p.stat_pitch = (a.tokens + 7) / 8 * 8;  // rows of statistics begin on sectors of 32 bytes
    p.stats = 2 * a.batch * a.heads * p.stat_pitch;
    const int64_t tile_floats = 2 * p.keys * ((a.d + 3) / 4 * 4);
    p.sink_partials = p.sink_parts > 1 ? bh * p.sink_tiles * p.sink_parts * tile_floats : 0;
    p.partials = p.parts > 1 ? bh * (p.key_tiles - p.sink_tiles) * p.parts * tile_floats : 0;
    p.query_blocks = bh * p.tiles;
    p.key_blocks = bh * (p.sink_tiles * p.sink_parts + (p.key_tiles - p.sink_tiles) * p.parts);
    const int64_t tile_joins = 2 * p.keys * ((a.d + 3) / 4);
    p.sink_joins = p.sink_parts > 1 ? bh * p.sink_tiles * tile_joins : 0;
    p.joins = p.parts > 1 ? bh * (p.key_tiles - p.sink_tiles) * tile_joins : 0;
    const int bytes = a.elem == 0 ? 4 : 2;
    p.fits = fits_launch(launched(p.query_blocks), grad_query_shape(bytes, pitch_of(blocks_of(a.d)), p.few_rows).threads()) &&
             fits_launch(launched(p.key_blocks), 2 * p.keys) && p.sink_joins + p.joins <= INT32_MAX;
    return p;
}

// ------------------------------------------------------------------------------------------------------------ large batches

// f(a, plan) for the launches that a call is made of: all sequences, or as many a launch as the half, the quarter, ... of them
// that fits, and what is left.  None where one sequence alone does not fit.  plan_of(a): plan_forward or plan_grad.
template <typename Plan, typename F>
void by_launches(const AttentionArgs& a, Plan&& plan_of, F&& f)
{
    AttentionArgs s = a;
    auto plan = plan_of(s);
    while (!plan.fits && s.batch > 1) {
        s.batch /= 2;
        plan = plan_of(s);
    }
    if (!plan.fits) {
        return;
    }
    f(s, plan);
    const int elem_bytes = a.elem == 0 ? 4 : 2;
    for (int64_t each = s.batch, b = each; b < a.batch; b += each) {
        for (Strided* x : {&s.q, &s.k, &s.v, &s.out, &s.grad_out, &s.grad_q, &s.grad_k, &s.grad_v, &s.lse}) {
            if (x->ptr != nullptr) {
                x->ptr = (char*)x->ptr + each * x->stride[0] * (x == &s.lse ? 4 : elem_bytes);
            }
        }
        for (Whole* x : {&s.q_lengths, &s.kv_lengths}) {
            if (x->ptr != nullptr) {
                x->ptr = (const char*)x->ptr + each * x->stride[0] * (x->wide != 0 ? 8 : 4);
            }
        }
        if (a.batch - b < each) {
            s.batch = a.batch - b;
            plan = plan_of(s);
        }
        f(s, plan);
    }
}

}  // namespace att
}  // namespace opscv
