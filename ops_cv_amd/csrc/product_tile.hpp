// Matrix products on the matrix cores, for the gated projections and their gradients:
//
//   out[t][f] = sum over k of Q[t][k] P[f][k]
//
// with "tokens" Q and "features" P.  An operand lies as it comes: as rows whose terms are side by side (t or f outside), or
// "turned", as rows of tokens or features, one a term (k outside).  Forward both are rows of terms; the gradient of x is a sum
// over the inner features, which are the weights' rows, and those of the weights sums over the rows of x and of the gradients.
//
// A workgroup makes a tile of results.  Stages of 128 bytes of terms (64 of 16 bits, 32 FLOAT) of both operands are copied
// straight to LDS, two stages in turn or more: while one is multiplied the others are under way.  Features are the rows of the 32 x 32
// results and tokens their columns, so that a lane holds four neighbouring features of a token.  In the gated forward product
// blocks of 32 features alternate between the two weights, so that a lane holds gate and up of the same features, and the
// activation and the product need no other lane.
//
// Bound by the products, at the clock that power allows (1.75 to 1.9 GHz; 63 % of a SIMD's cycles are products, LDS is busy for a
// quarter).  4096 rows of 4096 to 14336 bf16: 786 us, 1224 TFLOP/s; both gradients of 4096 rows of 2048 to 8192 474 us, 1160
// TFLOP/s; 10952 rows of 1280 to 3413 fp16 with gate and up 260, of which the results' way out is 80.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "acl_types.hpp"
#include "attention_tile.hpp"
#include "product_plan.hpp"
#include "token_elem.hpp"

namespace opscv {
namespace prod {

using att::acc_t;

struct ProductArgs {
    // features' rows of terms: gate and up.  Turned: rows of features, p[1] from term `p_turn` on, `p_terms` of each.
    const void* p[2] = {nullptr, nullptr};
    int64_t p_stride[2] = {0, 0};  // elements
    int64_t p_turn = 0, p_terms = 0;
    const void* q = nullptr;
    int64_t q_stride = 0;
    int64_t tokens = 0, features = 0;  // of the operands; gated: features of y
    int64_t columns = 0;               // features of the results that are written: turned rows may be padded
    int64_t terms = 0;                 // rows of terms: whole vectors of 16 bytes
    // plain: results of tokens below `turn` go to out[0], the others to out[1] from its first row on, `rows` to each;
    // gated: y, gate and up
    void* out[3] = {nullptr, nullptr, nullptr};
    int64_t out_stride[3] = {0, 0, 0};
    int64_t turn = INT64_MAX, rows = 0;  // turn: a multiple of 32
    const float* token_scale = nullptr;  // plain: factor of every token's results, or null
    const void* bias[2] = {nullptr, nullptr};
    int activation = 0;
    // the terms in parts of `part_stages` stages, whose sums go to `partial`, (parts, tokens, features), gated: gate's features
    // and then up's; or null
    float* partial = nullptr;
    uint32_t parts = 1, part_stages = 0;
    uint32_t token_tiles = 0, feature_tiles = 0;  // set by the launcher
};

// ------------------------------------------------------------------------------------------------- activations

// silu, gelu (erf) and gelu (tanh) in the order of opscvGateActivation: value, and derivative where wanted.

// By the hardware's exponential and reciprocal, a unit in the last place each; the product with log2 e loses up to 1.5 |x| 2^-24
// of the exponential (3.7e-6 measured at -80).  A workgroup has nothing to do beside its results' activations: with expf and a division the product of 4096
// rows, 4096 to 14336 bf16, takes 838 us.
__device__ __forceinline__ float sigmoid(float x)
{
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504f * x));
}

// The normal distribution's upper tail from a >= 0 on, and exp(-a^2 / 2), as exp(-a^2 / 2) t q(t) with t = 1 / (1 + 0.26 a): q
// is a polynomial fitted to the tail's relative error over 0 <= a <= 14.5, 3e-8 in exact arithmetic (from there on both are 0).
// In 32 bits the exponential's argument is rounded, and the tail is off by up to 1.25 a^2 2^-24 of itself more: 1.4e-6 at 5, 7e-6
// at 13, where it is 6e-39.  Sixteen instructions, where erfc with its branches takes the time of a fifth of a product over 1280
// terms.
__device__ __forceinline__ float upper_tail(float a, float* bell)
{
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.26f, a, 1.0f));
    float q = 0.03023091602825318f;
    q = __builtin_fmaf(q, t, -0.15149724028733202f);
    q = __builtin_fmaf(q, t, 0.2487386101963239f);
    q = __builtin_fmaf(q, t, -0.1477950848517748f);
    q = __builtin_fmaf(q, t, 0.15876242607995536f);
    q = __builtin_fmaf(q, t, 0.05196338416951116f);
    q = __builtin_fmaf(q, t, 0.10278901969593153f);
    q = __builtin_fmaf(q, t, 0.10305093049928157f);
    q = __builtin_fmaf(q, t, 0.10375702444392684f);
    *bell = __builtin_amdgcn_exp2f(-0.72134752f * (a * a));
    return *bell * (t * q);
}

__device__ __forceinline__ float activate(float g, int kind)
{
    if (kind == 0) {
        return g * sigmoid(g);
    }
    if (kind == 1) {
        float bell;
        const float tail = upper_tail(fabsf(g), &bell);
        return g * (g > 0.0f ? 1.0f - tail : tail);
    }
    // (1 + tanh(u)) / 2 = sigmoid(2 u)
    return g * sigmoid(1.5957691f * (g + 0.044715f * g * g * g));
}

__device__ __forceinline__ void activate_both(float g, int kind, float* value, float* slope)
{
    if (kind == 1) {
        float bell;
        const float tail = upper_tail(fabsf(g), &bell), below = g > 0.0f ? 1.0f - tail : tail;
        *value = g * below;
        *slope = below + g * (0.39894228f * bell);
        return;
    }
    float s, du;  // value g s, s = sigmoid(u), and u's derivative
    if (kind == 0) {
        s = sigmoid(g);
        du = 1.0f;
    } else {
        s = sigmoid(1.5957691f * (g + 0.044715f * g * g * g));
        // from 10 on s (1 - s) is 0: the square of a larger one may be infinite
        const float c = fminf(fmaxf(g, -10.0f), 10.0f);
        du = 1.5957691f * (1.0f + 3.0f * 0.044715f * c * c);
    }
    *value = g * s;
    *slope = s + g * (s * (1.0f - s)) * du;
}

// ------------------------------------------------------------------------------------------------- stages

typedef float f32x4 __attribute__((ext_vector_type(4)));

// 16 bytes of terms of 32 rows a lane: one step of 32 bytes of terms (half h of the lanes takes the second 16).
template <typename T>
struct Step;

template <>
struct Step<__bf16> {
    typedef att::bf16x8 Frag;
    static __device__ __forceinline__ acc_t mul(Frag a, Frag b, acc_t c)
    {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
};

template <>
struct Step<_Float16> {
    typedef att::f16x8 Frag;
    static __device__ __forceinline__ acc_t mul(Frag a, Frag b, acc_t c)
    {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
};

template <>
struct Step<float> {
    typedef f32x4 Frag;
    static __device__ __forceinline__ acc_t mul(Frag a, Frag b, acc_t c)
    {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
        }
        return c;
    }
};

struct alignas(16) Pack16 {
    uint32_t v[4];
};

constexpr uint32_t kInside = 0x80000000u;  // size of the descriptors: offsets of rows and terms that are there stay below it

// Vector c of row r lies at place c ^ swizzle(r), so that 16 neighbouring rows' vectors of one number fall on the 16 places of
// the 64 banks.
__device__ __forceinline__ int swizzle(int r) { return (r >> 1) & 7; }

// 16 bytes a lane from offset off + ahead of a buffer into LDS, as att::load_to_lds, which says why it is not the builtin.
__device__ __forceinline__ void load_to_lds(att::rsrc_t rsrc, uint32_t dst, uint32_t off, uint32_t ahead)
{
    __asm__ volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(dst), "v"(off), "s"(rsrc),
                     "s"(ahead)
                     : "memory", "m0");
}

// FB x TB blocks of 32 x 32 results a wavefront (features, tokens), WF x WT wavefronts a workgroup, places for STAGES stages.
template <int FB_, int TB_, int WF_, int WT_, int STAGES_ = 2>
struct Shape {
    static constexpr int FB = FB_, TB = TB_, WF = WF_, WT = WT_, STAGES = STAGES_;
    static constexpr int kWaves = WF * WT, kThreads = 64 * kWaves;
    static constexpr int kFeatures = 32 * FB * WF, kTokens = 32 * TB * WT;  // rows of the operands in a stage
    static constexpr int kStageBytes = (kFeatures + kTokens) * kRowBytes;
    static constexpr int kLds = STAGES * kStageBytes;
    static_assert(kWaves % 2 == 0 && kFeatures % (8 * kWaves) == 0 && kTokens % (8 * kWaves) == 0, "whole loads");
};
// 256 x 256, eight wavefronts, one workgroup a CU; gated: a wavefront has 64 features of y, so that its tokens leave in runs of
// 128 bytes of 16-bit numbers (10952 rows of 1280 to 3413 with both sums: 324 us with 32 features)
typedef Shape<2, 4, 4, 2> Large;
typedef Shape<4, 2, 2, 4> LargeGated;
// 128 x 128, four wavefronts, two workgroups a CU
typedef Shape<2, 2, 2, 2> Small;
// 128 x 128, eight wavefronts, more stages under way, one workgroup a CU: few tiles of the forward product (with four wavefronts, which
// wait for LDS with nothing beside them, 512 rows of 4096 to 4096 47 us, 80 of 1024 to 4096 13; with eight 44 and 12)
typedef Shape<2, 1, 2, 4, 4> Deep;
// 256 features of 32 tokens, four wavefronts, two workgroups a CU: FLOAT rows that would leave larger tiles empty
typedef Shape<2, 1, 4, 1> Slim;

// One operand's part of the stages: WIDTH tokens or features, BLOCKS blocks of 32 a wavefront, WAVES wavefronts.
template <typename T, bool TURNED, int WIDTH, int BLOCKS, int WAVES>
struct Side {
    typedef typename Step<T>::Frag Frag;
    static constexpr int kE = (int)sizeof(T);
    static constexpr int kLoads = WIDTH / 8 / WAVES;                      // of a wavefront and stage, 1024 bytes each
    static constexpr int kTerms = kRowBytes / kE;                         // of a stage
    static constexpr int kPitch = TURNED ? WIDTH * kE : kRowBytes;        // of a row in LDS
    static constexpr int kRowsALoad = 1024 / kPitch;                      // turned: 1, 2 or 4

    uint32_t off[kLoads];  // of this lane's vectors from the stage's base; kOutside: past the end of the tokens or features
    int first;             // rows of terms: the vector's number in its row; turned: the term of the first load
    int at[TURNED ? BLOCKS : 4];

    // Turned rows: vector c of row k lies at place c ^ turned_swizzle(k), so that what a half wavefront reads together, four
    // rows of 64 bytes (FLOAT: two of 128, four rows apart), falls on all 64 banks.
    static __device__ __forceinline__ int turned_swizzle(int k) { return kE == 2 ? (k & 3) << 2 : ((k >> 2) & 1) << 3; }

    // `left`: tokens or features from the tile's first on; `row`: which row of the operand row r of the tile is
    template <typename F>
    __device__ __forceinline__ void places(int64_t stride, int64_t left, int wave, int lane, F&& row)
    {
        if constexpr (TURNED) {
#pragma unroll
            for (int i = 0; i < kLoads; i++) {
                const int byte = (i * WAVES + wave) * 1024 + lane * 16, k = byte / kPitch;
                const int c = (byte % kPitch / 16) ^ turned_swizzle(k);
                off[i] = c * (16 / kE) < left ? (uint32_t)(k * stride * kE) + (uint32_t)(c * 16) : att::kOutside;
            }
            first = (wave * 1024 + lane * 16) / kPitch;
        } else {
            const int row8 = wave * 8 + (lane >> 3);  // of the first load
            first = (lane & 7) ^ swizzle(row8);       // the same in all loads: WAVES * 8 is a multiple of 16
#pragma unroll
            for (int i = 0; i < kLoads; i++) {
                const int64_t r = row(i * WAVES * 8 + row8);
                off[i] = r < left ? (uint32_t)(r * stride * kE) + (uint32_t)(first * 16) : att::kOutside;
            }
        }
    }

    // Copies a stage whose first term the buffer, `ahead` bytes on, begins with; `terms` are left from there on, and what is
    // behind them becomes zeros.  `rsrc` gives the buffer of load i.
    template <typename F>
    __device__ __forceinline__ void load(F&& rsrc, uint32_t to, uint32_t ahead, int terms) const
    {
#pragma unroll
        for (int i = 0; i < kLoads; i++) {
            const int own = TURNED ? first + i * WAVES * kRowsALoad : first * (16 / kE);
            load_to_lds(rsrc(i), to + (uint32_t)(i * WAVES * 1024), own < terms ? off[i] : att::kOutside, ahead);
        }
    }

    // Where this lane reads the blocks from `block` on.
    __device__ __forceinline__ void reads(int block, int lane)
    {
        if constexpr (!TURNED) {
            // row l % 32 of a block, vector 2 j + h of step j
#pragma unroll
            for (int j = 0; j < 4; j++) {
                at[j] = (block * 32 + (lane & 31)) * kRowBytes + (((2 * j + (lane >> 5)) ^ swizzle(lane & 31)) << 4);
            }
        } else {
            const int h = lane >> 5, i = lane & 15;
#pragma unroll
            for (int b = 0; b < BLOCKS; b++) {
                if constexpr (kE == 2) {
                    // Sixteen lanes together read four rows of sixteen elements, eight bytes a lane (row i / 4, elements
                    // 4 (i % 4) .. + 3), and the instruction hands lane i column i of them.
                    const int r = 8 * h + (i >> 2);
                    at[b] = r * kPitch + (((block + b) * 64) ^ (turned_swizzle(r) * 16)) + ((lane >> 4) & 1) * 32 + (i & 3) * 8;
                } else {
                    at[b] = 4 * h * kPitch + (((block + b) * 128) ^ (h * 128)) + (lane & 31) * 4;
                }
            }
        }
    }

    // Operand of step j of the stage at `from`, block b: terms 16 j + 8 h .. + 7 (FLOAT: 8 j + 4 h .. + 3) of token or
    // feature l % 32.
    __device__ __forceinline__ Frag read(const char* from, int j, int b) const
    {
        if constexpr (!TURNED) {
            return *reinterpret_cast<const Frag*>(from + at[j] + b * 32 * kRowBytes);
        } else if constexpr (kE == 2) {
            typedef __attribute__((address_space(3))) att::s16x4* place;
            const char* const here = from + at[b] + 16 * j * kPitch;
            const att::s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((place)(here));
            const att::s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((place)(here + 4 * kPitch));
            att::s16x8 both;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                both[e] = lo[e];
                both[4 + e] = hi[e];
            }
            return __builtin_bit_cast(Frag, both);
        } else {
            const char* const here = from + at[b] + 8 * j * kPitch;
            Frag f;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                f[e] = *reinterpret_cast<const float*>(here + e * kPitch);
            }
            return f;
        }
    }
};

// Where a workgroup's tile lies.
struct TileOf {
    uint32_t t, f, part;
};

// Workgroups are dealt to the eight XCDs in turn, and each XCD's share is a run of tiles that share operands in its L2: four
// rows of tiles, column by column.
__device__ __forceinline__ TileOf tile_of(const ProductArgs& a, uint32_t block)
{
    constexpr uint32_t kGroup = 4;
    const uint32_t tiles = a.token_tiles * a.feature_tiles, total = tiles * a.parts;
    const uint32_t xcd = block & 7, each = total >> 3, more = total & 7;
    uint32_t id = xcd * each + (xcd < more ? xcd : more) + (block >> 3);
    TileOf tile;
    tile.part = id / tiles;
    id -= tile.part * tiles;
    const uint32_t run = kGroup * a.feature_tiles, group = id / run, first = group * kGroup;
    const uint32_t high = a.token_tiles - first < kGroup ? a.token_tiles - first : kGroup;
    id -= group * run;
    tile.f = id / high;
    tile.t = first + id - tile.f * high;
    // the same for all lanes: in scalar registers, which the loads' bases have to be in
    tile.t = (uint32_t)__builtin_amdgcn_readfirstlane((int)tile.t);
    tile.f = (uint32_t)__builtin_amdgcn_readfirstlane((int)tile.f);
    tile.part = (uint32_t)__builtin_amdgcn_readfirstlane((int)tile.part);
    return tile;
}

template <typename T, bool GATED, bool P_TURNED, bool Q_TURNED, typename S>
__device__ __forceinline__ void product(const ProductArgs& a, uint32_t block, char* lds)
{
    typedef typename Step<T>::Frag Frag;
    constexpr int kE = (int)sizeof(T), FB = S::FB, TB = S::TB;
    constexpr int kResults = GATED ? S::kFeatures / 2 : S::kFeatures;  // features of the tile's results
    static_assert(!GATED || (FB % 2 == 0 && (S::kWaves == 4 || S::kWaves == 8) && !P_TURNED && !Q_TURNED), "gate and up in turn");
    const int lane = (int)threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int wf = wave % S::WF, wt = wave / S::WF;
    const TileOf tile = tile_of(a, block);
    const int64_t t0 = (int64_t)tile.t * S::kTokens, f0 = (int64_t)tile.f * kResults;

    typedef Side<T, P_TURNED, S::kFeatures, FB, S::kWaves> SideP;
    typedef Side<T, Q_TURNED, S::kTokens, TB, S::kWaves> SideQ;
    SideP side_p;
    SideQ side_q;
    constexpr int kTerms = kRowBytes / kE;
    uint32_t first_stage = 0, stages = (uint32_t)((a.terms + kTerms - 1) / kTerms);
    if (a.parts > 1) {
        first_stage = tile.part * a.part_stages;
        const uint32_t left = stages > first_stage ? stages - first_stage : 0;
        stages = left < a.part_stages ? left : a.part_stages;
    }
    // gate or up.  Rows of terms, 32 features of each in turn: with eight wavefronts by the wavefront, with four by the load.
    // Turned rows: one after the other; `own` is the one that side_p has the offsets of.
    int own = GATED ? (S::kWaves == 8 ? (wave >> 2) & 1 : 0) : (P_TURNED && (int64_t)first_stage * kTerms >= a.p_turn ? 1 : 0);
    const int64_t own_stride = own != 0 ? a.p_stride[1] : a.p_stride[0];
    side_p.places(own_stride, a.features - f0, wave, lane, [](int r) { return GATED ? (r >> 6) * 32 + (r & 31) : r; });
    if constexpr (GATED && S::kWaves == 4) {
#pragma unroll
        for (int i = 1; i < SideP::kLoads; i += 2) {  // of up, whose stride is its own
            const int r = i * 32 + wave * 8 + (lane >> 3);
            const int64_t f = (r >> 6) * 32 + (r & 31);
            side_p.off[i] = f < a.features - f0 ? (uint32_t)(f * a.p_stride[1] * kE) + (uint32_t)(side_p.first * 16) : att::kOutside;
        }
    }
    side_q.places(a.q_stride, a.tokens - t0, wave, lane, [](int r) { return r; });
    att::rsrc_t rsrc_p[2], rsrc_q;  // rows of terms: once; turned rows: stage by stage, further than 32 bits
    if constexpr (!P_TURNED) {
        rsrc_p[0] = att::buffer((const char*)(own != 0 ? a.p[1] : a.p[0]) + f0 * own_stride * kE, kInside);
        rsrc_p[1] = GATED && S::kWaves == 4 ? att::buffer((const char*)a.p[1] + f0 * a.p_stride[1] * kE, kInside) : rsrc_p[0];
    }
    if constexpr (!Q_TURNED) {
        rsrc_q = att::buffer((const char*)a.q + t0 * a.q_stride * kE, kInside);
    }
    const uint32_t lds0 = att::lds_place(lds);
    const auto load_stage = [&](uint32_t stage, int buffer) {
        const int64_t term = (int64_t)(first_stage + stage) * kTerms;
        const uint32_t to = lds0 + (uint32_t)(buffer * S::kStageBytes + wave * 1024);
        const int left = (int)(a.terms - term < kTerms ? a.terms - term : kTerms);
        if constexpr (P_TURNED) {
            const int half = term >= a.p_turn ? 1 : 0;
            const int64_t row = half != 0 ? term - a.p_turn : term;
            const int64_t there = a.p_terms - row;  // none or less where only zeros stand for the padding of the other operand
            const int64_t stride = half != 0 ? a.p_stride[1] : a.p_stride[0];
            if constexpr (!Q_TURNED) {  // the weights' gradients are sums over one operand's rows
                if (half != own) {      // stages are loaded in their order: once, if at all
                    own = half;
                    side_p.places(stride, a.features - f0, wave, lane, [](int r) { return r; });
                }
            }
            const att::rsrc_t rsrc = att::buffer((const char*)(half != 0 ? a.p[1] : a.p[0]) + (row * stride + f0) * kE, kInside);
            side_p.load([&](int) { return rsrc; }, to, 0, there < left ? (int)there : left);
        } else {
            side_p.load([&](int i) { return rsrc_p[S::kWaves == 4 ? i & 1 : 0]; }, to, (uint32_t)(term * kE), left);
        }
        const uint32_t to_q = to + S::kFeatures * kRowBytes;
        if constexpr (Q_TURNED) {
            const att::rsrc_t rsrc = att::buffer((const char*)a.q + (term * a.q_stride + t0) * kE, kInside);
            side_q.load([&](int) { return rsrc; }, to_q, 0, left);
        } else {
            side_q.load([&](int) { return rsrc_q; }, to_q, (uint32_t)(term * kE), left);
        }
    };

    side_p.reads(wf * FB, lane);
    side_q.reads(wt * TB, lane);
    Frag fp[2][FB], fq[2][TB];
    const auto read_step = [&](int j, int buffer, int slot) {
        const char* const from = lds + buffer * S::kStageBytes;
#pragma unroll
        for (int b = 0; b < FB; b++) {
            fp[slot][b] = side_p.read(from, j, b);
        }
#pragma unroll
        for (int b = 0; b < TB; b++) {
            fq[slot][b] = side_q.read(from + S::kFeatures * kRowBytes, j, b);
        }
    };
    // Register r of a block is feature 8 (r / 4) + 4 h + r % 4 of token l % 32.  The sums begin with the biases, whose loads are
    // under way together with the first stages' (10952 rows of 1280 to 3413 fp16: 232 us, added at the end 28 more).
    const int h = lane >> 5, n = lane & 31;
    constexpr int kRow = GATED ? FB / 2 : FB;  // blocks of 32 features of the results
    acc_t acc[FB][TB];
#pragma unroll
    for (int b = 0; b < FB; b++) {
        acc[b][0] = att::zeros();
        if constexpr (GATED) {
            if (a.bias[0] != nullptr && a.partial == nullptr) {
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    float x[4];
                    const int64_t f = f0 + (wf * kRow + b / 2) * 32 + 8 * q + 4 * h;
                    tok::load_part<T, 4, false>((const T*)a.bias[b % 2], f, a.features, x);
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        acc[b][0][4 * q + e] = x[e];
                    }
                }
            }
        }
#pragma unroll
        for (int c = 1; c < TB; c++) {
            acc[b][c] = acc[b][0];
        }
    }
    const auto multiply = [&](int slot) {
#pragma unroll
        for (int c = 0; c < TB; c++) {
#pragma unroll
            for (int b = 0; b < FB; b++) {
                acc[b][c] = Step<T>::mul(fp[slot][b], fq[slot][c], acc[b][c]);
            }
        }
    };

    // Steps j of a stage read the operands of step j + 1 before they multiply their own; the last step of a stage first waits
    // for the next stage (all wavefronts have read this one then, so its place is loaded again) and reads its first step.
    // Loads end in the order in which they were asked for, so the wait counts those of the stages behind the next one.
    constexpr int kLoads = SideP::kLoads + SideQ::kLoads;
    static_assert((S::STAGES - 1) * kLoads < 64, "the loads under way can be counted");
    if (stages > 0) {
#pragma unroll
        for (int i = 0; i < S::STAGES; i++) {
            if ((uint32_t)i < stages) {
                load_stage((uint32_t)i, i);
            }
        }
        if (stages >= (uint32_t)S::STAGES) {
            __asm__ volatile("s_waitcnt vmcnt(%0)" ::"n"((S::STAGES - 1) * kLoads) : "memory");
        } else {
            __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
        __builtin_amdgcn_s_barrier();
        __asm__ volatile("" ::: "memory");
        read_step(0, 0, 0);
        int buffer = 0;
        for (uint32_t stage = 0; stage < stages; stage++) {
            const int next = buffer + 1 < S::STAGES ? buffer + 1 : 0;
#pragma unroll
            for (int j = 0; j < 3; j++) {
                read_step(j + 1, buffer, (j + 1) & 1);
                multiply(j & 1);
            }
            if (stage + 1 < stages) {
                // of the stages behind the next one all are under way, or the last ones are waited for together
                if (S::STAGES > 2 && stage + S::STAGES <= stages) {
                    __asm__ volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((S::STAGES - 2) * kLoads) : "memory");
                } else {
                    __asm__ volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
                }
                __builtin_amdgcn_s_barrier();
                __asm__ volatile("" ::: "memory");
                if (stage + S::STAGES < stages) {
                    load_stage(stage + S::STAGES, buffer);
                }
                read_step(0, next, 0);
            }
            multiply(1);
            buffer = next;
        }
    }

    // ---------------------------------------------------------------------------------------------- results
    // A wavefront's results go out by way of a place of its own in LDS, 32 tokens at a time, so that neighbouring lanes write
    // neighbouring vectors of a token.
    if (a.partial != nullptr) {
        const int64_t pitch = GATED ? 2 * a.features : a.features;
        float* const to = a.partial + (int64_t)tile.part * a.tokens * pitch;
#pragma unroll
        for (int c = 0; c < TB; c++) {
            const int64_t t = t0 + (wt * TB + c) * 32 + n;
            if (t >= a.tokens) {
                continue;
            }
#pragma unroll
            for (int b = 0; b < FB; b++) {
                const int64_t first = f0 + (wf * kRow + (GATED ? b / 2 : b)) * 32;
                float* const row = to + t * pitch + (GATED && b % 2 != 0 ? a.features : 0);
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const int64_t f = first + 8 * q + 4 * h;
                    if (f + 4 <= a.features) {
                        tok::Loose<float> v;
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            v.v[e] = acc[b][c][4 * q + e];
                        }
                        *reinterpret_cast<tok::Loose<float>*>(row + f) = v;
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            if (f + e < a.features) {
                                row[f + e] = acc[b][c][4 * q + e];
                            }
                        }
                    }
                }
            }
        }
        return;
    }
    constexpr int kPitch = 32 * kRow * kE + 16;      // of a token on its way
    static_assert(S::kWaves * 32 * kPitch <= S::kLds, "the results' way out fits the stages");
    constexpr int kVec = 16 / kE, kChunks = 32 * kRow * kE / 16;  // vectors of a token
    __syncthreads();  // all have read their last stage
    char* const place = lds + wave * 32 * kPitch;
    // Writes out what lies there: tokens t.. , features f..  The 32 tokens are on one side of `turn`, a multiple of 32.
    const int put_token = lane / kChunks, put_vector = lane % kChunks;
    const auto put = [&](int which, int64_t t, int64_t f) {
        __asm__ volatile("" ::: "memory");  // the compiler keeps the order; LDS does for one wavefront
        const bool second = !GATED && t >= a.turn;
        const int64_t row = second ? t - a.turn : t, stride = second ? a.out_stride[1] : a.out_stride[which];
        T* to = (T*)(second ? a.out[1] : a.out[which]) + row * stride + f + (int64_t)put_token * stride + put_vector * kVec;
        const int left = (int)(a.rows - row < 32 ? a.rows - row : 32);
        const int64_t columns = a.columns - f - put_vector * kVec;
#pragma unroll
        for (int i = 0; i < 32 * kChunks / 64; i++) {
            constexpr int kTokens = 64 / kChunks;  // of an instruction
            const Pack16 v = *reinterpret_cast<const Pack16*>(place + (put_token + i * kTokens) * kPitch + put_vector * 16);
            if (put_token + i * kTokens < left) {
                if (columns >= kVec) {
                    *reinterpret_cast<tok::Loose<T>*>(to) = __builtin_bit_cast(tok::Loose<T>, v);
                } else {
                    const tok::Loose<T> each = __builtin_bit_cast(tok::Loose<T>, v);
#pragma unroll
                    for (int e = 0; e < kVec; e++) {
                        if (e < columns) {
                            to[e] = each.v[e];
                        }
                    }
                }
            }
            to += kTokens * stride;
        }
        __asm__ volatile("" ::: "memory");
    };
    const auto hold = [&](int b, int quarter, const float (&x)[4]) {
        tok::Pack<T, 4> k;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            k.v[e] = (T)x[e];
        }
        *reinterpret_cast<tok::Pack<T, 4>*>(place + n * kPitch + (b * 32 + 8 * quarter + 4 * h) * kE) = k;
    };
#pragma unroll
    for (int c = 0; c < TB; c++) {
        const int64_t t = t0 + (wt * TB + c) * 32;
        if constexpr (!GATED) {
            float scale = 1.0f;
            if (a.token_scale != nullptr) {
                const bool second = t + n >= a.turn;
                const int64_t row = second ? t + n - a.turn : t + n;
                scale = row < a.rows ? a.token_scale[second ? a.rows + row : row] : 1.0f;
            }
#pragma unroll
            for (int b = 0; b < FB; b++) {
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    float x[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        x[e] = acc[b][c][4 * q + e] * scale;
                    }
                    hold(b, q, x);
                }
            }
            put(0, t, f0 + wf * FB * 32);
        } else {
            const int64_t f = f0 + wf * kRow * 32;
            const auto hold_all = [&](auto value) {
#pragma unroll
                for (int b = 0; b < kRow; b++) {
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        float x[4];
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            x[e] = value(acc[2 * b][c][4 * q + e], acc[2 * b + 1][c][4 * q + e]);
                        }
                        hold(b, q, x);
                    }
                }
            };
            if (a.activation == 0) {
                hold_all([](float gate, float up) { return activate(gate, 0) * up; });
            } else if (a.activation == 1) {
                hold_all([](float gate, float up) { return activate(gate, 1) * up; });
            } else {
                hold_all([](float gate, float up) { return activate(gate, 2) * up; });
            }
            put(0, t, f);
            if (a.out[1] != nullptr) {
                hold_all([](float gate, float) { return gate; });
                put(1, t, f);
                hold_all([](float, float up) { return up; });
                put(2, t, f);
            }
        }
    }
}

template <typename T, typename S>
__global__ __launch_bounds__(S::kThreads) void gated_kernel(ProductArgs a)
{
    extern __shared__ __align__(16) char lds[];
    product<T, true, false, false, S>(a, blockIdx.x, lds);
}

// The gradients of x (`first` workgroups) and of the weights, in one launch: the long sums over the inner features first, so
// that the short ones over the rows fill up the CUs that are done.
template <typename T, typename SX, typename SW>
__global__ __launch_bounds__(SX::kThreads) void gradients_kernel(ProductArgs x, ProductArgs weights, uint32_t first)
{
    extern __shared__ __align__(16) char lds[];
    if (blockIdx.x < first) {
        product<T, false, true, false, SX>(x, blockIdx.x, lds);
    } else {
        product<T, false, true, true, SW>(weights, blockIdx.x - first, lds);
    }
}

}  // namespace prod
}  // namespace opscv
