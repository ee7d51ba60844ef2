// Matrix products on the matrix cores, for the gated projections and their gradients:
//
//   out[t][f] = sum over k of Q[t][k] P[f][k]
//
// Both operands are rows of terms that lie side by side ("tokens" Q and "features" P), so one kernel serves every product;
// where a gradient sums over another dimension, its operands are laid out so first (gated_layout.hip).
//
// A workgroup makes a tile of TOKENS x FEATURES results.  Stages of 128 bytes of terms (64 of 16 bits, 32 FLOAT) of both
// operands are copied straight to LDS, two stages in turn: while one is multiplied the other is under way.  Features are the
// rows of the 32 x 32 results and tokens their columns, so that a lane holds four neighbouring features of a token.  In the
// gated forward product blocks of 32 features alternate between the two weights, so that a lane holds gate and up of the same
// features, and the activation and the product need no other lane.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "acl_types.hpp"
#include "attention_tile.hpp"
#include "token_elem.hpp"

namespace opscv {
namespace prod {

using att::acc_t;

enum Kind { kPlain = 0, kGated = 1, kPartial = 2 };  // kPartial: 32-bit sums over a part of the terms

struct ProductArgs {
    const void* p[2] = {nullptr, nullptr};  // features' rows; kGated: gate and up
    int64_t p_stride[2] = {0, 0};           // elements
    const void* q = nullptr;
    int64_t q_stride = 0;
    int64_t tokens = 0, features = 0;  // results; kGated: features of y
    int64_t terms = 0;                 // whole vectors of 16 bytes
    // results of tokens below `turn` go to out[0], the others to out[1] from its first row on; kGated: y, gate and up
    void* out[3] = {nullptr, nullptr, nullptr};
    int64_t out_stride[3] = {0, 0, 0};
    int64_t turn = 0;
    const float* token_scale = nullptr;  // factor of every token's results, or null
    const void* bias[2] = {nullptr, nullptr};
    int activation = 0;
    int wide[3] = {0, 0, 0};  // the output's rows start on 16 bytes
    // launch
    uint32_t token_tiles = 0, feature_tiles = 0, parts = 1;
    int64_t part_stages = 0;  // kPartial: stages of a part
};

// ------------------------------------------------------------------------------------------------- activations

// silu, gelu (erf) and gelu (tanh) in the order of opscvGateActivation: value, and derivative where wanted.
__device__ __forceinline__ float sigmoid(float x) { return 1.0f / (1.0f + expf(-x)); }

__device__ __forceinline__ float activate(float g, int kind)
{
    if (kind == 0) {
        return g * sigmoid(g);
    }
    if (kind == 1) {
        return g * (0.5f * erfcf(-g * 0.70710678f));  // erfc: the lower tail keeps its bits
    }
    // (1 + tanh(u)) / 2 = sigmoid(2 u)
    return g * sigmoid(1.5957691f * (g + 0.044715f * g * g * g));
}

__device__ __forceinline__ void activate_both(float g, int kind, float* value, float* slope)
{
    if (kind == 1) {
        const float below = 0.5f * erfcf(-g * 0.70710678f);
        *value = g * below;
        *slope = below + g * (0.39894228f * expf(-0.5f * g * g));
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

constexpr int kRowBytes = 128;  // of a row in a stage: eight vectors of 16 bytes
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

// FB x TB blocks of 32 x 32 results a wavefront (features, tokens), WF x WT wavefronts a workgroup.
template <typename T, int KIND, int FB, int TB, int WF, int WT>
struct Shape {
    static constexpr int kWaves = WF * WT, kThreads = 64 * kWaves;
    static constexpr int kFeatures = 32 * FB * WF, kTokens = 32 * TB * WT;  // rows of the operands in a stage
    static constexpr int kResults = KIND == kGated ? kFeatures / 2 : kFeatures;  // features of the tile's results
    static constexpr int kStageBytes = (kFeatures + kTokens) * kRowBytes;
    static constexpr int kLds = 2 * kStageBytes;
    static constexpr int kLoadsP = kFeatures / 8 / kWaves, kLoadsQ = kTokens / 8 / kWaves;  // of a wavefront and stage
    static constexpr int kPitch = 32 * (KIND == kGated ? 1 : FB) * (int)sizeof(T) + 16;  // of a token's results on their way out
    static_assert(kWaves % 2 == 0 && kFeatures % (8 * kWaves) == 0 && kTokens % (8 * kWaves) == 0, "whole loads");
    static_assert(KIND != kGated || (FB % 2 == 0 && (kWaves == 4 || kWaves == 8)), "gate and up in turn");
    static_assert(kWaves * 32 * kPitch <= kLds, "the results' way out fits the stages");
};

template <typename T, int KIND, int FB, int TB, int WF, int WT>
__global__ __launch_bounds__(64 * WF * WT) void product_kernel(ProductArgs a)
{
    typedef Shape<T, KIND, FB, TB, WF, WT> S;
    typedef typename Step<T>::Frag Frag;
    constexpr int kE = (int)sizeof(T);
    extern __shared__ __align__(16) char lds[];
    const int lane = (int)threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int wf = wave % WF, wt = wave / WF;

    // Which tile: workgroups are dealt to the eight XCDs in turn, and each XCD's share is a run of tiles that share operands
    // in its L2: four rows of tiles, column by column.
    uint32_t tile_t, tile_f, part;
    {
        const uint32_t tiles = a.token_tiles * a.feature_tiles, total = tiles * a.parts;
        const uint32_t xcd = blockIdx.x & 7, each = total >> 3, more = total & 7;
        uint32_t id = xcd * each + (xcd < more ? xcd : more) + (blockIdx.x >> 3);
        part = id / tiles;
        id -= part * tiles;
        constexpr uint32_t kGroup = 4;
        const uint32_t run = kGroup * a.feature_tiles, group = id / run, first = group * kGroup;
        const uint32_t high = a.token_tiles - first < kGroup ? a.token_tiles - first : kGroup;
        id -= group * run;
        tile_f = id / high;
        tile_t = first + id - tile_f * high;
    }
    const int64_t t0 = (int64_t)tile_t * S::kTokens, f0 = (int64_t)tile_f * S::kResults;

    // What this lane copies of every stage: vector `chunk` of some rows; rows past the end become zeros.
    const int row8 = wave * 8 + (lane >> 3);  // of the first load
    const int chunk = (lane & 7) ^ swizzle(row8);  // the same in all loads: kWaves * 8 is a multiple of 16
    uint32_t off_p[S::kLoadsP], off_q[S::kLoadsQ];
    att::rsrc_t rsrc_p[2], rsrc_q;
    {
        const int64_t left = a.tokens - t0;
#pragma unroll
        for (int i = 0; i < S::kLoadsQ; i++) {
            const int r = i * S::kWaves * 8 + row8;
            off_q[i] = r < left ? (uint32_t)(r * a.q_stride * kE) + (uint32_t)(chunk * 16) : att::kOutside;
        }
        rsrc_q = att::buffer((const char*)a.q + t0 * a.q_stride * kE, kInside);
    }
    {
        const int64_t left = a.features - f0;
#pragma unroll
        for (int i = 0; i < S::kLoadsP; i++) {
            const int r = i * S::kWaves * 8 + row8;
            const int f = KIND == kGated ? (r >> 6) * 32 + (r & 31) : r;
            const int half = KIND == kGated ? (r >> 5) & 1 : 0;
            off_p[i] = f < left ? (uint32_t)(f * a.p_stride[half] * kE) + (uint32_t)(chunk * 16) : att::kOutside;
        }
        // gate or up: with eight wavefronts by the wavefront, with four by the load
        const int own = KIND == kGated && S::kWaves == 8 ? (wave >> 2) & 1 : 0;
        const void* const base = own != 0 ? a.p[1] : a.p[0];
        const int64_t stride = own != 0 ? a.p_stride[1] : a.p_stride[0];
        rsrc_p[0] = att::buffer((const char*)base + f0 * stride * kE, kInside);
        rsrc_p[1] = KIND == kGated && S::kWaves == 4
                        ? att::buffer((const char*)a.p[1] + f0 * a.p_stride[1] * kE, kInside)
                        : rsrc_p[0];
    }
    const uint32_t lds0 = att::lds_place(lds);
    const uint32_t term_bytes = (uint32_t)(a.terms * kE);
    uint32_t first_stage = 0, stages = (term_bytes + kRowBytes - 1) / kRowBytes;
    if (KIND == kPartial) {
        first_stage = part * (uint32_t)a.part_stages;
        const uint32_t left = stages > first_stage ? stages - first_stage : 0;
        stages = left < (uint32_t)a.part_stages ? left : (uint32_t)a.part_stages;
    }
    const auto load_stage = [&](uint32_t stage, int buffer) {
        const uint32_t at = (first_stage + stage) * kRowBytes;
        const bool there = at + (uint32_t)chunk * 16 < term_bytes;  // the last stage may end early: zeros, on both sides
        const uint32_t to = lds0 + (uint32_t)(buffer * S::kStageBytes + wave * 1024);
#pragma unroll
        for (int i = 0; i < S::kLoadsP; i++) {
            load_to_lds(rsrc_p[S::kWaves == 4 ? i & 1 : 0], to + (uint32_t)(i * S::kWaves * 1024),
                        there ? off_p[i] : att::kOutside, at);
        }
#pragma unroll
        for (int i = 0; i < S::kLoadsQ; i++) {
            load_to_lds(rsrc_q, to + (uint32_t)(S::kFeatures * kRowBytes + i * S::kWaves * 1024),
                        there ? off_q[i] : att::kOutside, at);
        }
    };

    // Where this lane reads: row l % 32 of a block, vector 2 j + h of step j.
    int at_step[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        at_step[j] = (lane & 31) * kRowBytes + (((2 * j + (lane >> 5)) ^ swizzle(lane & 31)) << 4);
    }
    const char* const from_p = lds + wf * FB * 32 * kRowBytes;
    const char* const from_q = lds + (S::kFeatures + wt * TB * 32) * kRowBytes;
    Frag fp[2][FB], fq[2][TB];
    const auto read_step = [&](int j, int buffer, int slot) {
        const int at = at_step[j] + buffer * S::kStageBytes;
#pragma unroll
        for (int b = 0; b < FB; b++) {
            fp[slot][b] = *reinterpret_cast<const Frag*>(from_p + at + b * 32 * kRowBytes);
        }
#pragma unroll
        for (int b = 0; b < TB; b++) {
            fq[slot][b] = *reinterpret_cast<const Frag*>(from_q + at + b * 32 * kRowBytes);
        }
    };
    acc_t acc[FB][TB];
#pragma unroll
    for (int b = 0; b < FB; b++) {
#pragma unroll
        for (int c = 0; c < TB; c++) {
            acc[b][c] = att::zeros();
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
    if (stages > 0) {
        load_stage(0, 0);
        if (stages > 1) {
            load_stage(1, 1);
            __asm__ volatile("s_waitcnt vmcnt(%0)" ::"n"(S::kLoadsP + S::kLoadsQ) : "memory");
        } else {
            __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
        __builtin_amdgcn_s_barrier();
        __asm__ volatile("" ::: "memory");
        read_step(0, 0, 0);
        for (uint32_t stage = 0; stage < stages; stage++) {
            const int buffer = (int)(stage & 1);
#pragma unroll
            for (int j = 0; j < 3; j++) {
                read_step(j + 1, buffer, (j + 1) & 1);
                multiply(j & 1);
            }
            if (stage + 1 < stages) {
                __asm__ volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
                __builtin_amdgcn_s_barrier();
                __asm__ volatile("" ::: "memory");
                if (stage + 2 < stages) {
                    load_stage(stage + 2, buffer);
                }
                read_step(0, buffer ^ 1, 0);
            }
            multiply(1);
        }
    }

    // ---------------------------------------------------------------------------------------------- results
    // A wavefront's results go out by way of a place of its own in LDS, 32 tokens at a time, so that neighbouring lanes write
    // neighbouring vectors of a token.  Register r of a block is feature 8 (r / 4) + 4 h + r % 4 of token l % 32.
    const int h = lane >> 5, n = lane & 31;
    if constexpr (KIND == kPartial) {
        float* const to = (float*)a.out[0] + ((int64_t)part * a.tokens) * a.features;
#pragma unroll
        for (int c = 0; c < TB; c++) {
            const int64_t t = t0 + (wt * TB + c) * 32 + n;
#pragma unroll
            for (int b = 0; b < FB; b++) {
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const int64_t f = f0 + (wf * FB + b) * 32 + 8 * (r / 4) + 4 * h + r % 4;
                    if (t < a.tokens && f < a.features) {
                        to[t * a.features + f] = acc[b][c][r];
                    }
                }
            }
        }
        return;
    } else {
        constexpr int kBlocks = KIND == kGated ? FB / 2 : FB;  // of results, a row of them; gated: one at a time
        constexpr int kRow = KIND == kGated ? 1 : FB;          // blocks of 32 features that go out together
        constexpr int kVec = 16 / kE;
        constexpr int kChunks = 32 * kRow * kE / 16;           // vectors of a token
        __syncthreads();  // all have read their last stage
        char* const own = lds + wave * 32 * S::kPitch;
        // Writes out what lies in `own`: tokens t.. , features f..
        const auto put = [&](int which, int64_t t, int64_t f) {
            __asm__ volatile("" ::: "memory");  // the compiler keeps the order; LDS does for one wavefront
#pragma unroll
            for (int i = 0; i < 32 * kChunks / 64; i++) {
                const int token = (i * 64 + lane) / kChunks, c = (i * 64 + lane) % kChunks;
                const Pack16 v = *reinterpret_cast<const Pack16*>(own + token * S::kPitch + c * 16);
                if (t + token < a.tokens) {
                    const bool second = KIND == kPlain && t + token >= a.turn;
                    const int64_t row = second ? t + token - a.turn : t + token;
                    const int64_t stride = second ? a.out_stride[1] : a.out_stride[which];
                    T* const to = (T*)(second ? a.out[1] : a.out[which]) + row * stride + f + c * kVec;
                    const int64_t left = a.features - (f + c * kVec);
                    if ((second ? a.wide[1] : a.wide[which]) != 0 && left >= kVec) {
                        *reinterpret_cast<Pack16*>(to) = v;
                    } else {
                        const T* const each = reinterpret_cast<const T*>(&v);
#pragma unroll
                        for (int e = 0; e < kVec; e++) {
                            if (e < left) {
                                to[e] = each[e];
                            }
                        }
                    }
                }
            }
            __asm__ volatile("" ::: "memory");
        };
        const auto hold = [&](int block, int quarter, const float (&x)[4]) {
            tok::Pack<T, 4> k;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                k.v[e] = (T)x[e];
            }
            *reinterpret_cast<tok::Pack<T, 4>*>(own + n * S::kPitch + (block * 32 + 8 * quarter + 4 * h) * kE) = k;
        };
#pragma unroll
        for (int c = 0; c < TB; c++) {
            const int64_t t = t0 + (wt * TB + c) * 32;
            if (t >= a.tokens) {
                break;
            }
            if constexpr (KIND == kPlain) {
                float scale = 1.0f;
                if (a.token_scale != nullptr && t + n < a.tokens) {
                    scale = a.token_scale[t + n];
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
#pragma unroll
                for (int b = 0; b < kBlocks; b++) {
                    const int64_t f = f0 + (wf * kBlocks + b) * 32;
                    if (a.bias[0] != nullptr) {
#pragma unroll
                        for (int r = 0; r < 16; r++) {
                            const int64_t own_f = f + 8 * (r / 4) + 4 * h + r % 4;
                            if (own_f < a.features) {
                                acc[2 * b][c][r] += (float)((const T*)a.bias[0])[own_f];
                                acc[2 * b + 1][c][r] += (float)((const T*)a.bias[1])[own_f];
                            }
                        }
                    }
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        float x[4];
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            x[e] = activate(acc[2 * b][c][4 * q + e], a.activation) * acc[2 * b + 1][c][4 * q + e];
                        }
                        hold(0, q, x);
                    }
                    put(0, t, f);
                    if (a.out[1] != nullptr) {
#pragma unroll
                        for (int which = 0; which < 2; which++) {
#pragma unroll
                            for (int q = 0; q < 4; q++) {
                                float x[4];
#pragma unroll
                                for (int e = 0; e < 4; e++) {
                                    x[e] = acc[2 * b + which][c][4 * q + e];
                                }
                                hold(0, q, x);
                            }
                            put(1 + which, t, f);
                        }
                    }
                }
            }
        }
    }
}

}  // namespace prod
}  // namespace opscv
