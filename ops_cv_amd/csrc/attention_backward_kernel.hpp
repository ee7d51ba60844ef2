// Gradients of attention, in two kernels and a join:
//
//   queries     as the forward pass walks keys:  P' = exp2(K Q' c - lse),  dP' = V gO',  dS' = P' (dP' - D),
//               gQ' += K' dS'.  Before that every row i's statistics, which the next kernel reads too: lse_i log2 e (infinity
//               where the row sees nothing) and D_i = sum gO_i O_i
//   keys        a wavefront keeps 32 keys and walks the queries that see them:  P, dS as above with rows and columns
//               exchanged,  gV' += gO' P,  gK' += Q' dS
//   join        where the queries of a tile of keys were cut into parts, their 32-bit sums in order
//
// Everything but the operands of the products is in 32 bits: P and dS are rounded to the type, because the matrix instructions
// take operands of one type (as in the forward pass).  P and dS are computed twice, once for each direction: seven products
// instead of five, but every sum has one owner and a fixed order, and no gradient is added up by atomics.
//
// 4096 tokens, 32 heads of 128 on 8, window 1024, bf16: 284 to 288 us (525 TFLOP/s of the five products); keys 160 to 167,
// queries 115 to 125, the join 15.  In both kernels 35 % of a SIMD's cycles are products and 30 % vector instructions,
// which two wavefronts a SIMD, all that the accumulators leave room for, cover in part; LDS is busy for 26 % in the keys'.
// FLOAT (2 x 777 tokens, 12 heads of 72 on 4, window 101: 91 us, queries 37, keys 50) is bound by single wavefronts that walk
// five or six tiles one after another: products, which take sixteen times as many cycles as those of 16-bit types, are half
// of a wavefront's time and loads that nothing covers a quarter (keys) to a third (queries), while fewer than half of the
// SIMDs have a wavefront at all.
//
// dS of FLOAT16 may be anything from P of a long row times a small gradient, for which FLOAT16 has few bits or none, to the
// products of large gradients and values, which are past its end.  So every sum's dS (of a row in the queries' kernel, of a
// key in the keys') is divided before it is rounded by a power of two that follows the largest |dS| met so far, and the sum
// multiplied by it (fit_unit).  P of the keys' kernel is never more than 1 and enters its products 2^14 times as large, so that
// it has its bits down to 2^-28, below which nothing that it is multiplied with makes more than FLOAT16's smallest numbers.
#pragma once

#include <atomic>
#include <type_traits>

#include "attention_plan.hpp"
#include "attention_tile.hpp"
#include "fast_div.hpp"
#include "kernels.hpp"

namespace opscv {
namespace att {

struct GradLaunch {
    AttentionArgs a;
    FastDiv group;
    uint32_t rows, tiles, kv_heads;
    uint32_t keys, key_tiles, sink_tiles, sink_parts, parts;
    uint32_t query_blocks, key_blocks;
    int64_t stat_pitch;
    float* stats;          // (batch, heads, 2, stat_pitch): lse log2 e - kWeightGain, and D
    float* sink_partials;  // (batch * kv_heads, sink_tiles, sink_parts, 2, keys, d rounded up to four)
    float* partials;       // the same of the other tiles
};

// binary logarithm of the factor that P of the keys' kernel has
template <typename T>
constexpr float kWeightGain = std::is_same<T, _Float16>::value ? 14.0f : 0.0f;

static __device__ __forceinline__ int64_t stats_row(const GradLaunch& p, int64_t b, int64_t head)
{
    return (b * p.a.heads + head) * 2 * p.stat_pitch;
}

// What dS of FLOAT16 is divided by before it is rounded, its unit: a power of two of the lane's column (a row or a key, whose
// 32 terms of a tile two lanes hold).  Terms past 2^15 units would not be numbers; those of less than 2^-14 lose bits.
constexpr float kMostUnits = 32768.0f;

// the column's largest |x| that is finite (a term that is not leaves a sum that is not, whatever the unit)
static __device__ __forceinline__ float largest_term(const acc_t& x)
{
    float highs[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int r = 0; r < 16; r += 2) {
        highs[r / 2 % 4] = fmaxf(fmaxf(highs[r / 2 % 4], fabsf(x[r])), fabsf(x[r + 1]));
    }
    float high = fmaxf(fmaxf(highs[0], highs[1]), fmaxf(highs[2], highs[3]));
    high = fmaxf(high, other_half(high));
    return high < INFINITY ? high : 0.0f;
}

// the unit of which a term of `size` has 2^steps to 2^(steps + 1)
static __device__ __forceinline__ float unit_of(float size, int steps)
{
    const float power = __uint_as_float(__float_as_uint(size) & 0x7f800000u);
    return size > 0.0f ? fmaxf(__builtin_amdgcn_ldexpf(power, -steps), 0x1p-100f) : 0.0f;
}

// Lets `unit` grow with the largest of x, what is seen of a tile's terms; `sum` holds what the column has so far, in units.  A
// new unit is 2^-8 of the largest term, so that it seldom has to grow again.
template <int NB>
static __device__ __forceinline__ void fit_unit(const acc_t& x, float& unit, acc_t (&sum)[NB])
{
    const float high = largest_term(x);
    const bool grows = high > unit * kMostUnits;
    if (__builtin_expect(__any(grows), 0)) {
        const float now = grows ? unit_of(high, 8) : unit, fade = grows ? unit / now : 1.0f;
#pragma unroll
        for (int i = 0; i < NB; i++) {
#pragma unroll
            for (int r = 0; r < 16; r++) {
                sum[i][r] *= fade;
            }
        }
        unit = now;
    }
}

// x in units
static __device__ __forceinline__ void to_units(acc_t& x, float unit)
{
    // 1 / unit of a power of two; 2^127 of 0, where x holds zeros or what is not finite
    const float per_unit = __uint_as_float(0x7f000000u - __float_as_uint(unit));
#pragma unroll
    for (int r = 0; r < 16; r++) {
        x[r] *= per_unit;
    }
}

// ---------------------------------------------------------------------------------------------------- queries' gradients

// gQ' += K' dS' for one block of features and 32 keys that some rows do not see and that may hold values that are not finite:
// the finite ones are multiplied as ever, and the rows that see one of the others (products of ones and zeros count them)
// get NaN, which is what a score that is not finite makes of them.
template <typename T, int PITCH>
static __device__ __forceinline__ acc_t add_seen_keys(acc_t sum, const acc_t& ds, const acc_t& seen, const T* tile, int block,
                                                      int lane)
{
    acc_t count = zeros();
#pragma unroll
    for (int g = 0; g < 2; g++) {
        Frag<T> f = Tile<T, PITCH>::column(tile, 16 * g, block, lane), special;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float v = (float)f[e];
            const bool finite = __builtin_amdgcn_classf(v, 0x1f8);
            f[e] = (T)(finite ? v : 0.0f);
            special[e] = (T)(finite ? 0.0f : 1.0f);
        }
        sum = Mma<T>::mul(f, operand<T>(ds, g), sum);
        count = Mma<T>::mul(special, operand<T>(seen, g), count);
    }
#pragma unroll
    for (int r = 0; r < 16; r++) {
        sum[r] = count[r] > 0.0f ? NAN : sum[r];
    }
    return sum;
}

template <typename T, int NB, bool FEW, bool VEC>
__global__ __launch_bounds__(grad_query_shape(sizeof(T), pitch_of(NB), FEW).threads(),
                             sizeof(T) * NB <= 8 ? 2 : 1) void attention_query_grad_kernel(GradLaunch p)
{
    constexpr int kPitch = pitch_of(NB);
    constexpr ForwardShape kShape = grad_query_shape(sizeof(T), kPitch, FEW);
    constexpr int kKeys = kShape.keys, kThreads = 64 * kShape.row_waves, kJoin = kShape.key_waves;
    // Units of dS: sums of up to 128 features are scaled as the unit grows.  Those of more, for which that would cost registers
    // in the loop (16 x 512 tokens, 2 heads of 256 on 1: 156 us for 119), have the unit of their first term's size, and
    // where a later one is past its range, all is done once more with the unit of the largest.
    constexpr bool kUnits = std::is_same<T, _Float16>::value, kOneUnit = kUnits && NB > 4;
    // FLOAT's products take so long that operands can come from memory as they are needed: the values of wider heads do,
    // which leaves LDS for the keys of four wavefronts, and gO of the widest, which leaves registers for the rest
    constexpr bool kDirect = grad_values_direct(sizeof(T), kPitch, FEW), kGradDirect = kDirect && NB > 4;
    constexpr int kTileElems = (kDirect ? 1 : 2) * kKeys * kPitch;
    extern __shared__ __align__(16) char lds[];

    const AttentionArgs& a = p.a;
    const uint32_t index = xcd_order(blockIdx.x, p.query_blocks);
    if (index >= p.query_blocks) {
        return;
    }
    const uint32_t tile = index % p.tiles, bh = index / p.tiles;
    const uint32_t b = bh / p.kv_heads, kv_head = bh % p.kv_heads;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = (int)threadIdx.x & 63;
    const int h = lane >> 5, own = lane & 31;
    const int d = (int)a.d, left = (int)a.left, right = (int)a.right, sinks = (int)a.sinks;
    const Sequence seq = sequence_at(a, b);

    const int row_wave = wave % kShape.row_waves, key_wave = wave / kShape.row_waves;
    const uint32_t row0 = tile * kShape.rows(), wave_row0 = row0 + row_wave * kBlock;
    const uint32_t row = min(wave_row0 + own, p.rows - 1);
    const int query = (int)fast_div(row, p.group);
    const int head = (int)(kv_head * p.group.div) + (int)(row - (uint32_t)query * p.group.div);
    const int pos = query < seq.q_len ? seq.first + query : INT32_MIN / 2;
    const auto query_of = [&](uint32_t r) { return (int)fast_div(min(r, p.rows - 1), p.group); };
    const int block_low = query_of(row0), block_high = min(query_of(row0 + kShape.rows() - 1), seq.q_len - 1);
    KeyRange range = key_range<kKeys>(seq.first + block_low, seq.first + block_high, seq.kv_len, left, right, sinks);
    if (block_high < block_low) {
        range.tiles = 0;
    }
    const int wave_low = seq.first + query_of(wave_row0);
    const int wave_high = seq.first + min(query_of(wave_row0 + kBlock - 1), seq.q_len - 1);
    const bool wave_whole = query_of(wave_row0 + kBlock - 1) < seq.q_len;

    const T* const k_base = (const T*)a.k.ptr + (int64_t)b * a.k.stride[0] + (int64_t)kv_head * a.k.stride[2];
    const T* const v_base = (const T*)a.v.ptr + (int64_t)b * a.v.stride[0] + (int64_t)kv_head * a.v.stride[2];
    const uint32_t k_pitch = (uint32_t)(a.k.stride[1] * (int64_t)sizeof(T));
    const uint32_t v_pitch = (uint32_t)(a.v.stride[1] * (int64_t)sizeof(T));
    T* const ring = reinterpret_cast<T*>(lds) + (size_t)key_wave * (kShape.stages * kTileElems);
    const auto fetch = [&](int t, int buffer) {
        const int key0 = range.key_of(t, kKeys), rows = range.end_of(t) - key0;
        T* const k_tile = ring + buffer * kTileElems;
        const int gt = row_wave * 64 + again(lane);
        stage<T, kPitch, kKeys, kThreads, VEC>(k_tile, at_bytes(k_base, (uint32_t)key0, k_pitch), gt, row_wave, d, k_pitch,
                                               min(rows, kKeys));
        if constexpr (!kDirect) {
            stage<T, kPitch, kKeys, kThreads, VEC>(k_tile + kKeys * kPitch, at_bytes(v_base, (uint32_t)key0, v_pitch), gt,
                                                   row_wave, d, v_pitch, min(rows, kKeys));
        }
    };
    const float c = a.scale * kLog2e;
    acc_t gq[NB];
    int buffer = 0;
    constexpr int kInFlight = kTileElems / kPitch * Tile<T, kPitch>::kChunks / kThreads;  // loads of one fetch, a wavefront
    if (key_wave < range.tiles) {
        fetch(key_wave, 0);
    }
    Frag<T> q[2 * NB], held[kGradDirect ? 1 : 2 * NB];
    const T* const grad_row = (const T*)a.grad_out.ptr + (int64_t)b * a.grad_out.stride[0] +
                              (int64_t)query * a.grad_out.stride[1] + (int64_t)head * a.grad_out.stride[2];
    const auto go = [&](int i) {
        if constexpr (kGradDirect) {
            return global_row<T, VEC>(grad_row, 16 * i + 8 * h, d);
        } else {
            return held[i];
        }
    };
    {
        const T* const src = (const T*)a.q.ptr + (int64_t)b * a.q.stride[0] + (int64_t)query * a.q.stride[1] +
                             (int64_t)head * a.q.stride[2];
#pragma unroll
        for (int i = 0; i < 2 * NB; i++) {
            q[i] = global_row<T, VEC>(src, 16 * i + 8 * h, d);
            if constexpr (!kGradDirect) {
                held[i] = global_row<T, VEC>(grad_row, 16 * i + 8 * h, d);
            }
        }
    }
    // the row's statistics, left for the keys' gradients too
    float lse, along;
    {
        const T* const out = (const T*)a.out.ptr + (int64_t)b * a.out.stride[0] + (int64_t)query * a.out.stride[1] +
                             (int64_t)head * a.out.stride[2];
        float sums[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < 2 * NB; i++) {
            const Frag<T> x = go(i), y = global_row<T, VEC>(out, 16 * i + 8 * h, d);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                sums[e % 4] += (float)x[e] * (float)y[e];
            }
        }
        along = (sums[0] + sums[1]) + (sums[2] + sums[3]);
        along += other_half(along);
        lse = ((const float*)a.lse.ptr)[(int64_t)b * a.lse.stride[0] + (int64_t)head * a.lse.stride[1] +
                                        (int64_t)query * a.lse.stride[2]];
        const bool live = query < seq.q_len && lse != -INFINITY;
        lse = live ? lse * kLog2e : INFINITY;
        along = live ? along : 0.0f;
        if (key_wave == 0 && h == 0 && wave_row0 + own < p.rows) {
            float* const stat = p.stats + stats_row(p, b, head) + query;
            stat[0] = lse - kWeightGain<T>;
            stat[p.stat_pitch] = along;
        }
    }
    wait_for_registers();
    // as in the forward pass: 32 keys of a tile, those of tiles that all of the wavefront's rows see whole in a loop of their own
    const auto whole = [&](int t) {
        const int key0 = range.key_of(t, kKeys);
        return wave_whole && key0 + kKeys <= range.end_of(t) && key0 + kKeys - 1 <= wave_low + right &&
               (key0 >= wave_high - left || key0 + kKeys <= sinks);
    };
    const auto unseen = [&](int key0, int end) {
        return wave_low > wave_high || key0 >= end || key0 > wave_high + right ||
               (key0 + kBlock - 1 < wave_low - left && key0 >= sinks);
    };
    bool careful = false;  // a second pass, for keys that are not finite
    float unit = 0.0f, most = 0.0f, first_unit = 0.0f;
    const auto attend = [&](auto part, int key0, int end, const T* k_tile, const T* v_tile, const Rows32<T, kPitch, NB>& rows,
                            const Columns32<T, kPitch, NB>& columns) {
        acc_t s = zeros(), dp = zeros();
        // keys that the lane's value stands in for past the end are not seen
        const T* const value = kDirect ? at_bytes(v_base, (uint32_t)min(key0 + own, end - 1), v_pitch) : nullptr;
        if constexpr (kGradDirect) {
            // the next operands are asked for before a product, and no earlier: their registers are few
            Frag<T> value_now = global_row<T, VEC>(value, 8 * h, d), grad_now = go(0);
#pragma unroll
            for (int i = 0; i < 2 * NB; i++) {
                const int next = i + 1 < 2 * NB ? i + 1 : i;
                const Frag<T> value_next = global_row<T, VEC>(value, 16 * next + 8 * h, d), grad_next = go(next);
                dp = Mma<T>::mul(value_now, grad_now, dp);
                s = Mma<T>::mul(rows(k_tile, 0, i), q[i], s);
                __builtin_amdgcn_sched_barrier(0);
                value_now = value_next;
                grad_now = grad_next;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 2 * NB; i++) {
                s = Mma<T>::mul(rows(k_tile, 0, i), q[i], s);
                if constexpr (kDirect) {
                    dp = Mma<T>::mul(global_row<T, VEC>(value, 16 * i + 8 * h, d), held[i], dp);
                } else {
                    dp = Mma<T>::mul(rows(v_tile, 0, i), held[i], dp);
                }
            }
        }
        if constexpr (sizeof(T) == 2) {
            read_ahead<4 * NB, 1, 4>();
        }
#pragma unroll
        for (int r = 0; r < 16; r++) {
            s[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], c, -lse)) * (dp[r] - along);
        }
        if constexpr (decltype(part)::value) {
            const Sight see = sight(pos, key0 + 4 * h, end, left, right, sinks);
#pragma unroll
            for (int r = 0; r < 16; r++) {
                s[r] = see.sees(8 * (r / 4) + r % 4) ? s[r] : 0.0f;
            }
        }
        if constexpr (kOneUnit) {
            const float high = largest_term(s);
            most = fmaxf(most, high);
            unit = unit == 0.0f ? unit_of(high, 0) : unit;
        } else if constexpr (kUnits) {
            fit_unit(s, unit, gq);
        }
        if constexpr (kUnits) {
            to_units(s, unit);
        }
        if (decltype(part)::value && __builtin_expect(careful, 0)) {
            const Sight see = sight(pos, key0 + 4 * h, end, left, right, sinks);
            acc_t seen;
#pragma unroll
            for (int r = 0; r < 16; r++) {
                seen[r] = see.sees(8 * (r / 4) + r % 4) ? 1.0f : 0.0f;
            }
#pragma unroll
            for (int i = 0; i < NB; i++) {
                gq[i] = add_seen_keys<T, kPitch>(gq[i], s, seen, k_tile, i, again(lane));
            }
        } else {
#pragma unroll
            for (int g = 0; g < 2; g++) {
                const Frag<T> w = operand<T>(s, g);
#pragma unroll
                for (int i = 0; i < NB; i++) {
                    gq[i] = Mma<T>::mul(columns(k_tile, 16 * g, i), w, gq[i]);
                }
            }
            if constexpr (sizeof(T) == 2) {
                read_ahead<2 * NB, 2, 3>();
            }
        }
    };
    int t = key_wave;
    const auto work = [&](auto part, const Rows32<T, kPitch, NB>& rows, const Columns32<T, kPitch, NB>& columns) {
        constexpr bool PART = decltype(part)::value;
        const bool more = t + kJoin < range.tiles;
        if constexpr (kJoin == 1) {
            wait_for_loads<0>();
            barrier();
            if (kShape.stages == 2 && more) {
                fetch(t + 1, buffer ^ 1);
            }
        } else {
            if (kShape.stages == 2 && more) {
                fetch(t + kJoin, buffer ^ 1);
                wait_for_loads<VEC ? kInFlight : 0>();
            } else {
                wait_for_loads<0>();
            }
        }
        const T* const k_tile = ring + buffer * kTileElems;
        const T* const v_tile = k_tile + kKeys * kPitch;
        const int key0 = range.key_of(t, kKeys), end = range.end_of(t);
        if constexpr (PART) {
#pragma unroll 1
            for (int j = 0; j < kKeys; j += kBlock) {
                if (!unseen(key0 + j, end)) {
                    attend(part, key0 + j, end, k_tile + j * kPitch, v_tile + j * kPitch, rows, columns);
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < kKeys; j += kBlock) {
                attend(part, key0 + j, end, k_tile + j * kPitch, v_tile + j * kPitch, rows, columns);
            }
        }
        if (kShape.stages == 1 && more) {
            if constexpr (kJoin == 1) {
                barrier();
            } else {
                wait_for_lds();
            }
            fetch(t + kJoin, 0);
        }
        buffer ^= kShape.stages - 1;
        t += kJoin;
    };
    while (true) {
#pragma unroll
        for (int i = 0; i < NB; i++) {
            gq[i] = zeros();
        }
        unit = first_unit;
        while (t < range.tiles) {
            {
                const Rows32<T, kPitch, NB> rows(again(lane));
                const Columns32<T, kPitch, NB> columns(again(lane));
                while (t < range.tiles && !whole(t)) {
                    work(std::true_type(), rows, columns);
                }
            }
            const Rows32<T, kPitch, NB> rows(again(lane));
            const Columns32<T, kPitch, NB> columns(again(lane));
            while (t < range.tiles && whole(t)) {
                work(std::false_type(), rows, columns);
            }
        }
        // as in the forward pass: gradients that are not finite may come from keys that a row does not see
        float check = 0.0f;
#pragma unroll
        for (int i = 0; i < NB; i++) {
#pragma unroll
            for (int r = 0; r < 16; r++) {
                check = __builtin_fmaf(gq[i][r], 0.0f, check);
            }
        }
        const auto any_row = [&](bool x) { return kShape.row_waves > 1 ? __syncthreads_or(x) != 0 : __any(x) != 0; };
        const bool past = most > unit * kMostUnits;
        if (kOneUnit && any_row(past)) {
            first_unit = past ? unit_of(most, 8) : unit;  // each row by its own terms alone
        } else if (any_row(!careful && check != 0.0f)) {
            careful = true;
        } else {
            break;
        }
        t = key_wave;
        buffer = 0;
        if (t < range.tiles) {
            fetch(t, 0);
        }
    }
    if constexpr (kUnits) {
#pragma unroll
        for (int i = 0; i < NB; i++) {
#pragma unroll
            for (int r = 0; r < 16; r++) {
                gq[i][r] *= unit;
            }
        }
    }
    if constexpr (kJoin > 1) {
        // sums of the wavefronts that shared the keys, [feature][row]; every one adds up a share of the features
        constexpr int kWaveFloats = NB * kBlock * kBlock;
        float* const sums = reinterpret_cast<float*>(lds);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NB; i++) {
#pragma unroll
            for (int r = 0; r < 16; r++) {
                sums[wave * kWaveFloats + (i * kBlock + 8 * (r / 4) + 4 * h + r % 4) * kBlock + own] = gq[i][r];
            }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NB; i++) {
            if (i % kJoin == wave) {
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    float x = 0.0f;
#pragma unroll
                    for (int w = 0; w < kJoin; w++) {
                        x += sums[w * kWaveFloats + (i * kBlock + 8 * (r / 4) + 4 * h + r % 4) * kBlock + own];
                    }
                    gq[i][r] = x;
                }
            }
        }
    }
    if (wave_row0 + own >= p.rows) {
        return;
    }
    const float f = a.scale;
    T* const to = (T*)a.grad_q.ptr + (int64_t)b * a.grad_q.stride[0] + (int64_t)query * a.grad_q.stride[1] +
                  (int64_t)head * a.grad_q.stride[2];
#pragma unroll
    for (int i = 0; i < NB; i++) {
        if (kJoin == 1 || i % kJoin == wave) {
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                put4<T, VEC>(to, i * kBlock + 8 * (r / 4) + 4 * h, d, gq[i][r] * f, gq[i][r + 1] * f, gq[i][r + 2] * f,
                             gq[i][r + 3] * f);
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------------- keys' gradients

// Both gradients in one pass, or, for heads of more than 128 features, whose two sums would not fit the registers, one after
// the other (the scores' product is done twice: five products instead of four).
enum KeyGradPass : int { kBothGrads = 0, kValueGrad = 1, kKeyGrad = 2 };

// The values of the keys are read from LDS for every product, which leaves 16-bit heads of up to 128 features within the
// 256 registers of two wavefronts a SIMD (with the values in registers too, one: the accumulators then lie in the other
// half of the register file and are copied to and fro; 4096 tokens, 32 heads on 8, window 1024: 366 us against 187).
// FLOAT keeps them in registers: LDS then holds four workgroups a CU.
constexpr bool key_grad_values_in_lds(int elem_bytes) { return elem_bytes == 2; }
constexpr int key_grad_stages(int elem_bytes) { return elem_bytes == 2 ? 2 : 1; }
constexpr int key_grad_waves(int elem_bytes, int nb) { return elem_bytes * nb <= 8 ? 2 : 1; }

template <typename T, int NB, int PASS, bool VEC>
__global__ __launch_bounds__(64 * grad_key_waves(sizeof(T) == 4, NB), key_grad_waves(sizeof(T), NB)) void
attention_key_grad_kernel(GradLaunch p)
{
    constexpr int kKeyWaves = grad_key_waves(sizeof(T) == 4, NB), kGradKeys = kBlock * kKeyWaves;
    constexpr int kPitch = pitch_of(NB), kThreads = 64 * kKeyWaves;
    constexpr int kStages = key_grad_stages(sizeof(T));
    constexpr bool kUnits = std::is_same<T, _Float16>::value;
    constexpr int kStatRows = 2;               // of 32 floats each, a wavefront and stage
    constexpr int kTile = kBlock * kPitch;     // elements
    constexpr bool kValuesInLds = key_grad_values_in_lds(sizeof(T)), kWithKeys = PASS != kValueGrad, kWithValues = PASS != kKeyGrad;
    extern __shared__ __align__(16) char lds[];

    const AttentionArgs& a = p.a;
    uint32_t index = xcd_order(blockIdx.x, p.key_blocks);
    if (index >= p.key_blocks) {
        return;
    }
    // of a key head: the parts of the sinks' tiles, then those of the others
    const uint32_t sink_items = p.sink_tiles * p.sink_parts;
    const uint32_t items = sink_items + (p.key_tiles - p.sink_tiles) * p.parts;
    const uint32_t bh = index / items, item = index % items;
    const bool sink_tile = item < sink_items;
    const uint32_t of = sink_tile ? p.sink_parts : p.parts, at = sink_tile ? item : item - sink_items;
    const uint32_t part = at % of, local_tile = at / of, tile = local_tile + (sink_tile ? 0 : p.sink_tiles);
    const uint32_t b = bh / p.kv_heads, kv_head = bh % p.kv_heads;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = (int)threadIdx.x & 63;
    const int h = lane >> 5, own = lane & 31;
    const int d = (int)a.d, left = (int)a.left, right = (int)a.right, sinks = (int)a.sinks;
    const Sequence seq = sequence_at(a, b);

    const int key0 = (int)tile * kGradKeys, wave_key0 = key0 + wave * kBlock, key = wave_key0 + own;
    // queries that see a key of the tile
    const int last = min(key0 + kGradKeys, seq.kv_len) - 1;
    int low = max(key0 - right - seq.first, 0);
    int high = key0 < sinks ? seq.q_len : min(seq.q_len, last + left + 1 - seq.first);
    if (last < key0) {
        high = low;
    }
    const int row_tiles = high > low ? (high - low + kBlock - 1) / kBlock : 0;
    const int steps = row_tiles * (int)p.group.div;
    const int s_begin = (int)((int64_t)steps * part / of), s_end = (int)((int64_t)steps * (part + 1) / of);

    T* const ring = reinterpret_cast<T*>(lds);
    float* const stat_ring = reinterpret_cast<float*>(lds + (size_t)kStages * 2 * kTile * sizeof(T)) +
                             wave * (kStages * kStatRows * kBlock);
    T* const v_tile = reinterpret_cast<T*>(lds + (size_t)kStages * 2 * kTile * sizeof(T) +
                                           kKeyWaves * kStages * kStatRows * kBlock * sizeof(float));
    const uint32_t q_pitch = (uint32_t)(a.q.stride[1] * (int64_t)sizeof(T));
    const uint32_t go_pitch = (uint32_t)(a.grad_out.stride[1] * (int64_t)sizeof(T));
    const int64_t head0 = (int64_t)kv_head * p.group.div;
    const T* const q_base = (const T*)a.q.ptr + (int64_t)b * a.q.stride[0] + head0 * a.q.stride[2];
    const T* const go_base = (const T*)a.grad_out.ptr + (int64_t)b * a.grad_out.stride[0] + head0 * a.grad_out.stride[2];
    const float* const stat_base = p.stats + stats_row(p, b, head0);
    // steps go through the tiles of one head's queries, then the next head's; `f_`: the step that is fetched next
    int f_head = s_begin < s_end ? s_begin / row_tiles : 0, f_query = low + (s_begin - f_head * row_tiles) * kBlock;
    int c_query = f_query;
    const auto fetch = [&](int buffer) {
        const int rows = min(seq.q_len - f_query, kBlock);
        T* const q_tile = ring + buffer * (2 * kTile);
        const int thread = wave * 64 + again(lane);
        stage<T, kPitch, kBlock, kThreads, VEC>(q_tile, at_bytes(q_base + f_head * a.q.stride[2], (uint32_t)f_query, q_pitch),
                                                thread, wave, d, q_pitch, rows);
        stage<T, kPitch, kBlock, kThreads, VEC>(q_tile + kTile,
                                                at_bytes(go_base + f_head * a.grad_out.stride[2], (uint32_t)f_query, go_pitch),
                                                thread, wave, d, go_pitch, rows);
        // statistics: lanes of the lower half read one kind, of the upper half the other; rows past the end read zeros,
        // which meet rows of zeros
        const rsrc_t rsrc = att::buffer(stat_base + f_head * (2 * p.stat_pitch) + f_query, 0x7fffffffu);
        load_to_lds<4, 0>(rsrc, lds_place(stat_ring + buffer * (kStatRows * kBlock)),
                          own < rows ? (uint32_t)(h * (int)p.stat_pitch + own) * 4u : kOutside);
        f_query += kBlock;
        if (f_query >= high) {
            f_query = low;
            f_head++;
        }
    };

    const float c = a.scale * kLog2e;
    acc_t gk[NB], gv[NB];
#pragma unroll
    for (int i = 0; i < NB; i++) {
        gk[i] = zeros();
        gv[i] = zeros();
    }
    float unit = 0.0f;
    int buffer = 0;
    if (s_begin < s_end) {
        fetch(0);
    }
    Frag<T> k[2 * NB], v[kValuesInLds || !kWithKeys ? 1 : 2 * NB];
    {
        const int64_t from = min(key, (int)a.kv_tokens - 1);
        const T* const k_first = (const T*)a.k.ptr + (int64_t)b * a.k.stride[0] + (int64_t)kv_head * a.k.stride[2];
        const T* const v_first = (const T*)a.v.ptr + (int64_t)b * a.v.stride[0] + (int64_t)kv_head * a.v.stride[2];
        if constexpr (kValuesInLds && kWithKeys) {
            if (last >= key0) {
                const uint32_t v_pitch = (uint32_t)(a.v.stride[1] * (int64_t)sizeof(T));
                stage<T, kPitch, kGradKeys, kThreads, VEC>(v_tile, at_bytes(v_first, (uint32_t)key0, v_pitch), wave * 64 + lane,
                                                           wave, d, v_pitch, last + 1 - key0);
            }
        }
#pragma unroll
        for (int i = 0; i < 2 * NB; i++) {
            k[i] = global_row<T, VEC>(k_first + from * a.k.stride[1], 16 * i + 8 * h, d);
            if constexpr (!kValuesInLds && kWithKeys) {
                v[i] = global_row<T, VEC>(v_first + from * a.v.stride[1], 16 * i + 8 * h, d);
            }
        }
    }
    wait_for_registers();
    for (int step = s_begin; step < s_end; step++) {
        const bool more = step + 1 < s_end;
        wait_for_loads<0>();
        barrier();
        if (kStages == 2 && more) {
            fetch(buffer ^ 1);
        }
        const T* const q_tile = ring + buffer * (2 * kTile);
        const T* const go_tile = q_tile + kTile;
        const float* const stat = stat_ring + buffer * (kStatRows * kBlock);
        const int i0 = c_query;
        c_query = c_query + kBlock < high ? c_query + kBlock : low;
        const int p_low = seq.first + i0, p_high = seq.first + min(i0 + kBlock, seq.q_len) - 1;
        // whether the wavefront's keys are seen by any of the rows, and by all of them
        const bool any = wave_key0 < seq.kv_len && wave_key0 <= p_high + right &&
                         (wave_key0 + kBlock - 1 >= p_low - left || wave_key0 < sinks);
        const bool all_seen = wave_key0 + kBlock <= seq.kv_len && wave_key0 + kBlock - 1 <= p_low + right &&
                              (wave_key0 >= p_high - left || wave_key0 + kBlock <= sinks);
        if (any) {
            acc_t s = zeros(), dp = zeros();
            const Rows32<T, kPitch, NB> rows(again(lane));
#pragma unroll
            for (int i = 0; i < 2 * NB; i++) {
                s = Mma<T>::mul(rows(q_tile, 0, i), k[i], s);
            }
            if constexpr (sizeof(T) == 2) {
                read_ahead<2 * NB, 1, 4>();
            }
            if constexpr (kWithKeys) {
#pragma unroll
                for (int i = 0; i < 2 * NB; i++) {
                    const Frag<T> g = rows(go_tile, 0, i);
                    if constexpr (kValuesInLds) {
                        dp = Mma<T>::mul(g, rows(v_tile, wave * kBlock, i), dp);
                    } else {
                        dp = Mma<T>::mul(g, v[i], dp);
                    }
                }
                if constexpr (sizeof(T) == 2) {
                    read_ahead<2 * NB, 2, 3>();
                }
            }
#pragma unroll
            for (int r = 0; r < 16; r++) {
                const int n = 8 * (r / 4) + 4 * h + r % 4;
                s[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], c, -stat[n]));
                if constexpr (kWithKeys) {
                    dp[r] = s[r] * (dp[r] - stat[kBlock + n]);
                }
            }
            if (__builtin_expect(!all_seen, 0)) {
                // query p_low + n sees the key: n >= first, n <= last or the key a sink, the key within the sequence
                const int first = key - right - p_low - 4 * h;
                const int last = key >= seq.kv_len ? -1 : key < sinks ? kBlock : key + left - p_low - 4 * h;
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const int n = 8 * (r / 4) + r % 4;
                    const bool seen = (n >= first) & (n <= last);
                    s[r] = seen ? s[r] : 0.0f;
                    dp[r] = seen ? dp[r] : 0.0f;
                }
            }
            if constexpr (kUnits && kWithKeys) {
                fit_unit(dp, unit, gk);
                to_units(dp, unit);
            }
            const Columns32<T, kPitch, NB> columns(again(lane));
#pragma unroll
            for (int g = 0; g < 2; g++) {
                const Frag<T> w = operand<T>(s, g), x = operand<T>(dp, g);
#pragma unroll
                for (int i = 0; i < NB; i++) {
                    if constexpr (kWithValues) {
                        gv[i] = Mma<T>::mul(columns(go_tile, 16 * g, i), w, gv[i]);
                    }
                    if constexpr (kWithKeys) {
                        gk[i] = Mma<T>::mul(columns(q_tile, 16 * g, i), x, gk[i]);
                    }
                }
            }
            if constexpr (sizeof(T) == 2) {
                read_ahead<(PASS == kBothGrads ? 4 : 2) * NB, 2, 4>();
            }
        }
        if (kStages == 1 && more) {
            barrier();
            fetch(0);
        }
        buffer ^= kStages - 1;
    }
    float f = a.scale;
    if constexpr (kUnits) {
        constexpr float kGain = 1.0f / (1 << (int)kWeightGain<T>);
        f *= unit * kGain;
#pragma unroll
        for (int i = 0; i < (kWithValues ? NB : 0); i++) {
#pragma unroll
            for (int r = 0; r < 16; r++) {
                gv[i][r] *= kGain;
            }
        }
    }
    if (of > 1) {
        const int64_t tile_index = sink_tile ? (int64_t)bh * p.sink_tiles + local_tile
                                             : (int64_t)bh * (p.key_tiles - p.sink_tiles) + local_tile;
        const int row_floats = (d + 3) / 4 * 4;
        float* const to = (sink_tile ? p.sink_partials : p.partials) +
                          ((tile_index * of + part) * 2 * kGradKeys + wave * kBlock + own) * row_floats;
#pragma unroll
        for (int i = 0; i < NB; i++) {
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const int el = i * kBlock + 8 * (r / 4) + 4 * h;
                if (el < d) {
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        if constexpr (kWithKeys) {
                            to[el + e] = gk[i][r + e] * f;
                        }
                        if constexpr (kWithValues) {
                            to[(int64_t)kGradKeys * row_floats + el + e] = gv[i][r + e];
                        }
                    }
                }
            }
        }
        return;
    }
    if (key >= (int)a.kv_tokens) {
        return;
    }
    T* const to_k = (T*)a.grad_k.ptr + (int64_t)b * a.grad_k.stride[0] + (int64_t)key * a.grad_k.stride[1] +
                    (int64_t)kv_head * a.grad_k.stride[2];
    T* const to_v = (T*)a.grad_v.ptr + (int64_t)b * a.grad_v.stride[0] + (int64_t)key * a.grad_v.stride[1] +
                    (int64_t)kv_head * a.grad_v.stride[2];
#pragma unroll
    for (int i = 0; i < NB; i++) {
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            const int el = i * kBlock + 8 * (r / 4) + 4 * h;
            if constexpr (kWithKeys) {
                put4<T, VEC>(to_k, el, d, gk[i][r] * f, gk[i][r + 1] * f, gk[i][r + 2] * f, gk[i][r + 3] * f);
            }
            if constexpr (kWithValues) {
                put4<T, VEC>(to_v, el, d, gv[i][r], gv[i][r + 1], gv[i][r + 2], gv[i][r + 3]);
            }
        }
    }
}

// Sums of the parts, of the sinks' tiles and of the others: four features of a key a thread.
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void attention_grad_join_kernel(GradLaunch p, uint32_t sink_joins, uint32_t quads, uint32_t total)
{
    const AttentionArgs& a = p.a;
    const uint32_t index = blockIdx.x * 256u + threadIdx.x;
    if (index >= total) {
        return;
    }
    const bool sinks = index < sink_joins;
    const float* const partials = sinks ? p.sink_partials : p.partials;
    const uint32_t first = sinks ? 0 : p.sink_tiles, tiles = sinks ? p.sink_tiles : p.key_tiles - p.sink_tiles;
    const uint32_t parts = sinks ? p.sink_parts : p.parts, local = sinks ? index : index - sink_joins;
    const uint32_t quad = local % quads;
    uint32_t rest = local / quads;
    const uint32_t local_key = rest % p.keys;
    rest /= p.keys;
    const uint32_t value = rest & 1, tile_index = rest >> 1;
    const uint32_t tile = first + tile_index % tiles, bh = tile_index / tiles;
    const int64_t key = (int64_t)tile * p.keys + local_key;
    if (key >= a.kv_tokens) {
        return;
    }
    const int row_floats = (int)quads * 4;
    const float* const from =
        partials + (((int64_t)tile_index * parts * 2 + value) * p.keys + local_key) * row_floats + quad * 4;
    float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (uint32_t i = 0; i < parts; i++) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            x[e] += from[(int64_t)i * 2 * p.keys * row_floats + e];
        }
    }
    const Strided& out = value != 0 ? a.grad_v : a.grad_k;
    T* const to = (T*)out.ptr + (int64_t)(bh / p.kv_heads) * out.stride[0] + key * out.stride[1] +
                  (int64_t)(bh % p.kv_heads) * out.stride[2];
    put4<T, VEC>(to, (int)quad * 4, (int)a.d, x[0], x[1], x[2], x[3]);
}

template <typename T, int NB, bool FEW, bool VEC>
hipError_t launch_query_grad(const GradLaunch& p, hipStream_t stream)
{
    constexpr ForwardShape kShape = grad_query_shape(sizeof(T), pitch_of(NB), FEW);
    constexpr int kOperands = grad_values_direct(sizeof(T), pitch_of(NB), FEW) ? 1 : 2;
    constexpr int kTiles = kShape.key_waves * kShape.stages * kOperands * kShape.keys * pitch_of(NB) * (int)sizeof(T);
    constexpr int kJoin = kShape.key_waves > 1 ? kShape.key_waves * NB * kBlock * kBlock * 4 : 0;
    constexpr int kBytes = kTiles > kJoin ? kTiles : kJoin;
    static_assert(kBytes <= 160 * 1024, "LDS of a CU");
    static std::atomic<uint32_t> done{0};
    const auto kernel = attention_query_grad_kernel<T, NB, FEW, VEC>;
    if (kBytes > 64 * 1024) {
        if (const hipError_t e = allow_dynamic_lds((const void*)kernel, kBytes, done); e != hipSuccess) {
            return e;
        }
    }
    hipLaunchKernelGGL(kernel, dim3((unsigned)launched(p.query_blocks)), dim3(kShape.threads()), kBytes, stream, p);
    return hipGetLastError();
}

template <typename T, int NB, int PASS, bool VEC>
hipError_t launch_key_grad(const GradLaunch& p, hipStream_t stream)
{
    constexpr int kPitch = pitch_of(NB);
    constexpr int kStages = key_grad_stages(sizeof(T)), kWaves = grad_key_waves(sizeof(T) == 4, NB);
    constexpr int kBytes = kStages * 2 * kBlock * kPitch * (int)sizeof(T) +
                           kWaves * kStages * 2 * kBlock * 4 +
                           (key_grad_values_in_lds(sizeof(T)) ? kWaves * kBlock * kPitch * (int)sizeof(T) : 0);
    static_assert(kBytes <= 160 * 1024, "LDS of a CU");
    static std::atomic<uint32_t> done{0};
    const auto kernel = attention_key_grad_kernel<T, NB, PASS, VEC>;
    if (kBytes > 64 * 1024) {
        if (const hipError_t e = allow_dynamic_lds((const void*)kernel, kBytes, done); e != hipSuccess) {
            return e;
        }
    }
    hipLaunchKernelGGL(kernel, dim3((unsigned)launched(p.key_blocks)), dim3(64 * kWaves), kBytes, stream, p);
    return hipGetLastError();
}

template <typename T, int NB, bool VEC>
hipError_t run_backward_shape(const GradLaunch& p, bool few, hipStream_t stream)
{
    hipError_t e = hipSuccess;
    if (p.query_blocks > 0) {
        if constexpr (sizeof(T) == 2 || NB > 2) {
            e = few ? launch_query_grad<T, NB, true, VEC>(p, stream) : launch_query_grad<T, NB, false, VEC>(p, stream);
        } else {
            e = few ? launch_query_grad<T, NB, true, VEC>(p, stream) : hipErrorInvalidValue;
        }
    }
    if (e == hipSuccess && p.key_blocks > 0) {
        if constexpr (NB <= 4) {
            e = launch_key_grad<T, NB, kBothGrads, VEC>(p, stream);
        } else {
            e = launch_key_grad<T, NB, kValueGrad, VEC>(p, stream);
            if (e == hipSuccess) {
                e = launch_key_grad<T, NB, kKeyGrad, VEC>(p, stream);
            }
        }
    }
    return e;
}

template <typename T, bool VEC>
hipError_t run_backward(const AttentionArgs& a, const GradPlan& plan, hipStream_t stream)
{
    // two rows of statistics are reached with 32-bit offsets in bytes
    if (!plan.fits || plan.stat_pitch > ((int64_t)1 << 28) || (a.scratch == nullptr && plan.stats > 0)) {
        return hipErrorInvalidValue;
    }
    GradLaunch p;
    p.a = a;
    p.group = make_fast_div((uint32_t)(a.heads / a.kv_heads));
    p.rows = (uint32_t)plan.rows;
    p.tiles = (uint32_t)plan.tiles;
    p.kv_heads = (uint32_t)a.kv_heads;
    p.keys = (uint32_t)plan.keys;
    p.key_tiles = (uint32_t)plan.key_tiles;
    p.sink_tiles = (uint32_t)plan.sink_tiles;
    p.sink_parts = (uint32_t)plan.sink_parts;
    p.parts = (uint32_t)plan.parts;
    p.query_blocks = (uint32_t)plan.query_blocks;
    p.key_blocks = (uint32_t)plan.key_blocks;
    p.stat_pitch = plan.stat_pitch;
    p.stats = a.scratch;
    p.sink_partials = a.scratch + plan.stats;
    p.partials = p.sink_partials + plan.sink_partials;
    hipError_t e = hipErrorInvalidValue;
    switch (blocks_of(a.d)) {
        case 8: e = run_backward_shape<T, 8, VEC>(p, plan.few_rows, stream); break;
        case 4: e = run_backward_shape<T, 4, VEC>(p, plan.few_rows, stream); break;
        case 3: e = run_backward_shape<T, 3, VEC>(p, plan.few_rows, stream); break;
        case 2: e = run_backward_shape<T, 2, VEC>(p, plan.few_rows, stream); break;
        default: e = run_backward_shape<T, 1, VEC>(p, plan.few_rows, stream); break;
    }
    if (e != hipSuccess) {
        return e;
    }
    if (plan.sink_joins + plan.joins > 0) {
        const uint32_t total = (uint32_t)(plan.sink_joins + plan.joins);
        hipLaunchKernelGGL((attention_grad_join_kernel<T, VEC>), dim3((total + 255) / 256), dim3(256), 0, stream, p,
                           (uint32_t)plan.sink_joins, (uint32_t)((a.d + 3) / 4), total);
    }
    return hipGetLastError();
}

}  // namespace att

// one translation unit a type
hipError_t run_attention_grad_f32(const AttentionArgs& a, const att::GradPlan& plan, bool vectors, hipStream_t stream);
hipError_t run_attention_grad_f16(const AttentionArgs& a, const att::GradPlan& plan, bool vectors, hipStream_t stream);
hipError_t run_attention_grad_bf16(const AttentionArgs& a, const att::GradPlan& plan, bool vectors, hipStream_t stream);

}  // namespace opscv
