// Attention forward: softmax over the keys that a query sees, in one pass over them with a running maximum and sum.
//
// The rows of a workgroup are queries of all heads that share a key head (row r: query r / G of head r % G of the group),
// so a tile of keys and values in LDS serves them all, and their windows span few keys beyond one query's.  A wavefront
// has 32 rows, one per lane of a half:
//   S' = K Q'        (32 keys x 32 rows; K from LDS in "row" order, Q in registers)
//   m, l             running reference of a row (near its largest score) and sum of exp2(S c - m), c = scale log2 e; a
//                    row's keys are spread over two lanes, which exchange their maxima
//   O' = O' f + V' P (head features x 32 rows; V from LDS in "column" order, P are S's registers, rounded to the type)
// m, l and O stay in 32 bits; P is rounded to the type, because the matrix instructions take operands of one type: with it in
// two parts of 16 bits the second product would be done twice.  Against 64 bits that makes results 1.4 times as far off as
// the rounding of the result alone does (bf16 0.0023 for 0.0017, FLOAT16 0.00029 for 0.00021, on heads of 64 and 128).
//
// Why so: O' in registers, its columns being rows of the product, is scaled by one number a lane, and S' becomes the
// operand P without leaving the registers.  Bound by memory for single tokens (32 caches of up to 16384 tokens, window
// 4096, 32 heads of 128 on 8, bf16: 104 us, 5.2 TB/s), where the keys are shared out over wavefronts and workgroups.  Of
// prompts (8192 tokens, the same heads, window 1024: 165 to 172 us, 750 to 785 TFLOP/s) by the issue of vector instructions
// and products: of a SIMD's cycles 40 % go to vector instructions (a fifth of those to exponentials) and 35 % to products,
// and two wavefronts a SIMD cover each other only in part.  LDS is busy for 18 %: 1 KB for every product is half of the
// 256 bytes a cycle that it gives.  Wavefronts of 64 rows read half as much, but leave the registers of one a SIMD, whose
// loads and exponentials are then not behind the products (235 us).  Heads of 64 (8 images of 1369 tokens, 16 heads, window
// 513: 51 us) have twice the exponentials to a product: vector instructions 40 %, products 16 %, and for 29 % of the time a
// CU has no work (start and end, and 1408 workgroups are five and a half for each).
#pragma once

#include <atomic>
#include <type_traits>

#include "attention_plan.hpp"
#include "attention_tile.hpp"
#include "fast_div.hpp"
#include "kernels.hpp"

namespace opscv {
namespace att {

struct ForwardLaunch {
    AttentionArgs a;
    FastDiv group;    // heads that share a key head
    uint32_t rows;    // queries times those
    uint32_t tiles, splits, kv_heads;
    uint32_t blocks;  // workgroups with work
};

// O' += V' P for one block of features of a tile that some rows do not see whole and that holds values that are not finite.
// Such a value must not reach the rows that do not see it through its product with their weight 0: the finite values are
// multiplied as ever, and which kinds of the others each row gives weight to is counted by products of ones and zeros.
template <typename T, int PITCH, int SUBS>
static __device__ __forceinline__ acc_t add_seen_values(acc_t o, const Frag<T> (&w)[2 * SUBS], const T* tile, int block, int lane)
{
    // the finite ones, then +infinity, -infinity and NaN, one class at a time
#pragma unroll 1
    for (int kind = 0; kind < 4; kind++) {
        const int mask = kind == 0 ? 0x1f8 : kind == 1 ? 0x200 : kind == 2 ? 0x004 : 0x003;
        const float special = kind == 1 ? INFINITY : kind == 2 ? -INFINITY : NAN;
        lane = again(lane);  // the values are read again for every class: held through the loop they cost registers
        acc_t count = kind == 0 ? o : zeros();
#pragma unroll 1
        for (int n = 0; n < 2 * SUBS; n++) {
            Frag<T> f = Tile<T, PITCH>::column(tile, 16 * n, block, lane), has = w[0];
#pragma unroll
            for (int m = 1; m < 2 * SUBS; m++) {
                has = n == m ? w[m] : has;
            }
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float v = (float)f[e];
                f[e] = (T)(__builtin_amdgcn_classf(v, mask) ? (kind == 0 ? v : 1.0f) : 0.0f);
                has[e] = (kind == 0 || !((float)has[e] > 0.0f)) ? has[e] : (T)1.0f;
            }
            count = Mma<T>::mul(f, has, count);
        }
#pragma unroll
        for (int r = 0; r < 16; r++) {
            o[r] = kind == 0 ? count[r] : (count[r] > 0.0f ? o[r] + special : o[r]);
        }
    }
    return o;
}

// Two wavefronts a SIMD (256 registers each) where a row's share fits: 16-bit heads of up to 128 features, FLOAT of up to 64.
constexpr int waves_per_simd(int elem_bytes, int nb) { return elem_bytes * nb <= 8 ? 2 : 1; }

template <typename T, int NB, bool FEW, bool VEC>
__global__ __launch_bounds__(forward_shape(sizeof(T), pitch_of(NB), FEW).threads(), waves_per_simd(sizeof(T), NB)) void attention_kernel(
    ForwardLaunch p)
{
    constexpr int kPitch = pitch_of(NB);
    constexpr ForwardShape kShape = forward_shape(sizeof(T), kPitch, FEW);
    constexpr int kKeys = kShape.keys, kSubs = kKeys / kBlock, kGroupThreads = 64 * kShape.row_waves;
    typedef Tile<T, kPitch> L;
    extern __shared__ __align__(16) char lds[];

    const AttentionArgs& a = p.a;
    const uint32_t index = xcd_order(blockIdx.x, p.blocks);
    if (index >= p.blocks) {
        return;
    }
    const uint32_t tile = index % p.tiles, rest = index / p.tiles;
    const uint32_t split = rest % p.splits, bh = rest / p.splits;
    const uint32_t b = bh / p.kv_heads, kv_head = bh % p.kv_heads;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = (int)threadIdx.x & 63;
    const int h = lane >> 5, own = lane & 31;
    const int row_wave = wave % kShape.row_waves, key_wave = wave / kShape.row_waves;
    const int d = (int)a.d, left = (int)a.left, right = (int)a.right, sinks = (int)a.sinks;
    const Sequence seq = sequence_at(a, b);

    // the row of this lane; rows past the last repeat it and are not written
    const uint32_t row0 = tile * kShape.rows(), wave_row0 = row0 + row_wave * kBlock;
    const uint32_t row = min(wave_row0 + own, p.rows - 1);
    const int query = (int)fast_div(row, p.group), in_group = (int)(row - (uint32_t)query * p.group.div);
    const int head = (int)(kv_head * p.group.div) + in_group;
    const int pos = query < seq.q_len ? seq.first + query : INT32_MIN / 2;  // a padding query sees nothing

    // queries of the workgroup and of the wavefront
    const auto query_of = [&](uint32_t r) { return (int)fast_div(min(r, p.rows - 1), p.group); };
    const int block_low = query_of(row0), block_high = min(query_of(row0 + kShape.rows() - 1), seq.q_len - 1);
    KeyRange range = key_range<kKeys>(seq.first + block_low, seq.first + block_high, seq.kv_len, left, right, sinks);
    if (block_high < block_low) {
        range.tiles = 0;
    }
    const int wave_first = seq.first + query_of(wave_row0);
    const bool rows_whole = query_of(wave_row0 + kBlock - 1) < seq.q_len;
    const int wave_last = seq.first + min(query_of(wave_row0 + kBlock - 1), seq.q_len - 1);
    const int t_begin = (int)((int64_t)range.tiles * split / p.splits);
    const int t_end = (int)((int64_t)range.tiles * (split + 1) / p.splits);

    const T* const k_base = (const T*)a.k.ptr + (int64_t)b * a.k.stride[0] + (int64_t)kv_head * a.k.stride[2];
    const T* const v_base = (const T*)a.v.ptr + (int64_t)b * a.v.stride[0] + (int64_t)kv_head * a.v.stride[2];
    const uint32_t k_pitch = (uint32_t)(a.k.stride[1] * (int64_t)sizeof(T));
    const uint32_t v_pitch = (uint32_t)(a.v.stride[1] * (int64_t)sizeof(T));

    T* const ring = reinterpret_cast<T*>(lds) + (size_t)key_wave * (kShape.stages * 2 * kKeys * kPitch);
    const auto fetch = [&](int t, int buffer) {
        const int key0 = range.key_of(t, kKeys), rows = range.end_of(t) - key0;
        T* const k_tile = ring + buffer * (2 * kKeys * kPitch);
        const int thread = row_wave * 64 + again(lane);
        stage<T, kPitch, kKeys, kGroupThreads, VEC>(k_tile, at_bytes(k_base, (uint32_t)key0, k_pitch), thread, row_wave, d,
                                                    k_pitch, min(rows, kKeys));
        stage<T, kPitch, kKeys, kGroupThreads, VEC>(k_tile + kKeys * kPitch, at_bytes(v_base, (uint32_t)key0, v_pitch), thread,
                                                    row_wave, d, v_pitch, min(rows, kKeys));
    };
    constexpr int kInFlight = 2 * kKeys * L::kChunks / kGroupThreads;  // loads of one fetch, a wavefront

    const float c = a.scale * kLog2e;
    // Scores are taken relative to `base`, a score of the row: not its largest, but at most kSlack (in powers of two) below,
    // so that sums seldom have to be scaled again.  -infinity: the row has seen nothing.
    constexpr float kSlack = 8.0f;
    // Weights of FLOAT16 are 2^7 times as large, and so at most 2^15: those of 2^-21 of the largest still have all their bits,
    // for long rows of which a few keys take the most.
    constexpr float kGain = std::is_same<T, _Float16>::value ? 7.0f : 0.0f;
    float base, total;  // `total`: of this lane's keys only
    acc_t o[NB];

    int t = t_begin + key_wave, buffer = 0;
    if (t < t_end) {
        fetch(t, 0);
    }
    Frag<T> q[2 * NB];
    {
        const T* const src = (const T*)a.q.ptr + (int64_t)b * a.q.stride[0] + (int64_t)query * a.q.stride[1] +
                             (int64_t)head * a.q.stride[2];
#pragma unroll
        for (int i = 0; i < 2 * NB; i++) {
            q[i] = global_row<T, VEC>(src, 16 * i + 8 * h, d);
        }
    }
    wait_for_registers();
    bool careful = false;  // a second pass, for values that are not finite
    // whether all rows of the wavefront see all keys of a tile, and whether none of them sees any of 32 keys: wavefronts of a
    // workgroup meet once a tile, but each spends on it what its own rows see of it
    const auto whole = [&](int tile_index) {
        const int key0 = range.key_of(tile_index, kKeys);
        return rows_whole && key0 + kKeys <= range.end_of(tile_index) && key0 + kKeys - 1 <= wave_first + right &&
               (key0 >= wave_last - left || key0 + kKeys <= sinks);
    };
    const auto unseen = [&](int key0, int end) {
        return wave_first > wave_last || key0 >= end || key0 > wave_last + right ||
               (key0 + kBlock - 1 < wave_first - left && key0 >= sinks);
    };
    // SUBS times 32 keys of a tile; PART: some rows may not see some of them
    const auto attend = [&](auto part, auto subs, int key0, int end, const T* k_tile, const T* v_tile,
                            const Rows32<T, kPitch, NB>& k_rows, const Columns32<T, kPitch, NB>& v_columns) {
        constexpr bool PART = decltype(part)::value;
        constexpr int SUBS = decltype(subs)::value;
        acc_t s[SUBS];
#pragma unroll
        for (int j = 0; j < SUBS; j++) {
            s[j] = zeros();
#pragma unroll
            for (int i = 0; i < 2 * NB; i++) {
                s[j] = Mma<T>::mul(k_rows(k_tile, j * kBlock, i), q[i], s[j]);
            }
        }
        if constexpr (sizeof(T) == 2) {
            read_ahead<2 * NB * SUBS, 1, 4>();
        }
        if constexpr (PART) {
            const Sight see = sight(pos, key0 + 4 * h, end, left, right, sinks);
#pragma unroll
            for (int j = 0; j < SUBS; j++) {
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    s[j][r] = see.sees(j * kBlock + 8 * (r / 4) + r % 4) ? s[j][r] : -INFINITY;
                }
            }
        }
        float highs[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};  // four chains: one would wait for itself
#pragma unroll
        for (int j = 0; j < SUBS; j++) {
#pragma unroll
            for (int r = 0; r < 16; r += 2) {
                highs[r / 2 % 4] = largest(highs[r / 2 % 4], s[j][r], s[j][r + 1]);
            }
        }
        const float high = larger_of_halves(largest(highs[0], highs[1], largest(highs[2], highs[3], highs[3]))) * c;
        const bool grows = !(high <= base + kSlack);
        if (__any(grows)) {
            // each row by its own scores alone: what it sees beside it does not change its result
            const float now = grows ? __builtin_elementwise_maximum(base, high) : base;
            const float fade = base == -INFINITY ? 0.0f : exp2f(base - now);
            total *= fade;
#pragma unroll
            for (int i = 0; i < NB; i++) {
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    o[i][r] *= fade;
                }
            }
            base = now;
        }
        const float from = base == -INFINITY ? 0.0f : base - kGain;  // exp2(-inf - 0) = 0
        Frag<T> w[2 * SUBS];
        float sums[4] = {total, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int n = 0; n < 2 * SUBS; n++) {
            acc_t& x = s[n / 2];
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int r = 8 * (n % 2) + e;
                x[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[r], c, -from));
                sums[e % 4] += x[r];
            }
            w[n] = operand<T>(x, n % 2);
        }
        total = (sums[0] + sums[1]) + (sums[2] + sums[3]);
        if (PART && __builtin_expect(careful, 0)) {
#pragma unroll
            for (int i = 0; i < NB; i++) {
                o[i] = add_seen_values<T, kPitch, SUBS>(o[i], w, v_tile, i, again(lane));
            }
        } else {
#pragma unroll
            for (int n = 0; n < 2 * SUBS; n++) {
#pragma unroll
                for (int i = 0; i < NB; i++) {
                    o[i] = Mma<T>::mul(v_columns(v_tile, 16 * n, i), w[n], o[i]);
                }
            }
            if constexpr (sizeof(T) == 2) {
                read_ahead<2 * NB * SUBS, 2, 3>();
            }
        }
    };
    // one tile; PART: some rows may not see some keys
    const auto work = [&](auto part, const Rows32<T, kPitch, NB>& k_rows, const Columns32<T, kPitch, NB>& v_columns) {
        constexpr bool PART = decltype(part)::value;
        const bool more = t + kShape.key_waves < t_end;
        if constexpr (kShape.row_waves > 1) {
            // tile t is there for all wavefronts, and all have done with the tile before it, whose place is filled again
            // while they work on this one
            wait_for_loads<0>();
            barrier();
            if (kShape.stages == 2 && more) {
                fetch(t + 1, buffer ^ 1);
            }
        } else {
            // a ring of its own: the next tile is asked for before this one has come
            if (kShape.stages == 2 && more) {
                fetch(t + kShape.key_waves, buffer ^ 1);
                wait_for_loads<VEC ? kInFlight : 0>();
            } else {
                wait_for_loads<0>();
            }
        }
        const T* const k_tile = ring + buffer * (2 * kKeys * kPitch);
        const T* const v_tile = k_tile + kKeys * kPitch;
        const int key0 = range.key_of(t, kKeys), end = range.end_of(t);
        if constexpr (PART) {
#pragma unroll 1
            for (int j = 0; j < kKeys; j += kBlock) {
                if (!unseen(key0 + j, end)) {
                    attend(part, std::integral_constant<int, 1>(), key0 + j, end, k_tile + j * kPitch, v_tile + j * kPitch, k_rows,
                           v_columns);
                }
            }
        } else {
            attend(part, std::integral_constant<int, kSubs>(), key0, end, k_tile, v_tile, k_rows, v_columns);
        }
        if (kShape.stages == 1 && more) {
            if constexpr (kShape.row_waves > 1) {
                barrier();
            } else {
                wait_for_lds();  // what was read of the tile is back before its place is filled again
            }
            fetch(t + kShape.key_waves, 0);
        }
        buffer ^= kShape.stages - 1;
        t += kShape.key_waves;
    };
    while (true) {
        base = -INFINITY;
        total = 0.0f;
#pragma unroll
        for (int i = 0; i < NB; i++) {
            o[i] = zeros();
        }
        // two loops, so that the one for whole tiles has its registers to itself
        while (t < t_end) {
            {
                const Rows32<T, kPitch, NB> k_rows(again(lane));
                const Columns32<T, kPitch, NB> v_columns(again(lane));
                while (t < t_end && !whole(t)) {
                    work(std::true_type(), k_rows, v_columns);
                }
            }
            const Rows32<T, kPitch, NB> k_rows(again(lane));
            const Columns32<T, kPitch, NB> v_columns(again(lane));
            while (t < t_end && whole(t)) {
                work(std::false_type(), k_rows, v_columns);
            }
        }
        // Sums that are not finite may come from values that a row does not see, through their products with its weight 0
        // (0 times infinity is NaN): then all is done once more, and tiles that not all rows see whole with care.
        float check = 0.0f;
#pragma unroll
        for (int i = 0; i < NB; i++) {
#pragma unroll
            for (int r = 0; r < 16; r++) {
                check = __builtin_fmaf(o[i][r], 0.0f, check);
            }
        }
        const bool odd = !careful && check != 0.0f;
        if (!(kShape.row_waves > 1 ? __syncthreads_or(odd) : __any(odd))) {
            break;
        }
        careful = true;
        t = t_begin + key_wave;
        buffer = 0;
        if (t < t_end) {
            fetch(t, 0);
        }
    }
    total += other_half(total);
    base -= kGain;  // what the sums are relative to

    // join the wavefronts that shared the keys: every one leaves its sums in LDS, [feature][row], and takes a share of
    // the features for all of them
    constexpr int kJoin = kShape.key_waves;
    float* const sums = reinterpret_cast<float*>(lds);
    if constexpr (kJoin > 1) {
        constexpr int kWaveFloats = (NB * kBlock + 2) * kBlock;
        __syncthreads();
        float* const mine = sums + wave * kWaveFloats;
        if (h == 0) {
            mine[own] = base;
            mine[kBlock + own] = total;
        }
#pragma unroll
        for (int i = 0; i < NB; i++) {
#pragma unroll
            for (int r = 0; r < 16; r++) {
                mine[(2 + i * kBlock + 8 * (r / 4) + 4 * h + r % 4) * kBlock + own] = o[i][r];
            }
        }
        __syncthreads();
        float high = -INFINITY;
#pragma unroll
        for (int w = 0; w < kJoin; w++) {
            high = fmaxf(high, sums[w * kWaveFloats + own]);
        }
        const float from = high == -INFINITY ? 0.0f : high;
        float share[kJoin];
        total = 0.0f;
        base = high;
#pragma unroll
        for (int w = 0; w < kJoin; w++) {
            share[w] = exp2f(sums[w * kWaveFloats + own] - from);
            total += share[w] * sums[w * kWaveFloats + kBlock + own];
        }
#pragma unroll
        for (int i = 0; i < NB; i++) {
            if (i % kJoin == wave) {
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    float x = 0.0f;
#pragma unroll
                    for (int w = 0; w < kJoin; w++) {
                        x += share[w] * sums[w * kWaveFloats + (2 + i * kBlock + 8 * (r / 4) + 4 * h + r % 4) * kBlock + own];
                    }
                    o[i][r] = x;
                }
            }
        }
    }

    if (wave_row0 + own >= p.rows) {
        return;
    }
    const bool first_wave = kJoin == 1 || wave == 0;
    if (p.splits > 1) {
        float* const part = a.scratch + (((int64_t)bh * p.splits + split) * p.rows + row) * partial_floats(d);
        if (first_wave && h == 0) {
            part[0] = base;
            part[1] = total;
        }
#pragma unroll
        for (int i = 0; i < NB; i++) {
            if (kJoin == 1 || i % kJoin == wave) {
#pragma unroll
                for (int r = 0; r < 16; r += 4) {
                    const int at = i * kBlock + 8 * (r / 4) + 4 * h;
                    if (at < d) {  // rows of partial results have room for whole groups of four
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            part[2 + at + e] = o[i][r + e];
                        }
                    }
                }
            }
        }
        return;
    }
    const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
    if (first_wave && h == 0 && a.lse.ptr != nullptr) {
        ((float*)a.lse.ptr)[(int64_t)b * a.lse.stride[0] + (int64_t)head * a.lse.stride[1] +
                            (int64_t)query * a.lse.stride[2]] =
            total == 0.0f ? -INFINITY : (base + log2f(total)) * kLn2;
    }
    T* const out = (T*)a.out.ptr + (int64_t)b * a.out.stride[0] + (int64_t)query * a.out.stride[1] +
                   (int64_t)head * a.out.stride[2];
#pragma unroll
    for (int i = 0; i < NB; i++) {
        if (kJoin == 1 || i % kJoin == wave) {
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                put4<T, VEC>(out, i * kBlock + 8 * (r / 4) + 4 * h, d, o[i][r] * inverse, o[i][r + 1] * inverse,
                             o[i][r + 2] * inverse, o[i][r + 3] * inverse);
            }
        }
    }
}

// Joins the parts of a split: four features of a row a thread.
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void attention_join_kernel(ForwardLaunch p, uint32_t quads, uint32_t total)
{
    const AttentionArgs& a = p.a;
    const uint32_t index = blockIdx.x * 256u + threadIdx.x;
    if (index >= total) {
        return;
    }
    const uint32_t quad = index % quads, rest = index / quads;
    const uint32_t row = rest % p.rows, bh = rest / p.rows;
    const uint32_t b = bh / p.kv_heads, kv_head = bh % p.kv_heads;
    const int d = (int)a.d;
    const int64_t step = partial_floats(d) * (int64_t)p.rows;
    const float* const part = a.scratch + ((int64_t)bh * p.splits * p.rows + row) * partial_floats(d);
    float high = -INFINITY;
#pragma unroll 8
    for (uint32_t s = 0; s < p.splits; s++) {
        high = fmaxf(high, part[s * step]);
    }
    const float base = high == -INFINITY ? 0.0f : high;
    float sum = 0.0f, x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 8
    for (uint32_t s = 0; s < p.splits; s++) {
        const float* const at = part + s * step;
        const float share = exp2f(at[0] - base);
        sum += share * at[1];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            x[e] += share * at[2 + 4 * quad + e];
        }
    }
    const uint32_t query = fast_div(row, p.group), head = kv_head * p.group.div + (row - query * p.group.div);
    const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
    if (quad == 0 && a.lse.ptr != nullptr) {
        ((float*)a.lse.ptr)[(int64_t)b * a.lse.stride[0] + (int64_t)head * a.lse.stride[1] +
                            (int64_t)query * a.lse.stride[2]] =
            sum == 0.0f ? -INFINITY : (high + log2f(sum)) * kLn2;
    }
    T* const out = (T*)a.out.ptr + (int64_t)b * a.out.stride[0] + (int64_t)query * a.out.stride[1] +
                   (int64_t)head * a.out.stride[2];
    put4<T, VEC>(out, (int)(4 * quad), d, x[0] * inverse, x[1] * inverse, x[2] * inverse, x[3] * inverse);
}

template <typename T, int NB, bool FEW, bool VEC>
hipError_t run_forward_shape(const ForwardLaunch& p, hipStream_t stream)
{
    constexpr ForwardShape kShape = forward_shape(sizeof(T), pitch_of(NB), FEW);
    constexpr int kTiles = kShape.key_waves * kShape.stages * 2 * kShape.keys * pitch_of(NB) * (int)sizeof(T);
    constexpr int kJoin = kShape.key_waves > 1 ? kShape.key_waves * (NB * kBlock + 2) * kBlock * 4 : 0;
    constexpr int kBytes = kTiles > kJoin ? kTiles : kJoin;
    static_assert(kBytes <= 160 * 1024, "LDS of a CU");
    static std::atomic<uint32_t> done{0};
    const auto kernel = attention_kernel<T, NB, FEW, VEC>;
    if (kBytes > 64 * 1024) {
        if (const hipError_t e = allow_dynamic_lds((const void*)kernel, kBytes, done); e != hipSuccess) {
            return e;
        }
    }
    hipLaunchKernelGGL(kernel, dim3((unsigned)launched(p.blocks)), dim3(kShape.threads()), kBytes, stream, p);
    return hipGetLastError();
}

template <typename T, bool VEC>
hipError_t run_forward(const AttentionArgs& a, const ForwardPlan& plan, hipStream_t stream)
{
    if (!plan.fits || (plan.splits > 1 && a.scratch == nullptr)) {
        return hipErrorInvalidValue;
    }
    ForwardLaunch p;
    p.a = a;
    p.group = make_fast_div((uint32_t)(a.heads / a.kv_heads));
    p.rows = (uint32_t)plan.rows;
    p.tiles = (uint32_t)plan.tiles;
    p.splits = (uint32_t)plan.splits;
    p.kv_heads = (uint32_t)a.kv_heads;
    p.blocks = (uint32_t)plan.blocks;
    hipError_t e = hipErrorInvalidValue;
    const auto pick = [&](auto few) {
        constexpr bool kFew = decltype(few)::value;
        switch (blocks_of(a.d)) {
            case 8: e = run_forward_shape<T, 8, kFew, VEC>(p, stream); break;
            case 4: e = run_forward_shape<T, 4, kFew, VEC>(p, stream); break;
            case 3: e = run_forward_shape<T, 3, kFew, VEC>(p, stream); break;
            case 2: e = run_forward_shape<T, 2, kFew, VEC>(p, stream); break;
            default: e = run_forward_shape<T, 1, kFew, VEC>(p, stream); break;
        }
    };
    if (plan.few_rows) {
        pick(std::true_type());
    } else if constexpr (sizeof(T) == 2) {
        pick(std::false_type());
    }
    if (e != hipSuccess || plan.splits == 1) {
        return e;
    }
    hipLaunchKernelGGL((attention_join_kernel<T, VEC>), dim3((unsigned)((plan.joins + 255) / 256)), dim3(256), 0, stream, p,
                       (uint32_t)((a.d + 3) / 4), (uint32_t)plan.joins);
    return hipGetLastError();
}

}  // namespace att

// one translation unit a type
hipError_t run_attention_f32(const AttentionArgs& a, const att::ForwardPlan& plan, bool vectors, hipStream_t stream);
hipError_t run_attention_f16(const AttentionArgs& a, const att::ForwardPlan& plan, bool vectors, hipStream_t stream);
hipError_t run_attention_bf16(const AttentionArgs& a, const att::ForwardPlan& plan, bool vectors, hipStream_t stream);

}  // namespace opscv
