// Rotary positions: pairs of features of every head turned by their token's angles, and the table of those angles.
//
//   (a, b) -> (a cos - b sin, b cos + a sin)
//
// Bound by memory: queries and keys are read once and written once.  The table is read instead of computing angles from
// positions, because a 32-bit product of a position and a frequency loses the angle's fraction far into a long context
// (position 100000: a hundredth of a radian); the table is computed in 64 bits and costs rot * 4 bytes a token against
// the heads' 4 d bytes each.  A thread owns a few features (16 bytes, or two halves of a pair group of 16 bytes each) of
// up to eight heads of one token, so that it reads its cosines and sines once for them.  Two prompts of 4096 tokens, 32 and
// 8 heads of 128, bf16: 34.4 us, 5.0 TB/s; one token of each of 64 sequences: 6.3, the launch.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "fast_div.hpp"
#include "launch_limits.hpp"
#include "opscv_tokens.h"
#include "token_elem.hpp"
#include "token_kernels.hpp"

namespace opscv {

using namespace tok;

namespace {

constexpr int kThreads = 256;

// Frequency of pair i: the angle of position 1.
double rotary_frequency(const RotaryTableArgs& a, int64_t i)
{
    double base = a.base;
    if (a.scaling == OPSCV_ROTARY_BASE) {
        base *= pow(a.factor, (double)a.rot / (double)(a.rot - 2));
    }
    const double f = pow(base, -2.0 * (double)i / (double)a.rot);
    if (a.scaling == OPSCV_ROTARY_LINEAR) {
        return f / a.factor;
    }
    if (a.scaling == OPSCV_ROTARY_BY_PARTS) {
        const double turns = (double)a.original_length * f / (2.0 * M_PI);
        const double keep = fmin(fmax((turns - 1.0) / (32.0 - 1.0), 0.0), 1.0);
        return f * keep + f / a.factor * (1.0 - keep);
    }
    return f;
}

constexpr int kMostPairs = 512;  // rot <= 1024

struct Frequencies {
    double f[kMostPairs];
};

__global__ __launch_bounds__(kThreads) void rotary_table_kernel(RotaryTableArgs a, Frequencies f)
{
    const int64_t half = a.rot / 2;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < a.positions * half;
         i += (int64_t)gridDim.x * kThreads) {
        const int64_t p = i / half, c = i % half;
        double s, k;
        sincos((double)p * f.f[c], &s, &k);
        float* const row = a.table + p * a.row_stride;
        row[c] = (float)(k * a.magnitude);
        row[half + c] = (float)(s * a.magnitude);
    }
}

struct RotaryPlan {
    RotaryArgs a;
    FastDiv units, groups, tokens;  // units of a head, groups of heads, tokens of a sequence
    uint32_t turned;                // units that turn; the others copy
    int wide_table;                 // the table's rows start on 16 bytes
    int streaming;
    uint32_t total;                 // threads with work
};

__device__ __forceinline__ int64_t whole_at(const Whole& w, int64_t i, int64_t j)
{
    const int64_t at = i * w.stride[0] + j * w.stride[1];
    return w.wide != 0 ? ((const int64_t*)w.ptr)[at] : (int64_t)((const int32_t*)w.ptr)[at];
}

// HEADS heads a thread, VEC features a vector.  A unit that turns is VEC / 2 interleaved pairs (one vector), or VEC pairs
// of features half a rotation apart (two vectors); a unit that copies is one vector.  Single elements (VEC 1) serve both
// orders as two vectors.
template <typename T, int VEC, int HEADS, bool INTERLEAVED>
__global__ __launch_bounds__(kThreads) void rotary_kernel(RotaryPlan p)
{
    constexpr int kPairs = INTERLEAVED ? VEC / 2 : VEC;
    const RotaryArgs& a = p.a;
    const uint32_t index = blockIdx.x * (uint32_t)kThreads + threadIdx.x;
    if (index >= p.total) {
        return;
    }
    const uint32_t rest = fast_div(index, p.units), unit = index - rest * p.units.div;
    const uint32_t token = fast_div(rest, p.groups), group = rest - token * p.groups.div;
    const uint32_t b = fast_div(token, p.tokens), t = token - b * p.tokens.div;
    const int half = (int)(a.rot / 2);
    const bool turns = unit < p.turned;
    float cosine[kPairs], sine[kPairs];
    int first, second = 0;  // features of the unit's vectors
    if (turns) {
        const int pair = (int)unit * kPairs;
        const bool neighbours = INTERLEAVED || (VEC == 1 && a.interleaved != 0);
        first = neighbours ? 2 * pair : pair;
        second = neighbours ? first + 1 : half + pair;
        const int64_t at = a.position.ptr != nullptr ? whole_at(a.position, b, t) : (int64_t)t;
        if (at >= 0 && at < a.positions) {
            const float* const row = a.table + at * a.table_stride + pair;
            bool read = false;
            if constexpr (kPairs % 4 == 0) {
                if (p.wide_table != 0) {
                    read = true;
#pragma unroll
                    for (int i = 0; i < kPairs; i += 4) {
                        const Pack<float, 4> x = *reinterpret_cast<const Pack<float, 4>*>(row + i);
                        const Pack<float, 4> y = *reinterpret_cast<const Pack<float, 4>*>(row + half + i);
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            cosine[i + e] = x.v[e];
                            sine[i + e] = y.v[e];
                        }
                    }
                }
            }
            if (!read) {
#pragma unroll
                for (int i = 0; i < kPairs; i++) {
                    cosine[i] = row[i];
                    sine[i] = row[half + i];
                }
            }
            if (a.inverse != 0) {
#pragma unroll
                for (int i = 0; i < kPairs; i++) {
                    sine[i] = -sine[i];
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < kPairs; i++) {
                cosine[i] = sine[i] = NAN;
            }
        }
    } else {
        first = (int)a.rot + (int)(unit - p.turned) * VEC;
    }
    const int total = (int)(a.heads + a.kv_heads), begin = (int)group * HEADS;
    float x[HEADS][VEC], y[HEADS][VEC];
    T* to[HEADS];
#pragma unroll
    for (int i = 0; i < HEADS; i++) {
        const int h = begin + i;
        if (h >= total) {
            break;
        }
        const bool query = h < (int)a.heads;
        const Strided& from = query ? a.query : a.key;
        const Strided& out = query ? a.query_out : a.key_out;
        const int64_t own = query ? h : h - (int)a.heads;
        const T* const src = (const T*)from.ptr + b * from.stride[0] + t * from.stride[1] + own * from.stride[2];
        to[i] = (T*)out.ptr + b * out.stride[0] + t * out.stride[1] + own * out.stride[2];
        load<T, VEC>(src + first, x[i]);
        if (!INTERLEAVED && turns) {
            load<T, VEC>(src + second, y[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < HEADS; i++) {
        if (begin + i >= total) {
            break;
        }
        if (turns) {
#pragma unroll
            for (int j = 0; j < kPairs; j++) {
                float& u = INTERLEAVED ? x[i][2 * j] : x[i][j];
                float& v = INTERLEAVED ? x[i][(2 * j + 1) % VEC] : y[i][j];
                const float s = u * cosine[j] - v * sine[j];
                v = v * cosine[j] + u * sine[j];
                u = s;
            }
            if (!INTERLEAVED) {
                store<T, VEC>(to[i] + second, y[i], p.streaming != 0);
            }
        }
        store<T, VEC>(to[i] + first, x[i], p.streaming != 0);
    }
}

template <typename T, int VEC, bool INTERLEAVED>
hipError_t run(const RotaryArgs& a, hipStream_t stream)
{
    const int64_t pairs = INTERLEAVED ? VEC / 2 : VEC;
    const int64_t turned = a.rot / 2 / pairs, units = turned + (a.d - a.rot) / VEC, heads = a.heads + a.kv_heads;
    const int64_t tokens = a.batch * a.tokens;
    // heads a thread takes one after the other: as many as still leave a wavefront for every SIMD (four a CU, 256 CUs)
    int each = 8;
    while (each > 1 && tokens * units * ((heads + each - 1) / each) < 256 * 4 * 64) {
        each /= 2;
    }
    // 31-bit indices and the division's range: large calls go sequence by sequence, then span by span of tokens
    const int64_t groups = (heads + each - 1) / each, per_token = units * groups, most = INT32_MAX / per_token;
    const int64_t span = a.tokens < most ? a.tokens : most;
    const int64_t sequences = span < a.tokens ? 1 : (most / a.tokens < a.batch ? most / a.tokens : a.batch);
    if (span < 1 || sequences < 1) {
        return hipErrorInvalidValue;
    }
    const auto shift = [](Strided& s, int64_t b, int64_t t) {
        if (s.ptr != nullptr) {
            s.ptr = (T*)s.ptr + b * s.stride[0] + t * s.stride[1];
        }
    };
    for (int64_t b = 0; b < a.batch; b += sequences) {
        for (int64_t t = 0; t < a.tokens; t += span) {
            RotaryPlan p;
            p.a = a;
            p.a.batch = a.batch - b < sequences ? a.batch - b : sequences;
            p.a.tokens = a.tokens - t < span ? a.tokens - t : span;
            for (Strided* s : {&p.a.query, &p.a.key, &p.a.query_out, &p.a.key_out}) {
                shift(*s, b, t);
            }
            if (a.position.ptr != nullptr) {
                p.a.position.ptr = (const char*)a.position.ptr +
                                   (b * a.position.stride[0] + t * a.position.stride[1]) * (a.position.wide != 0 ? 8 : 4);
            } else {
                p.a.table = a.table + t * a.table_stride;
                p.a.positions = a.positions - t;
            }
            p.units = make_fast_div((uint32_t)units);
            p.groups = make_fast_div((uint32_t)groups);
            p.tokens = make_fast_div((uint32_t)p.a.tokens);
            p.turned = (uint32_t)turned;
            p.streaming = tokens * heads * a.d * (int64_t)sizeof(T) >= kStreamBytes ? 1 : 0;
            p.wide_table = aligned(p.a.table, a.table_stride, 4, 16) && a.rot / 2 % 4 == 0 ? 1 : 0;
            p.total = (uint32_t)(p.a.batch * p.a.tokens * per_token);
            const dim3 grid((p.total + kThreads - 1) / kThreads);
            if (each == 8) {
                hipLaunchKernelGGL((rotary_kernel<T, VEC, 8, INTERLEAVED>), grid, dim3(kThreads), 0, stream, p);
            } else if (each == 4) {
                hipLaunchKernelGGL((rotary_kernel<T, VEC, 4, INTERLEAVED>), grid, dim3(kThreads), 0, stream, p);
            } else if (each == 2) {
                hipLaunchKernelGGL((rotary_kernel<T, VEC, 2, INTERLEAVED>), grid, dim3(kThreads), 0, stream, p);
            } else {
                hipLaunchKernelGGL((rotary_kernel<T, VEC, 1, INTERLEAVED>), grid, dim3(kThreads), 0, stream, p);
            }
        }
    }
    return hipGetLastError();
}

// the widest vector, of 16 bytes down to one element, that every head's parts are made of whole and aligned
template <typename T, bool INTERLEAVED, int VEC>
hipError_t run_widest(const RotaryArgs& a, hipStream_t stream)
{
    if constexpr (VEC > 1) {
        const int e = (int)sizeof(T), bytes = VEC * e;
        bool fits = (INTERLEAVED ? a.rot : a.rot / 2) % VEC == 0 && a.d % VEC == 0;
        for (const Strided* s : {&a.query, &a.key, &a.query_out, &a.key_out}) {
            fits = fits && aligned(s->ptr, s->stride[0], e, bytes) && aligned(s->ptr, s->stride[1], e, bytes) &&
                   aligned(s->ptr, s->stride[2], e, bytes);
        }
        return fits ? run<T, VEC, INTERLEAVED>(a, stream) : run_widest<T, INTERLEAVED, VEC / 2>(a, stream);
    } else {
        return run<T, 1, false>(a, stream);
    }
}

template <typename T>
hipError_t run_type(const RotaryArgs& a, hipStream_t stream)
{
    constexpr int kVec = 16 / (int)sizeof(T);
    return a.interleaved != 0 ? run_widest<T, true, kVec>(a, stream) : run_widest<T, false, kVec>(a, stream);
}

}  // namespace

hipError_t launch_rotary_table(const RotaryTableArgs& a, hipStream_t stream)
{
    if (a.table == nullptr || a.rot < 2 || a.rot / 2 > kMostPairs) {
        return hipErrorInvalidValue;
    }
    Frequencies f;
    for (int64_t i = 0; i < a.rot / 2; i++) {
        f.f[i] = rotary_frequency(a, i);
    }
    const int64_t blocks = (a.positions * (a.rot / 2) + kThreads - 1) / kThreads;
    hipLaunchKernelGGL(rotary_table_kernel, dim3((unsigned)(blocks < 65536 ? blocks : 65536)), dim3(kThreads), 0, stream, a,
                       f);
    return hipGetLastError();
}

hipError_t launch_rotary(const RotaryArgs& a, hipStream_t stream)
{
    if (a.rot < 2 || a.rot % 2 != 0 || a.rot > a.d || a.batch < 1 || a.tokens < 1) {
        return hipErrorInvalidValue;
    }
    // a launch takes one token at least, whose threads have 31-bit numbers: more heads than those reach go span by span, keys
    // as queries of their own
    constexpr int64_t kMostHeads = (int64_t)1 << 20;
    if (a.heads + a.kv_heads > kMostHeads) {
        const int64_t e = a.elem == (int)Elem::F32 ? 4 : 2;
        for (const bool keys : {false, true}) {
            const int64_t heads = keys ? a.kv_heads : a.heads;
            for (int64_t h = 0; h < heads; h += kMostHeads) {
                RotaryArgs s = a;
                s.heads = heads - h < kMostHeads ? heads - h : kMostHeads;
                s.kv_heads = 0;
                s.query = keys ? a.key : a.query;
                s.query_out = keys ? a.key_out : a.query_out;
                s.key = s.key_out = Strided();
                s.query.ptr = (char*)s.query.ptr + h * s.query.stride[2] * e;
                s.query_out.ptr = (char*)s.query_out.ptr + h * s.query_out.stride[2] * e;
                if (const hipError_t status = launch_rotary(s, stream); status != hipSuccess) {
                    return status;
                }
            }
        }
        return hipSuccess;
    }
    switch ((Elem)a.elem) {
        case Elem::F32: return run_type<float>(a, stream);
        case Elem::F16: return run_type<_Float16>(a, stream);
        default: return run_type<__bf16>(a, stream);
    }
}

}  // namespace opscv
