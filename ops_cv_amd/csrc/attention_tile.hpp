// Tiles of attention on the matrix cores: fragments, staging through LDS, and what a query sees.
//
// Every product is made of 32 x 32 results over 16 terms: result[m][n] += sum over slots of A[m][slot] B[slot][n].  Lane l
// holds row m = l % 32 of A (or column n of B) and the eight slots (h, 0..7) of its half h = l / 32; of the result it
// holds column n = l % 32 and rows m = 8 (r / 4) + 4 h + r % 4 for r = 0..15.  16-bit types take one instruction
// (32x32x16); FLOAT takes eight of 32x32x2, one for each slot of a lane, so the three types share all code.
//
// Which term a slot stands for is free as long as A and B agree.  Two orders are used: "row": slot (h, e) is term
// 8 h + e, for operands whose terms lie side by side in memory; "column": slot (h, e) is term 4 h + e % 4 + 8 (e / 4),
// the order in which a result of the instruction holds its rows.  So eight registers of one product's result are, rounded
// to the type, the B operand of the next product as they stand, and nothing moves between lanes.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>
#include <utility>

#include "acl_types.hpp"

namespace opscv {
namespace att {

typedef float acc_t __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) void* lds_ptr_t;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr uint32_t kOutside = 0x80000000u;  // an offset past every buffer: the load returns zeros
constexpr int kBufferFlags = 0x00027000;    // raw buffer, 32-bit elements

template <typename T>
struct Mma;

template <>
struct Mma<__bf16> {
    typedef bf16x8 Frag;
    static __device__ __forceinline__ acc_t mul(Frag a, Frag b, acc_t c)
    {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
};

template <>
struct Mma<_Float16> {
    typedef f16x8 Frag;
    static __device__ __forceinline__ acc_t mul(Frag a, Frag b, acc_t c)
    {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
};

template <>
struct Mma<float> {
    typedef f32x8 Frag;
    static __device__ __forceinline__ acc_t mul(Frag a, Frag b, acc_t c)
    {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
        }
        return c;
    }
};

template <typename T>
using Frag = typename Mma<T>::Frag;

static __device__ __forceinline__ acc_t zeros()
{
    acc_t z;
#pragma unroll
    for (int i = 0; i < 16; i++) {
        z[i] = 0.0f;
    }
    return z;
}

// registers 8 g .. 8 g + 7 of a result as an operand, rounded to the type (to nearest: the products that follow take the
// type's numbers, and their sums stay in 32 bits)
template <typename T>
static __device__ __forceinline__ Frag<T> operand(const acc_t& x, int g)
{
    Frag<T> f;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        f[e] = (T)x[8 * g + e];
    }
    return f;
}

// x of the other half's lane with the same l % 32
static __device__ __forceinline__ float other_half(float x)
{
    const uint32_t u = __float_as_uint(x);
    const auto both = __builtin_amdgcn_permlane32_swap(u, u, false, false);  // halves: lower twice, upper twice
    return __uint_as_float((threadIdx.x & 32) != 0 ? both[0] : both[1]);
}

// the larger of x and of the other half's lane, for both
static __device__ __forceinline__ float larger_of_halves(float x)
{
    const uint32_t u = __float_as_uint(x);
    const auto both = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return __builtin_elementwise_maximum(__uint_as_float(both[0]), __uint_as_float(both[1]));
}

// the largest of three, NaN where any is
static __device__ __forceinline__ float largest(float a, float b, float c)
{
    return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c);
}

// ---------------------------------------------------------------------------------------------------- loads into LDS

typedef int rsrc_t __attribute__((ext_vector_type(4)));

// Descriptor of `bytes` bytes from an address that the wavefront shares.
static __device__ __forceinline__ rsrc_t buffer(const void* base, uint32_t bytes)
{
    const uint64_t at = (uint64_t)base;
    rsrc_t r;
    r[0] = __builtin_amdgcn_readfirstlane((int)(uint32_t)at);
    r[1] = __builtin_amdgcn_readfirstlane((int)(uint32_t)(at >> 32));  // addresses have 48 bits: no stride, no swizzle
    r[2] = __builtin_amdgcn_readfirstlane((int)bytes);
    r[3] = kBufferFlags;
    // the loads that use it are not instructions whose hazards the compiler looks after: five wait states between a vector
    // instruction that writes a scalar register and a load that reads it
    __asm__ volatile("s_nop 4" : "+s"(r));
    return r;
}

// BYTES bytes a lane from offset `off` of a buffer into LDS, the wavefront's first at place dst + AT and the lanes in order; lanes
// whose offset is out of range write zeros.  It has no result for the compiler to wait for, and as an instruction that the
// compiler does not look into it makes it wait for nothing: with the builtin, every transposed read of LDS is preceded by
// a wait for all loads under way (a prompt of 8192 tokens took 203 us so where it took 193 without, before later steps).  The
// caller waits.
template <int BYTES, int AT>
static __device__ __forceinline__ void load_to_lds(rsrc_t rsrc, uint32_t dst, uint32_t off)
{
    if constexpr (BYTES == 16) {
        __asm__ volatile("s_add_u32 m0, %0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(dst), "v"(off),
                         "s"(rsrc), "n"(AT)
                         : "memory", "m0", "scc");
    } else {
        __asm__ volatile("s_add_u32 m0, %0, %3\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(dst), "v"(off),
                         "s"(rsrc), "n"(AT)
                         : "memory", "m0", "scc");
    }
}

// where a place in LDS begins, for load_to_lds
static __device__ __forceinline__ uint32_t lds_place(const void* at)
{
    return (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(uintptr_t)(lds_ptr_t)const_cast<void*>(at));
}

// Order of the instructions around it: AHEAD products' reads of LDS (READS each) first, then a product and the reads of
// the one AHEAD behind it in turn.  Left alone, the compiler reads, waits and multiplies in turn.
template <int PRODUCTS, int READS, int AHEAD>
static __device__ __forceinline__ void read_ahead()
{
    constexpr int kAhead = AHEAD < PRODUCTS ? AHEAD : PRODUCTS;
    __builtin_amdgcn_sched_group_barrier(0x100, kAhead * READS, 0);
#pragma unroll
    for (int i = 0; i < PRODUCTS - kAhead; i++) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, kAhead, 0);
}

// ---------------------------------------------------------------------------------------------------------------- LDS
//
// A tile is rows of PITCH elements (a power of two, the head size rounded up) in 16-byte chunks; chunk c of row r lies at
// place c ^ swizzle(r).  The swizzle spreads both ways of reading over the 64 banks: whole rows by neighbouring lanes
// (16 rows of one chunk number fall on 16 places of a 256-byte span) and columns (four neighbouring rows of the same 64
// bytes fall on the four quarters of such a span).

template <typename T, int PITCH>
struct Tile {
    static constexpr int kPerChunk = 16 / (int)sizeof(T);
    static constexpr int kChunks = PITCH / kPerChunk;  // of a row: 8 or more
    static_assert(kChunks >= 8 && (kChunks & (kChunks - 1)) == 0, "rows of a power of two, 128 bytes or more");

    static __device__ __forceinline__ int swizzle(int row)
    {
        return kChunks == 8 ? ((((row >> 1) & 1) << 2) | ((row >> 2) & 3)) : (((row & 3) << 2) | ((row >> 2) & 3));
    }

    static constexpr int bytes(int rows) { return rows * PITCH * (int)sizeof(T); }

    // element 32 block + l % 32 of rows base + 4 h + {0..3, 8..11}: an operand in "column" order, m or n = the element
    static __device__ __forceinline__ Frag<T> column(const T* tile, int base, int block, int lane)
    {
        const int h = lane >> 5;
        if constexpr (sizeof(T) == 2) {
            // Sixteen lanes together read four rows of sixteen elements, eight bytes a lane (row i / 4, elements
            // 4 (i % 4) .. + 3), and the instruction hands lane i column i of them.
            const int i = lane & 15;
            const int r = base + 4 * h + (i >> 2);
            const int c = 4 * block + ((lane >> 4) & 1) * 2 + ((i & 3) >> 1);
            const T* const a = tile + r * PITCH + ((c ^ swizzle(r)) * 8) + (i & 1) * 4;
            const T* const b = tile + (r + 8) * PITCH + ((c ^ swizzle(r + 8)) * 8) + (i & 1) * 4;
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(a));
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(b));
            s16x8 both;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                both[e] = lo[e];
                both[4 + e] = hi[e];
            }
            return __builtin_bit_cast(Frag<T>, both);
        } else {
            const int d = 32 * block + (lane & 31);
            Frag<T> f;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int r = base + 4 * h + (e & 3) + 8 * (e >> 2);
                f[e] = tile[r * PITCH + (((d >> 2) ^ swizzle(r)) * 4) + (d & 3)];
            }
            return f;
        }
    }
};

// Where a lane reads whole rows (row base + l % 32) or columns of a tile: places that a loop computes once.  NB blocks of
// 32 elements.  FLOAT has eight places a column and computes them as it goes: its products take sixteen times as many cycles.
template <typename T, int PITCH, int NB>
struct Rows32 {
    int at[2 * NB];
    __device__ __forceinline__ explicit Rows32(int lane)
    {
        const int r = lane & 31, h = lane >> 5;
#pragma unroll
        for (int i = 0; i < 2 * NB; i++) {
            constexpr int kPer8 = 8 / Tile<T, PITCH>::kPerChunk;  // chunks of eight elements: 1, FLOAT 2
            at[i] = r * PITCH * (int)sizeof(T) + (((kPer8 * (2 * i + h)) ^ Tile<T, PITCH>::swizzle(r)) * 16);
        }
    }
    // operand i (elements 16 i .. 16 i + 15) of rows base + l % 32, base a multiple of 32
    __device__ __forceinline__ Frag<T> operator()(const T* tile, int base, int i) const
    {
        const char* const from = reinterpret_cast<const char*>(tile) + at[i] + base * PITCH * (int)sizeof(T);
        if constexpr (sizeof(T) == 2) {
            return *reinterpret_cast<const Frag<T>*>(from);
        } else {
            typedef float f32x4 __attribute__((ext_vector_type(4)));
            const f32x4 a = *reinterpret_cast<const f32x4*>(from);
            const f32x4 b = *reinterpret_cast<const f32x4*>(reinterpret_cast<const char*>(tile) + (at[i] ^ 16) +
                                                            base * PITCH * (int)sizeof(T));
            Frag<T> f;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                f[e] = a[e];
                f[4 + e] = b[e];
            }
            return f;
        }
    }
};

template <typename T, int PITCH, int NB>
struct Columns32 {
    int at[sizeof(T) == 2 ? 2 * NB : 1];
    __device__ __forceinline__ explicit Columns32(int lane)
    {
        if constexpr (sizeof(T) == 2) {
            const int i = lane & 15, r = 4 * (lane >> 5) + (i >> 2);
#pragma unroll
            for (int n = 0; n < NB; n++) {
                const int c = 4 * n + ((lane >> 4) & 1) * 2 + ((i & 3) >> 1);
                at[2 * n] = r * PITCH * 2 + ((c ^ Tile<T, PITCH>::swizzle(r)) * 16) + (i & 1) * 8;
                at[2 * n + 1] = (r + 8) * PITCH * 2 + ((c ^ Tile<T, PITCH>::swizzle(r + 8)) * 16) + (i & 1) * 8;
            }
        } else {
            at[0] = lane;
        }
    }
    // block n of the sixteen rows from base on, a multiple of 16
    __device__ __forceinline__ Frag<T> operator()(const T* tile, int base, int n) const
    {
        if constexpr (sizeof(T) == 2) {
            typedef __attribute__((address_space(3))) s16x4* place;
            const char* const from = reinterpret_cast<const char*>(tile) + base * PITCH * 2;
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((place)(from + at[2 * n]));
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((place)(from + at[2 * n + 1]));
            s16x8 both;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                both[e] = lo[e];
                both[4 + e] = hi[e];
            }
            return __builtin_bit_cast(Frag<T>, both);
        } else {
            return Tile<T, PITCH>::column(tile, base, n, at[0]);
        }
    }
};

// the address `n` rows of `pitch` bytes behind another
template <typename T>
static __device__ __forceinline__ const T* at_bytes(const T* base, uint32_t n, uint32_t pitch)
{
    return reinterpret_cast<const T*>(reinterpret_cast<const char*>(base) + (uint64_t)n * pitch);
}

// the loads of stage(): chunk `place` (swizzled) of rows r0, r0 + STEP, ..., BYTES apart in LDS
template <typename T, int PITCH, int STEP, int BYTES, int... I>
static __device__ __forceinline__ void stage_chunks(rsrc_t rsrc, uint32_t dst, int r0, int place, int d, uint32_t pitch,
                                                    uint32_t row0, std::integer_sequence<int, I...>)
{
    typedef Tile<T, PITCH> L;
    const auto one = [&](auto i) {
        constexpr int kI = decltype(i)::value;
        const int c = place ^ L::swizzle(r0 + kI * STEP);
        const uint32_t off = (c * L::kPerChunk >= d ? kOutside : row0 + (uint32_t)c * 16u) + (uint32_t)(kI * STEP) * pitch;
        load_to_lds<16, kI * BYTES>(rsrc, dst, off);
    };
    (one(std::integral_constant<int, I>()), ...);
}

// Copies ROWS rows into a tile by THREADS threads (thread `gt` of them, in their wavefront `wave`): row r from base + r * pitch
// bytes, rows from `rows` (one or more) on and elements from d on as zeros.  VEC: 16-byte loads that write LDS themselves
// (asynchronous: the caller waits), pitch at least the row's own bytes; else element by element.
template <typename T, int PITCH, int ROWS, int THREADS, bool VEC>
static __device__ __forceinline__ void stage(T* tile, const T* base, int gt, int wave, int d, uint32_t pitch, int rows)
{
    typedef Tile<T, PITCH> L;
    constexpr int kChunks = ROWS * L::kChunks;
    constexpr int kStep = THREADS / L::kChunks;  // rows between a thread's chunks
    static_assert(kChunks % THREADS == 0 && THREADS % L::kChunks == 0, "every thread copies as many chunks");
    const int r0 = gt / L::kChunks, place = gt % L::kChunks;
    if constexpr (VEC) {
        // What lies behind the last row's last element is out of the buffer's range, and such loads return zeros; so do
        // chunks behind the head's end, by an offset that no range holds.
        const uint32_t bytes = (uint32_t)(rows - 1) * pitch + (uint32_t)d * (uint32_t)sizeof(T);
        const rsrc_t rsrc = buffer(base, bytes);
        const uint32_t row0 = (uint32_t)r0 * pitch;
        const uint32_t dst = lds_place(tile + wave * 64 * L::kPerChunk);  // the wavefront's; lanes follow in order
        stage_chunks<T, PITCH, kStep, THREADS * 16>(rsrc, dst, r0, place, d, pitch, row0,
                                                    std::make_integer_sequence<int, kChunks / THREADS>());
    } else {
#pragma unroll 1
        for (int i = 0; i < kChunks / THREADS; i++) {
            const int r = r0 + i * kStep, c = place ^ L::swizzle(r);
            alignas(16) T x[L::kPerChunk];
#pragma unroll
            for (int e = 0; e < L::kPerChunk; e++) {
                const int el = c * L::kPerChunk + e;
                x[e] = (r >= rows || el >= d) ? (T)0.0f : at_bytes(base, (uint32_t)r, pitch)[el];
            }
            typedef float f32x4 __attribute__((ext_vector_type(4)));
            *reinterpret_cast<f32x4*>(tile + (i * THREADS + gt) * L::kPerChunk) = *reinterpret_cast<const f32x4*>(x);
        }
    }
}

// Eight elements from element `first` of a row on, zeros from element d on.
template <typename T, bool VEC>
static __device__ __forceinline__ Frag<T> global_row(const T* row, int first, int d)
{
    Frag<T> f;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        f[e] = (T)0.0f;
    }
    if constexpr (VEC) {
        // d is a multiple of the 16-byte vector: four elements of FLOAT, eight of the others
        if constexpr (sizeof(T) == 2) {
            if (first < d) {
                f = *reinterpret_cast<const Frag<T>*>(row + first);
            }
        } else {
            typedef float f32x4 __attribute__((ext_vector_type(4)));
#pragma unroll
            for (int i = 0; i < 2; i++) {
                if (first + 4 * i < d) {
                    const f32x4 x = *reinterpret_cast<const f32x4*>(row + first + 4 * i);
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        f[4 * i + e] = x[e];
                    }
                }
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            if (first + e < d) {
                f[e] = row[first + e];
            }
        }
    }
    return f;
}

// Writes four neighbouring elements of a row from `first` on, none from element d on.
template <typename T, bool VEC>
static __device__ __forceinline__ void put4(T* row, int first, int d, float a, float b, float c, float e)
{
    float x[4] = {a, b, c, e};
    // products are rounded to 32 bits before they are rounded to the type: without this the compiler fuses the two for
    // FLOAT16 in one of the ways below and not in the other, and results would depend on the strides
#pragma unroll
    for (int i = 0; i < 4; i++) {
        __asm__("" : "+v"(x[i]));
    }
    if constexpr (VEC) {
        if (first < d) {  // d is a multiple of four
            struct alignas(4 * sizeof(T)) Four {
                T v[4];
            } k;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                k.v[i] = (T)x[i];
            }
            *reinterpret_cast<Four*>(row + first) = k;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (first + i < d) {
                row[first + i] = (T)x[i];
            }
        }
    }
}

// Waits until at most N loads to memory or LDS are under way, or none of LDS; nothing that follows is moved before it.
template <int N>
static __device__ __forceinline__ void wait_for_loads()
{
    __asm__ volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// Waits for all loads, in a way that the compiler knows: it has then no reason to wait for registers loaded before a loop
// inside the loop, where such a wait would be one for the loop's own loads.
static __device__ __forceinline__ void wait_for_registers() { __builtin_amdgcn_s_waitcnt(0x0f70); }
static __device__ __forceinline__ void wait_for_lds() { __asm__ volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// The same number, which the compiler takes for another: what is computed from it inside a loop is computed there, in a few
// instructions, and holds no registers through the rest of the loop.
static __device__ __forceinline__ int again(int x)
{
    __asm__ volatile("" : "+v"(x));
    return x;
}

// ---------------------------------------------------------------------------------------------------------- visibility

static __device__ __forceinline__ int length_at(const Whole& w, int64_t b, int64_t most)
{
    if (w.ptr == nullptr) {
        return (int)most;
    }
    const int64_t v = w.wide != 0 ? ((const int64_t*)w.ptr)[b * w.stride[0]] : (int64_t)((const int32_t*)w.ptr)[b * w.stride[0]];
    return (int)(v < 0 ? 0 : (v > most ? most : v));
}

// One sequence: its lengths and the position of query 0.
struct Sequence {
    int q_len, kv_len, first;
};

static __device__ __forceinline__ Sequence sequence_at(const AttentionArgs& a, int64_t b)
{
    Sequence s;
    s.q_len = length_at(a.q_lengths, b, a.tokens);
    s.kv_len = length_at(a.kv_lengths, b, a.kv_tokens);
    s.first = s.kv_len - s.q_len;
    return s;
}

// What a query at position p sees of 64 keys from key0 on, of which those before `end` count: key key0 + n for
// n <= last and (n >= first or n < sinks).
struct Sight {
    int first, last, sinks;
    __device__ __forceinline__ bool sees(int n) const { return (n <= last) & ((n >= first) | (n < sinks)); }
};

static __device__ __forceinline__ Sight sight(int p, int key0, int end, int left, int right, int sinks)
{
    return Sight{p - left - key0, min(p + right, end - 1) - key0, sinks - key0};
}

// Barrier of the workgroup that waits for the wavefront's LDS operations, but not for loads under way into LDS, as
// __syncthreads would.
static __device__ __forceinline__ void barrier() { __asm__ volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Workgroups go round the eight XCDs; this gives every XCD a run of neighbouring numbers, so that the tiles of rows that
// read the same keys share an L2.
static __device__ __forceinline__ uint32_t xcd_order(uint32_t index, uint32_t count)
{
    const uint32_t each = (count + 7) / 8;
    return (index & 7u) * each + (index >> 3);
}

// Keys that a range of rows sees, as tiles: the first `sink_tiles` start at key 0, the others at `first`.  Tiles hold
// nothing between the sinks and the window: what lies there is seen by none of the rows, and may be anything.
struct KeyRange {
    int first, end;  // window
    int sink_end;    // sinks in front of it
    int sink_tiles, tiles;

    __device__ __forceinline__ int key_of(int t, int keys) const
    {
        return t < sink_tiles ? t * keys : first + (t - sink_tiles) * keys;
    }
    __device__ __forceinline__ int end_of(int t) const { return t < sink_tiles ? sink_end : end; }
};

template <int KEYS>
static __device__ __forceinline__ KeyRange key_range(int p_low, int p_high, int kv_len, int left, int right, int sinks)
{
    KeyRange k;
    k.end = min(max(p_high + right + 1, 0), kv_len);
    k.first = min(max(p_low - left, 0), k.end);
    k.sink_end = min(sinks, k.first);
    if (k.sink_end == k.first) {  // the window follows the sinks: one run of tiles
        k.sink_end = k.first = 0;
    }
    k.sink_tiles = (k.sink_end + KEYS - 1) / KEYS;
    k.tiles = k.sink_tiles + (k.end - k.first + KEYS - 1) / KEYS;
    return k;
}

}  // namespace att
}  // namespace opscv
