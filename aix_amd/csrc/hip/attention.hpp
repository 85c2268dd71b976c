// attention.hpp -- what the forward and backward kernels of attention share: the shape and its mask, matrix
// instructions over fragments of eight elements for f16 / bf16 / f32, and tiles in LDS that can be read along their rows
// and along their columns.
//
// Notation: query i of a sequence stands at position p = start + i.  It sees key j when
//     j < length, p >= 0, (not causal or j <= p) and (no window or |p - j| < window or j < sinks).
#pragma once

#include "common.hpp"

namespace aixk {
namespace attn {

using namespace aixd;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
constexpr int kFar = 1 << 29;                 // lengths are below this, positions within +- this: sums of two stay in 32 bits

// [batch, heads, sequence, head dim]: strides in elements.  Operands the kernels read have d = 1 and 16-byte rows;
// results are written through any strides.
struct View {
    char* p;
    u64 b, h, s, d;
};

struct Shape {
    u32 B, H, HK, G, D, DW;                   // heads, key heads, heads per key head, head dim; DW: D in whole 16-byte words, as operands are read
    i32 SQ, SK;
    i32 causal, window, sinks;                // window 0: none
    float scale;
    const i32* lengths; i64 lengths_step;     // null: SK everywhere
    const i32* starts; i64 starts_step;       // null: length - SQ
};

struct Row { i32 length, start; };
__device__ __forceinline__ i32 clampi(i32 v, i32 lo, i32 hi) { return v < lo ? lo : v > hi ? hi : v; }
__device__ __forceinline__ Row row_of(const Shape& s, u32 b)
{
    Row r;
    r.length = s.lengths ? clampi(s.lengths[(i64)b * s.lengths_step], 0, s.SK) : s.SK;
    r.start = s.starts ? clampi(s.starts[(i64)b * s.starts_step], -kFar, kFar) : r.length - s.SQ;
    return r;
}

// Masks as words of 32 bits, one bit per key (per query): formed once for 32 elements, then two instructions per element -- the
// bit as a word of ones or zeros, and a select or an and -- where the definition's comparisons take five and, written out per
// element, a branch per condition.
__device__ __forceinline__ u32 ones_below(i32 n) { return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1u; }
__device__ __forceinline__ u32 spread(u32 word, int bit) { return (u32)((i32)(word << (31 - bit)) >> 31); }
__device__ __forceinline__ float hide(float x, u32 word, int bit)         // -infinity where the bit is not set
{
    const u32 t = spread(word, bit);
    return __builtin_bit_cast(float, (__builtin_bit_cast(u32, x) & t) | (0xFF800000u & ~t));
}
__device__ __forceinline__ float drop(float x, u32 word, int bit) { return __builtin_bit_cast(float, __builtin_bit_cast(u32, x) & spread(word, bit)); }

// The keys the query at position p sees: lo <= j < hi, and j < sink.
struct Keys {
    i32 lo, hi, sink;
    // keys j0 .. j0 + 31
    __device__ __forceinline__ u32 word(i32 j0) const { return (ones_below(hi - j0) & ~ones_below(lo - j0)) | ones_below(sink - j0); }
};
__device__ __forceinline__ Keys keys_of(const Shape& s, i32 length, i32 p)
{
    Keys k{0, 0, 0};
    if (p < 0) return k;
    i32 hi = length;
    if (s.causal && p + 1 < hi) hi = p + 1;
    if (s.window) {
        k.sink = s.sinks < hi ? s.sinks : hi;
        if ((i64)p + s.window < hi) hi = p + s.window;
        if (p >= s.window) k.lo = p - s.window + 1;
    }
    k.hi = hi;
    return k;
}
// The positions that see key j: lo <= p < hi.
struct Queries {
    i32 lo, hi;
    __device__ __forceinline__ u32 word(i32 p0) const { return ones_below(hi - p0) & ~ones_below(lo - p0); }
};
__device__ __forceinline__ Queries queries_of(const Shape& s, i32 length, i32 j)
{
    if (j >= length) return Queries{0, 0};
    const bool near = s.window && j >= s.sinks;
    const i32 lo = s.causal ? j : near && j >= s.window ? j - s.window + 1 : 0;
    constexpr i32 kEnd = 0x50000000;                           // behind every position (2^30), and within 32 bits of the first (-2^29)
    return Queries{lo, near && (i64)j + s.window < kEnd ? j + s.window : kEnd};
}
// every / no pair of the rows at positions [p0, p1] and the keys [j0, j1] is visible
__device__ __forceinline__ bool all_visible(const Shape& s, i32 length, i32 p0, i32 p1, i32 j0, i32 j1)
{
    if (j1 >= length || p0 < 0 || (s.causal && j1 > p0)) return false;
    return !s.window || j1 < s.sinks || (p1 - j0 < s.window && j1 - p0 < s.window);
}
__device__ __forceinline__ bool none_visible(const Shape& s, i32 length, i32 p0, i32 p1, i32 j0, i32 j1)
{
    if (j0 >= length || p1 < 0 || (s.causal && j0 > p1)) return true;
    return s.window && j0 >= s.sinks && ((p0 > j1 && p0 - j1 >= s.window) || (j0 > p1 && j0 - p1 >= s.window));
}

// The key tiles of `step` keys that rows at positions [p0, p1] can see: the tiles of the first keys, then a run that starts
// at tile `first`.
struct Tiles { i32 sink, first, n; };
__device__ __forceinline__ Tiles tiles_of(const Shape& s, i32 length, i32 p0, i32 p1, i32 step)
{
    Tiles t{0, 0, 0};
    if (length <= 0 || p1 < 0) return t;
    if (p0 < 0) p0 = 0;
    i32 hi = length, lo = 0, sink_end = 0;
    if (s.causal && p1 + 1 < hi) hi = p1 + 1;
    if (s.window) {
        sink_end = s.sinks < hi ? s.sinks : hi;
        if (!s.causal && (i64)p1 + s.window < hi) hi = p1 + s.window;
        if (hi < sink_end) hi = sink_end;
        lo = p0 - s.window + 1 > 0 ? p0 - s.window + 1 : 0;
    }
    if (lo < hi) {
        const i32 sink_tiles = (sink_end + step - 1) / step;
        t.first = lo / step;
        t.sink = sink_tiles < t.first ? sink_tiles : t.first;
        t.n = t.sink + (hi + step - 1) / step - t.first;
    } else t.n = t.sink = t.first = (sink_end + step - 1) / step;
    return t;
}
__device__ __forceinline__ i32 tile_at(const Tiles& t, i32 i) { return i < t.sink ? i : t.first + i - t.sink; }

// A grid of `heads` x ranks: workgroup id stands for the (id / heads)-th rank -- the heaviest first -- of head id % heads.  Ids go
// round the XCDs, so with a multiple of eight key heads a key head and all query heads on it stay on one XCD, whose L2 then
// holds its keys, and every XCD gets every rank.  Sequences of different lengths are moved on by one from rank to rank: the long
// ones do not stay on the XCDs of their heads (777 padded f32, of four sequences: 43.4 -> 29.2 us).
struct Place { u32 rank, head; };
__device__ __forceinline__ Place place_of(const Shape& s, u32 id, u32 heads)
{
    Place p;
    p.rank = id / heads;
    p.head = id % heads;
    if (s.lengths) p.head = (p.head + p.rank) % heads;
    return p;
}

// ---- matrix instructions over fragments of eight elements ------------------------------------------------------------
// Lane l of a wave feeds row (column) l % 32 (l % 16) with eight consecutive elements of the summed dimension.  The f32
// instructions take one element per lane, so eight of them go through a fragment; which k they call which does not
// matter, as both operands agree.
template <class T> struct Mma;
template <> struct Mma<bf16> {
    typedef u32x4 Frag;
    static __device__ __forceinline__ Frag zero() { return Frag{0, 0, 0, 0}; }
    static __device__ __forceinline__ f32x16 run32(const Frag& a, const Frag& b, f32x16 c)
    { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0); }
    static __device__ __forceinline__ f32x4 run16(const Frag& a, const Frag& b, f32x4 c)
    { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0); }
    // (the operands of the inline conversion come from vector arithmetic, never straight from a matrix instruction)
    static __device__ __forceinline__ u32 pack(float lo, float hi) { u32 r; asm("v_cvt_pk_bf16_f32 %0, %1, %2" : "=v"(r) : "v"(lo), "v"(hi)); return r; }
    static __device__ __forceinline__ Frag pack8(const float* x) { return Frag{pack(x[0], x[1]), pack(x[2], x[3]), pack(x[4], x[5]), pack(x[6], x[7])}; }
    static __device__ __forceinline__ float at(const Frag& f, int j) { return __builtin_bit_cast(float, (j & 1) ? f[j >> 1] & 0xFFFF0000u : f[j >> 1] << 16); }
};
template <> struct Mma<f16> {
    typedef u32x4 Frag;
    static __device__ __forceinline__ Frag zero() { return Frag{0, 0, 0, 0}; }
    static __device__ __forceinline__ f32x16 run32(const Frag& a, const Frag& b, f32x16 c)
    { return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0); }
    static __device__ __forceinline__ f32x4 run16(const Frag& a, const Frag& b, f32x4 c)
    { return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0); }
    static __device__ __forceinline__ u32 pack(float lo, float hi) { return __builtin_bit_cast(u32, f16x2{(f16)lo, (f16)hi}); }
    static __device__ __forceinline__ Frag pack8(const float* x) { return Frag{pack(x[0], x[1]), pack(x[2], x[3]), pack(x[4], x[5]), pack(x[6], x[7])}; }
    static __device__ __forceinline__ float at(const Frag& f, int j) { return (float)__builtin_bit_cast(f16x2, (u32)f[j >> 1])[j & 1]; }
};
template <> struct Mma<float> {
    struct Frag { f32x4 lo, hi; };
    static __device__ __forceinline__ Frag zero() { return Frag{{0, 0, 0, 0}, {0, 0, 0, 0}}; }
    static __device__ __forceinline__ float at(const Frag& f, int j) { return j < 4 ? f.lo[j] : f.hi[j - 4]; }
    static __device__ __forceinline__ f32x16 run32(const Frag& a, const Frag& b, f32x16 c)
    {
#pragma unroll
        for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(at(a, j), at(b, j), c, 0, 0, 0);
        return c;
    }
    static __device__ __forceinline__ f32x4 run16(const Frag& a, const Frag& b, f32x4 c)
    {
#pragma unroll
        for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(at(a, j), at(b, j), c, 0, 0, 0);
        return c;
    }
    static __device__ __forceinline__ Frag pack8(const float* x) { return Frag{{x[0], x[1], x[2], x[3]}, {x[4], x[5], x[6], x[7]}}; }
};

// eight consecutive elements of a row in memory, zeros past the head dim (D is a whole number of 16-byte words)
template <class T> __device__ __forceinline__ typename Mma<T>::Frag load8(const T* row, u32 d, u32 D, bool on)
{
    typedef typename Mma<T>::Frag Frag;
    Frag f = Mma<T>::zero();
    if constexpr (sizeof(T) == 2) { if (on && d < D) f = *(const u32x4*)(row + d); }
    else {
        if (on && d < D) f.lo = *(const f32x4*)(row + d);
        if (on && d + 4 < D) f.hi = *(const f32x4*)(row + d + 4);
    }
    return f;
}

// Elements from d on lie past the head dim and their products are left out: f32, whose matrix instructions take 16 times as
// long as the branch does, and head dims above 128, where the branches also keep the compiler from holding every operand of a
// loop at once (attention_dkdv_k at 256: 263 spilled registers, 16 with them).  There they have a price: loops that end at
// such a branch stay rolled, and the register arrays they index become private memory (bytes per lane at 256 dims: attention_split_k 272 in
// 16 bits; attention_dq_k 528, f32 1040; attention_dkdv_k 336, f16 384, f32 1104).  The other kernels multiply the zeros and stay free of branches.
template <class T, int DP> __device__ __forceinline__ bool past(int d, u32 DW) { return (sizeof(T) == 4 || DP > 128) && d >= (int)DW; }

// Waves per SIMD a kernel is compiled for: two where a wave's share of the 512 registers then holds its accumulators, fragments
// and staged words (rows of up to 256 bytes), else one.  Two waves cover each other's exponentials, barriers and LDS reads:
// 8192 queries on 32 heads of 128, window 2048, bf16: 407 us with one, 284 with two.
template <class T, int DP> constexpr int waves_per_simd() { return DP * (int)sizeof(T) <= 256 ? 2 : 1; }

// ---- a tile of ROWS x DP elements in LDS --------------------------------------------------------------------------------
// 16-byte word c of row r is kept in slot c ^ turn(r).  Reading one word from each of 16 consecutive rows then touches all
// banks once, and so does reading 64 bytes from each of four consecutive rows (what a transposed read of 32 columns does).
template <class T, int DP> struct Tile {
    static constexpr int WORDS = DP * (int)sizeof(T) / 16, PITCH = DP * (int)sizeof(T), PER = 16 / (int)sizeof(T);
    static __device__ __forceinline__ int turn(int r)
    {
        if constexpr (WORDS >= 16) return ((r & 3) << 2) | ((r >> 2) & 3);
        else return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
    }
    static __device__ __forceinline__ int at(int r, int word) { return r * PITCH + ((word ^ turn(r)) << 4); }
    // elements 8 f .. 8 f + 7 of row r
    static __device__ __forceinline__ typename Mma<T>::Frag row(const char* lds, int r, int f)
    {
        if constexpr (sizeof(T) == 2) return *(const u32x4*)(lds + at(r, f));
        else return {*(const f32x4*)(lds + at(r, 2 * f)), *(const f32x4*)(lds + at(r, 2 * f + 1))};
    }
    // column 32 block + lane % 32, the eight rows r0 + 8 (j / 4) + 4 (lane / 32) + j % 4: what a 32 x 32 accumulator's
    // elements 8 c .. 8 c + 7 (r0 = 16 c) number in a lane, so that accumulators feed the other operand as they are.
    // 16-bit: two transposed reads; in every group of 16 lanes lane i points at four elements of row i / 4 and receives
    // column i of the four rows.
    static __device__ __forceinline__ typename Mma<T>::Frag column(const char* lds, int r0, int block, int lane)
    {
        if constexpr (sizeof(T) == 2) {
            const int i = lane & 15, r = r0 + 4 * (lane >> 5) + (i >> 2), word = 4 * block + 2 * ((lane >> 4) & 1) + ((i & 3) >> 1);
            const char* lo = lds + at(r, word) + 8 * (i & 1);
            const char* hi = lds + at(r + 8, word) + 8 * (i & 1);
            const u32x2 l = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)lo));
            const u32x2 h = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)hi));
            return u32x4{l.x, l.y, h.x, h.y};
        } else {
            const int c = 32 * block + (lane & 31);
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = *(const float*)(lds + at(r0 + 8 * (j >> 2) + 4 * (lane >> 5) + (j & 3), c >> 2) + 4 * (c & 3));
            return Mma<T>::pack8(x);
        }
    }
    // the same for 16 x 16 accumulators: column 16 block + lane % 16, the rows r0 + 16 (j / 4) + 4 (lane / 16) + j % 4
    static __device__ __forceinline__ typename Mma<T>::Frag column16(const char* lds, int r0, int block, int lane)
    {
        const int g = lane >> 4, i = lane & 15;
        if constexpr (sizeof(T) == 2) {
            const int r = r0 + 4 * g + (i >> 2), word = 2 * block + ((i & 3) >> 1);
            const char* lo = lds + at(r, word) + 8 * (i & 1);
            const char* hi = lds + at(r + 16, word) + 8 * (i & 1);
            const u32x2 l = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)lo));
            const u32x2 h = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)hi));
            return u32x4{l.x, l.y, h.x, h.y};
        } else {
            const int c = 16 * block + i;
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = *(const float*)(lds + at(r0 + 16 * (j >> 2) + 4 * g + (j & 3), c >> 2) + 4 * (c & 3));
            return Mma<T>::pack8(x);
        }
    }
};

// ROWS rows of DP elements on their way from memory into such a tile through the registers of NT threads.  A tile whose rows
// all exist and whose rows are DP elements is fetched from a uniform address and one offset per thread; at an edge the
// addresses stay inside the operand and zeros are chosen when the words are stored.
template <class T, int DP, int ROWS, int NT, bool WHOLE = true> struct Stage {
    typedef Tile<T, DP> L;
    static constexpr int N = ROWS * L::WORDS / NT, STEP = NT / L::WORDS;                // rows between a thread's words
    static_assert(ROWS * L::WORDS % NT == 0 && NT % L::WORDS == 0, "whole words per thread, all in one column");
    u32x4 w[N];
    static __device__ __forceinline__ bool inside(i32 r0, i32 rows, u32 D) { return WHOLE && r0 + ROWS <= rows && D == (u32)DP; }
    // rows [r0, ...) of `base`, of which those below `rows` exist (rows > 0)
    __device__ __forceinline__ void load(const T* base, u64 step, i32 r0, i32 rows, u32 D, int tid)
    {
        if (inside(r0, rows, D) && step < (1u << 24)) {
            const char* from = (const char*)(base + (u64)(u32)r0 * step);
            const u32 at = ((u32)(tid / L::WORDS) * (u32)step + (u32)(tid % L::WORDS) * L::PER) * (u32)sizeof(T);
#pragma unroll
            for (int n = 0; n < N; ++n) w[n] = *(const u32x4*)(from + (u64)(n * STEP) * step * sizeof(T) + at);
            return;
        }
        const int last = (int)D / L::PER - 1, word = tid % L::WORDS < last ? tid % L::WORDS : last;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const i32 r = r0 + tid / L::WORDS + n * STEP;
            w[n] = *(const u32x4*)(base + (u64)(u32)(r < rows ? r : rows - 1) * step + word * L::PER);
        }
    }
    __device__ __forceinline__ void store(char* lds, i32 r0, i32 rows, u32 D, int tid)
    {
        if (!inside(r0, rows, D)) {
            const bool on = tid % L::WORDS < (int)D / L::PER;
#pragma unroll
            for (int n = 0; n < N; ++n) if (!(on & (r0 + tid / L::WORDS + n * STEP < rows))) w[n] = u32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int n = 0; n < N; ++n) *(u32x4*)(lds + L::at(tid / L::WORDS + n * STEP, tid % L::WORDS)) = w[n];
    }
};

// the larger value, and the sum, of a lane and the lane 32 away: one instruction swaps the upper half of one register with the
// lower half of another (the copy has to be another register, so the compiler may not see that it is one)
struct Halves { float lo, hi; };
__device__ __forceinline__ Halves halves(float v)
{
    u32 x = __builtin_bit_cast(u32, v), y = x;
    asm("" : "+v"(y));
    const auto r = __builtin_amdgcn_permlane32_swap(x, y, false, false);
    x = r[0];                                                  // (a bit cast of a vector's element would always take the first)
    y = r[1];
    return Halves{__builtin_bit_cast(float, x), __builtin_bit_cast(float, y)};
}
__device__ __forceinline__ float max_of_halves(float v) { const Halves h = halves(v); return fmaxf(h.lo, h.hi); }
__device__ __forceinline__ float sum_of_halves(float v) { const Halves h = halves(v); return h.lo + h.hi; }
__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

// element e of a result row: rounded once from f32
template <class T> __device__ __forceinline__ void put4(char* base, u64 step, bool whole, u32 d, u32 D, float a, float b, float c, float e)
{
    T* p = (T*)base;
    if (whole) {                                             // unit step, 4-element groups aligned
        if (d < D) {
            if constexpr (sizeof(T) == 2) *(u32x2*)(p + d) = u32x2{Mma<T>::pack(a, b), Mma<T>::pack(c, e)};
            else *(f32x4*)(p + d) = f32x4{a, b, c, e};
        }
        return;
    }
    if (d < D) p[d * step] = down<T>(a);
    if (d + 1 < D) p[(d + 1) * step] = down<T>(b);
    if (d + 2 < D) p[(d + 2) * step] = down<T>(c);
    if (d + 3 < D) p[(d + 3) * step] = down<T>(e);
}

} // namespace attn
} // namespace aixk
