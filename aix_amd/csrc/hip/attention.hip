// attention.hip -- softmax(scale q k^T + mask) v over 4-D views [batch, heads, sequence, head dim], with causal masks,
// sliding windows, leading keys that stay visible, shared key heads and a length per sequence, in one pass over the keys:
// running maximum m and sum l per query, out = sum_j exp(x_j - m) v_j / l, lse = m + log l.
//
//   attention_k        many queries: 128 queries of one head per workgroup, tiles of 64 keys through LDS;
//   attention_split_k  few queries (single tokens over a cache): the queries of all heads that share a key head are the
//                      rows of one 16-row tile, waves and workgroups split the keys, attention_join_k adds them up.
#pragma clang fp contract(fast)

#include "attention.hpp"
#include "attention_host.hpp"

#include <algorithm>

using namespace aixd;
using namespace aixk;
using namespace aixk::attn;

namespace {

struct ForwardArgs {
    Shape s;
    View q, k, v, out;
    float* lse;
    u32 tiles;                                // 128-row tiles per head
    i32 whole;                                // results in 4-element groups
};

// Scores are formed transposed, S^T = K Q^T with v_mfma 32x32: a lane then holds 16 of 32 keys of ONE query (lane % 32), the
// row statistics are lane-local but for one exchange between the halves of the wave, and the accumulators, rounded, are
// the second operand of O^T = V^T P^T as they lie -- the transposed reads of V number the keys the same way.  The running
// maximum is only raised when some query of the wave passes it by a factor 2^8 (exact either way: any reference that
// keeps exp in range gives the same quotient), so the accumulators are rarely rescaled.  P is rounded to the operands'
// type for the second product, as the matrix unit takes it; the sum is taken from the f32 values.
template <class T, int DP>
__global__ __launch_bounds__(256, (waves_per_simd<T, DP>())) void attention_k(ForwardArgs a)
{
    typedef Mma<T> M;
    typedef typename M::Frag Frag;
    typedef Tile<T, DP> L;
    constexpr int KT = DP <= 128 ? 64 : 32, KB = KT / 32, DB = DP / 32, DC = DP / 16;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    char* ks = lds;
    char* vs = lds + KT * L::PITCH;
    const Shape& s = a.s;
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

    const Place at = place_of(s, blockIdx.x, s.B * s.H);                     // (the last rows of a causal mask are the longest)
    const u32 keys = s.B * s.HK, tile = a.tiles - 1 - at.rank;
    const u32 b = at.head % keys / s.HK, hk = at.head % keys % s.HK, h = hk * s.G + at.head / keys;
    const Row r = row_of(s, b);
    const T* K = (const T*)a.k.p + b * a.k.b + hk * a.k.h;
    const T* V = (const T*)a.v.p + b * a.v.b + hk * a.v.h;

    const i32 i0 = (i32)tile * 128, i1 = i0 + 127 < s.SQ ? i0 + 127 : s.SQ - 1;
    const i32 w0 = i0 + wave * 32, w1 = w0 + 31 < s.SQ ? w0 + 31 : s.SQ - 1;      // this wave's queries (w0 > w1: none)
    const i32 i = w0 + (lane & 31);
    const i32 p = r.start + i;
    const bool on = i < s.SQ;

    Frag q[DC];
    {
        const T* row = (const T*)a.q.p + b * a.q.b + h * a.q.h + (u64)(on ? i : 0) * a.q.s;
#pragma unroll
        for (int c = 0; c < DC; ++c) q[c] = load8<T>(row, c * 16 + half * 8, s.DW, on);
    }
    f32x16 o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) o[d] = f32x16{};
    float m = -__builtin_inff(), l = 0.0f;                    // m in units of log2, l this half's part of the sum
    const float c2 = s.scale * kLog2e;

    const Keys seen = keys_of(s, r.length, p);
    const Tiles t = tiles_of(s, r.length, r.start + i0, r.start + i1, KT);
    Stage<T, DP, KT, 256> sk, sv;
    if (t.n) {
        const i32 j0 = tile_at(t, 0) * KT;
        sk.load(K, a.k.s, j0, r.length, s.DW, tid);
        sv.load(V, a.v.s, j0, r.length, s.DW, tid);
    }
    for (i32 n = 0; n < t.n; ++n) {
        const i32 j0 = tile_at(t, n) * KT;
        __syncthreads();
        sk.store(ks, j0, r.length, s.DW, tid);
        sv.store(vs, j0, r.length, s.DW, tid);
        __syncthreads();
        if (n + 1 < t.n) {
            const i32 next = tile_at(t, n + 1) * KT;
            sk.load(K, a.k.s, next, r.length, s.DW, tid);
            sv.load(V, a.v.s, next, r.length, s.DW, tid);
        }
        if (w0 > w1 || none_visible(s, r.length, r.start + w0, r.start + w1, j0, j0 + KT - 1)) continue;

        f32x16 x[KB];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            x[kb] = f32x16{};
#pragma unroll
            for (int c = 0; c < DC; ++c) if (!past<T, DP>(c * 16, s.DW)) x[kb] = M::run32(L::row(ks, kb * 32 + (lane & 31), 2 * c + half), q[c], x[kb]);
        }
        if (!all_visible(s, r.length, r.start + w0, r.start + w1, j0, j0 + KT - 1)) {
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
                const u32 word = seen.word(j0 + kb * 32) >> (4 * half);
#pragma unroll
                for (int v = 0; v < 16; ++v) x[kb][v] = hide(x[kb][v], word, 8 * (v >> 2) + (v & 3));
            }
        }
        float top = x[0][0];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int v = 0; v < 16; ++v) top = fmaxf(top, x[kb][v]);
        top = max_of_halves(top) * c2;
        if (__any(top > m + 8.0f)) {                          // (m = -inf: any visible key)
            const float raised = fmaxf(m, top);
            const float keep = raised == -__builtin_inff() ? 0.0f : exp2_of(m - raised);
            m = raised;
            l *= keep;
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int v = 0; v < 16; ++v) o[d][v] *= keep;
        }
        const float ref = m == -__builtin_inff() ? 0.0f : m;   // a row without a visible key so far: every term is exp(-inf)
        Frag w[2 * KB];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            float e[16];
#pragma unroll
            for (int v = 0; v < 16; ++v) { e[v] = exp2_of(x[kb][v] * c2 - ref); l += e[v]; }
            w[2 * kb] = M::pack8(e);
            w[2 * kb + 1] = M::pack8(e + 8);
        }
#pragma unroll
        for (int c = 0; c < 2 * KB; ++c)
#pragma unroll
            for (int d = 0; d < DB; ++d) if (!past<T, DP>(d * 32, s.DW)) o[d] = M::run32(L::column(vs, c * 16, d, lane), w[c], o[d]);
    }

    l = sum_of_halves(l);
    if (!on) return;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;            // a row that sees nothing: zeros
    if (a.lse && half == 0) a.lse[((u64)b * s.H + h) * (u64)s.SQ + (u32)i] = l == 0.0f ? -__builtin_inff() : (m + log2f(l)) * kLn2;
    char* row = a.out.p + (b * a.out.b + h * a.out.h + (u64)(u32)i * a.out.s) * sizeof(T);
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            put4<T>(row, a.out.d, a.whole, d * 32 + g * 8 + half * 4, s.D, o[d][4 * g] * inv, o[d][4 * g + 1] * inv, o[d][4 * g + 2] * inv, o[d][4 * g + 3] * inv);
}

// The same on 16 queries per wave, 64 per workgroup, with v_mfma 16x16: for f32, whose matrix instructions are a sixteenth as
// fast (a wave of 32 queries takes 7 us for a tile of 64 keys: half the queries are twice the waves to fill the chip with, and
// the head dim's tail is left out), and up to 128 head dims for grids of 128-query workgroups that leave compute units without one.
template <class T, int DP>
__global__ __launch_bounds__(256, DP * sizeof(T) <= 512 ? 2 : 1) void attention16_k(ForwardArgs a)
{
    typedef Mma<T> M;
    typedef typename M::Frag Frag;
    typedef Tile<T, DP> L;
    constexpr int KT = DP * sizeof(T) <= 256 ? 64 : 32, SUB = KT / 16, DB = DP / 16, DC = DP / 32;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    char* ks = lds;
    char* vs = lds + KT * L::PITCH;
    const Shape& s = a.s;
    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, c15 = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

    const Place at = place_of(s, blockIdx.x, s.B * s.H);                     // (the last rows of a causal mask are the longest)
    const u32 keys = s.B * s.HK, tile = a.tiles - 1 - at.rank;
    const u32 b = at.head % keys / s.HK, hk = at.head % keys % s.HK, h = hk * s.G + at.head / keys;
    const Row r = row_of(s, b);
    const T* K = (const T*)a.k.p + b * a.k.b + hk * a.k.h;
    const T* V = (const T*)a.v.p + b * a.v.b + hk * a.v.h;
    const i32 i0 = (i32)tile * 64, i1 = i0 + 63 < s.SQ ? i0 + 63 : s.SQ - 1;
    const i32 w0 = i0 + wave * 16, w1 = w0 + 15 < s.SQ ? w0 + 15 : s.SQ - 1;
    const i32 i = w0 + c15, p = r.start + i;
    const bool on = i < s.SQ;

    Frag q[DC];
    {
        const T* row = (const T*)a.q.p + b * a.q.b + h * a.q.h + (u64)(on ? i : 0) * a.q.s;
#pragma unroll
        for (int c = 0; c < DC; ++c) q[c] = load8<T>(row, c * 32 + g * 8, s.DW, on);
    }
    f32x4 o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) o[d] = f32x4{};
    float m = -__builtin_inff(), l = 0.0f;
    const float c2 = s.scale * kLog2e;

    const Keys seen = keys_of(s, r.length, p);
    const Tiles t = tiles_of(s, r.length, r.start + i0, r.start + i1, KT);
    Stage<T, DP, KT, 256> sk, sv;
    if (t.n) {
        const i32 j0 = tile_at(t, 0) * KT;
        sk.load(K, a.k.s, j0, r.length, s.DW, tid);
        sv.load(V, a.v.s, j0, r.length, s.DW, tid);
    }
    for (i32 n = 0; n < t.n; ++n) {
        const i32 j0 = tile_at(t, n) * KT;
        __syncthreads();
        sk.store(ks, j0, r.length, s.DW, tid);
        sv.store(vs, j0, r.length, s.DW, tid);
        __syncthreads();
        if (n + 1 < t.n) {
            const i32 next = tile_at(t, n + 1) * KT;
            sk.load(K, a.k.s, next, r.length, s.DW, tid);
            sv.load(V, a.v.s, next, r.length, s.DW, tid);
        }
        if (w0 > w1 || none_visible(s, r.length, r.start + w0, r.start + w1, j0, j0 + KT - 1)) continue;

        f32x4 x[SUB];
#pragma unroll
        for (int k = 0; k < SUB; ++k) x[k] = f32x4{};
#pragma unroll
        for (int c = 0; c < DC; ++c) {
            if (past<T, DP>(c * 32, s.DW)) break;
#pragma unroll
            for (int k = 0; k < SUB; ++k) x[k] = M::run16(L::row(ks, k * 16 + c15, 4 * c + g), q[c], x[k]);
        }
        const bool masked = !all_visible(s, r.length, r.start + w0, r.start + w1, j0, j0 + KT - 1);
        if (masked) {
#pragma unroll
            for (int k = 0; k < SUB; k += 2) {
                const u32 word = seen.word(j0 + k * 16) >> (4 * g);
#pragma unroll
                for (int v = 0; v < 8; ++v) x[k + (v >> 2)][v & 3] = hide(x[k + (v >> 2)][v & 3], word, 16 * (v >> 2) + (v & 3));
            }
        }
        float top = -__builtin_inff();
#pragma unroll
        for (int k = 0; k < SUB; ++k)
#pragma unroll
            for (int v = 0; v < 4; ++v) top = fmaxf(top, x[k][v]);
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = max_of_halves(top) * c2;
        if (__any(top > m + 8.0f)) {
            const float raised = fmaxf(m, top);
            const float keep = raised == -__builtin_inff() ? 0.0f : exp2_of(m - raised);
            m = raised;
            l *= keep;
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int v = 0; v < 4; ++v) o[d][v] *= keep;
        }
        const float ref = m == -__builtin_inff() ? 0.0f : m;
#pragma unroll
        for (int k = 0; k < SUB / 2; ++k) {
            float e[8];
#pragma unroll
            for (int v = 0; v < 8; ++v) { e[v] = exp2_of(x[2 * k + (v >> 2)][v & 3] * c2 - ref); l += e[v]; }
            const Frag w = M::pack8(e);
#pragma unroll
            for (int d = 0; d < DB; ++d) {
                if (past<T, DP>(d * 16, s.DW)) break;
                o[d] = M::run16(L::column16(vs, k * 32, d, lane), w, o[d]);
            }
        }
    }
    l += __shfl_xor(l, 16, 64);
    l = sum_of_halves(l);
    if (!on) return;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    if (a.lse && g == 0) a.lse[((u64)b * s.H + h) * (u64)s.SQ + (u32)i] = l == 0.0f ? -__builtin_inff() : (m + log2f(l)) * kLn2;
    char* row = a.out.p + (b * a.out.b + h * a.out.h + (u64)(u32)i * a.out.s) * sizeof(T);
#pragma unroll
    for (int d = 0; d < DB; ++d) put4<T>(row, a.out.d, a.whole, d * 16 + g * 4, s.D, o[d].x * inv, o[d].y * inv, o[d].z * inv, o[d].w * inv);
}

// ---- few queries ----------------------------------------------------------------------------------------------------------

struct SplitArgs {
    Shape s;
    View q, k, v, out;
    float* lse;
    u32 tiles, splits;                        // 16-row tiles per key head, shares of the keys
    i32 whole;
    float* part_o;                            // [split][batch * heads * queries][DP]
    float* part_ml;                           // [split][batch * heads * queries][2]: maximum (log2), sum
};

constexpr int kSplitKeys = 32;        // keys per wave and step

// WAVES: 4, several workgroups to a row's keys; or 8 for one workgroup that takes all of them
template <class T, int DP, int WAVES> struct SplitLds {
    static constexpr int kSlab = kSplitKeys * DP * (int)sizeof(T);                        // a wave's keys of V
    static constexpr int kJoin = WAVES * (16 * DP + 32) * 4;                                 // accumulators, maxima and sums of all waves
    static constexpr int kBytes = kSlab * WAVES > kJoin ? kSlab * WAVES : kJoin;
};
template <class T, int DP> constexpr int most_waves() { return DP * sizeof(T) <= 256 ? 8 : 4; }

// Row r of a key head's R = G * SQ rows is query r % SQ of head r / SQ of the group.  16 rows against 32 keys with v_mfma
// 16x16: keys are read from memory straight as the first operand; V goes through a slab of LDS that belongs to the wave
// alone (no barrier in the loop) to be read transposed.  Reading the cache is the bound, so the next step's words are in
// flight while a step is computed.
template <class T, int DP, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void attention_split_k(SplitArgs a)
{
    typedef Mma<T> M;
    typedef typename M::Frag Frag;
    constexpr int KT = kSplitKeys, DC = DP / 32, DB = DP / 16, WORDS = DP * (int)sizeof(T) / 16, PER = 16 / (int)sizeof(T), PITCH = DP * (int)sizeof(T);
    constexpr int NV = KT * WORDS / 64;                        // 16-byte words of V per lane
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const Shape& s = a.s;
    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, c15 = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    char* slab = lds + wave * SplitLds<T, DP, WAVES>::kSlab;

    const u32 id = blockIdx.x, split = id % a.splits, rest = id / a.splits;
    const u32 tile = rest % a.tiles, bk = rest / a.tiles, b = bk / s.HK, hk = bk % s.HK;
    const Row r = row_of(s, b);
    const u32 R = s.G * (u32)s.SQ, r0 = tile * 16, r1 = r0 + 15 < R ? r0 + 15 : R - 1;
    const u32 rr = r0 + c15;
    const bool on = rr < R;
    const i32 i = (i32)((on ? rr : 0) % (u32)s.SQ), p = r.start + i;
    const u32 h = hk * s.G + (on ? rr : 0) / (u32)s.SQ;
    const bool one_head = r0 / (u32)s.SQ == r1 / (u32)s.SQ;
    const i32 p0 = r.start + (one_head ? (i32)(r0 % (u32)s.SQ) : 0), p1 = r.start + (one_head ? (i32)(r1 % (u32)s.SQ) : s.SQ - 1);

    Frag q[DC];
    {
        const T* row = (const T*)a.q.p + b * a.q.b + h * a.q.h + (u64)(u32)i * a.q.s;
#pragma unroll
        for (int c = 0; c < DC; ++c) q[c] = load8<T>(row, c * 32 + g * 8, s.DW, on);
    }
    const T* K = (const T*)a.k.p + b * a.k.b + hk * a.k.h;
    const T* V = (const T*)a.v.p + b * a.v.b + hk * a.v.h;
    f32x4 o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) o[d] = f32x4{};
    float m = -__builtin_inff(), l = 0.0f;
    const float c2 = s.scale * kLog2e;

    // this workgroup's share of the visible steps; its waves take them in turn
    const Keys seen = keys_of(s, r.length, p);
    const Tiles t = tiles_of(s, r.length, p0, p1, KT);
    const u32 each = (u32)t.n / a.splits, over = (u32)t.n % a.splits;
    const i32 from = (i32)(split * each + (split < over ? split : over)), to = from + (i32)(each + (split < over ? 1 : 0));

    // slot of 16-byte word c of key k in the slab: the transposed reads take 32 bytes from each of eight keys at a time
    auto turn = [](int k) { return WORDS >= 16 ? ((k & 7) << 1) | ((k >> 3) & 1) : ((k >> 1) & 3) << 1; };
    const int last = (int)s.DW / PER - 1;
    // rows of 1 KB: the registers hold no next step beside this one.  Keys and values come within their step, V in two turns (a
    // step of the four waves is 256 KB, several times what a compute unit's share of the bandwidth brings in the time of a load)
    constexpr bool LATE = DP * sizeof(T) > 512;
    constexpr int TURNS = LATE ? 2 : 1, NW = NV / TURNS;
    Frag kf[2][DC];
    u32x4 vf[NW];
    auto load_v = [&](i32 j0, int turn) {
#pragma unroll
        for (int n = 0; n < NW; ++n) {
            const int e = lane + (turn * NW + n) * 64, w = e % WORDS;
            const i32 j = j0 + e / WORDS;
            vf[n] = *(const u32x4*)(V + (u64)(u32)(j < r.length ? j : r.length - 1) * a.v.s + (w < last ? w : last) * PER);
        }
    };
    auto load = [&](i32 j0) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            const i32 j = j0 + kb * 16 + c15;
            const T* row = K + (u64)(u32)(j < r.length ? j : r.length - 1) * a.k.s;
#pragma unroll
            for (int c = 0; c < DC; ++c) {
                if constexpr (sizeof(T) == 2) { const int w = c * 4 + g; kf[kb][c] = *(const u32x4*)(row + (w < last ? w : last) * 8); }
                else {
                    const int w = c * 8 + g * 2;
                    kf[kb][c].lo = *(const f32x4*)(row + (w < last ? w : last) * 4);
                    kf[kb][c].hi = *(const f32x4*)(row + (w + 1 < last ? w + 1 : last) * 4);
                }
            }
        }
        if constexpr (!LATE) load_v(j0, 0);
    };
    i32 n = from + wave;
    if (!LATE && n < to) load(tile_at(t, n) * KT);
    for (; n < to; n += WAVES) {
        const i32 j0 = tile_at(t, n) * KT;
        if constexpr (LATE) load(j0);
        f32x4 x[2];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            x[kb] = f32x4{};
#pragma unroll
            for (int c = 0; c < DC; ++c) {
                if (past<T, DP>(c * 32, s.DW)) break;
                // (words past the head dim repeat the last one: the query's zeros would meet an infinity there as a NaN)
                Frag f = kf[kb][c];
                if constexpr (sizeof(T) == 2) { if (c * 32 + g * 8 >= (int)s.DW) f = M::zero(); }
                else { if (c * 32 + g * 8 >= (int)s.DW) f.lo = f32x4{}; if (c * 32 + g * 8 + 4 >= (int)s.DW) f.hi = f32x4{}; }
                x[kb] = M::run16(f, q[c], x[kb]);
            }
        }
#pragma unroll
        for (int u = 0; u < TURNS; ++u) {
            if constexpr (LATE) load_v(j0, u);
#pragma unroll
            for (int e = 0; e < NW; ++e) {
                const int at = lane + (u * NW + e) * 64, k = at / WORDS, w = at % WORDS;
                *(u32x4*)(slab + k * PITCH + ((w ^ turn(k)) << 4)) = j0 + k < r.length && w <= last ? vf[e] : u32x4{0, 0, 0, 0};
            }
        }
        if (!LATE && n + WAVES < to) load(tile_at(t, n + WAVES) * KT);

        float top = -__builtin_inff();
        const u32 word = seen.word(j0) >> (4 * g);
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                x[kb][v] = hide(x[kb][v] * c2, word, 16 * kb + v);
                top = fmaxf(top, x[kb][v]);
            }
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = max_of_halves(top);
        if (__any(top > m + 8.0f)) {
            const float raised = fmaxf(m, top);
            const float keep = raised == -__builtin_inff() ? 0.0f : exp2_of(m - raised);
            m = raised;
            l *= keep;
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int v = 0; v < 4; ++v) o[d][v] *= keep;
        }
        const float ref = m == -__builtin_inff() ? 0.0f : m;
        float e[8];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int v = 0; v < 4; ++v) { e[4 * kb + v] = exp2_of(x[kb][v] - ref); l += e[4 * kb + v]; }
        const Frag w = M::pack8(e);
        // column 16 d + lane % 16 of V, the keys 16 (j / 4) + 4 g + j % 4 of element j
#pragma unroll
        for (int d = 0; d < DB; ++d) {
            if (past<T, DP>(d * 16, s.DW)) break;
            Frag f;
            if constexpr (sizeof(T) == 2) {
                const int k = 4 * g + (c15 >> 2), word = 2 * d + ((c15 & 3) >> 1);
                const char* lo = slab + k * PITCH + ((word ^ turn(k)) << 4) + 8 * (c15 & 1);
                const char* hi = slab + (k + 16) * PITCH + ((word ^ turn(k + 16)) << 4) + 8 * (c15 & 1);
                const u32x2 lw = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)lo));
                const u32x2 hw = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)hi));
                f = u32x4{lw.x, lw.y, hw.x, hw.y};
            } else {
                float y[8];
                const int c = 16 * d + c15;
#pragma unroll
                for (int j = 0; j < 8; ++j) { const int k = 16 * (j >> 2) + 4 * g + (j & 3); y[j] = *(const float*)(slab + k * PITCH + (((c >> 2) ^ turn(k)) << 4) + 4 * (c & 3)); }
                f = M::pack8(y);
            }
            o[d] = M::run16(f, w, o[d]);
        }
    }
    l += __shfl_xor(l, 16, 64);
    l = sum_of_halves(l);

    // the waves' shares: [wave][16 rows][DP] accumulators, then maxima and sums
    __syncthreads();
    float* all = (float*)lds;
    float* ml = all + WAVES * 16 * DP;
#pragma unroll
    for (int d = 0; d < DB; ++d) *(f32x4*)(all + (wave * 16 + c15) * DP + ((d * 16 + 4 * g) ^ (4 * (c15 & 7)))) = o[d];
    if (g == 0) { ml[(wave * 16 + c15) * 2] = m; ml[(wave * 16 + c15) * 2 + 1] = l; }
    __syncthreads();
    const u64 rows = (u64)s.B * s.H * (u32)s.SQ;
    for (int e = tid; e < 16 * DP / 4; e += WAVES * 64) {
        const int row = e / (DP / 4), d = e % (DP / 4) * 4;
        if (r0 + row >= R) continue;
        float top = -__builtin_inff();
#pragma unroll
        for (int w = 0; w < WAVES; ++w) top = fmaxf(top, ml[(w * 16 + row) * 2]);
        // (no maximum: a row without a visible key, whose sums are zeros, or one of NaN scores, whose sums are NaNs and stay so)
        const float ref = top == -__builtin_inff() ? 0.0f : top;
        f32x4 sum = f32x4{};
        float total = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const float f = exp2_of(ml[(w * 16 + row) * 2] - ref);
            total += f * ml[(w * 16 + row) * 2 + 1];
            sum += f * *(const f32x4*)(all + (w * 16 + row) * DP + (d ^ (4 * (row & 7))));
        }
        const u32 qi = (r0 + row) % (u32)s.SQ, qh = hk * s.G + (r0 + row) / (u32)s.SQ;
        const u64 at = ((u64)b * s.H + qh) * (u32)s.SQ + qi;
        if (a.splits > 1) {
            *(f32x4*)(a.part_o + (split * rows + at) * DP + d) = sum;
            if (d == 0) *(f32x2*)(a.part_ml + (split * rows + at) * 2) = f32x2{top, total};
        } else {
            const float inv = total == 0.0f ? 0.0f : 1.0f / total;
            if (a.lse && d == 0) a.lse[at] = total == 0.0f ? -__builtin_inff() : (top + log2f(total)) * kLn2;
            put4<T>(a.out.p + (b * a.out.b + qh * a.out.h + (u64)qi * a.out.s) * sizeof(T), a.out.d, a.whole, d, s.D, sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv);
        }
    }
}

// The shares of the keys added up: a workgroup per row, DP / 4 lanes side by side in several groups that take the shares in turn
// and meet in LDS (one group alone waits for a load per share: 9.2 us for 512 rows of 8 shares).
template <class T, int DP>
__global__ __launch_bounds__(256) void attention_join_k(SplitArgs a)
{
    constexpr int LANES = DP / 4, GROUPS = 256 / LANES;
    __shared__ f32x4 part[GROUPS][LANES];
    const Shape& s = a.s;
    const u64 rows = (u64)s.B * s.H * (u32)s.SQ, at = blockIdx.x;
    const int group = threadIdx.x / LANES, lane = threadIdx.x % LANES;
    const u32 d = lane * 4;
    float top = -__builtin_inff(), total = 0.0f;
#pragma unroll 8
    for (u32 k = 0; k < a.splits; ++k) top = fmaxf(top, a.part_ml[(k * rows + at) * 2]);
    const float ref = top == -__builtin_inff() ? 0.0f : top;       // as where the waves' shares meet
    f32x4 sum = f32x4{};
#pragma unroll 8
    for (u32 k = 0; k < a.splits; ++k) {
        const f32x2 ml = *(const f32x2*)(a.part_ml + (k * rows + at) * 2);
        total += exp2_of(ml.x - ref) * ml.y;
    }
#pragma unroll 2
    for (u32 k = group; k < a.splits; k += GROUPS)
        sum += exp2_of(a.part_ml[(k * rows + at) * 2] - ref) * *(const f32x4*)(a.part_o + (k * rows + at) * DP + d);
    part[group][lane] = sum;
    __syncthreads();
    if (group) return;
#pragma unroll
    for (int g = 1; g < GROUPS; ++g) sum += part[g][lane];
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    if (a.lse && d == 0) a.lse[at] = total == 0.0f ? -__builtin_inff() : (top + log2f(total)) * kLn2;
    const u32 i = (u32)(at % (u32)s.SQ), h = (u32)(at / (u32)s.SQ % s.H), b = (u32)(at / (u32)s.SQ / s.H);
    put4<T>(a.out.p + (b * a.out.b + h * a.out.h + (u64)i * a.out.s) * sizeof(T), a.out.d, a.whole, d, s.D, sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv);
}

// ---- operands the kernels cannot read where they lie ----------------------------------------------------------------------
// [batch, heads, rows, D] through any strides into dense rows of DW elements (whole 16-byte words), zeros behind D.  A group of
// `lanes` lanes takes a row, a word per lane and turn, so the row's place is worked out once per row.
template <class T>
__global__ __launch_bounds__(256) void attention_pack_k(View src, T* dst, u32 H, u32 S, u32 D, u32 DW, u64 rows, u32 lanes)
{
    constexpr u32 PER = 16 / sizeof(T);
    const u32 lane = threadIdx.x % lanes, each = 256 / lanes;
    for (u64 row = (u64)blockIdx.x * each + threadIdx.x / lanes; row < rows; row += (u64)gridDim.x * each) {
        const u32 i = (u32)(row % S), bh = (u32)(row / S), h = bh % H, b = bh / H;
        const T* from = (const T*)src.p + b * src.b + h * src.h + i * src.s;
        T* to = dst + row * DW;
        for (u32 w = lane; w < DW / PER; w += lanes) {
            union { u32x4 word; T x[PER]; } v;
            if (src.d == 1 && w * PER + PER <= D) __builtin_memcpy(&v, from + w * PER, 16);        // (any alignment)
            else
#pragma unroll
            for (u32 j = 0; j < PER; ++j) { const u32 d = w * PER + j; v.x[j] = d < D ? from[(u64)d * src.d] : zero<T>(); }
            *(u32x4*)(to + w * PER) = v.word;
        }
    }
}

// The same for rows that lie side by side (unit stride from row to row): 64 x 64 elements at a time turned in LDS, so that both
// the loads and the stores are of whole lines.
template <class T>
__global__ __launch_bounds__(256) void attention_pack_turned_k(View src, T* dst, u32 H, u32 S, u32 D, u32 DW, u32 across, u32 down, u64 tiles)
{
    constexpr u32 PER = 16 / sizeof(T), WORDS = 64 / PER;
    __shared__ T tile[64][64 + 4 / sizeof(T)];
    for (u64 at = blockIdx.x; at < tiles; at += gridDim.x) {
        const u32 tx = (u32)(at % across), ty = (u32)(at / across % down), bh = (u32)(at / across / down), h = bh % H, b = bh / H;
        const u32 s0 = ty * 64, d0 = tx * 64, lane = threadIdx.x & 63;
        const T* from = (const T*)src.p + b * src.b + h * src.h + s0 + lane;
        for (u32 d = threadIdx.x >> 6; d < 64; d += 4) tile[d][lane] = s0 + lane < S && d0 + d < D ? from[(u64)(d0 + d) * src.d] : zero<T>();
        __syncthreads();
        for (u32 c = threadIdx.x; c < 64 * WORDS; c += 256) {
            const u32 r = c / WORDS, w = c % WORDS;
            if (s0 + r >= S || d0 + w * PER >= DW) continue;
            union { u32x4 word; T x[PER]; } v;
#pragma unroll
            for (u32 j = 0; j < PER; ++j) v.x[j] = tile[w * PER + j][r];
            *(u32x4*)(dst + ((u64)bh * S + s0 + r) * DW + d0 + w * PER) = v.word;
        }
        __syncthreads();
    }
}

} // namespace

namespace aixk {
namespace attn {

int pack(aixk_ctx* ctx, int dtype, const View& src, void* dst, u32 B, u32 H, u64 S, u32 D, u32 DW)
{
    const u64 rows = (u64)B * H * S;
    if (!rows || !DW) return AIXK_OK;
    AIXK_REQUIRE(S < (1ull << 31) && (u64)B * H < (1ull << 32), "operand copy: shape too large");
    const u32 words = DW / (16 / (u32)aixk_dtype_size(dtype));
    u32 lanes = 1;
    while (lanes < words && lanes < 64) lanes *= 2;
    const unsigned blocks = grid_for((rows * lanes + 255) / 256, 1, (unsigned)ctx->cus * 16u);
    const u32 across = (DW + 63) / 64, down = (u32)((S + 63) / 64);
    const u64 tiles = (u64)across * down * B * H;
    auto run = [&](auto type) -> int {
        typedef decltype(type) T;
        if (src.s == 1 && src.d != 1 && S > 1 && D > 1) hipLaunchKernelGGL((attention_pack_turned_k<T>), dim3(grid_for(tiles, 1, (unsigned)ctx->cus * 16u)), dim3(256), 0, ctx->stream, src, (T*)dst, H, (u32)S, D, DW, across, down, tiles);
        else hipLaunchKernelGGL((attention_pack_k<T>), dim3(blocks), dim3(256), 0, ctx->stream, src, (T*)dst, H, (u32)S, D, DW, rows, lanes);
        AIXK_HIP(hipGetLastError());
        return AIXK_OK;
    };
    return dtype == AIXK_F32 ? run(float{}) : dtype == AIXK_F16 ? run(f16{}) : run(bf16{});
}

namespace {

// Microseconds of the two ways, by bytes per element and padded head dim: a workgroup's launch and ends and each of its steps of 64
// keys; the two launches of shares and each step of 16 rows and 32 keys for every wave of (up to) two workgroups per compute unit.  Fitted to both, each
// forced, on 8 heads of n x n (256, 512), n x 1024 (64, 128), 256 x 2048 and 1024 x 4096, 32 on 8 of 128 and 256 x 8192 and 12 of 40 x 512:
// the choice is the faster one or within 10 % of it there.  Split / not, us:
//                       16-bit, 64    128         256        f32, 64     128         256
//   8 of 512 x 512      16.5 / 10.6   20.4 / 16.1  51 / 45   23 / 29     41 / 48     62 / 97
//   8 of 1024 x 4096    56.9 / 56.9   92 / 94     441 / 306  135 / 200   400 / 351   820 / 724
//   32 on 8, 128 x 8192   52 / 108    89 / 182    449 / 603  129 / 394   402 / 698   897 / 1440
//   32 on 8, 256 x 8192   90 / 108   160 / 182    808 / 603  235 / 395   717 / 698  1729 / 1443
template <size_t BYTES, int DP> struct SplitOrNot;
template <> struct SplitOrNot<2, 64>  { static constexpr double block = 3.8, block_step = 0.82, split = 8.0, split_step = 1.4; };
template <> struct SplitOrNot<2, 128> { static constexpr double block = 5.0, block_step = 1.38, split = 12.0, split_step = 2.45; };
template <> struct SplitOrNot<2, 256> { static constexpr double block = 8.0, block_step = 4.65, split = 22.0, split_step = 12.4; };
template <> struct SplitOrNot<4, 64>  { static constexpr double block = 4.5, block_step = 3.04, split = 10.0, split_step = 3.6; };
template <> struct SplitOrNot<4, 128> { static constexpr double block = 5.0, block_step = 5.41, split = 15.0, split_step = 11.2; };
template <> struct SplitOrNot<4, 256> { static constexpr double block = 6.0, block_step = 11.2, split = 15.0, split_step = 13.2; };

template <class T, int DP> int forward(aixk_ctx* ctx, const Call& c)
{
    const Shape& s = c.s;
    const u64 rows = (u64)s.B * s.H * (u32)s.SQ;
    const u64 R = (u64)s.G * (u32)s.SQ;
    const u64 wide = (u64)s.B * s.H * (((u32)s.SQ + 127) / 128), narrow = (u64)s.B * s.HK * ((R + 15) / 16);
    // Split or not, by the time either takes (SplitOrNot): rows are worth a workgroup each 64 queries if its chain of steps is shorter
    // than the rows' shares of the chip.  Up to 32 rows per key head, a single token among them, are split in any case.
    constexpr int most = most_waves<T, DP>();
    constexpr u64 resident = 163840 / SplitLds<T, DP, 4>::kBytes < 4 ? 163840 / SplitLds<T, DP, 4>::kBytes : 4;
    // what a row can see at most: the whole cache, or the window and the leading keys
    auto reach = [&](u64 span) {
        const u64 inside = s.window ? (u64)s.window + span + (u64)s.sinks : (u64)s.SK;
        return inside < (u64)s.SK ? inside : (u64)s.SK;
    };
    const u64 keys = reach(std::min<u64>((u64)(u32)s.SQ, 16));
    const bool one = most > 4 && narrow < (u64)ctx->cus && keys > 4 * kSplitKeys && keys <= 3u * most * kSplitKeys;
    typedef SplitOrNot<sizeof(T), DP> Us;
    const u64 split_steps = (keys + kSplitKeys - 1) / kSplitKeys;
    const double block_cost = Us::block + Us::block_step * (double)((reach(64) + 63) / 64);
    const double split_cost = one ? 4.5 + Us::split_step * (double)((split_steps + most - 1) / most)
                                  : Us::split + Us::split_step * (double)narrow * (double)split_steps / (double)((u64)ctx->cus * 4 * std::min<u64>(resident, 2));
    if (R > 32 && (split_cost >= block_cost || R >= (1ull << 31))) {
        // 32 queries to a wave where that leaves a workgroup for every compute unit, and above 128 head dims, where 16 queries to a
        // wave read too much LDS for what they multiply (8 heads of 1000 x 192, few workgroups: 25.3 us against 36.0); f32 and
        // small grids: 16 queries to a wave.
        if constexpr (sizeof(T) == 4 || DP <= 128) {
            if (sizeof(T) == 4 || wide < (u64)ctx->cus) {
                const u64 grid = (u64)s.B * s.H * (((u32)s.SQ + 63) / 64);
                AIXK_REQUIRE(grid < (1ull << 31), "attention: too many rows");
                ForwardArgs a{s, c.q, c.k, c.v, c.out, c.lse, ((u32)s.SQ + 63) / 64, c.whole_out};
                constexpr size_t lds = 2 * (DP * sizeof(T) <= 256 ? 64 : 32) * DP * sizeof(T);
                AIXK_TRY(allow_lds(attention16_k<T, DP>, lds));
                hipLaunchKernelGGL((attention16_k<T, DP>), dim3((unsigned)grid), dim3(256), lds, ctx->stream, a);
                AIXK_HIP(hipGetLastError());
                return AIXK_OK;
            }
        }
        if constexpr (sizeof(T) == 2) {
            AIXK_REQUIRE(wide < (1ull << 31), "attention: too many rows");
            ForwardArgs a{s, c.q, c.k, c.v, c.out, c.lse, ((u32)s.SQ + 127) / 128, c.whole_out};
            constexpr size_t lds = 2 * (DP <= 128 ? 64 : 32) * DP * sizeof(T);
            AIXK_TRY(allow_lds(attention_k<T, DP>, lds));
            hipLaunchKernelGGL((attention_k<T, DP>), dim3((unsigned)wide), dim3(256), lds, ctx->stream, a);
            AIXK_HIP(hipGetLastError());
            return AIXK_OK;
        }
    }
    SplitArgs a{s, c.q, c.k, c.v, c.out, c.lse, (u32)((R + 15) / 16), 1, c.whole_out, nullptr, nullptr};
    auto launch = [&](auto waves_tag) -> int {
        constexpr int WAVES = decltype(waves_tag)::value;
        constexpr size_t lds = SplitLds<T, DP, WAVES>::kBytes;
        AIXK_TRY(allow_lds(attention_split_k<T, DP, WAVES>, lds));
        hipLaunchKernelGGL((attention_split_k<T, DP, WAVES>), dim3((unsigned)(narrow * a.splits)), dim3(WAVES * 64), lds, ctx->stream, a);
        AIXK_HIP(hipGetLastError());
        return AIXK_OK;
    };
    AIXK_REQUIRE(narrow < (1ull << 31) && rows < (1ull << 31), "attention: too many rows");
    // Few keys and few workgroups: one workgroup of as many waves as it holds takes them all in at most three steps, where
    // sharing them out costs a second launch (12 heads of 64 on 512 keys: 6.4 us with eight waves, 7.2 with sixteen, 4.8 + 3.4 in 4 shares).
    if (one) return launch(std::integral_constant<int, most>{});
    // Otherwise shares of the keys until every compute unit has the workgroups its LDS holds, four at most (f32 at 256 dims holds one:
    // 4 x 8 heads on 4 of 8192 keys 72 us), but no share below one step of all waves; up to eight workgroups where a share still has eight steps (16 sequences of any length up to 32768: 193 us with shares for four
    // workgroups, 172 for eight, which even the lengths out; 2052 keys: 31.0 us with four, 34.2 with eight).
    const u64 steps = (keys + kSplitKeys * 4 - 1) / (kSplitKeys * 4);
    u64 splits = ((u64)ctx->cus * resident + narrow - 1) / narrow;
    splits = std::max<u64>(splits, std::min<u64>(((u64)ctx->cus * 8 + narrow - 1) / narrow, steps / 8));
    if (splits > steps) splits = steps;
    if (splits < 1) splits = 1;
    AIXK_REQUIRE(narrow * splits < (1ull << 31), "attention: too many rows");
    a.splits = (u32)splits;
    if (splits > 1) {
        const size_t o_bytes = (size_t)splits * rows * DP * sizeof(float);
        void* ws;
        AIXK_TRY(block_scratch(ctx, kScratchParts, o_bytes + (size_t)splits * rows * 2 * sizeof(float), &ws));
        a.part_o = (float*)ws;
        a.part_ml = (float*)((char*)ws + o_bytes);
    }
    AIXK_TRY(launch(std::integral_constant<int, 4>{}));
    if (splits > 1) {
        hipLaunchKernelGGL((attention_join_k<T, DP>), dim3((unsigned)rows), dim3(256), 0, ctx->stream, a);
        AIXK_HIP(hipGetLastError());
    }
    return AIXK_OK;
}

} // namespace
} // namespace attn
} // namespace aixk

extern "C" int32_t aixk_attention(aixk_ctx* ctx, const aixhip_tensor* q, const aixhip_tensor* k, const aixhip_tensor* v, const aixk_attention_spec* spec,
                                  const aixhip_tensor* out, const aixhip_tensor* lse)
{
    Call c;
    AIXK_TRY(c.shape("attention", q, k, v, spec));
    AIXK_TRY(c.result("attention", out, q, "the result", &c.out, &c.whole_out));
    if (lse) AIXK_TRY(c.statistics("attention", lse, q, &c.lse));
    const aixhip_tensor* inputs[] = {q, k, v, spec->lengths, spec->starts};
    for (const aixhip_tensor* in : inputs) AIXK_REQUIRE(!overlap(out, in) && !overlap(lse, in), "attention: a result overlaps an operand");
    AIXK_REQUIRE(!overlap(out, lse), "attention: the results overlap");
    AIXK_TRY(set_device(ctx));
    if (c.s.B == 0 || c.s.H == 0 || c.s.SQ == 0) return AIXK_OK;
    AIXK_TRY(c.operand(ctx, q, kScratchQ, &c.q));
    AIXK_TRY(c.operand(ctx, k, kScratchK, &c.k));
    AIXK_TRY(c.operand(ctx, v, kScratchV, &c.v));
    return c.by_type([&](auto type, auto width) { return forward<decltype(type), decltype(width)::value>(ctx, c); });
}
