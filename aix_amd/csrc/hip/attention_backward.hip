// attention_backward.hip -- the gradients of attention.hip's softmax(scale q k^T + mask) v from the saved lse:
//     P = exp(scale q k^T - lse)     delta = sum_d grad out     dS = P (grad v^T - delta)
//     dq = scale dS k                dk = scale dS^T q          dv = P^T grad
// in two passes without atomics: attention_dq_k walks the keys for a block of queries (and leaves delta for the other),
// attention_dkdv_k walks the queries of all heads that share a block of keys.  Each forms the scores again; seven products
// instead of the five of a single pass that would add dq with atomics in an order of their own.
#pragma clang fp contract(fast)

#include "attention.hpp"
#include "attention_host.hpp"

#include <algorithm>
#include <cmath>

using namespace aixd;
using namespace aixk;
using namespace aixk::attn;

namespace {

struct BackwardArgs {
    Shape s;
    View grad, q, k, v, y, dq, dk, dv;
    const float* lse;
    float* delta;
    u32 tiles;                                // row tiles per head (dq), key tiles per key head (dk, dv)
    u32 splits;                               // shares of the queries (dk, dv)
    u32 lead, lead_splits, lead_keys;         // key tiles with leading keys that a window does not hide: every query sees them, so they have more shares
    i32 whole_dq, whole_dk, whole_dv;
    float* part;                              // [split][dk, dv][batch * key heads * keys][DP] if there are several; the lead tiles' further shares
                                              // follow, [share][dk, dv][batch * key heads * lead_keys][DP] (see share_of)
};

// P and dS are rounded to the operands' type to feed the matrix unit.  bf16 has the range of f32; f16 holds 2^-24 to 65504, and dS
// has no such bounds: loss-scaled gradients on a peaked row pass the upper end, an even row over some thousand keys the lower.  So
// for f16 a lane (a query in attention_dq_k, a key in attention_dkdv_k) has its dS, and its sums, times a power of two of its own: 2^75
// at first, which no product of f16 numbers takes out of f32, and lowered when a tile's largest passes 2^15, so that it comes to
// 2^11 .. 2^12.  What is left of the range below is 2^-36 of the lane's largest dS.  P is at most 1 and has 2^15.  (The factor
// enters with the exponential's argument where that is dS's alone.  Looking for the largest costs f16 11 %: 16 x 12 heads of 512 x 64,
// window 128, 57.4 us where bf16 takes 50.7; 16 heads on 4 of 4096 x 128, window 1024, 200 and 179; 21 % at 256 dims.)
template <class T> struct Unit {
    static constexpr int kProbability = 0;
    __device__ __forceinline__ float in_exponent(float lse2) const { return lse2; }
    __device__ __forceinline__ float times(float x) const { return x; }
    template <int DB> __device__ __forceinline__ void fit(float*, f32x16 (&)[DB]) {}
    __device__ __forceinline__ float taken_out(float x) const { return x; }
};
template <> struct Unit<f16> {
    static constexpr int kProbability = 15;
    int exponent = 75;
    __device__ __forceinline__ float in_exponent(float lse2) const { return lse2 - (float)exponent; }
    __device__ __forceinline__ float times(float x) const { return x * __builtin_amdgcn_ldexpf(1.0f, exponent - kProbability); }      // of x with P's factor
    // a tile of one query's or key's dS, half of it in this lane, and its sums so far
    template <int DB> __device__ __forceinline__ void fit(float* e, f32x16 (&sums)[DB])
    {
        float top = fabsf(e[0]);
#pragma unroll
        for (int v = 1; v < 16; ++v) top = fmaxf(top, fabsf(e[v]));
        if (!__any(top > 32768.0f)) return;
        top = max_of_halves(top);
        int lower = top > 32768.0f ? 12 - __builtin_amdgcn_frexp_expf(top) : 0;
        lower = lower < 0 ? lower : 0;                         // (an infinity has no exponent)
        exponent += lower;
#pragma unroll
        for (int v = 0; v < 16; ++v) e[v] = __builtin_amdgcn_ldexpf(e[v], lower);
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int v = 0; v < 16; ++v) sums[d][v] = __builtin_amdgcn_ldexpf(sums[d][v], lower);
    }
    __device__ __forceinline__ float taken_out(float x) const { return __builtin_amdgcn_ldexpf(x, -exponent); }
};

// As in attention_k the scores are transposed (a lane = one query): dS^T, rounded, feeds dq^T = K^T dS^T as it lies.
// (Rows of 128 bytes: three waves per SIMD, which bf16 comes to by itself; f16 at two 63.6 us for the 16 x 12 heads.)
template <class T, int DP, int KT>
__global__ __launch_bounds__(256, (DP * sizeof(T) == 128 ? 3 : waves_per_simd<T, DP>())) void attention_dq_k(BackwardArgs a)
{
    typedef Mma<T> M;
    typedef typename M::Frag Frag;
    typedef Tile<T, DP> L;
    constexpr int DB = DP / 32, DC = DP / 16;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    char* ks = lds;
    char* vs = lds + KT * L::PITCH;
    const Shape& s = a.s;
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

    const Place place = place_of(s, blockIdx.x, s.B * s.H);
    const u32 keys = s.B * s.HK, tile = a.tiles - 1 - place.rank;
    const u32 b = place.head % keys / s.HK, hk = place.head % keys % s.HK, h = hk * s.G + place.head / keys;
    const Row r = row_of(s, b);
    const T* K = (const T*)a.k.p + b * a.k.b + hk * a.k.h;
    const T* V = (const T*)a.v.p + b * a.v.b + hk * a.v.h;
    const i32 i0 = (i32)tile * 128, i1 = i0 + 127 < s.SQ ? i0 + 127 : s.SQ - 1;
    const i32 w0 = i0 + wave * 32, w1 = w0 + 31 < s.SQ ? w0 + 31 : s.SQ - 1;
    const i32 i = w0 + (lane & 31), p = r.start + i;
    const bool on = i < s.SQ;
    const u64 at = ((u64)b * s.H + h) * (u64)(u32)s.SQ + (u32)i;

    Frag q[DC], go[DC];
    float delta = 0.0f;
    {
        const u64 row = (u64)(u32)(on ? i : 0);
        const T* rq = (const T*)a.q.p + b * a.q.b + h * a.q.h + row * a.q.s;
        const T* rg = (const T*)a.grad.p + b * a.grad.b + h * a.grad.h + row * a.grad.s;
        const T* ry = (const T*)a.y.p + b * a.y.b + h * a.y.h + row * a.y.s;
#pragma unroll
        for (int c = 0; c < DC; ++c) {
            q[c] = load8<T>(rq, c * 16 + half * 8, s.DW, on);
            go[c] = load8<T>(rg, c * 16 + half * 8, s.DW, on);
            const Frag y = load8<T>(ry, c * 16 + half * 8, s.DW, on);
#pragma unroll
            for (int j = 0; j < 8; ++j) delta += M::at(go[c], j) * M::at(y, j);
        }
        delta = sum_of_halves(delta);
    }
    float lse2 = __builtin_inff();                            // exp(x - inf) = 0: a query that sees nothing has no gradient
    if (on) {
        const float saved = a.lse[at];
        if (saved != -__builtin_inff()) lse2 = saved * kLog2e;
        if (half == 0) a.delta[at] = delta;
    }
    f32x16 acc[DB], less;                                     // (grad v^T starts from -delta: the products subtract it)
#pragma unroll
    for (int d = 0; d < DB; ++d) acc[d] = f32x16{};
#pragma unroll
    for (int v = 0; v < 16; ++v) less[v] = -delta;
    Unit<T> unit;
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
        if (w0 > w1) continue;
#pragma unroll
        for (int kb = 0; kb < KT / 32; ++kb) {
            const i32 k0 = j0 + kb * 32;
            if (none_visible(s, r.length, r.start + w0, r.start + w1, k0, k0 + 31)) continue;
            f32x16 x = f32x16{}, dp = less;
#pragma unroll
            for (int c = 0; c < DC; ++c) {
                if (past<T, DP>(c * 16, s.DW)) break;
                x = M::run32(L::row(ks, kb * 32 + (lane & 31), 2 * c + half), q[c], x);
                dp = M::run32(L::row(vs, kb * 32 + (lane & 31), 2 * c + half), go[c], dp);
            }
            const bool masked = !all_visible(s, r.length, r.start + w0, r.start + w1, k0, k0 + 31);
            float e[16];
            const float ref = unit.in_exponent(lse2);
#pragma unroll
            for (int v = 0; v < 16; ++v) e[v] = exp2_of(x[v] * c2 - ref) * dp[v];
            if (masked) {
                const u32 word = seen.word(k0) >> (4 * half);
#pragma unroll
                for (int v = 0; v < 16; ++v) e[v] = drop(e[v], word, 8 * (v >> 2) + (v & 3));
            }
            unit.fit(e, acc);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const Frag ds = M::pack8(e + 8 * c);
#pragma unroll
                for (int d = 0; d < DB; ++d) if (!past<T, DP>(d * 32, s.DW)) acc[d] = M::run32(L::column(ks, kb * 32 + c * 16, d, lane), ds, acc[d]);
            }
        }
    }
    if (!on) return;
    char* row = a.dq.p + (b * a.dq.b + h * a.dq.h + (u64)(u32)i * a.dq.s) * sizeof(T);
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int v = 0; v < 16; ++v) acc[d][v] = unit.taken_out(acc[d][v]);
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            put4<T>(row, a.dq.d, a.whole_dq, d * 32 + g * 8 + half * 4, s.D, acc[d][4 * g] * s.scale, acc[d][4 * g + 1] * s.scale, acc[d][4 * g + 2] * s.scale, acc[d][4 * g + 3] * s.scale);
}

// A wave keeps both sums of its 32 keys in registers, and the keys and values where the registers hold them beside that.  Rows of
// 256 bytes: sums of 128 registers leave room for two waves per SIMD only with keys and values in LDS (32 more registers for the
// keys alone cost eight spilled ones and 18 %: each reload waits for the loads in flight), 144 KB for eight waves; one wave
// per SIMD with everything in registers takes 1.4 times as long.  Rows of 128 bytes: keys and values in LDS make room for a third
// wave per SIMD (16 x 12 heads of 512 x 64, window 128: 28.2 us, with them in registers and two waves 32.6).  The queries and gradients of every head of the group come by in tiles of QT rows.  Here a lane is one key: P and
// dS, rounded, feed dv^T = grad^T P and dk^T = q^T dS as they lie.
template <class T, int DP> struct KeyBlock {
    static constexpr size_t kRow = DP * sizeof(T);
    static constexpr int kThreads = kRow == 256 ? 512 : 256, kKeys = kThreads / 2;
    static constexpr int kWaves = kRow == 128 ? 3 : kRow == 256 ? 2 : 1;                 // per SIMD
    static constexpr bool kKeysInLds = kRow <= 256, kValuesInLds = kRow <= 512;
    static constexpr int kRows = kRow <= 128 ? 64 : 32;                                  // QT
    static constexpr size_t kLds = 2 * kRows * kRow + 2 * kRows * sizeof(float) + (kKeysInLds + kValuesInLds) * kKeys * kRow;
};
// where share `split` of key j of a (batch, key head) lies
template <int DP> __device__ __forceinline__ void share_of(const BackwardArgs& a, u32 split, u64 head, u32 j, float** pk, float** pv)
{
    const u64 heads = (u64)a.s.B * a.s.HK, lead_rows = heads * a.lead_keys;
    const u64 rows = a.splits > 1 ? heads * (u32)a.s.SK : 0;
    if (a.splits > 1 && split < a.splits) {
        *pk = a.part + ((u64)split * 2 * rows + head * (u32)a.s.SK + j) * DP;
        *pv = *pk + rows * DP;
    } else {
        *pk = a.part + ((u64)a.splits * 2 * rows + (u64)(a.splits > 1 ? split - a.splits : split) * 2 * lead_rows + head * a.lead_keys + j) * DP;
        *pv = *pk + lead_rows * DP;
    }
}

template <class T, int DP>
__global__ __launch_bounds__((KeyBlock<T, DP>::kThreads), (KeyBlock<T, DP>::kWaves)) void attention_dkdv_k(BackwardArgs a)
{
    constexpr int NT = KeyBlock<T, DP>::kThreads, KB = KeyBlock<T, DP>::kKeys, QT = KeyBlock<T, DP>::kRows;
    typedef Mma<T> M;
    typedef typename M::Frag Frag;
    typedef Tile<T, DP> L;
    constexpr int DB = DP / 32, DC = DP / 16;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    char* qs = lds;
    char* gs = lds + QT * L::PITCH;
    float* ls = (float*)(lds + 2 * QT * L::PITCH);            // lse (log2), delta of the tile's rows
    float* ds = ls + QT;
    constexpr bool KL = KeyBlock<T, DP>::kKeysInLds, VL = KeyBlock<T, DP>::kValuesInLds;
    char* vs = (char*)(ds + QT);                              // the values and keys of the block, if they are kept here
    char* ks = vs + KB * L::PITCH;
    const Shape& s = a.s;
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

    // a head's workgroups: the lead tiles with lead_splits shares each, then the others with `splits`
    const Place place = place_of(s, blockIdx.x, s.B * s.HK);
    const u32 head = place.head, in = place.rank;
    const bool leads = in < a.lead * a.lead_splits;
    const u32 splits = leads ? a.lead_splits : a.splits, in2 = leads ? in : in - a.lead * a.lead_splits;
    const u32 split = in2 % splits, tile = in2 / splits + (leads ? 0 : a.lead);
    const u32 b = head / s.HK, hk = head % s.HK;
    const Row r = row_of(s, b);
    const i32 k0 = (i32)tile * KB, k1 = k0 + KB - 1 < r.length - 1 ? k0 + KB - 1 : r.length - 1;      // keys in use
    const i32 j0 = k0 + wave * 32, j = j0 + (lane & 31);
    const bool on = j < r.length;

    Frag kf[KL ? 1 : DC], vf[VL ? 1 : DC];
    {
        const u64 row = (u64)(u32)(on ? j : 0);
        const T* rk = (const T*)a.k.p + b * a.k.b + hk * a.k.h + row * a.k.s;
        const T* rv = (const T*)a.v.p + b * a.v.b + hk * a.v.h + row * a.v.s;
#pragma unroll
        for (int c = 0; c < DC; ++c) {
            if constexpr (!KL) kf[c] = load8<T>(rk, c * 16 + half * 8, s.DW, on);
            if constexpr (!VL) vf[c] = load8<T>(rv, c * 16 + half * 8, s.DW, on);
        }
    }
    if constexpr (VL) {                                       // (each wave reads its own rows only, but the loop's first barrier comes in between anyway)
        if (k0 <= k1) {
            Stage<T, DP, KB, NT> sv;
            sv.load((const T*)a.v.p + b * a.v.b + hk * a.v.h, a.v.s, k0, r.length, s.DW, tid);
            sv.store(vs, k0, r.length, s.DW, tid);
            if constexpr (KL) {
                sv.load((const T*)a.k.p + b * a.k.b + hk * a.k.h, a.k.s, k0, r.length, s.DW, tid);
                sv.store(ks, k0, r.length, s.DW, tid);
            }
        }
    }
    auto key = [&](int c) {
        if constexpr (KL) return L::row(ks, wave * 32 + (lane & 31), 2 * c + half);
        else return kf[c];
    };
    auto value = [&](int c) {
        if constexpr (VL) return L::row(vs, wave * 32 + (lane & 31), 2 * c + half);
        else return vf[c];
    };
    f32x16 dk[DB], dv[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) { dk[d] = f32x16{}; dv[d] = f32x16{}; }
    Unit<T> unit;
    const float c2 = s.scale * kLog2e;

    // the queries that can see a key of this block: positions [lo, hi)
    i32 i_lo = 0, i_hi = 0;
    if (k0 <= k1) {
        i64 lo = s.causal ? k0 : 0, hi = (i64)r.start + s.SQ;
        if (s.window && k0 >= s.sinks) {
            if ((i64)k0 - s.window + 1 > lo) lo = (i64)k0 - s.window + 1;
            if ((i64)k1 + s.window < hi) hi = (i64)k1 + s.window;
        }
        if (lo < r.start) lo = r.start;
        if (lo < hi) { i_lo = (i32)(lo - r.start); i_hi = (i32)(hi - r.start); }
    }
    const Queries seen = queries_of(s, r.length, j);
    // Shares of the queries, whole tiles of QT.  With shares for lead tiles alone the first takes all the queries that see more
    // than the leading keys, so that the others, and the partial sums, are about those keys only.
    const bool apart = leads && a.splits == 1 && splits > 1;
    i32 first = i_lo / QT, last = i_lo < i_hi ? (i_hi + QT - 1) / QT : first;
    u32 parts = splits, part = split;
    if (apart) {
        i64 far = (i64)k1 + s.window - r.start;               // (positions from k1 + window on see no other key of the tile)
        far = far < i_lo ? i_lo : far > i_hi ? i_hi : far;
        i32 near = ((i32)far + QT - 1) / QT;
        near = near < first ? first : near > last ? last : near;
        if (split == 0) last = near; else first = near;
        parts = split == 0 ? 1 : splits - 1;
        part = split == 0 ? 0 : split - 1;
    }
    const i32 per = last - first;
    const u64 total = (u64)(u32)per * s.G;
    const u64 from = total * part / parts, to = total * (part + 1) / parts;

    // the (head of the group, tile) of a step, stepped on by counting (a division per step costs more than its products)
    struct At { u32 g; i32 tile; };
    auto on_from = [&](At& at) { if (++at.tile == per) { at.tile = 0; ++at.g; } };
    Stage<T, DP, QT, NT, !KL> sq, sg;                       // (with the keys in LDS the second way to fetch costs registers there are not)
    float next_l = 0.0f, next_d = 0.0f;
    auto load = [&](const At& at) {
        const u32 h = hk * s.G + at.g;
        const i32 i0 = (first + at.tile) * QT;
        sq.load((const T*)a.q.p + b * a.q.b + h * a.q.h, a.q.s, i0, s.SQ, s.DW, tid);
        sg.load((const T*)a.grad.p + b * a.grad.b + h * a.grad.h, a.grad.s, i0, s.SQ, s.DW, tid);
        if (tid < QT) {
            const i32 i = i0 + tid < s.SQ ? i0 + tid : s.SQ - 1;
            const u64 row = ((u64)b * s.H + h) * (u64)(u32)s.SQ + (u32)i;
            next_l = a.lse[row];                               // (looked at when it is stored: here it would wait for every load in flight)
            next_d = a.delta[row];
        }
    };
    At now{0, 0};
    if (from < to) { now.g = (u32)(from / (u32)per); now.tile = (i32)(from % (u32)per); load(now); }
    At next = now;
    for (u64 n = from; n < to; ++n, now = next) {
        const i32 i0 = (first + now.tile) * QT;
        __syncthreads();
        sq.store(qs, i0, s.SQ, s.DW, tid);
        sg.store(gs, i0, s.SQ, s.DW, tid);
        if (tid < QT) { ls[tid] = i0 + tid < s.SQ && next_l != -__builtin_inff() ? next_l * kLog2e - Unit<T>::kProbability : __builtin_inff(); ds[tid] = next_d; }
        __syncthreads();
        if (n + 1 < to) { on_from(next); load(next); }
#pragma unroll
        for (int qb = 0; qb < QT / 32; ++qb) {
            const i32 q0 = i0 + qb * 32, q1 = q0 + 31 < s.SQ ? q0 + 31 : s.SQ - 1;
            if (q0 > q1 || none_visible(s, r.length, r.start + q0, r.start + q1, j0, j0 + 31)) continue;
            f32x16 x = f32x16{}, dp = f32x16{};
#pragma unroll
            for (int c = 0; c < DC; ++c) {
                if (past<T, DP>(c * 16, s.DW)) break;
                x = M::run32(L::row(qs, qb * 32 + (lane & 31), 2 * c + half), key(c), x);
                dp = M::run32(L::row(gs, qb * 32 + (lane & 31), 2 * c + half), value(c), dp);
            }
            const bool masked = !all_visible(s, r.length, r.start + q0, r.start + q1, j0, j0 + 31);
            float e[16], w[16];
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const f32x4 l4 = *(const f32x4*)(ls + qb * 32 + g * 8 + half * 4), d4 = *(const f32x4*)(ds + qb * 32 + g * 8 + half * 4);
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    e[4 * g + v] = exp2_of(x[4 * g + v] * c2 - l4[v]);
                    w[4 * g + v] = unit.times(e[4 * g + v] * (dp[4 * g + v] - d4[v]));
                }
            }
            if (masked) {
                const u32 word = seen.word(r.start + q0) >> (4 * half);
#pragma unroll
                for (int v = 0; v < 16; ++v) {
                    e[v] = drop(e[v], word, 8 * (v >> 2) + (v & 3));
                    w[v] = drop(w[v], word, 8 * (v >> 2) + (v & 3));
                }
            }
            unit.fit(w, dk);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const Frag fp = M::pack8(e + 8 * c), fs = M::pack8(w + 8 * c);
#pragma unroll
                for (int d = 0; d < DB; ++d) {
                    if (past<T, DP>(d * 32, s.DW)) break;
                    dv[d] = M::run32(L::column(gs, qb * 32 + c * 16, d, lane), fp, dv[d]);
                    dk[d] = M::run32(L::column(qs, qb * 32 + c * 16, d, lane), fs, dk[d]);
                }
            }
        }
    }
    if constexpr (Unit<T>::kProbability != 0) {
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                dk[d][v] = unit.taken_out(dk[d][v]);
                dv[d][v] = __builtin_amdgcn_ldexpf(dv[d][v], -Unit<T>::kProbability);
            }
    }
    if (j >= s.SK) return;
    if (apart && split && j >= (i32)a.lead_keys) return;
    if (splits > 1 && !(apart && j >= (i32)a.lead_keys)) {
        float *pk, *pv;
        share_of<DP>(a, split, head, (u32)j, &pk, &pv);
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int c = d * 32 + g * 8 + half * 4;
                *(f32x4*)(pk + c) = f32x4{dk[d][4 * g], dk[d][4 * g + 1], dk[d][4 * g + 2], dk[d][4 * g + 3]};
                *(f32x4*)(pv + c) = f32x4{dv[d][4 * g], dv[d][4 * g + 1], dv[d][4 * g + 2], dv[d][4 * g + 3]};
            }
        return;
    }
    char* rk = a.dk.p + (b * a.dk.b + hk * a.dk.h + (u64)(u32)j * a.dk.s) * sizeof(T);
    char* rv = a.dv.p + (b * a.dv.b + hk * a.dv.h + (u64)(u32)j * a.dv.s) * sizeof(T);
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const u32 c = d * 32 + g * 8 + half * 4;
            put4<T>(rk, a.dk.d, a.whole_dk, c, s.D, dk[d][4 * g] * s.scale, dk[d][4 * g + 1] * s.scale, dk[d][4 * g + 2] * s.scale, dk[d][4 * g + 3] * s.scale);
            put4<T>(rv, a.dv.d, a.whole_dv, c, s.D, dv[d][4 * g] * 1.0f, dv[d][4 * g + 1] * 1.0f, dv[d][4 * g + 2] * 1.0f, dv[d][4 * g + 3] * 1.0f);
        }
}

// the shares of the queries added up in their order
template <class T, int DP>
__global__ __launch_bounds__(256) void attention_dkdv_join_k(BackwardArgs a)
{
    constexpr int LANES = DP / 4;
    const Shape& s = a.s;
    const u64 row = (u64)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
    const u32 keys = a.splits > 1 ? (u32)s.SK : a.lead_keys;       // per head, those with shares
    const u32 c = threadIdx.x % LANES * 4;
    if (row >= (u64)s.B * s.HK * keys) return;
    const u64 j = row % keys, head = row / keys, hk = head % s.HK, b = head / s.HK;
    f32x4 k = f32x4{}, v = f32x4{};
    const u32 splits = j < a.lead_keys ? a.lead_splits : a.splits;
    for (u32 n = 0; n < splits; ++n) {
        float *pk, *pv;
        share_of<DP>(a, n, head, (u32)j, &pk, &pv);
        k += *(const f32x4*)(pk + c);
        v += *(const f32x4*)(pv + c);
    }
    put4<T>(a.dk.p + (b * a.dk.b + hk * a.dk.h + j * a.dk.s) * sizeof(T), a.dk.d, a.whole_dk, c, s.D, k.x * s.scale, k.y * s.scale, k.z * s.scale, k.w * s.scale);
    put4<T>(a.dv.p + (b * a.dv.b + hk * a.dv.h + j * a.dv.s) * sizeof(T), a.dv.d, a.whole_dv, c, s.D, v.x, v.y, v.z, v.w);
}

template <class T, int DP> int backward(aixk_ctx* ctx, const Call& c, BackwardArgs a)
{
    const Shape& s = c.s;
    // rows per LDS tile: 32 where 64 would leave less than two workgroups' worth of registers or LDS
    constexpr int KT = DP * sizeof(T) <= 256 ? 64 : 32;
    if (s.SQ > 0 && s.B > 0 && s.H > 0) {
        a.tiles = ((u32)s.SQ + 127) / 128;
        const u64 grid = (u64)s.B * s.H * a.tiles;
        AIXK_REQUIRE(grid < (1ull << 31), "attention_backward: too many rows");
        constexpr size_t lds = 2 * (size_t)KT * DP * sizeof(T);
        AIXK_TRY(allow_lds(attention_dq_k<T, DP, KT>, lds));
        hipLaunchKernelGGL((attention_dq_k<T, DP, KT>), dim3((unsigned)grid), dim3(256), lds, ctx->stream, a);
        AIXK_HIP(hipGetLastError());
    }
    if (s.SK == 0 || s.B == 0 || s.HK == 0) return AIXK_OK;
    constexpr u32 keys = KeyBlock<T, DP>::kKeys;
    a.tiles = ((u32)s.SK + keys - 1) / keys;
    const u64 heads = (u64)s.B * s.HK, rows = heads * (u32)s.SK;
    // Shares of the queries by a cost in microseconds: rounds of workgroups, each of its steps (about 2 us, three of them the
    // workgroup's own), and the shares written and read again (4 TB/s, and the joining launch).  Key tiles with leading keys, which
    // every query sees, take up to as many more shares as they have more queries: they start first, so that a chip full of other
    // work hides their longer chains.  16 heads on 4 of 4096 x 128, window 1024: 3 shares 98 us and 13 for joining them, 8 shares 148 in all.
    constexpr u64 resident = KeyBlock<T, DP>::kWaves * 256 / KeyBlock<T, DP>::kThreads;
    const u64 slots = (u64)ctx->cus * resident;
    const u64 seen = s.window && (u64)s.window + keys < (u64)(u32)s.SQ ? (u64)s.window + keys : (u64)(u32)s.SQ;      // queries of a tile at most
    const u64 steps = ((u64)s.G * seen + KeyBlock<T, DP>::kRows - 1) / KeyBlock<T, DP>::kRows;
    if (s.window && s.sinks && seen) {
        a.lead = ((u32)s.sinks + keys - 1) / keys;
        if (a.lead > a.tiles) a.lead = a.tiles;
    }
    const u64 more = a.lead ? std::min<u64>(((u32)s.SQ + seen - 1) / seen, 32) : 1;      // shares of a tile with leading keys for each of another's, at most
    // keys with shares of their own: whole tiles if the other tiles have shares too, else the leading keys
    auto lead_keys = [&](u64 sp) { return a.lead ? std::min<u64>(sp > 1 ? (u64)a.lead * keys : (u64)(u32)s.sinks, (u64)(u32)s.SK) : 0; };
    struct Plan { u64 splits, more, planes, grid; };
    // the cheapest shares whose partial sums take no more than `most` bytes (fewer on leading keys than more queries only for a twentieth:
    // 16 x 16 heads of 8192 x 128, window 256, 1024 leading keys: 5.7 ms with one share, 7.4 with 16 of 4 GB in all; 2 x 32 heads on 8 of
    // 8192 x 128, window 512, four leading keys, equal by this count: 767 us with 11, 788 with 6)
    auto cheapest = [&](u64 most) {
        Plan best{};
        double least = -1.0;
        for (u64 sp = 1; sp <= 64 && (sp == 1 || sp * 4 <= steps); ++sp)
            for (u64 mo = more;; mo = (mo + 1) / 2) {
                const u64 n = heads * (a.lead * sp * mo + (a.tiles - a.lead) * sp);
                const u64 shares = (sp > 1 ? sp * rows : 0) + (sp * mo > 1 ? (sp > 1 ? sp * (mo - 1) : mo) * heads * lead_keys(sp) : 0);
                // steps of a workgroup, and of one on leading keys: all queries of theirs over its shares, or (one share for the
                // other tiles) the first share's as anywhere and the rest over the others
                const double chain = (double)((steps + sp - 1) / sp + 3);
                const double reach = mo == more ? 1.0 : sp > 1 ? (double)more / (double)mo : mo > 1 ? (double)(more - 1) / (double)(mo - 1) : (double)more;
                const double led = a.lead ? std::ceil((double)steps * reach / (double)sp) + 3.0 : chain;
                const double full = std::ceil((double)heads * ((double)(a.lead * sp * mo) * led / chain + (double)((a.tiles - a.lead) * sp)));
                const double cost = 2.0 * std::max(std::ceil(full / (double)slots) * chain, led) + (shares ? 3.0 + (double)shares * (16.0 * DP / 4e6) : 0.0);
                if (shares * 2 * DP * sizeof(float) <= most && (least < 0.0 || cost < least * (mo == more ? 1.0 : 0.95))) { least = cost; best = Plan{sp, mo, shares, n}; }
                if (mo == 1) break;
            }
        return best;
    };
    // At most as much as the gradients in f32, or 256 MB: many leading keys on many heads came to 16 GB (4 x 32 heads of 16384 x 128,
    // window 1024, 4096 leading keys), though every head's own tiles fill the chip.  Without that memory: no shares.
    const u64 gradients = rows * 2 * DP * sizeof(float);
    void* ws = nullptr;
    Plan plan = cheapest(std::max<u64>(u64(256) << 20, gradients));
    if (plan.planes) {
        int rc = block_scratch(ctx, kScratchParts, (size_t)plan.planes * 2 * DP * sizeof(float), &ws);
        if (rc == AIXK_ENOMEM) { plan = cheapest(0); rc = AIXK_OK; ws = nullptr; }
        AIXK_TRY(rc);
    }
    a.splits = (u32)plan.splits;
    a.lead_keys = (u32)lead_keys(plan.splits);
    a.lead_splits = (u32)(a.lead ? plan.splits * plan.more : plan.splits);
    a.part = (float*)ws;
    const u64 grid = plan.grid;
    AIXK_REQUIRE(grid < (1ull << 31), "attention_backward: too many rows");
    constexpr size_t lds = KeyBlock<T, DP>::kLds;
    AIXK_TRY(allow_lds(attention_dkdv_k<T, DP>, lds));
    hipLaunchKernelGGL((attention_dkdv_k<T, DP>), dim3((unsigned)grid), dim3(KeyBlock<T, DP>::kThreads), lds, ctx->stream, a);
    AIXK_HIP(hipGetLastError());
    if (a.part) {
        constexpr u32 per = 256 / (DP / 4);
        const u64 joined = heads * (plan.splits > 1 ? (u64)(u32)s.SK : a.lead_keys);
        hipLaunchKernelGGL((attention_dkdv_join_k<T, DP>), dim3((unsigned)((joined + per - 1) / per)), dim3(256), 0, ctx->stream, a);
        AIXK_HIP(hipGetLastError());
    }
    return AIXK_OK;
}

} // namespace

extern "C" int32_t aixk_attention_backward(aixk_ctx* ctx, const aixhip_tensor* grad, const aixhip_tensor* q, const aixhip_tensor* k, const aixhip_tensor* v,
                                           const aixhip_tensor* out, const aixhip_tensor* lse, const aixk_attention_spec* spec,
                                           const aixhip_tensor* dq, const aixhip_tensor* dk, const aixhip_tensor* dv)
{
    const char* what = "attention_backward";
    Call c;
    AIXK_TRY(c.shape(what, q, k, v, spec));
    for (const aixhip_tensor* t : {grad, out}) {
        AIXK_REQUIRE(valid_tensor(t) && t->rank == 4 && t->dtype == c.dtype && t->size == numel(t), "%s: bad descriptor of grad or out", what);
        for (int d = 0; d < 4; ++d) AIXK_REQUIRE(t->shape[d] == q->shape[d], "%s: grad and out must have the shape of the queries", what);
    }
    AIXK_REQUIRE(lse != nullptr, "%s: the forward pass's lse is needed", what);
    AIXK_TRY(c.statistics(what, lse, q, &c.lse));
    i32 wq = 0, wk = 0, wv = 0;
    AIXK_TRY(c.result(what, dq, q, "dq", &c.dq, &wq));
    AIXK_TRY(c.result(what, dk, k, "dk", &c.dk, &wk));
    AIXK_TRY(c.result(what, dv, v, "dv", &c.dv, &wv));
    const aixhip_tensor* inputs[] = {grad, q, k, v, out, lse, spec->lengths, spec->starts};
    for (const aixhip_tensor* in : inputs)
        AIXK_REQUIRE(!overlap(dq, in) && !overlap(dk, in) && !overlap(dv, in), "%s: a result overlaps an operand", what);
    // (the three may be views side by side in one buffer)
    AIXK_REQUIRE(!overlap(dq, dk) && !overlap(dq, dv) && !overlap(dk, dv), "%s: results share their memory", what);
    AIXK_TRY(set_device(ctx));
    AIXK_TRY(c.operand(ctx, q, kScratchQ, &c.q));
    AIXK_TRY(c.operand(ctx, k, kScratchK, &c.k));
    AIXK_TRY(c.operand(ctx, v, kScratchV, &c.v));
    AIXK_TRY(c.operand(ctx, grad, kScratchGrad, &c.grad));
    AIXK_TRY(c.operand(ctx, out, kScratchOut, &c.y));
    void* delta;
    AIXK_TRY(block_scratch(ctx, kScratchDelta, (size_t)(numel(lse) + 1) * sizeof(float), &delta));
    BackwardArgs a{c.s, c.grad, c.q, c.k, c.v, c.y, c.dq, c.dk, c.dv, c.lse, (float*)delta, 0, 1, 0, 1, 0, wq, wk, wv, nullptr};
    return c.by_type([&](auto type, auto width) { return backward<decltype(type), decltype(width)::value>(ctx, c, a); });
}
