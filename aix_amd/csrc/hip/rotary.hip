// rotary.hip -- rotary positions: pairs of elements of every head turned by an angle that grows with the position,
//     (x, y) -> (x cos t - y sin t, x sin t + y cos t),   t = position * frequency_i,
// for queries and keys in one launch.
//
// Angles.  The host forms the frequencies in 64 bits and hands each over as a fraction of a turn in units of 2^-64; position
// times that, in wrapping 64-bit integer arithmetic, IS the angle modulo a turn, exactly, however far the position: no range
// reduction, and f32 enters only with the sine and cosine of the fraction.
//
// Reading and writing q and k once is the bound, so a position's sines and cosines are formed once (into LDS) and
// serve all heads: forming them per element costs more than the transfer of the element.
#pragma clang fp contract(fast)

#include "common.hpp"

#include <cmath>

using namespace aixd;
using namespace aixk;

namespace {

constexpr int kPairs = 128;                    // dims up to 256

struct HeadView { const char* in; char* out; u64 ib, ih, is, id, ob, oh, os, od; };
struct RotaryArgs {
    HeadView q, k;
    const i32* positions; u64 pb, ps;
    u64 S, rows;                               // positions per sequence, batch * S
    u32 HQ, HK, D, pairs;
    u32 span, heads;                           // positions and heads per workgroup
    i32 inverse;
    float magnitude;
    u64 turn[kPairs];                          // frequency in 2^-64 turns
};

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

template <class T> struct Word {               // a 16-byte word as f32 values
    static constexpr int N = 16 / (int)sizeof(T);
    float x[N];
    __device__ __forceinline__ void get(const T* p)
    {
        const u32x4 w = *(const u32x4*)p;
        if constexpr (sizeof(T) == 4) { for (int j = 0; j < N; ++j) x[j] = __builtin_bit_cast(float, (u32)w[j]); }
        else {
#pragma unroll
            for (int j = 0; j < N; ++j) { const u16 h = (u16)(w[j >> 1] >> (16 * (j & 1))); x[j] = up<T>(__builtin_bit_cast(T, h)); }
        }
    }
    __device__ __forceinline__ void put(T* p) const
    {
        u32x4 w;
        if constexpr (sizeof(T) == 4) { for (int j = 0; j < N; ++j) w[j] = __builtin_bit_cast(u32, x[j]); }
        else {
#pragma unroll
            for (int j = 0; j < N / 2; ++j) w[j] = (u32)__builtin_bit_cast(u16, down<T>(x[2 * j])) | ((u32)__builtin_bit_cast(u16, down<T>(x[2 * j + 1])) << 16);
        }
        *(u32x4*)p = w;
    }
};

// A workgroup turns `heads` heads (queries first, then keys) of `span` consecutive positions.  VEC: a lane moves whole 16-byte
// words -- a word of pairs (INTER) or a word of first and a word of second elements; otherwise a pair or a copied element.
template <class T, bool INTER, bool VEC>
__global__ __launch_bounds__(256) void rotary_k(RotaryArgs a)
{
    extern __shared__ f32x2 table[];           // [span][pairs] cosine, sine
    const u64 row0 = (u64)blockIdx.x * a.span;
    const u32 span = (u32)(a.rows - row0 < a.span ? a.rows - row0 : a.span);
    for (u32 e = threadIdx.x; e < span * a.pairs; e += 256) {
        const u64 row = row0 + e / a.pairs, b = row / a.S, i = row % a.S;
        const i64 position = a.positions[b * a.pb + i * a.ps];
        const i64 phase = (i64)((u64)position * a.turn[e % a.pairs]);
        float sine, cosine;
        sincospif((float)phase * 0x1p-63f, &sine, &cosine);
        if (a.inverse) sine = -sine;
        table[e] = f32x2{cosine * a.magnitude, sine * a.magnitude};
    }
    __syncthreads();

    constexpr u32 N = Word<T>::N;
    // units of a head: (words of) pairs, then the (words of) elements that are copied
    const u32 turned = VEC ? (INTER ? 2 * a.pairs / N : a.pairs / N) : a.pairs;
    const u32 copied = VEC ? (a.D - 2 * a.pairs) / N : a.D - 2 * a.pairs;
    const u32 units = turned + copied, heads = a.HQ + a.HK;
    const u32 h0 = blockIdx.y * a.heads, here = heads - h0 < a.heads ? heads - h0 : a.heads;
    for (u32 e = threadIdx.x; e < span * here * units; e += 256) {
        const u32 unit = e % units, rest = e / units, h = h0 + rest % here, at = rest / here;
        const u64 row = row0 + at, b = row / a.S, i = row % a.S;
        const bool key = h >= a.HQ;
        const HeadView& v = key ? a.k : a.q;
        const u64 hh = key ? h - a.HQ : h;
        const T* in = (const T*)v.in + b * v.ib + hh * v.ih + i * v.is;
        T* out = (T*)v.out + b * v.ob + hh * v.oh + i * v.os;
        const f32x2* cs = table + at * a.pairs;
        if constexpr (VEC) {
            if (unit >= turned) {
                const u32 d = 2 * a.pairs + (unit - turned) * N;
                *(u32x4*)(out + d) = *(const u32x4*)(in + d);
            } else if constexpr (INTER) {
                Word<T> w;
                w.get(in + unit * N);
#pragma unroll
                for (u32 j = 0; j < N / 2; ++j) {
                    const f32x2 t = cs[unit * (N / 2) + j];
                    const float x = w.x[2 * j], y = w.x[2 * j + 1];
                    w.x[2 * j] = x * t.x - y * t.y;
                    w.x[2 * j + 1] = x * t.y + y * t.x;
                }
                w.put(out + unit * N);
            } else {
                Word<T> lo, hi;
                lo.get(in + unit * N);
                hi.get(in + a.pairs + unit * N);
#pragma unroll
                for (u32 j = 0; j < N; ++j) {
                    const f32x2 t = cs[unit * N + j];
                    const float x = lo.x[j], y = hi.x[j];
                    lo.x[j] = x * t.x - y * t.y;
                    hi.x[j] = x * t.y + y * t.x;
                }
                lo.put(out + unit * N);
                hi.put(out + a.pairs + unit * N);
            }
        } else {
            if (unit >= turned) {
                const u64 d = 2 * a.pairs + (unit - turned);
                out[d * v.od] = in[d * v.id];
            } else {
                const u64 first = INTER ? 2 * unit : unit, second = INTER ? 2 * unit + 1 : unit + a.pairs;
                const float x = up<T>(in[first * v.id]), y = up<T>(in[second * v.id]);
                const f32x2 t = cs[unit];
                out[first * v.od] = down<T>(x * t.x - y * t.y);
                out[second * v.od] = down<T>(x * t.y + y * t.x);
            }
        }
    }
}

bool same_view(const aixhip_tensor* a, const aixhip_tensor* b)
{
    if (a->data != b->data || a->offset != b->offset || a->dtype != b->dtype) return false;
    for (int d = 0; d < a->rank; ++d) if (a->shape[d] > 1 && a->strides[d] != b->strides[d]) return false;
    return true;
}

int check_pair(const aixhip_tensor* in, const aixhip_tensor* out, const char* name)
{
    AIXK_REQUIRE(valid_tensor(in) && in->rank == 4 && in->size == numel(in), "rotary: %s must be [batch, heads, sequence, head dim]", name);
    AIXK_REQUIRE(in->dtype == AIXK_F32 || in->dtype == AIXK_F16 || in->dtype == AIXK_BF16, "rotary: the element type must be f32, f16 or bf16");
    AIXK_REQUIRE(valid_tensor(out) && out->rank == 4 && out->size == in->size && out->dtype == in->dtype, "rotary: bad descriptor of the result for %s", name);
    for (int d = 0; d < 4; ++d) {
        AIXK_REQUIRE(out->shape[d] == in->shape[d], "rotary: the shape of the result for %s differs", name);
        AIXK_REQUIRE(out->size == 0 || out->shape[d] <= 1 || out->strides[d] != 0, "rotary: the result for %s cannot be a broadcast view", name);
    }
    AIXK_REQUIRE(distinct(out), "rotary: the result for %s meets an element twice", name);
    return AIXK_OK;
}

} // namespace

extern "C" int32_t aixk_rotary(aixk_ctx* ctx, const aixhip_tensor* q, const aixhip_tensor* k, const aixhip_tensor* positions, const aixk_rotary_spec* spec,
                               const aixhip_tensor* q_out, const aixhip_tensor* k_out)
{
    AIXK_REQUIRE(spec != nullptr, "rotary: null spec");
    AIXK_TRY(check_pair(q, q_out, "the queries"));
    AIXK_REQUIRE((k == nullptr) == (k_out == nullptr), "rotary: keys and their result belong together");
    if (k) {
        AIXK_TRY(check_pair(k, k_out, "the keys"));
        AIXK_REQUIRE(k->dtype == q->dtype && k->shape[0] == q->shape[0] && k->shape[2] == q->shape[2] && k->shape[3] == q->shape[3],
                     "rotary: queries and keys differ in type, batch, sequence or head dim");
    }
    const uint64_t B = q->shape[0], S = q->shape[2], D = q->shape[3], HQ = q->shape[1], HK = k ? k->shape[1] : 0;
    AIXK_REQUIRE(valid_tensor(positions) && positions->dtype == AIXK_I32 && positions->rank == 2 && positions->shape[0] == B && positions->shape[1] == S &&
                 positions->size == B * S, "rotary: positions must be int32 [batch, sequence]");
    AIXK_REQUIRE(spec->dims >= 2 && spec->dims % 2 == 0 && spec->dims <= 2 * kPairs && spec->dims <= D, "rotary: the turned part must be even, 2 .. 256 and within the head dim");
    AIXK_REQUIRE(D < (1u << 16) && HQ < (1u << 20) && HK < (1u << 20) && B < (1ull << 31) && S < (1ull << 31) && B * S < (1ull << 40), "rotary: shape too large");
    AIXK_REQUIRE(std::isfinite(spec->base) && spec->base > 0.0 && std::isfinite(spec->magnitude) && spec->magnitude > 0.0f, "rotary: base and magnitude must be positive numbers");
    AIXK_REQUIRE(spec->scaling >= AIXK_ROTARY_PLAIN && spec->scaling <= AIXK_ROTARY_PARTS, "rotary: unknown scaling %d", spec->scaling);
    if (spec->scaling != AIXK_ROTARY_PLAIN) AIXK_REQUIRE(std::isfinite(spec->factor) && spec->factor > 0.0, "rotary: the factor must be a positive number");
    if (spec->scaling == AIXK_ROTARY_PARTS)
        AIXK_REQUIRE(std::isfinite(spec->original_length) && spec->original_length > 0.0 && std::isfinite(spec->low_turns) && std::isfinite(spec->high_turns) && spec->high_turns > spec->low_turns,
                     "rotary: the original length must be positive and high_turns above low_turns");
    const aixhip_tensor* results[] = {q_out, k_out};
    const aixhip_tensor* operands[] = {q, k, positions};
    for (int r = 0; r < 2; ++r)
        for (int o = 0; o < 3; ++o)
            if (results[r] && operands[o] && overlap(results[r], operands[o]))
                AIXK_REQUIRE(r == o && same_view(results[r], operands[o]), "rotary: a result overlaps an operand (in place means the same view)");
    AIXK_REQUIRE(!k || !overlap(q_out, k_out), "rotary: the results share their memory");
    AIXK_TRY(set_device(ctx));
    if (B * S == 0 || HQ + HK == 0) return AIXK_OK;

    RotaryArgs a{};
    const size_t e = aixk_dtype_size(q->dtype);
    const uint64_t word = 16 / e, pairs = spec->dims / 2;
    bool vec = spec->interleaved ? spec->dims % word == 0 : pairs % word == 0;
    vec = vec && (D - spec->dims) % word == 0;
    auto view = [&](const aixhip_tensor* in, const aixhip_tensor* out, HeadView* v) {
        v->in = (const char*)in->data + in->offset * e; v->out = (char*)out->data + out->offset * e;
        v->ib = in->strides[0]; v->ih = in->strides[1]; v->is = in->strides[2]; v->id = in->strides[3];
        v->ob = out->strides[0]; v->oh = out->strides[1]; v->os = out->strides[2]; v->od = out->strides[3];
        if (in->size == 0) return;
        for (const aixhip_tensor* t : {in, out}) {
            vec = vec && t->strides[3] == 1 && (uintptr_t)((const char*)t->data + t->offset * e) % 16 == 0;
            for (int d = 0; d < 3; ++d) vec = vec && (t->shape[d] <= 1 || t->strides[d] % word == 0);
        }
    };
    view(q, q_out, &a.q);
    if (k) view(k, k_out, &a.k);
    a.positions = (const i32*)positions->data + positions->offset; a.pb = positions->strides[0]; a.ps = positions->strides[1];
    a.S = S; a.rows = B * S; a.HQ = (u32)HQ; a.HK = (u32)HK; a.D = (u32)D; a.pairs = (u32)pairs;
    a.inverse = spec->inverse != 0; a.magnitude = spec->magnitude;
    // the frequencies are a geometric series, stepped in extended precision (a power per pair takes the host longer than the
    // kernel takes for a token)
    double base = spec->base;
    if (spec->scaling == AIXK_ROTARY_BASE && spec->dims > 2) base *= std::pow(spec->factor, (double)spec->dims / ((double)spec->dims - 2.0));
    const long double ratio = powl((long double)base, -2.0L / (long double)spec->dims), per_turn = 0.15915494309189533576888L;      // 1 / (2 pi)
    long double f = 1.0L;
    for (uint64_t i = 0; i < pairs; ++i, f *= ratio) {
        long double turns = f * per_turn;
        if (spec->scaling == AIXK_ROTARY_LINEAR) turns /= (long double)spec->factor;
        if (spec->scaling == AIXK_ROTARY_PARTS) {
            double kept = (spec->original_length * (double)turns - spec->low_turns) / (spec->high_turns - spec->low_turns);
            kept = kept < 0.0 ? 0.0 : kept > 1.0 ? 1.0 : kept;
            turns *= (long double)(kept + (1.0 - kept) / spec->factor);
        }
        if (turns >= 1.0L) turns -= floorl(turns);                             // whole turns per position do nothing
        a.turn[i] = (u64)(turns * 18446744073709551616.0L);
    }
    // Positions per workgroup: about 16 KB of elements, a table of at most 32 KB, and, if there are few positions, the heads
    // spread over workgroups until every compute unit has two.
    const u64 heads = HQ + HK, bytes = heads * D * e;
    u64 span = bytes >= 16384 ? 1 : 16384 / bytes;
    if (span > 4096 / pairs) span = 4096 / pairs;
    if (span > a.rows) span = a.rows;
    while (span > 1 && (a.rows + span - 1) / span < (u64)ctx->cus * 4) span = span / 2;
    u64 per = heads;
    const u64 groups = (a.rows + span - 1) / span;
    if (groups < (u64)ctx->cus * 2) { const u64 parts = ((u64)ctx->cus * 2 + groups - 1) / groups; per = (heads + parts - 1) / parts; }
    while (span * per * D >= (1ull << 31)) per = (per + 1) / 2;
    if ((heads + per - 1) / per > 65535) per = (heads + 65534) / 65535;
    AIXK_REQUIRE(groups < (1ull << 31), "rotary: too many positions");
    a.span = (u32)span; a.heads = (u32)per;
    const dim3 grid((unsigned)groups, (unsigned)((heads + per - 1) / per));
    const size_t lds = (size_t)span * pairs * sizeof(f32x2);
    auto launch = [&](auto type) -> int {
        typedef decltype(type) T;
        if (vec && spec->interleaved) hipLaunchKernelGGL((rotary_k<T, true, true>), grid, dim3(256), lds, ctx->stream, a);
        else if (vec) hipLaunchKernelGGL((rotary_k<T, false, true>), grid, dim3(256), lds, ctx->stream, a);
        else if (spec->interleaved) hipLaunchKernelGGL((rotary_k<T, true, false>), grid, dim3(256), lds, ctx->stream, a);
        else hipLaunchKernelGGL((rotary_k<T, false, false>), grid, dim3(256), lds, ctx->stream, a);
        AIXK_HIP(hipGetLastError());
        return AIXK_OK;
    };
    if (q->dtype == AIXK_F32) return launch(float{});
    if (q->dtype == AIXK_F16) return launch(f16{});
    return launch(bf16{});
}
