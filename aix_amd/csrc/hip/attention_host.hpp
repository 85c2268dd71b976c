// attention_host.hpp -- what the entry points of attention check, and how they make operands readable for the kernels.
#pragma once

#include "attention.hpp"

#include <cmath>
#include <type_traits>

namespace aixk {
namespace attn {

// slots of the context's scratch memory (block_scratch)
enum { kScratchQ = 0, kScratchK, kScratchV, kScratchGrad, kScratchOut, kScratchParts, kScratchDelta, kScratchProduct, kScratchColumns, kScratchLeft, kScratchRight };

int pack(aixk_ctx* ctx, int dtype, const View& src, void* dst, u32 B, u32 H, u64 S, u32 D, u32 DW);      // attention.hip

struct Call {
    Shape s{};
    int dtype{0};
    View q{}, k{}, v{}, grad{}, y{}, out{}, dq{}, dk{}, dv{};
    i32 whole_out{0};
    float* lse{nullptr};

    int shape(const char* what, const aixhip_tensor* tq, const aixhip_tensor* tk, const aixhip_tensor* tv, const aixk_attention_spec* spec)
    {
        AIXK_REQUIRE(valid_tensor(tq) && valid_tensor(tk) && valid_tensor(tv), "%s: bad operand descriptor", what);
        AIXK_REQUIRE(spec != nullptr, "%s: null spec", what);
        AIXK_REQUIRE(tq->rank == 4 && tk->rank == 4 && tv->rank == 4, "%s: queries, keys and values must be [batch, heads, sequence, head dim]", what);
        dtype = tq->dtype;
        AIXK_REQUIRE(dtype == AIXK_F32 || dtype == AIXK_F16 || dtype == AIXK_BF16, "%s: the element type must be f32, f16 or bf16", what);
        AIXK_REQUIRE(tk->dtype == dtype && tv->dtype == dtype, "%s: queries, keys and values must have one element type", what);
        for (const aixhip_tensor* t : {tq, tk, tv}) AIXK_REQUIRE(t->size == numel(t), "%s: size and shape of an operand differ", what);
        for (int d = 0; d < 4; ++d) AIXK_REQUIRE(tk->shape[d] == tv->shape[d], "%s: shapes of keys and values differ", what);
        AIXK_REQUIRE(tq->shape[0] == tk->shape[0] && tq->shape[3] == tk->shape[3], "%s: batch or head dim of queries and keys differ", what);
        AIXK_REQUIRE(tq->shape[3] >= 1 && tq->shape[3] <= 256, "%s: the head dim must be in 1 .. 256", what);
        AIXK_REQUIRE(tq->shape[2] < (uint64_t)kFar && tk->shape[2] < (uint64_t)kFar, "%s: sequences must be shorter than 2^29", what);
        AIXK_REQUIRE(tq->shape[0] < (1u << 20) && tq->shape[1] < (1u << 20) && tq->shape[0] * tq->shape[1] < (1u << 28), "%s: too many sequences or heads", what);
        AIXK_REQUIRE((tk->shape[1] > 0 || tq->shape[1] == 0) && (tk->shape[1] == 0 || tq->shape[1] % tk->shape[1] == 0),
                     "%s: the heads of the queries must be a multiple of those of the keys", what);
        // (the kernels' exponentials are powers of two: a factor beyond f32 would turn a score of zero into a NaN)
        AIXK_REQUIRE(std::isfinite(spec->scale * kLog2e) && spec->scale > 0.0f, "%s: the scale must be a positive number, at most 2^127", what);
        s.B = (u32)tq->shape[0]; s.H = (u32)tq->shape[1]; s.HK = (u32)tk->shape[1]; s.G = s.HK ? s.H / s.HK : 0;
        s.SQ = (i32)tq->shape[2]; s.SK = (i32)tk->shape[2];
        s.D = (u32)tq->shape[3];
        const u32 per = 16 / (u32)aixk_dtype_size(dtype);
        s.DW = (s.D + per - 1) / per * per;
        s.causal = spec->causal != 0;
        s.window = spec->window > 0x7FFFFFFFull ? 0x7FFFFFFF : (i32)spec->window;          // positions are within +- 2^30: nothing is further away
        s.sinks = spec->sinks > (uint64_t)s.SK ? s.SK : (i32)spec->sinks;
        s.scale = spec->scale;
        for (const aixhip_tensor* t : {spec->lengths, spec->starts})
            AIXK_REQUIRE(!t || (valid_tensor(t) && t->dtype == AIXK_I32 && t->rank == 1 && t->shape[0] == tq->shape[0] && t->size == t->shape[0]),
                         "%s: lengths and starts must be int32 [batch]", what);
        if (spec->lengths) { s.lengths = (const i32*)spec->lengths->data + spec->lengths->offset; s.lengths_step = (i64)spec->lengths->strides[0]; }
        if (spec->starts) { s.starts = (const i32*)spec->starts->data + spec->starts->offset; s.starts_step = (i64)spec->starts->strides[0]; }
        return AIXK_OK;
    }

    View view(const aixhip_tensor* t) const
    {
        return View{(char*)t->data + t->offset * aixk_dtype_size(t->dtype), t->strides[0], t->strides[1], t->strides[2], t->strides[3]};
    }

    // a result of the shape of `like`, through its strides; *whole: it may be written in aligned groups of four elements
    int result(const char* what, const aixhip_tensor* t, const aixhip_tensor* like, const char* name, View* out_view, i32* whole) const
    {
        AIXK_REQUIRE(valid_tensor(t) && t->rank == 4 && t->dtype == dtype && t->size == numel(t), "%s: bad descriptor of %s", what, name);
        for (int d = 0; d < 4; ++d) {
            AIXK_REQUIRE(t->shape[d] == like->shape[d], "%s: the shape of %s does not match the operands", what, name);
            AIXK_REQUIRE(t->size == 0 || t->shape[d] <= 1 || t->strides[d] != 0, "%s: %s cannot be a broadcast view", what, name);
        }
        AIXK_REQUIRE(distinct(t), "%s: %s meets an element twice", what, name);
        *out_view = view(t);
        const size_t e = aixk_dtype_size(dtype);
        bool w = (t->strides[3] == 1 || t->shape[3] == 1) && t->shape[3] % 4 == 0 && (uintptr_t)out_view->p % (4 * e) == 0;
        for (int d = 0; d < 3; ++d) w = w && (t->shape[d] <= 1 || t->strides[d] % 4 == 0);
        *whole = w ? 1 : 0;
        return AIXK_OK;
    }

    int statistics(const char* what, const aixhip_tensor* t, const aixhip_tensor* like, float** p) const
    {
        AIXK_REQUIRE(valid_tensor(t) && t->rank == 3 && t->dtype == AIXK_F32 && t->size == numel(t), "%s: bad descriptor of lse", what);
        uint64_t run = 1;
        for (int d = 2; d >= 0; --d) {
            AIXK_REQUIRE(t->shape[d] == like->shape[d] && (t->shape[d] <= 1 || t->strides[d] == run), "%s: lse must be a dense f32 [batch, heads, queries]", what);
            run *= t->shape[d];
        }
        *p = (float*)t->data + t->offset;
        return AIXK_OK;
    }

    // Kernels read 16-byte words of rows with unit stride; anything else -- another innermost stride, rows that do not start
    // on 16 bytes, a head dim that is no whole number of words -- is copied into dense rows first.
    int operand(aixk_ctx* ctx, const aixhip_tensor* t, int slot, View* out_view) const
    {
        const size_t e = aixk_dtype_size(dtype);
        const uint64_t per = 16 / e;
        View src = view(t);
        bool direct = (t->strides[3] == 1 || t->shape[3] == 1) && t->shape[3] % per == 0 && (uintptr_t)src.p % 16 == 0;
        for (int d = 0; d < 3; ++d) direct = direct && (t->shape[d] <= 1 || t->strides[d] % per == 0);
        if (direct || numel(t) == 0) { *out_view = src; return AIXK_OK; }
        const uint64_t heads = t->shape[1], len = t->shape[2];
        void* p;
        AIXK_TRY(block_scratch(ctx, slot, (size_t)(t->shape[0] * heads * len * s.DW) * e, &p));
        AIXK_TRY(pack(ctx, dtype, src, p, (u32)t->shape[0], (u32)heads, len, s.D, s.DW));
        *out_view = View{(char*)p, heads * len * s.DW, len * s.DW, s.DW, 1};
        return AIXK_OK;
    }

    // element type x padded head dim
    template <class F> int by_type(F&& f) const
    {
        auto by_width = [&](auto type) -> int {
            if (s.D <= 64) return f(type, std::integral_constant<int, 64>{});
            if (s.D <= 128) return f(type, std::integral_constant<int, 128>{});
            return f(type, std::integral_constant<int, 256>{});
        };
        if (dtype == AIXK_F32) return by_width(float{});
        if (dtype == AIXK_F16) return by_width(f16{});
        return by_width(bf16{});
    }
};

// dynamic LDS beyond the 64 KB every kernel may use
template <class K> int allow_lds(K kernel, size_t bytes)
{
    if (bytes > 65536) AIXK_HIP(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
    return AIXK_OK;
}

} // namespace attn
} // namespace aixk
