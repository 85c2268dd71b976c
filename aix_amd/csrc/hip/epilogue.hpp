// epilogue.hpp -- what follows a matrix product while its accumulators are still in registers:
//     z = product + bias,   out = act(z) + residual,   z kept for the backward pass on request,
// formed in f32 and rounded once per result.
#pragma once

#include "common.hpp"

namespace aixk {

using aixd::i32;
using aixd::u32;
using aixd::u64;

struct EpiArgs {
    const void* bias; u64 bias_step;           // null: none
    const void* res; u64 rs0, rs1;             // null: none; element strides of rows and columns
    void* pre;                                 // null: not kept; dense like the result
    i32 act;
    i32 whole;                                 // bias, residual, pre and result in aligned groups of eight columns
};

// The tanh form of GELU, 0.5 z (1 + tanh(c (z + 0.044715 z^3))), c = sqrt(2 / pi), is z sigmoid(2 c (z + 0.044715 z^3)).  The
// reciprocal instruction is good to one unit of f32, which is what a correctly rounded quotient's dozen instructions save.
__device__ __forceinline__ float exp_minus(float w) { return __builtin_amdgcn_exp2f(-1.44269504088896340736f * w); }
__device__ __forceinline__ float gelu_argument(float z) { return 1.59576912160573071176f * (z + 0.044715f * z * z * z); }

// (an exponential that leaves f32 is an infinity, its reciprocal the right zero)
__device__ __forceinline__ float activate(float z, int act)
{
    if (act == AIXK_ACT_RELU) return z < 0.0f ? 0.0f : z;                          // (a NaN stays one)
    if (act == AIXK_ACT_NONE) return z;
    return z * __builtin_amdgcn_rcpf(1.0f + exp_minus(act == AIXK_ACT_GELU ? gelu_argument(z) : z));
}
// with s = sigmoid(w): s + z s (1 - s) w', 1 - s = e s without cancellation; 0 or 1 to f32 where the exponential leaves it
__device__ __forceinline__ float slope(float z, int act)
{
    if (act == AIXK_ACT_RELU) return z > 0.0f ? 1.0f : 0.0f;
    if (act == AIXK_ACT_NONE) return 1.0f;
    const bool gelu = act == AIXK_ACT_GELU;
    const float w = gelu ? gelu_argument(z) : z;
    const float e = exp_minus(w), s = __builtin_amdgcn_rcpf(1.0f + e);
    const float inner = gelu ? 1.59576912160573071176f * (1.0f + 3.0f * 0.044715f * z * z) : 1.0f;
    const float y = s + z * s * (e * s) * inner;
    return w < -87.0f ? 0.0f : w > 87.0f ? 1.0f : y;
}

// sixteen bytes of 16-bit elements, or 32 of f32, as eight f32 values
template <class T> __device__ __forceinline__ void get8(const T* p, float* x)
{
    typedef unsigned int w4 __attribute__((ext_vector_type(4)));
    if constexpr (sizeof(T) == 4) {
        typedef float v4 __attribute__((ext_vector_type(4)));
        const v4 lo = *(const v4*)p, hi = *(const v4*)(p + 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) { x[j] = lo[j]; x[4 + j] = hi[j]; }
    } else {
        const w4 w = *(const w4*)p;
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = aixd::up<T>(__builtin_bit_cast(T, (aixd::u16)(w[j >> 1] >> (16 * (j & 1)))));
    }
}
template <class T> __device__ __forceinline__ void put8(T* p, const float* x)
{
    typedef unsigned int w4 __attribute__((ext_vector_type(4)));
    if constexpr (sizeof(T) == 4) {
        typedef float v4 __attribute__((ext_vector_type(4)));
        *(v4*)p = v4{x[0], x[1], x[2], x[3]};
        *(v4*)(p + 4) = v4{x[4], x[5], x[6], x[7]};
    } else {
        w4 w;
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = (aixd::u32)__builtin_bit_cast(aixd::u16, aixd::down<T>(x[2 * j])) | ((aixd::u32)__builtin_bit_cast(aixd::u16, aixd::down<T>(x[2 * j + 1])) << 16);
        *(w4*)p = w;
    }
}

// x: the products of columns col .. col + 7 of a row (e.whole), on return the results
template <class T> __device__ __forceinline__ void epilogue8(float* x, const EpiArgs& e, u64 row, u64 col, u64 N)
{
    if (e.bias) {
        float b[8];
        get8((const T*)e.bias + col, b);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] += b[j];
    }
    if (e.pre) put8((T*)e.pre + row * N + col, x);
    if (e.act) {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = activate(x[j], e.act);
    }
    if (e.res) {
        float r[8];
        get8((const T*)e.res + row * e.rs0 + col, r);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] += r[j];
    }
}
template <class T> __device__ __forceinline__ float epilogue1(float x, const EpiArgs& e, u64 row, u64 col, u64 N)
{
    using namespace aixd;
    if (e.bias) x += up<T>(((const T*)e.bias)[col * e.bias_step]);
    if (e.pre) ((T*)e.pre)[row * N + col] = down<T>(x);
    if (e.act) x = activate(x, e.act);
    if (e.res) x += up<T>(((const T*)e.res)[row * e.rs0 + col * e.rs1]);
    return x;
}

} // namespace aixk
