// kv_terms.cuh -- f32 values as sums of f16 or bf16 terms, for matrix instructions on a cache of that type.
//
// Two f16 terms hold 22 bits of a value, three bf16 terms 24. For f16 the rows of q are scaled by a power of two to
// [2^13, 2^14) and softmax weights by 2^14, which keeps the terms out of f16's subnormal range; the factors are taken
// out of the scores (exactly) and cancel between the weighted sum and the total. bf16 has f32's range, so that rows scaled
// up could overflow beside large keys: only those below 2^-64 are, to there (their last terms would be subnormal; products with
// any key stay below 2^65), and those from 2^126 on are scaled below it (rounded to bf16 they could be infinite).
#pragma once
#include "common.cuh"

namespace hoard {

template <typename KT> struct Terms;
template <> struct Terms<__half> {
    static constexpr int N = 2, Q_MIN = 13, Q_MAX = 13;
    static constexpr float P_EXP = 14.f;
    static constexpr uint32_t INF2 = 0x7C007C00u;        // exponent bits of two values
};
template <> struct Terms<__nv_bfloat16> {
    static constexpr int N = 3, Q_MIN = -64, Q_MAX = 125;
    static constexpr float P_EXP = 0.f;
    static constexpr uint32_t INF2 = 0x7F807F80u;
};

// two f32 -> packed terms: a's rounding in the low half, b's in the high half; a and b become the remainders
template <typename KT> __device__ __forceinline__ uint32_t take_term(float& a, float& b);
template <> __device__ __forceinline__ uint32_t take_term<__half>(float& a, float& b) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    a -= f.x;
    b -= f.y;
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t take_term<__nv_bfloat16>(float& a, float& b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    const float2 f = __bfloat1622float2(h);
    a -= f.x;
    b -= f.y;
    return *reinterpret_cast<const uint32_t*>(&h);
}

template <typename KT> __device__ __forceinline__ float kv_lo(uint32_t w);
template <> __device__ __forceinline__ float kv_lo<__half>(uint32_t w) { return h2f(w); }
template <> __device__ __forceinline__ float kv_lo<__nv_bfloat16>(uint32_t w) { return __uint_as_float(w << 16); }

// whether either of two packed values is an infinity or NaN
template <typename KT> __device__ __forceinline__ bool odd_pair(uint32_t w) {
    const uint32_t e = w & Terms<KT>::INF2;
    return (e & 0xFFFFu) == (Terms<KT>::INF2 & 0xFFFFu) || (e >> 16) == (Terms<KT>::INF2 >> 16);
}

// The power of two that brings a row with largest magnitude am (2^e <= am < 2^(e + 1)) to an exponent of Q_MIN .. Q_MAX, and
// its inverse (both normal numbers: 2^113 at most). Rows of zeros, and rows with infinities or NaN (bad), are left as they are.
struct RowScale {
    float up, down;
};
template <typename KT> __device__ __forceinline__ RowScale row_scale(float am, bool bad) {
    const int e = (int)(__float_as_uint(am) >> 23) - 127;
    const int by = bad || am == 0.f ? 0 : min(min(max(e, Terms<KT>::Q_MIN), Terms<KT>::Q_MAX) - e, 113);
    return {__uint_as_float((uint32_t)(127 + by) << 23), __uint_as_float((uint32_t)(127 - by) << 23)};
}
// n things in `parts` shares that differ by one at most: the first of share i (one 32-bit division, before the first load)
struct Share {
    unsigned each, more;
    __device__ __forceinline__ Share(unsigned n, unsigned parts) : each(n / parts), more(n - each * parts) {}
    __device__ __forceinline__ int first(unsigned i) const { return (int)(each * i + min(i, more)); }
};

// four floats to an address of any alignment that floats have
__device__ __forceinline__ void store4(float* p, const float* v) {
    if ((reinterpret_cast<uintptr_t>(p) & 15) == 0) {
        *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = v[i];
    }
}
__device__ __forceinline__ float ex2f(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The weight of a score beside the largest one, times 2^P_EXP. The difference is formed first: top - P_EXP rounded at scores of
// 2^24 and more makes the largest weight 2^16, which is no f16.
template <typename KT> __device__ __forceinline__ float weight(float s, float top) {
    if constexpr (Terms<KT>::P_EXP == 0.f) return ex2f(s - top);
    else return ex2f((s - top) + Terms<KT>::P_EXP);
}

}  // namespace hoard
