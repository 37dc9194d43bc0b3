// What the kernels of INT8 arithmetic with a scale for each token share: the quantiser's steps and the layers' results.
#pragma once

#include "device_utils.hpp"

namespace trtamd
{

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

constexpr uint32_t kF16Inf = 0x7c00u;

// The larger of the absolute values' bits in each half: as integers they are ordered as the values are, with infinity and
// the NaNs above all others, so that a row's maximum says whether it holds any.
__device__ inline u16x2 max_abs(u16x2 m, uint32_t pair)
{
    return __builtin_elementwise_max(m, bits_as<u16x2>(pair & 0x7fff7fffu));
}

// What a row's values are multiplied by, 127 / amax in two parts: the second is what the first is off by, so a product with
// both is the quotient rounded once.  A quotient half way between two integers therefore comes out as such (a product with one
// rounded factor misses now and then, and amax / 2 is a common value: 63.5), and any other is further from half way than a
// rounding moves it: 127 x / amax has operands of 11 bits.
struct RowScale
{
    float high, low;
};

// From the bits of amax.  Rows of zeros have factors of 0, and so have rows with an infinity or a NaN.  The scale, amax / 127,
// is rounded correctly: a product with 1 / 127, corrected by its exact remainder.
__device__ inline RowScale row_scale(uint32_t bits, float& scale)
{
    float const amax = (float) bits_as<f16>((uint16_t) bits);
    bool const finite = bits < kF16Inf;
    constexpr float k127th = 1.f / 127.f;
    float const s = amax * k127th;
    scale = finite ? fmaf(fmaf(-s, 127.f, amax), k127th, s) : __builtin_nanf("");
    float const inverse = __builtin_amdgcn_rcpf(amax);
    float const high = 127.f * inverse;
    return finite && bits ? RowScale{high, fmaf(-high, amax, 127.f) * inverse} : RowScale{0.f, 0.f};
}

// Adding 1.5 * 2^23 rounds to an integer, ties to even, and leaves it in the lowest byte.  What is not a number (an infinity or
// a NaN times the factors of its row, 0) has zeros there.
__device__ inline uint32_t quantized_bits(f16 x, RowScale const& r)
{
    float const low = fmaf((float) x, r.low, 0.f); // as a multiply-add it takes the binary16 as it is
    return bits_as<uint32_t>(fmaf((float) x, r.high, low) + 12582912.f);
}

// The lowest bytes of four dwords in one.
__device__ inline uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d)
{
    uint32_t const ab = __builtin_amdgcn_perm(b, a, 0x0c0c0400u), cd = __builtin_amdgcn_perm(d, c, 0x0c0c0400u);
    return ab | cd << 16;
}

__device__ inline u32x2 quantize8(f16x8 v, RowScale const& r)
{
    uint32_t b[8];
#pragma unroll
    for (int e = 0; e < 8; ++e)
    {
        b[e] = quantized_bits(v[e], r);
    }
    return {low_bytes(b[0], b[1], b[2], b[3]), low_bytes(b[4], b[5], b[6], b[7])};
}

__device__ inline uint32_t wave_max_bits(u16x2 m)
{
    uint32_t const both = max((uint32_t) m[0], (uint32_t) m[1]);
    return group_allreduce<kWaveSize>(both, [](uint32_t a, uint32_t b) { return max(a, b); });
}

__device__ inline u16x2 max_abs(u16x2 m, u32x4 const& v)
{
#pragma unroll
    for (int e = 0; e < 4; ++e)
    {
        m = max_abs(m, v[e]);
    }
    return m;
}

// GELU for FP16 results: gelu(y) = max(y, 0) - |y| Phi(-|y|), with log2(Phi(-a)) as a polynomial of degree 5 whose error counts
// by what it does to the result: 8.5e-5 of it where that is a normal binary16 (a sixth to a third of the half step that rounding
// costs), 5.2e-9 below (a sixth): 5.1 % of the results for normal values are the neighbour of the nearest binary16.  Degree 7 gives
// 4e-6 (0.2 %) for two more multiply-adds, which are 6 of 170 us at 33289 tokens x 1024 -> 4096: the vector ALU and the matrix
// cores take turns there.  The leading coefficient is negative, so the term vanishes for
// larger a, also of infinities (an infinity times nothing would be a NaN); a NaN stays one, through the IEEE minimum.
__device__ inline float gelu_f16(float y)
{
    float const a = __builtin_elementwise_minimum(fabsf(y), 0x1p126f);
    float p = fmaf(a, -3.205105604e-04f, 5.827311892e-03f);
    p = fmaf(p, a, -4.823749512e-02f);
    p = fmaf(p, a, -4.641202092e-01f);
    p = fmaf(p, a, -1.149176598e+00f);
    p = fmaf(p, a, -1.000120640e+00f);
    return fmaf(-a, __builtin_amdgcn_exp2f(p), fmaxf(y, 0.f));
}

// The result of a token-scaled layer for four consecutive channels of a token: y = acc * tokenScale[t] * channelScale[n] +
// bias[n], or gelu(y). Converted in pairs: one by one the compiler now and then makes the multiply-add and the conversion one
// instruction, and a token's bits would depend on the kernel.
template <bool GELU, typename Acc4>
__device__ __forceinline__ u32x2 token_results(Acc4 const& acc, float const ts, f32x4 const& al, f32x4 const& be)
{
    u32x2 r;
#pragma unroll
    for (int pair = 0; pair < 2; ++pair)
    {
        f32x2 y;
#pragma unroll
        for (int e = 0; e < 2; ++e)
        {
            int const c = 2 * pair + e;
            y[e] = fmaf((float) acc[c] * ts, al[c], be[c]);
            if constexpr (GELU)
            {
                y[e] = gelu_f16(y[e]);
            }
        }
        r[pair] = bits_as<uint32_t>(__builtin_convertvector(y, f16x2));
    }
    return r;
}

} // namespace trtamd
