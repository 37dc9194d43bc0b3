// Quantisation of FP16 activations to INT8 with a scale for each token, and the linear layer that starts with it.
//
//   amax[t] = max_c |x[t][c]|,   s[t] = amax[t] / 127,   q[t][c] = rne(127 x[t][c] / amax[t])
//
// Two passes over a row, the second out of the L2 or registers: HBM streaming of 2 bytes in and 1 byte out per value.
#include "device_utils.hpp"
#include "host_utils.hpp"
#include "network_ops.hpp"
#include "trtamd_encoder_ops.h"

#include <limits>

namespace trtamd
{
namespace
{

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

constexpr uint32_t kF16Inf = 0x7c00u;

// The larger of the absolute values' bits in each half: as integers they are ordered as the values are, with infinity and
// the NaNs above all others, so that a row's maximum says whether it holds any.
__device__ inline u16x2 max_abs(u16x2 m, uint32_t pair)
{
    return __builtin_elementwise_max(m, bits_as<u16x2>(pair & 0x7fff7fffu));
}

// What a row is divided by: q = 127 x / amax, with 1 / amax at hand.  amax = 0 stands for rows whose values all become 0.
struct RowScale
{
    float amax, inverse;
};

__device__ inline RowScale row_scale(uint32_t bits, float& scale)
{
    float const amax = (float) bits_as<f16>((uint16_t) bits);
    bool const finite = bits < kF16Inf;
    scale = finite ? __fdiv_rn(amax, 127.f) : __builtin_nanf("");
    return finite && bits ? RowScale{amax, __fdiv_rn(1.f, amax)} : RowScale{0.f, 0.f};
}

// The quotient is corrected by its exact remainder, which makes it the correctly rounded one (Markstein's step): 127 x
// is exact, and so is what is half way between two integers, which the product with a rounded reciprocal misses now and then
// (amax / 2 is a common value, and is 63.5).  What is not half way is further from it than this rounding moves it: 127 x / amax has
// 11-bit operands.  Adding 1.5 * 2^23 rounds to an integer, ties to even, and leaves it in the lowest byte.
__device__ inline uint32_t quantized_bits(float x, RowScale const& r)
{
    float const n = x * 127.f;
    float const y = n * r.inverse;
    return bits_as<uint32_t>(fmaf(fmaf(-y, r.amax, n), r.inverse, y) + 12582912.f);
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
        // 0 * NaN and 0 * infinity: a row that holds them has no quotients
        b[e] = r.amax > 0.f ? quantized_bits((float) v[e], r) : 0u;
    }
    return {low_bytes(b[0], b[1], b[2], b[3]), low_bytes(b[4], b[5], b[6], b[7])};
}

__device__ inline uint32_t wave_max_bits(u16x2 m)
{
    uint32_t const both = max((uint32_t) m[0], (uint32_t) m[1]);
    return group_allreduce<kWaveSize>(both, [](uint32_t a, uint32_t b) { return max(a, b); });
}

// One workgroup per row of any length.
__global__ __launch_bounds__(256) void token_quantize_kernel(
    f16 const* __restrict__ in, int64_t stride, int C, int8_t* __restrict__ out, float* __restrict__ scales)
{
    __shared__ uint32_t part[4];
    size_t const t = blockIdx.x;
    f16 const* src = in + t * stride;
    u16x2 m = {0, 0};
    for (int c = threadIdx.x * 8; c < C; c += 256 * 8)
    {
        u32x4 const v = *reinterpret_cast<u32x4 const*>(src + c);
#pragma unroll
        for (int e = 0; e < 4; ++e)
        {
            m = max_abs(m, v[e]);
        }
    }
    uint32_t const own = wave_max_bits(m);
    if ((threadIdx.x & 63) == 0)
    {
        part[threadIdx.x >> 6] = own;
    }
    __syncthreads();
    float scale;
    RowScale const r = row_scale(max(max(part[0], part[1]), max(part[2], part[3])), scale);
    if (threadIdx.x == 0)
    {
        scales[t] = scale;
    }
    for (int c = threadIdx.x * 8; c < C; c += 256 * 8)
    {
        *reinterpret_cast<u32x2*>(out + t * C + c) = quantize8(*reinterpret_cast<f16x8 const*>(src + c), r);
    }
}

int check_quantize(char const* what, int32_t T, int32_t C, void const* in, int64_t stride, void const* out, void const* scales)
{
    if (T < 0 || C <= 0 || C % 32 != 0)
    {
        return set_error(TRTAMD_STATUS_BAD_PARAM, "%s: T=%d C=%d (C must be a positive multiple of 32)", what, T, C);
    }
    if (stride < C || stride % 8 != 0)
    {
        return set_error(TRTAMD_STATUS_BAD_PARAM, "%s: row stride %lld (a multiple of 8, no less than %d)", what,
            (long long) stride, C);
    }
    if (T == 0)
    {
        return TRTAMD_STATUS_SUCCESS; // tensors without a token may have no address
    }
    if (in == nullptr || out == nullptr || scales == nullptr)
    {
        return set_error(TRTAMD_STATUS_BAD_PARAM, "%s: null pointer", what);
    }
    if (!aligned16(in) || !aligned16(out) || (reinterpret_cast<uintptr_t>(scales) & 3u) != 0)
    {
        return set_error(TRTAMD_STATUS_BAD_PARAM, "%s: pointers must be 16-byte aligned (scales: 4)", what);
    }
    return TRTAMD_STATUS_SUCCESS;
}

int launch_quantize(trtamd_stream_t stream, int32_t T, int32_t C, trtamd_half_t const* in, int64_t stride, int8_t* out, float* scales)
{
    hipLaunchKernelGGL(token_quantize_kernel, dim3((unsigned) T), dim3(256), 0, as_stream(stream),
        reinterpret_cast<f16 const*>(in), stride, C, out, scales);
    return check_launch("token_quantize_kernel");
}

// The workspace of a dynamic layer: the quantised tokens, then their scales.
size_t quantized_bytes(int32_t T, int32_t K)
{
    return ((size_t) T * K + 255) / 256 * 256;
}

} // namespace
} // namespace trtamd

using namespace trtamd;

extern "C" int trtamd_quantize_fp16_per_token(trtamd_stream_t stream, int32_t T, int32_t C, trtamd_half_t const* in,
    int64_t in_stride, int8_t* out, float* scales)
{
    int const st = check_quantize("quantize_fp16_per_token", T, C, in, in_stride, out, scales);
    return st || T == 0 ? st : launch_quantize(stream, T, C, in, in_stride, out, scales);
}

extern "C" size_t trtamd_int8_dynamic_linear_workspace_size(int32_t T, int32_t K, int32_t N)
{
    return T > 0 && K > 0 && N > 0 ? quantized_bytes(T, K) + (size_t) T * sizeof(float) : 0;
}

extern "C" int trtamd_int8_dynamic_linear(trtamd_stream_t stream, trtamd_int8_dynamic_linear_params const* p)
{
    if (p == nullptr)
    {
        return set_error(TRTAMD_STATUS_BAD_PARAM, "int8_dynamic_linear: null pointer");
    }
    if (p->T > 0
        && (p->workspace == nullptr || !aligned16(p->workspace)
            || p->workspace_bytes < trtamd_int8_dynamic_linear_workspace_size(p->T, p->K, p->N)))
    {
        return set_error(TRTAMD_STATUS_BAD_PARAM, "int8_dynamic_linear: T=%d K=%d N=%d need a 16-byte aligned workspace of %zu bytes",
            p->T, p->K, p->N, trtamd_int8_dynamic_linear_workspace_size(p->T, p->K, p->N));
    }
    int8_t* const quantized = static_cast<int8_t*>(p->workspace);
    float* const scales = p->T > 0 ? reinterpret_cast<float*>(quantized + quantized_bytes(p->T, p->K)) : nullptr;
    trtamd_int8_token_linear_params const q = {quantized, p->w, scales, p->channel_scale, p->bias, p->out, p->T, p->K, p->N, p->epilogue};
    int st = int8_token_linear_check(q);
    st = st ? st : check_quantize("int8_dynamic_linear", p->T, p->K, p->a, p->a_stride, quantized, scales);
    if (st || p->T == 0)
    {
        return st;
    }
    st = launch_quantize(stream, p->T, p->K, p->a, p->a_stride, quantized, scales);
    return st ? st : trtamd_int8_token_linear(stream, &q);
}
