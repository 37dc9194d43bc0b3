// INT8 linear layers on FP16 activations that are quantised token by token: the quantiser and the token-scaled layer behind it,
// or for few tokens both in one launch.
#include "device_utils.hpp"
#include "host_utils.hpp"
#include "network_ops.hpp"
#include "token_ops.hpp"
#include "trtamd_encoder_ops.h"

namespace trtamd
{
namespace
{

// ---- Few tokens ----
//
// A launch of its own for the quantiser is as long as the layer itself (1024 -> 4096 channels, one token: 2.5 of 5.1 us, and 3
// us of the host), so every workgroup quantises all tokens for itself.  What bounds it is one trip to memory for the weights,
// which are requested before the tokens are looked at.
//
// A workgroup has 16 output channels and 16 TB tokens.  Its eight wavefronts share k: wavefront w multiplies the stretches w, w
// + 8, .. of 128 values with v_mfma_i32_16x16x64_i8, whose operands are 16 values of one row per lane: weights, and tokens that
// the lane has quantised itself.  They meet twice in LDS, for the tokens' maxima and for the sums.
constexpr int kFewWaves = 8;
constexpr int kFewK = 128 * kFewWaves; // values of k in one stretch of each wavefront

// D: stretches a wavefront has at most, all of them in registers.
template <bool GELU, int TB, int D>
__global__ __launch_bounds__(kFewWaves * 64) void dynamic_few_kernel(uint64_t const aAddress, uint64_t const wAddress, int64_t const stride,
    int const T, int const K, int const N, float const* channelScale, float const* bias, f16* out)
{
    __shared__ i32x4 part[kFewWaves][TB][64];
    __shared__ uint32_t tops[kFewWaves][TB][16];
    int const lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int const row = lane & 15, group = lane >> 4;
    int const n0 = (int) blockIdx.x * 16;

    // Both operands' lanes hold the values 16 group .. +15 of either half of a stretch.  Loads come back in order, and the
    // tokens are needed first.  Columns behind the last token are the last one's; their sums are not used.  What lies behind
    // the last value is the last half of a stretch again, which is loaded (the maxima stay what they are) and not multiplied:
    // no load stands behind a branch.
    f16 const* const a = global_ptr<f16 const>(aAddress) + group * 16;
    int8_t const* const w = global_ptr<int8_t const>(wAddress) + (size_t) (n0 + row) * K + group * 16;
    auto const k_of = [&](int d, int h) { return (wave + d * kFewWaves) * 128 + h * 64; };
    u32x4 x[TB][D][2][2];
    i32x4 weights[D][2];
#pragma unroll
    for (int b = 0; b < TB; ++b)
    {
        f16 const* const token = a + min(16 * b + row, T - 1) * stride;
#pragma unroll
        for (int d = 0; d < D; ++d)
        {
#pragma unroll
            for (int h = 0; h < 2; ++h)
            {
                u32x4 const* const from = reinterpret_cast<u32x4 const*>(token + min(k_of(d, h), K - 64));
                x[b][d][h][0] = from[0];
                x[b][d][h][1] = from[1];
            }
        }
    }
#pragma unroll
    for (int d = 0; d < D; ++d)
    {
#pragma unroll
        for (int h = 0; h < 2; ++h)
        {
            weights[d][h] = *reinterpret_cast<i32x4 const*>(w + min(k_of(d, h), K - 64));
        }
    }
    f32x4 al = {}, be = {};
    if (wave < TB)
    {
        al = *reinterpret_cast<f32x4 const*>(channelScale + n0 + 4 * group);
        if (bias)
        {
            be = *reinterpret_cast<f32x4 const*>(bias + n0 + 4 * group);
        }
    }

    // maxima: over the four lanes of a token, then over the wavefronts
    auto const larger = [](uint32_t p, uint32_t q) { return max(p, q); };
#pragma unroll
    for (int b = 0; b < TB; ++b)
    {
        u16x2 m = {0, 0};
#pragma unroll
        for (int d = 0; d < D; ++d)
        {
#pragma unroll
            for (int h = 0; h < 2; ++h)
            {
                m = max_abs(max_abs(m, x[b][d][h][0]), x[b][d][h][1]);
            }
        }
        uint32_t const top = reduce_step<32>(reduce_step<16>(max((uint32_t) m[0], (uint32_t) m[1]), larger), larger);
        if (lane < 16)
        {
            tops[wave][b][lane] = top;
        }
    }
    __syncthreads();
    RowScale r[TB];
    float scale[TB];
#pragma unroll
    for (int b = 0; b < TB; ++b)
    {
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < kFewWaves; ++i)
        {
            top = max(top, tops[i][b][row]);
        }
        r[b] = row_scale(top, scale[b]);
    }

    i32x4 acc[TB] = {};
#pragma unroll
    for (int d = 0; d < D; ++d)
    {
#pragma unroll
        for (int h = 0; h < 2; ++h)
        {
            if (k_of(d, h) < K) // uniform
            {
#pragma unroll
                for (int b = 0; b < TB; ++b)
                {
                    u32x2 const lo = quantize8(bits_as<f16x8>(x[b][d][h][0]), r[b]), hi = quantize8(bits_as<f16x8>(x[b][d][h][1]), r[b]);
                    i32x4 const q = {(int) lo[0], (int) lo[1], (int) hi[0], (int) hi[1]};
                    acc[b] = __builtin_amdgcn_mfma_i32_16x16x64_i8(weights[d][h], q, acc[b], 0, 0, 0);
                }
            }
        }
    }
#pragma unroll
    for (int b = 0; b < TB; ++b)
    {
        part[wave][b][lane] = acc[b];
    }
    __syncthreads();
    // wavefront b adds up and stores block b; register e: channel 4 group + e, token `row`, whose scale this lane has worked out
#pragma unroll
    for (int b = 0; b < TB; ++b)
    {
        int const t = 16 * b + row;
        if (wave == b && t < T)
        {
            i32x4 sum = part[0][b][lane];
#pragma unroll
            for (int i = 1; i < kFewWaves; ++i)
            {
                sum += part[i][b][lane];
            }
            *reinterpret_cast<u32x2*>(out + (size_t) t * N + n0 + 4 * group) = token_results<GELU>(sum, scale[b], al, be);
        }
    }
}

// Where one launch takes about as long as two on the GPU or less (the host's 3 us are saved either way): 32768 values at most
// and no more weights than one round of workgroups has, in two blocks of tokens only rows of one stretch and no more workgroups
// than CUs.  us, graph replays, one launch / two: 1 x 1024 -> 4096 3.4 / 5.2, 16 x 1024 -> 4096 4.1 / 5.3, 1 x 4096 -> 1024 6.4
// / 6.8, 8 x 4096 -> 1024 7.7 / 7.2, 16 x 2048 -> 1024 5.5 / 5.9, 32 x 1024 -> 4096 5.7 / 5.5; not taken: 16 x 4096 -> 1024 9.1
// / 7.1, 32 x 2048 -> 1024 8.4 / 6.2, 32 x 1024 -> 8192 7.9 / 5.5, 64 x 1024 -> 4096 8.9 / 5.7, 1 x 4096 -> 16384 17.5 / 14.4.
bool few_tokens(trtamd_int8_dynamic_linear_params const& p)
{
    if (p.T <= 16)
    {
        return p.K <= 4 * kFewK && p.T * p.K <= 8 * 4 * kFewK && (int64_t) p.N * p.K <= (int64_t) 16 * num_cus() * 4 * kFewK;
    }
    return p.T <= 32 && p.K <= kFewK && p.N <= 16 * num_cus();
}

template <int TB, int D>
int launch_few(trtamd_stream_t stream, trtamd_int8_dynamic_linear_params const& p)
{
    auto const kernel = p.epilogue == TRTAMD_LINEAR_GELU ? dynamic_few_kernel<true, TB, D> : dynamic_few_kernel<false, TB, D>;
    hipLaunchKernelGGL(kernel, dim3((unsigned) (p.N / 16)), dim3(kFewWaves * 64), 0, as_stream(stream), address(p.a), address(p.w),
        p.a_stride, p.T, p.K, p.N, p.channel_scale, p.bias, reinterpret_cast<f16*>(p.out));
    return check_launch("dynamic_few_kernel");
}

int dynamic_few(trtamd_stream_t stream, trtamd_int8_dynamic_linear_params const& p)
{
    if (p.T > 16)
    {
        return launch_few<2, 1>(stream, p);
    }
    return p.K <= kFewK ? launch_few<1, 1>(stream, p) : p.K <= 2 * kFewK ? launch_few<1, 2>(stream, p) : launch_few<1, 4>(stream, p);
}

// The workspace of a dynamic layer: the quantised tokens, then their scales.
size_t quantized_bytes(int32_t T, int32_t K)
{
    return ((size_t) T * K + 255) / 256 * 256;
}

} // namespace
} // namespace trtamd

using namespace trtamd;

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
    int st = int8_token_linear_check("int8_dynamic_linear", q);
    st = st ? st : token_quantize_check("int8_dynamic_linear", p->T, p->K, p->a, p->a_stride, quantized, scales);
    if (st || p->T == 0)
    {
        return st;
    }
    if (few_tokens(*p))
    {
        return dynamic_few(stream, *p);
    }
    st = token_quantize(stream, p->T, p->K, p->a, p->a_stride, quantized, scales);
    return st ? st : trtamd_int8_token_linear(stream, &q);
}
