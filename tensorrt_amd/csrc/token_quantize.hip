// Quantisation of FP16 activations to INT8 with a scale for each token.
//
//   amax[t] = max_c |x[t][c]|,   s[t] = amax[t] / 127,   q[t][c] = rne(127 x[t][c] / amax[t])
//
// HBM streaming of 2 bytes in and 1 byte out per value.
#include "device_utils.hpp"
#include "host_utils.hpp"
#include "network_ops.hpp"
#include "token_ops.hpp"
#include "trtamd_encoder_ops.h"

#include <type_traits>

namespace trtamd
{
namespace
{

// Rows whose values stay in registers between the maximum and the quotients: WPR wavefronts a row, NV chunks of 8 values a lane.
// PAST_CACHE: loads that leave nothing in the caches; `through`: stores through the L2.
template <int WPR, int NV, bool PAST_CACHE>
__global__ __launch_bounds__(256) void token_quantize_kernel(f16 const* __restrict__ in, int64_t stride, int T, int C, int8_t* __restrict__ out,
    float* __restrict__ scales, bool through)
{
    constexpr int kRows = 4 / WPR;
    int const lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int const part = (wave % WPR) * 64 + lane;
    size_t const t = (size_t) blockIdx.x * kRows + wave / WPR;
    if (t >= (size_t) T)
    {
        return; // WPR = 4: none; otherwise no barrier follows
    }
    f16 const* src = in + t * stride;
    u32x4 v[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i)
    {
        int const c = (part + i * 64 * WPR) * 8;
        u32x4 const* const from = reinterpret_cast<u32x4 const*>(src + (c < C ? c : 0)); // twice the first chunk leaves the maximum as it is
        v[i] = PAST_CACHE ? __builtin_nontemporal_load(from) : *from;
    }
    u16x2 m = {0, 0};
#pragma unroll
    for (int i = 0; i < NV; ++i)
    {
        m = max_abs(m, v[i]);
    }
    uint32_t top = wave_max_bits(m);
    if constexpr (WPR > 1)
    {
        __shared__ uint32_t tops[4];
        static_assert(WPR == 4, "one row a workgroup");
        if (lane == 0)
        {
            tops[wave] = top;
        }
        __syncthreads();
        top = max(max(tops[0], tops[1]), max(tops[2], tops[3]));
    }
    float scale;
    RowScale const r = row_scale(top, scale);
    if (part == 0)
    {
        scales[t] = scale;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
    {
        int const c = (part + i * 64 * WPR) * 8;
        if (c < C)
        {
            u32x2 const q = quantize8(bits_as<f16x8>(v[i]), r);
            if (through)
            {
                store_through_l2(out + t * C + c, q);
            }
            else
            {
                *reinterpret_cast<u32x2*>(out + t * C + c) = q;
            }
        }
    }
}

// Rows of any length, read twice, a workgroup each.
__global__ __launch_bounds__(256) void token_quantize_long_kernel(
    f16 const* __restrict__ in, int64_t stride, int T, int C, int8_t* __restrict__ out, float* __restrict__ scales, bool)
{
    __shared__ uint32_t part[4];
    size_t const t = blockIdx.x;
    f16 const* src = in + t * stride;
    u16x2 m = {0, 0};
    for (int c = threadIdx.x * 8; c < C; c += 256 * 8)
    {
        m = max_abs(m, *reinterpret_cast<u32x4 const*>(src + c));
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

} // namespace

int token_quantize_check(
    char const* what, int32_t T, int32_t C, void const* in, int64_t stride, void const* out, void const* scales)
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
    if (T >= 1 << 24 || C >= 1 << 30)
    {
        return set_error(TRTAMD_STATUS_NOT_SUPPORTED, "%s: 2^24 tokens or 2^30 values of one or more", what); // a launch has 2^32 threads
    }
    if (!aligned16(in) || !aligned16(out) || (reinterpret_cast<uintptr_t>(scales) & 3u) != 0)
    {
        return set_error(TRTAMD_STATUS_BAD_PARAM, "%s: pointers must be 16-byte aligned (scales: 4)", what);
    }
    return TRTAMD_STATUS_SUCCESS;
}

int token_quantize(trtamd_stream_t stream, int32_t T, int32_t C, trtamd_half_t const* in, int64_t stride, int8_t* out, float* scales)
{
    bool const few = T <= 4 * num_cus();
    // Tokens of more than a quarter of the last-level cache push out what the layer behind them could find there; below that
    // stores that stay in the L2 are written back when the kernel has nothing else to do, which launches that do not fill the chip
    // do not notice.  Whole layers (projection, feed-forward layers, quantisers, norms) of 33289 tokens of 1024 and 4096 values 537 -> 520
    // us, 16384 of them 257 -> 247, 33289 of 768 and 2304 299 -> 295, 4963 of them 61.0 -> 60.4, 1500 of 1024 49.1 -> 48.7.
    bool const pastCache = (int64_t) T * C * (int64_t) sizeof(f16) > (int64_t) 64 << 20;
    auto const run = [&](auto kernel, int rows) {
        hipLaunchKernelGGL(kernel, dim3((unsigned) ceil_div(T, rows)), dim3(256), 0, as_stream(stream),
            reinterpret_cast<f16 const*>(in), stride, T, C, out, scales, !few && !pastCache);
        return check_launch("token_quantize_kernel");
    };
    // A wavefront a row where it holds one; four from 1025 values on where there are too few rows to fill the chip (graph replays,
    // 1024 tokens of 4096: 3.8 us against 4.4; of 1024 values: 3.0 against 2.7), which are never past the cache.
    if (few && C > 1024 && C <= 4096)
    {
        return C <= 2048 ? run(token_quantize_kernel<4, 1, false>, 1) : run(token_quantize_kernel<4, 2, false>, 1);
    }
    if (C > 16384)
    {
        return run(token_quantize_long_kernel, 1);
    }
    auto const by_length = [&](auto past) {
        constexpr bool P = decltype(past)::value;
        return C <= 512 ? run(token_quantize_kernel<1, 1, P>, 4)
            : C <= 1024 ? run(token_quantize_kernel<1, 2, P>, 4)
            : C <= 2048 ? run(token_quantize_kernel<1, 4, P>, 4)
            : C <= 4096 ? run(token_quantize_kernel<1, 8, P>, 4)
            : C <= 8192 ? run(token_quantize_kernel<4, 4, P>, 1)
                        : run(token_quantize_kernel<4, 8, P>, 1);
    };
    return pastCache ? by_length(std::true_type{}) : by_length(std::false_type{});
}

} // namespace trtamd

using namespace trtamd;

extern "C" int trtamd_quantize_fp16_per_token(trtamd_stream_t stream, int32_t T, int32_t C, trtamd_half_t const* in,
    int64_t in_stride, int8_t* out, float* scales)
{
    int const st = token_quantize_check("quantize_fp16_per_token", T, C, in, in_stride, out, scales);
    return st || T == 0 ? st : token_quantize(stream, T, C, in, in_stride, out, scales);
}
