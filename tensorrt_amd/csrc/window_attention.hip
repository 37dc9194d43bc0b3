// Attention in windows over packed sequences in FP16.
//
//   o_i = sum_j 2^(c s_ij - m) v_j / sum_j 2^(c s_ij - m),   s_ij = scale * q_i k_j,   c = log2(e),
//   over i - left <= j <= i + right and j < min(sinks, i + right + 1)
//
// 128 rows of a key head a workgroup, (token, query head) with the heads of a group side by side, 32 a wavefront
// (attention_rows.hpp). Keys and values come in chunks of 64 straight into LDS, in two slots; of the keys in front of a tile's
// windows only the chunks with sinks. Values lie in LDS as in memory and become the second product's operand by transposing reads.
// What bounds it: long windows the matrix and the vector instructions (34 and 35 % of the cycles, in turns), short ones the trips to memory
// of a workgroup's few chunks. 8001 tokens of 16 heads of 128 on 4, 1024 keys back and 4 sinks: 260 us with branches on the head size
// between the products, 99 without, 91 with rows of LDS in all 64 banks and masks as bits (694 TFLOP/s); all 8001 keys, causal, 302 (869). 128
// sequences, 16621 tokens, 16 heads of 64, 64 keys on either side: 44 us (3.1 TB/s), 2 to 4 workgroups a CU at once; a third slot of LDS
// instead of the fourth workgroup 47, both, with 34 registers spilled, 99.
#include "attention_rows.hpp"
#include "host_utils.hpp"
#include "trtamd_encoder_ops.h"

#include <algorithm>
#include <cmath>

namespace trtamd
{
namespace
{

typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef short i16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) i16x4 lds_i16x4;

constexpr int kThreads = 256, kWaves = kThreads / kWaveSize;
constexpr int kTileRows = 128;
__device__ u32x4 const kZeros[1] = {}; // 8 binary16 zeros, in memory

struct Rows
{
    uint8_t const* p;    // FP16
    int64_t token, head; // bytes
};

struct WindowArgs
{
    Rows q, k, v;
    uint8_t* out;
    int64_t outToken, outHead; // bytes
    int32_t const* cu;
    int32_t T, maxTokens, d;
    int32_t left, right, sinks; // beyond any length where there is no limit
    float scale;                // in powers of 2
    bool near;                  // whole chunks lie within 32-bit offsets, and heads fill their rows in LDS
    FastDiv group, kvHeads;
};

template <int DP>
struct WindowLds
{
    static constexpr int kRow = 2 * DP;
    static constexpr int kMatrix = kChunkKeys * kRow;
    static constexpr int kTotal = 4 * kMatrix;
};

// One row over the keys it sees and no others, a lane's elements lane, lane + 64, ..: what rows take that have infinities or NaNs
// near them, where a weight of 0 in the products above is not enough. A key is a trip to memory: 8001 tokens of 16 heads of 128 in windows of
// 1024, all of them NaN, 38 ms.
template <int DP>
__device__ void one_row(WindowArgs const& a, int first, int token, int head, int kvHead, Seen const& seen)
{
    constexpr int N = (DP + 63) / 64;
    int const lane = threadIdx.x & 63;
    auto load = [&](Rows const& r, int t, int h, float (&x)[N]) {
        f16 const* const from = reinterpret_cast<f16 const*>(r.p + (int64_t) (first + t) * r.token + (int64_t) h * r.head);
#pragma unroll
        for (int e = 0; e < N; ++e)
        {
            x[e] = lane + 64 * e < a.d ? (float) from[lane + 64 * e] : 0.f;
        }
    };
    float q[N], o[N] = {};
    load(a.q, token, head, q);
    float negMax = kNothingSeen, sum = 0.f;
    int const sinks = min(seen.sinks, min(seen.lo, seen.hi));
    for (int key = sinks > 0 ? 0 : seen.lo; key < seen.hi; key = key + 1 == sinks ? max(seen.lo, sinks) : key + 1)
    {
        float x[N], s = 0.f;
        load(a.k, key, kvHead, x);
#pragma unroll
        for (int e = 0; e < N; ++e)
        {
            s = lane + 64 * e < a.d ? fmaf(q[e], x[e], s) : s;
        }
        s = wave_sum(s) * a.scale;
        float const to = fminf(negMax, fminf(-s, kNothingSeen));
        float const by = __builtin_amdgcn_exp2f(to - negMax), w = __builtin_amdgcn_exp2f(s + to);
        load(a.v, key, kvHead, x);
#pragma unroll
        for (int e = 0; e < N; ++e)
        {
            o[e] = fmaf(w, x[e], o[e] * by);
        }
        sum = fmaf(sum, by, w);
        negMax = to;
    }
    f16* const out = reinterpret_cast<f16*>(a.out + (int64_t) (first + token) * a.outToken + (int64_t) head * a.outHead);
#pragma unroll
    for (int e = 0; e < N; ++e)
    {
        if (lane + 64 * e < a.d)
        {
            out[lane + 64 * e] = (f16) (sum == 0.f ? 0.f : o[e] / sum);
        }
    }
}

template <int KS /* 16 of the head's values */>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(KS <= 4 ? 4 : KS <= 8 ? 2 : 1))) void window_attention_kernel(
    WindowArgs const a)
{
    constexpr int DP = padded_head(KS);
    using Lds = WindowLds<DP>;
    constexpr int kRow = Lds::kRow, DV = (KS + 1) / 2;
    constexpr int kChunks = DP / 8;              // of 16 bytes in a row
    constexpr int kRowsPerLoad = 64 / kChunks;   // of a wavefront's load into LDS
    constexpr int NL = kChunkKeys / kRowsPerLoad / kWaves;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    int const b = blockIdx.z;
    int const first = min(max(a.cu[b], 0), a.T);
    int const n = min(min(max(a.cu[b + 1], first), a.T) - first, a.maxTokens);
    int const group = a.group.d;
    int const rows = n * group;
    int const fromEnd = (int) (blockIdx.x / a.kvHeads), h = (int) (blockIdx.x - fromEnd * a.kvHeads.d);
    int const tiles = (int) (((int64_t) rows + kTileRows - 1) / kTileRows);
    if (fromEnd >= tiles)
    {
        return;
    }
    int const row0 = (tiles - 1 - fromEnd) * kTileRows, rowEnd = min(row0 + kTileRows, rows);
    auto seen_by = [&](int row) {
        int const i = (int) ((uint32_t) row / a.group);
        return Seen{max(i - a.left, 0), (int) min((int64_t) i + a.right + 1, (int64_t) n), a.sinks};
    };
    Chunks const chunks = chunks_of(seen_by(row0).lo, seen_by(rowEnd - 1).hi, a.sinks);
    int const tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int const lq = lane & 31, half = lane >> 5;
    int const wRow = row0 + 32 * wave;
    bool const active = wRow < rowEnd;
    int const row = min(wRow + lq, rowEnd - 1);
    int const token = (int) ((uint32_t) row / a.group), head = h * group + row - token * group;
    Seen const seen = seen_by(row), least = seen_by(min(wRow, rowEnd - 1)), most = seen_by(min(wRow + 31, rowEnd - 1));

    f16x8 q[KS]; // row lq, elements 16 s + 8 half .. + 7
    {
        uint8_t const* const from = a.q.p + (int64_t) (first + token) * a.q.token + (int64_t) head * a.q.head;
#pragma unroll
        for (int s = 0; s < KS; ++s)
        {
            q[s] = f16x8{};
            if (16 * s + 8 * half < a.d)
            {
                q[s] = *reinterpret_cast<f16x8 const*>(from + 2 * (16 * s + 8 * half));
            }
        }
    }

    uint32_t const ldsBase = (uint32_t) (size_t) (lds_u8*) lds;
    int const rowInLoad = lane / kChunks, place = lane & (kChunks - 1);
    // where this lane's pieces of a whole chunk lie from its first row on
    uint32_t kAt[NL], vAt[NL];
#pragma unroll
    for (int l = 0; l < NL; ++l)
    {
        int const r = (l * kWaves + wave) * kRowsPerLoad + rowInLoad;
        // both are their own inverses
        kAt[l] = (uint32_t) ((r & 32) + key_of_row(r & 31)) * (uint32_t) a.k.token + 16u * (uint32_t) swizzled<kRow>(r, place);
        vAt[l] = (uint32_t) r * (uint32_t) a.v.token + 16u * (uint32_t) swizzled_turned<kRow>(r, place);
    }
    uint8_t const* const kUnit = a.k.p + (int64_t) first * a.k.token + (int64_t) h * a.k.head;
    uint8_t const* const vUnit = a.v.p + (int64_t) first * a.v.token + (int64_t) h * a.v.head;
    auto request = [&](int i, int slot) {
        int const key0 = chunks.key0(i);
        uint32_t const to = ldsBase + (uint32_t) (2 * slot * Lds::kMatrix);
        if (a.near && key0 + kChunkKeys <= n)
        {
#pragma unroll
            for (int l = 0; l < NL; ++l)
            {
                uint32_t const at = to + (uint32_t) ((l * kWaves + wave) * kRowsPerLoad * kRow);
                load_to_lds16_sbase(kUnit + (int64_t) key0 * a.k.token, kAt[l], at);
                load_to_lds16_sbase(vUnit + (int64_t) key0 * a.v.token, vAt[l], at + (uint32_t) Lds::kMatrix);
            }
            return;
        }
#pragma unroll
        for (int l = 0; l < NL; ++l)
        {
            int const r0 = (l * kWaves + wave) * kRowsPerLoad, r = r0 + rowInLoad;
            int const kChunk = swizzled<kRow>(r, place), vChunk = swizzled_turned<kRow>(r, place);
            int const kKey = min(key0 + (r & 32) + key_of_row(r & 31), n - 1), vKey = key0 + r;
            uint8_t const* const k = kUnit + (int64_t) kKey * a.k.token + 16 * kChunk;
            // 0, the weight of a key behind the sequence, times an infinite value would not be 0
            uint8_t const* const v = vUnit + (int64_t) vKey * a.v.token + 16 * vChunk;
            uint8_t const* const zeros = reinterpret_cast<uint8_t const*>(kZeros);
            load_to_lds16(8 * kChunk < a.d ? k : zeros, to + (uint32_t) (r0 * kRow));
            load_to_lds16(8 * vChunk < a.d && vKey < n ? v : zeros, to + (uint32_t) (Lds::kMatrix + r0 * kRow));
        }
    };

    RowSums<DV> sums;
    sums.clear();
    int const tr = (lane & 15) >> 2; // transposing reads: 16 lanes take 4 rows of 16 elements
    int const trChunk = 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1), trByte = (lane & 1) * 8;
    if (chunks.total > 0)
    {
        request(0, 0);
    }
    for (int i = 0; i < chunks.total; ++i)
    {
        wait_vmcnt<0>();
        __syncthreads(); // everybody's rows of chunk i have landed, and everybody has read chunk i - 1
        int const key0 = chunks.key0(i);
        uint8_t const* const keys = lds + 2 * (i & 1) * Lds::kMatrix;
        uint8_t const* const values = keys + Lds::kMatrix;
        if (i + 1 < chunks.total)
        {
            request(i + 1, (i + 1) & 1);
        }
        if (!active || key0 >= most.hi || (key0 + kChunkKeys <= least.lo && key0 >= a.sinks))
        {
            continue;
        }
        f32x16 s[2];
#pragma unroll
        for (int v = 0; v < 16; ++v)
        {
            s[0][v] = s[1][v] = 0.f;
        }
#pragma unroll
        for (int e = 0; e < KS; ++e)
        {
#pragma unroll
            for (int t = 0; t < 2; ++t)
            {
                int const kRowAt = 32 * t + lq;
                f16x8 const k = *reinterpret_cast<f16x8 const*>(keys + kRowAt * kRow + 16 * swizzled<kRow>(kRowAt, 2 * e + half));
                s[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, q[e], s[t], 0, 0, 0);
            }
        }
        if (!(key0 + kChunkKeys <= least.hi && (key0 >= most.lo || key0 + kChunkKeys <= a.sinks)))
        {
            hide(s, seen, key0 + 16 * half, 16, 16);
        }
        float mx = -__builtin_inff();
#pragma unroll
        for (int v = 0; v < 32; ++v)
        {
            mx = fmaxf(mx, s[v >> 4][v & 15]);
        }
        sums.move(reduce_step<32>(mx, max_of) * a.scale);
#pragma unroll
        for (int t = 0; t < 2; ++t)
        {
#pragma unroll
            for (int w = 0; w < 2; ++w)
            {
                float p[8];
#pragma unroll
                for (int e = 0; e < 8; ++e)
                {
                    p[e] = __builtin_amdgcn_exp2f(fmaf(s[t][8 * w + e], a.scale, sums.negMax));
                    sums.sum += p[e];
                }
                f16x8 const weights = weights_f16(p);
#pragma unroll
                for (int d = 0; d < DV; ++d)
                {
                    int const r = 32 * t + 16 * half + 8 * w + tr;
                    i16x4 const lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                        (lds_i16x4*) (values + r * kRow + 16 * swizzled_turned<kRow>(r, 4 * d + trChunk) + trByte));
                    i16x4 const hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                        (lds_i16x4*) (values + (r + 4) * kRow + 16 * swizzled_turned<kRow>(r + 4, 4 * d + trChunk) + trByte));
                    i16x8 const both = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
                    sums.out[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(bits_as<f16x8>(both), weights, sums.out[d], 0, 0, 0);
                }
            }
        }
    }
    if (!active)
    {
        return;
    }
    float const total = reduce_step<32>(sums.sum, [](float x, float y) { return x + y; });
    float const inverse = total == 0.f ? 0.f : 1.f / total;
    f16x4 y[4 * DV];
    // Whatever is not finite leaves a NaN here: an infinity of a value that is not seen leaves one in its row.
    float odd = inverse * 0.f;
#pragma unroll
    for (int i = 0; i < 4 * DV; ++i)
    {
        f32x16 const& o = sums.out[i >> 2];
        int const v = 4 * (i & 3);
        f16x2 const lo = __builtin_convertvector(f32x2{o[v] * inverse, o[v + 1] * inverse}, f16x2);
        f16x2 const hi = __builtin_convertvector(f32x2{o[v + 2] * inverse, o[v + 3] * inverse}, f16x2);
        odd = __builtin_amdgcn_fdot2(lo, f16x2{}, __builtin_amdgcn_fdot2(hi, f16x2{}, odd, false), false);
        y[i] = f16x4{lo[0], lo[1], hi[0], hi[1]};
    }
    if (__ballot(odd != 0.f) != 0)
    {
        for (int r = wRow; r < min(wRow + 32, rowEnd); ++r)
        {
            int const t = (int) ((uint32_t) r / a.group);
            one_row<DP>(a, first, t, h * group + r - t * group, h, seen_by(r));
        }
        return;
    }
    if (wRow + lq >= rowEnd)
    {
        return;
    }
    uint8_t* const to = a.out + (int64_t) (first + token) * a.outToken + (int64_t) head * a.outHead + 8 * half;
#pragma unroll
    for (int i = 0; i < 4 * DV; ++i)
    {
        if (8 * i + 4 * half < a.d)
        {
            *reinterpret_cast<f16x4*>(to + 16 * i) = y[i];
        }
    }
}

// LDS that a workgroup asks for where it needs `need` bytes. Fewer workgroups than the CUs could hold at once are not spread evenly by
// themselves: some CUs get as many as fit and others none. With no more than their share fitting they are: 16 sequences of up to 512, 12
// heads of 64, all keys (some 360 tiles) 20.0 us without, 17.2 with two a CU; 32 of up to 384 in windows (760) 17.1, three 15.4; 8
// (190) 10.7, one 9.9.
constexpr int kCuLds = 160 << 10, kMostLds = kCuLds / 2 + 1024;
size_t spreading_lds(size_t need, int64_t workgroups, int cus)
{
    int64_t const share = std::max<int64_t>((workgroups + cus - 1) / cus, 1);
    return share >= 4 ? need : std::max(need, (size_t) (kCuLds / (share + 1) + 1024));
}

template <int KS>
int launch(hipStream_t stream, dim3 grid, int64_t tiles, WindowArgs const& a)
{
    constexpr int kBytes = WindowLds<padded_head(KS)>::kTotal;
    if (int const st = reserve_lds<window_attention_kernel<KS>>("window_attention", std::max(kBytes, kMostLds)))
    {
        return st;
    }
    hipLaunchKernelGGL(window_attention_kernel<KS>, grid, dim3(kThreads), spreading_lds(kBytes, tiles, num_cus()), stream, a);
    return check_launch("window_attention_kernel");
}

int window_check(trtamd_window_attention_params const& p)
{
    char const* const what = "window_attention";
    if (p.B < 0 || p.T < 0 || p.max_tokens < 0)
    {
        return set_error(TRTAMD_STATUS_BAD_PARAM, "%s: B=%d T=%d max_tokens=%d", what, p.B, p.T, p.max_tokens);
    }
    if (p.kv_heads <= 0 || p.q_heads <= 0 || p.q_heads % p.kv_heads != 0)
    {
        return set_error(TRTAMD_STATUS_BAD_PARAM, "%s: q_heads=%d (a multiple of kv_heads=%d)", what, p.q_heads, p.kv_heads);
    }
    if (p.d <= 0 || p.d % 8 != 0 || p.d > 256)
    {
        return set_error(TRTAMD_STATUS_BAD_PARAM, "%s: d=%d (a multiple of 8, at most 256)", what, p.d);
    }
    if (!(p.scale >= 0.f) || !std::isfinite(p.scale))
    {
        return set_error(TRTAMD_STATUS_BAD_PARAM, "%s: scale %g (finite and not negative)", what, p.scale);
    }
    if (p.left < -1 || p.right < -1 || p.sinks < 0)
    {
        return set_error(TRTAMD_STATUS_BAD_PARAM, "%s: left=%d right=%d (-1 or more) sinks=%d", what, p.left, p.right, p.sinks);
    }
    for (int64_t s : {p.q_token_stride, p.q_head_stride, p.k_token_stride, p.k_head_stride, p.v_token_stride, p.v_head_stride,
             p.out_token_stride, p.out_head_stride})
    {
        if (s < 0 || s % 8 != 0)
        {
            return set_error(TRTAMD_STATUS_BAD_PARAM, "%s: strides must be multiples of 8 elements, and not negative", what);
        }
    }
    if (p.B == 0 || p.T == 0 || p.max_tokens == 0)
    {
        return TRTAMD_STATUS_SUCCESS;
    }
    if (p.B > 65535 || (int64_t) p.T * p.q_heads >= (int64_t) 1 << 30 || p.kv_heads > 65535) // a launch has 2^32 threads
    {
        return set_error(TRTAMD_STATUS_NOT_SUPPORTED, "%s: B=%d kv_heads=%d (at most 65535), T * q_heads=%lld (less than 2^30)", what, p.B, p.kv_heads,
            (long long) p.T * p.q_heads);
    }
    for (void const* x : {(void const*) p.q, (void const*) p.k, (void const*) p.v, (void const*) p.out, (void const*) p.cu_seqlens})
    {
        if (x == nullptr)
        {
            return set_error(TRTAMD_STATUS_BAD_PARAM, "%s: null pointer", what);
        }
    }
    if (!aligned16(p.q) || !aligned16(p.k) || !aligned16(p.v) || !aligned16(p.out) || (reinterpret_cast<uintptr_t>(p.cu_seqlens) & 3u) != 0)
    {
        return set_error(TRTAMD_STATUS_BAD_PARAM, "%s: pointers must be 16-byte aligned (cu_seqlens: 4)", what);
    }
    return TRTAMD_STATUS_SUCCESS;
}

} // namespace
} // namespace trtamd

using namespace trtamd;

extern "C" int trtamd_window_attention(trtamd_stream_t stream, trtamd_window_attention_params const* params)
{
    if (params == nullptr)
    {
        return set_error(TRTAMD_STATUS_BAD_PARAM, "window_attention: null params");
    }
    trtamd_window_attention_params const& p = *params;
    if (int const st = window_check(p))
    {
        return st;
    }
    if (p.B == 0 || p.T == 0 || p.max_tokens == 0)
    {
        return TRTAMD_STATUS_SUCCESS;
    }
    auto const rows = [](trtamd_half_t const* x, int64_t token, int64_t head) {
        return Rows{reinterpret_cast<uint8_t const*>(x), 2 * token, 2 * head};
    };
    WindowArgs a{};
    a.q = rows(p.q, p.q_token_stride, p.q_head_stride);
    a.k = rows(p.k, p.k_token_stride, p.k_head_stride);
    a.v = rows(p.v, p.v_token_stride, p.v_head_stride);
    a.out = reinterpret_cast<uint8_t*>(p.out);
    a.outToken = 2 * p.out_token_stride, a.outHead = 2 * p.out_head_stride;
    a.cu = p.cu_seqlens;
    a.T = p.T, a.maxTokens = p.max_tokens, a.d = p.d;
    a.left = p.left < 0 ? INT32_MAX : p.left;
    a.right = p.right < 0 ? INT32_MAX : p.right;
    a.sinks = p.sinks;
    // a scale of 0 times a score of -infinity is no number, nor is an infinite one times 0
    a.scale = std::min(std::max(p.scale * 1.44269504088896f, 0x1p-126f), kLargest);
    int const group = p.q_heads / p.kv_heads;
    a.group = fast_div((uint32_t) group);
    a.kvHeads = fast_div((uint32_t) p.kv_heads);
    int64_t const tiles = ceil_div((int64_t) std::min(p.max_tokens, p.T) * group, (int64_t) kTileRows);
    a.near = p.d == padded_head(head_steps(p.d)) && std::max(a.k.token, a.v.token) < (int64_t) 1 << 25;
    dim3 const grid((unsigned) (tiles * p.kv_heads), 1, (unsigned) p.B);
    // about as many tiles as there are: one of each sequence is half full
    int64_t const there = ((int64_t) p.T * group / kTileRows + (p.B + 1) / 2) * p.kv_heads;
    return by_head(p.d, [&](auto steps) { return launch<decltype(steps)::value>(as_stream(stream), grid, there, a); });
}
