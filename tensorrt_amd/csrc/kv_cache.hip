// The 8-bit cache of keys and values: new tokens quantised into its pages, and tokens read back.
//
//   scale[page][head] = max|x| / top,   byte = rne(x / scale);   a page that goes on keeps its scale, or doubles it until its new
//   values fit, and rounds what it held to that.
//
// Both are HBM streaming, of 2 bytes on one side and 1 on the other. A workgroup takes a page of a head, its keys or its values:
// they share a scale, so nothing is exchanged between workgroups, and whatever has to be read again lies in one place.
#include "host_utils.hpp"
#include "kv_cache.hpp"
#include "token_ops.hpp"

#include <algorithm>
#include <type_traits>

namespace trtamd
{
namespace
{

constexpr int kThreads = 256;

struct Strided
{
    uint8_t* p; // FP16
    int64_t token, head; // elements
};

struct CopyArgs
{
    CacheArgs cache;
    Strided kv[2];
    FastDiv chunks; // d / 8
};

template <bool FP8>
constexpr float kTop = FP8 ? 448.f : 127.f;

// Four values, already divided by their scale, as bytes.
template <bool FP8>
__device__ inline uint32_t round_codes(f32x4 y)
{
    if constexpr (FP8)
    {
#pragma unroll
        for (int e = 0; e < 4; ++e)
        {
            y[e] = __builtin_amdgcn_fmed3f(y[e], -448.f, 448.f);
        }
        int const lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
        return (uint32_t) __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], lo, true);
    }
    else
    {
        // 1.5 * 2^23 more: rounded to an integer, ties to even, in the lowest byte. What rounds to 128 is brought back before.
        uint32_t b[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
        {
            b[e] = bits_as<uint32_t>(__builtin_amdgcn_fmed3f(y[e], -127.f, 127.f) + 12582912.f);
        }
        return low_bytes(b[0], b[1], b[2], b[3]);
    }
}

// x is a NaN or an infinity only where inverse is 0 (see scale_of): 0 * it is a NaN, which is 0 as a byte.
template <bool FP8>
__device__ inline uint32_t quantize_codes(f16x4 x, float inverse)
{
    f32x4 y;
#pragma unroll
    for (int e = 0; e < 4; ++e)
    {
        y[e] = (float) x[e] * inverse;
    }
    return round_codes<FP8>(y);
}

// Bytes of a page whose scale became 2^n times itself, shrink = 2^-n.
template <bool FP8>
__device__ inline uint32_t requantize_codes(uint32_t w, float shrink)
{
    f16x4 const x = code_values<FP8>(w);
    return quantize_codes<FP8>(x, shrink);
}

struct PageScale
{
    float scale, inverse, shrink;
    bool grown, zeros; // what was held changes; new bytes are zeros
};

// bits: of the largest absolute value among the new ones, as binary16. old: the page's scale, or 0 where the new tokens begin it.
template <bool FP8>
__device__ inline PageScale page_scale(uint32_t bits, float old)
{
    PageScale r = {old, 0.f, 1.f, false, true};
    if (bits >= kF16Inf || old != old)
    {
        r.scale = __builtin_nanf("");
        return r;
    }
    float const a = (float) bits_as<f16>((uint16_t) bits), limit = old * kTop<FP8>;
    if (!(limit > 0.f))
    {
        r.scale = a / kTop<FP8>;
    }
    else if (a > limit)
    {
        int const n = __builtin_amdgcn_frexp_expf(a) - __builtin_amdgcn_frexp_expf(limit)
            + (__builtin_amdgcn_frexp_mantf(a) > __builtin_amdgcn_frexp_mantf(limit) ? 1 : 0);
        r.scale = __builtin_amdgcn_ldexpf(old, n);
        r.shrink = __builtin_amdgcn_ldexpf(1.f, -n);
        r.grown = true;
    }
    r.zeros = !(r.scale > 0.f);
    r.inverse = r.zeros ? 0.f : 1.f / r.scale;
    return r;
}

// The bytes of w whose bit in `take` is set from a, the others from b.
__device__ inline uint32_t merge_bytes(uint32_t a, uint32_t b, uint32_t take)
{
    uint32_t const m = ((take & 1u) | (take & 2u) << 7 | (take & 4u) << 14 | (take & 8u) << 21) * 255u;
    return (a & m) | (b & ~m);
}

// NV: chunks of 8 values a thread, P * d / 8 / 256 or more.
template <int NV, bool FP8>
__global__ __launch_bounds__(kThreads) void kv_cache_write_kernel(CopyArgs const a)
{
    extern __shared__ __attribute__((aligned(16))) uint8_t turned[]; // values: [d][P + 4] bytes
    __shared__ uint32_t tops[kThreads / kWaveSize];
    CacheArgs const& c = a.cache;
    int const b = blockIdx.y, h = blockIdx.z >> 1, which = blockIdx.z & 1;
    int const P = 1 << c.shift, tid = threadIdx.x;
    CacheRows const r = cache_rows(c, b);
    int const begin = max(r.begin, 0), end = min(r.begin + r.n, r.len);
    uint8_t const* const src = a.kv[which].p + 2 * (int64_t) h * a.kv[which].head;
    int const n8 = a.chunks.d;
    for (int64_t block = (begin >> c.shift) + blockIdx.x; block * P < end && block < c.maxPages; block += gridDim.x)
    {
        int const page = c.table[(int64_t) b * c.maxPages + block];
        if ((uint32_t) page >= (uint32_t) c.pages)
        {
            continue;
        }
        int const first = (int) block * P, lo = max(begin - first, 0), hi = min(end - first, P);
        float* const scaleAt = (which ? c.vScale : c.kScale) + (size_t) page * c.heads + h;
        uint8_t* const codes = (which ? c.v : c.k) + page_offset(c, page, h);
        float const old = lo > 0 ? *scaleAt : 0.f;
        f16x8 x[NV];
        u16x2 m = {0, 0};
#pragma unroll
        for (int i = 0; i < NV; ++i)
        {
            uint32_t const at = tid + i * kThreads, row = at / a.chunks, chunk = at - row * n8;
            int const token = lo + (int) row;
            x[i] = f16x8{};
            if (token < hi)
            {
                int64_t const t = (int64_t) r.row0 + (first + token - r.begin);
                x[i] = *reinterpret_cast<f16x8 const*>(src + 2 * (t * a.kv[which].token + 8 * chunk));
            }
            m = max_abs(m, bits_as<u32x4>(x[i]));
        }
        uint32_t const own = wave_max_bits(m);
        if ((tid & 63) == 0)
        {
            tops[tid >> 6] = own;
        }
        __syncthreads();
        PageScale const s = page_scale<FP8>(max(max(tops[0], tops[1]), max(tops[2], tops[3])), old);
        if (tid == 0)
        {
            *scaleAt = s.scale; // everybody has read it
        }
#pragma unroll
        for (int i = 0; i < NV; ++i)
        {
            uint32_t const at = tid + i * kThreads, row = at / a.chunks, chunk = at - row * n8;
            int const token = lo + (int) row;
            if (token >= hi)
            {
                continue;
            }
            u32x2 w = {quantize_codes<FP8>(f16x4{x[i][0], x[i][1], x[i][2], x[i][3]}, s.inverse),
                quantize_codes<FP8>(f16x4{x[i][4], x[i][5], x[i][6], x[i][7]}, s.inverse)};
            w = s.zeros ? u32x2{0, 0} : w;
            if (which == 0)
            {
                *reinterpret_cast<u32x2*>(codes + (uint32_t) token * c.d + 8 * chunk) = w;
            }
            else
            {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                {
                    turned[(8 * chunk + e) * (P + 4) + token] = (uint8_t) (w[e >> 2] >> (8 * (e & 3)));
                }
            }
        }
        if (which == 0)
        {
            for (uint32_t at = tid; s.grown && at < (uint32_t) lo * n8; at += kThreads)
            {
                u32x2* const p = reinterpret_cast<u32x2*>(codes) + at;
                *p = u32x2{requantize_codes<FP8>((*p)[0], s.shrink), requantize_codes<FP8>((*p)[1], s.shrink)};
            }
            __syncthreads(); // tops
            continue;
        }
        __syncthreads();
        // 16 tokens of a row at a time: the page and head are this workgroup's, so bytes on either side of the new ones are as well
        int const groups = P >> 4, from = (s.grown ? 0 : lo) >> 4, to = (hi + 15) >> 4;
        for (int at = tid; at < c.d * groups; at += kThreads)
        {
            int const row = at >> (c.shift - 4), group = at & (groups - 1);
            if (group < from || group >= to)
            {
                continue;
            }
            u32x4* const p = reinterpret_cast<u32x4*>(codes + (uint32_t) row * P) + group;
            uint32_t const* const t = reinterpret_cast<uint32_t const*>(turned + row * (P + 4) + 16 * group);
            int const l = min(max(lo - 16 * group, 0), 16), u = min(hi - 16 * group, 16);
            u32x4 w = {t[0], t[1], t[2], t[3]};
            if (l > 0 || u < 16)
            {
                uint32_t const isNew = l < u ? (1u << u) - (1u << l) : 0u;
                u32x4 const was = *p;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                {
                    // behind the new ones nothing is held: whatever lies there stays
                    uint32_t held = was[e];
                    if (s.grown)
                    {
                        held = merge_bytes(requantize_codes<FP8>(held, s.shrink), held, ((1u << l) - 1u) >> (4 * e));
                    }
                    w[e] = merge_bytes(w[e], held, isNew >> (4 * e));
                }
            }
            *p = w;
        }
        __syncthreads(); // tops and turned
    }
}

template <bool FP8>
__global__ __launch_bounds__(kThreads) void kv_cache_read_kernel(CopyArgs const a)
{
    extern __shared__ __attribute__((aligned(16))) uint8_t turned[]; // values: [d][P + 4] bytes
    CacheArgs const& c = a.cache;
    int const b = blockIdx.y, h = blockIdx.z >> 1, which = blockIdx.z & 1;
    int const P = 1 << c.shift, tid = threadIdx.x;
    CacheRows const r = cache_rows(c, b);
    uint8_t* const out = a.kv[which].p + 2 * (int64_t) h * a.kv[which].head;
    int const n8 = a.chunks.d;
    // by position, so that rows without a place in the table get their zeros as well
    int64_t const begin = r.begin, end = begin + r.n;
    for (int64_t block = (begin >> c.shift) + blockIdx.x; block * P < end; block += gridDim.x)
    {
        int const page = block >= 0 && block < c.maxPages ? c.table[(int64_t) b * c.maxPages + block] : -1;
        int64_t const first = block * P;
        int const lo = (int) max(begin - first, (int64_t) 0), hi = (int) min(end - first, (int64_t) P);
        bool const there = (uint32_t) page < (uint32_t) c.pages;
        int const at0 = there ? page : 0;
        float const scale = there ? (which ? c.vScale : c.kScale)[(size_t) at0 * c.heads + h] : 0.f;
        uint8_t const* const codes = (which ? c.v : c.k) + page_offset(c, at0, h);
        if (which && there)
        {
            int const groups = P >> 4, from = lo >> 4, to = (hi + 15) >> 4;
            for (int at = tid; at < c.d * groups; at += kThreads)
            {
                int const row = at >> (c.shift - 4), group = at & (groups - 1);
                if (group >= from && group < to)
                {
                    u32x4 const w = *(reinterpret_cast<u32x4 const*>(codes + (uint32_t) row * P) + group);
                    uint32_t* const t = reinterpret_cast<uint32_t*>(turned + row * (P + 4) + 16 * group);
                    t[0] = w[0], t[1] = w[1], t[2] = w[2], t[3] = w[3];
                }
            }
            __syncthreads();
        }
        for (uint32_t at = tid; at < (uint32_t) (hi - lo) * n8; at += kThreads)
        {
            uint32_t const row = at / a.chunks, chunk = at - row * n8;
            int const token = lo + (int) row;
            u32x2 w = {0, 0};
            if (there && which == 0)
            {
                w = *reinterpret_cast<u32x2 const*>(codes + (uint32_t) token * c.d + 8 * chunk);
            }
            else if (there)
            {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                {
                    w[e >> 2] |= (uint32_t) turned[(8 * chunk + e) * (P + 4) + token] << (8 * (e & 3));
                }
            }
            f16x8 const v = code_values8<FP8>(w[0], w[1]);
            f16x8 y;
#pragma unroll
            for (int e = 0; e < 8; ++e)
            {
                y[e] = (f16) ((float) v[e] * scale);
            }
            *reinterpret_cast<f16x8*>(out + 2 * ((r.row0 + (first + token - begin)) * a.kv[which].token + 8 * chunk)) = y;
        }
        __syncthreads(); // turned
    }
}

int copy_check(char const* what, trtamd_kv_cache const& c, void const* k, void const* v, int64_t const (&strides)[4])
{
    if (int const st = cache_check(what, c))
    {
        return st;
    }
    for (int64_t s : strides)
    {
        if (s < 0 || s % 8 != 0)
        {
            return set_error(TRTAMD_STATUS_BAD_PARAM, "%s: strides must be multiples of 8 elements, and not negative", what);
        }
    }
    if (c.B == 0 || c.T == 0 || c.max_tokens == 0)
    {
        return TRTAMD_STATUS_SUCCESS;
    }
    if (k == nullptr || v == nullptr)
    {
        return set_error(TRTAMD_STATUS_BAD_PARAM, "%s: null pointer", what);
    }
    if (!aligned16(k) || !aligned16(v))
    {
        return set_error(TRTAMD_STATUS_BAD_PARAM, "%s: k and v must be 16-byte aligned", what);
    }
    return TRTAMD_STATUS_SUCCESS;
}

dim3 copy_grid(trtamd_kv_cache const& c)
{
    // pages that max_tokens tokens can touch, and no more than a sequence has
    int64_t const touched = ((int64_t) std::min(c.max_tokens, c.T) + c.page_tokens - 2) / c.page_tokens + 1;
    return dim3((unsigned) std::min<int64_t>(touched, 65536), (unsigned) c.B, (unsigned) c.kv_heads * 2);
}

size_t turned_bytes(trtamd_kv_cache const& c)
{
    return (size_t) c.d * (c.page_tokens + 4);
}

} // namespace

int cache_check(char const* what, trtamd_kv_cache const& c)
{
    if (c.data_type != kCacheInt8 && c.data_type != kCacheFp8)
    {
        return set_error(TRTAMD_STATUS_BAD_PARAM, "%s: data_type %d (2 = INT8 or 6 = FP8)", what, c.data_type);
    }
    if (c.page_tokens != 16 && c.page_tokens != 32 && c.page_tokens != 64 && c.page_tokens != 128)
    {
        return set_error(TRTAMD_STATUS_BAD_PARAM, "%s: page_tokens=%d (16, 32, 64 or 128)", what, c.page_tokens);
    }
    if (c.d <= 0 || c.d % 16 != 0 || c.d > 256 || c.kv_heads <= 0)
    {
        return set_error(
            TRTAMD_STATUS_BAD_PARAM, "%s: kv_heads=%d d=%d (d a multiple of 16, at most 256)", what, c.kv_heads, c.d);
    }
    if (c.B < 0 || c.T < 0 || c.max_tokens < 0 || c.max_pages < 0 || c.pages < 0)
    {
        return set_error(TRTAMD_STATUS_BAD_PARAM, "%s: B=%d T=%d max_tokens=%d max_pages=%d pages=%d", what, c.B, c.T, c.max_tokens,
            c.max_pages, c.pages);
    }
    if (c.B == 0 || c.T == 0 || c.max_tokens == 0)
    {
        return TRTAMD_STATUS_SUCCESS; // a call without a token: its tensors may have no address
    }
    if (c.max_pages == 0 || c.pages == 0)
    {
        return set_error(TRTAMD_STATUS_BAD_PARAM, "%s: max_pages=%d pages=%d", what, c.max_pages, c.pages);
    }
    if (c.B > 65535 || c.kv_heads > 32767)
    {
        return set_error(TRTAMD_STATUS_NOT_SUPPORTED, "%s: B=%d kv_heads=%d (at most 65535 and 32767)", what, c.B, c.kv_heads);
    }
    if ((int64_t) c.pages * c.kv_heads >= (int64_t) 1 << 31)
    {
        return set_error(TRTAMD_STATUS_NOT_SUPPORTED, "%s: pages * kv_heads of 2^31 or more", what);
    }
    for (void const* p : {(void const*) c.k, (void const*) c.v, (void const*) c.k_scale, (void const*) c.v_scale,
             (void const*) c.page_table, (void const*) c.lengths, (void const*) c.cu_seqlens})
    {
        if (p == nullptr)
        {
            return set_error(TRTAMD_STATUS_BAD_PARAM, "%s: null pointer in the cache", what);
        }
        if ((reinterpret_cast<uintptr_t>(p) & 3u) != 0)
        {
            return set_error(TRTAMD_STATUS_BAD_PARAM, "%s: scales, page_table, lengths and cu_seqlens must be 4-byte aligned", what);
        }
    }
    if (!aligned16(c.k) || !aligned16(c.v))
    {
        return set_error(TRTAMD_STATUS_BAD_PARAM, "%s: the cache must be 16-byte aligned", what);
    }
    return TRTAMD_STATUS_SUCCESS;
}

CacheArgs cache_args(trtamd_kv_cache const& c)
{
    int shift = 4;
    while (1 << shift < c.page_tokens)
    {
        ++shift;
    }
    return {static_cast<uint8_t*>(c.k), static_cast<uint8_t*>(c.v), c.k_scale, c.v_scale, c.page_table, c.lengths, c.cu_seqlens,
        c.pages, shift, c.kv_heads, c.d, c.max_pages, c.max_tokens, c.T};
}

} // namespace trtamd

using namespace trtamd;

extern "C" int trtamd_kv_cache_write(trtamd_stream_t stream, trtamd_kv_cache_write_params const* params)
{
    if (params == nullptr)
    {
        return set_error(TRTAMD_STATUS_BAD_PARAM, "kv_cache_write: null params");
    }
    trtamd_kv_cache_write_params const& p = *params;
    trtamd_kv_cache const& c = p.cache;
    if (int const st = copy_check("kv_cache_write", c, p.k, p.v, {p.k_token_stride, p.k_head_stride, p.v_token_stride, p.v_head_stride}))
    {
        return st;
    }
    if (c.B == 0 || c.T == 0 || c.max_tokens == 0)
    {
        return TRTAMD_STATUS_SUCCESS;
    }
    CopyArgs const a = {cache_args(c),
        {{reinterpret_cast<uint8_t*>(const_cast<trtamd_half_t*>(p.k)), p.k_token_stride, p.k_head_stride},
            {reinterpret_cast<uint8_t*>(const_cast<trtamd_half_t*>(p.v)), p.v_token_stride, p.v_head_stride}},
        fast_div((uint32_t) c.d / 8)};
    int const tokens = std::min(c.page_tokens, std::min(c.max_tokens, c.T));
    int const perThread = ceil_div(tokens * c.d / 8, kThreads);
    auto const run = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, copy_grid(c), dim3(kThreads), turned_bytes(c), as_stream(stream), a);
        return check_launch("kv_cache_write_kernel");
    };
    auto const by_size = [&](auto type) {
        constexpr bool F = decltype(type)::value;
        return perThread <= 1 ? run(kv_cache_write_kernel<1, F>)
            : perThread <= 2  ? run(kv_cache_write_kernel<2, F>)
            : perThread <= 4  ? run(kv_cache_write_kernel<4, F>)
            : perThread <= 8  ? run(kv_cache_write_kernel<8, F>)
                              : run(kv_cache_write_kernel<16, F>);
    };
    return c.data_type == kCacheFp8 ? by_size(std::true_type{}) : by_size(std::false_type{});
}

extern "C" int trtamd_kv_cache_read(trtamd_stream_t stream, trtamd_kv_cache_read_params const* params)
{
    if (params == nullptr)
    {
        return set_error(TRTAMD_STATUS_BAD_PARAM, "kv_cache_read: null params");
    }
    trtamd_kv_cache_read_params const& p = *params;
    trtamd_kv_cache const& c = p.cache;
    if (int const st = copy_check("kv_cache_read", c, p.k, p.v, {p.k_token_stride, p.k_head_stride, p.v_token_stride, p.v_head_stride}))
    {
        return st;
    }
    if (c.B == 0 || c.T == 0 || c.max_tokens == 0)
    {
        return TRTAMD_STATUS_SUCCESS;
    }
    CopyArgs const a = {cache_args(c),
        {{reinterpret_cast<uint8_t*>(p.k), p.k_token_stride, p.k_head_stride},
            {reinterpret_cast<uint8_t*>(p.v), p.v_token_stride, p.v_head_stride}},
        fast_div((uint32_t) c.d / 8)};
    auto const run = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, copy_grid(c), dim3(kThreads), turned_bytes(c), as_stream(stream), a);
        return check_launch("kv_cache_read_kernel");
    };
    return c.data_type == kCacheFp8 ? run(kv_cache_read_kernel<true>) : run(kv_cache_read_kernel<false>);
}
