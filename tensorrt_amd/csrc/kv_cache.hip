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

// Four values, divided by their scale, as bytes. None is past the largest by more than three roundings to binary32, and what is that
// little past it is rounded to it.
template <bool FP8>
__device__ inline uint32_t round_codes(f32x4 y)
{
    if constexpr (FP8)
    {
        int const lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
        return (uint32_t) __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], lo, true);
    }
    else
    {
        // 1.5 * 2^23 more: rounded to an integer, ties to even, in the lowest byte. Not as one operation with the product before it.
#pragma clang fp contract(off)
        uint32_t b[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
        {
            b[e] = bits_as<uint32_t>(y[e] + 12582912.f);
        }
        return low_bytes(b[0], b[1], b[2], b[3]);
    }
}

template <bool FP8>
__device__ inline uint32_t quantize_codes(f16x4 x, float inverse)
{
#pragma clang fp contract(off)
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

typedef __attribute__((address_space(3))) i32x2 lds_i32x2;
constexpr int kRowPad = 16; // rows of bytes in LDS this much further apart: eight of them, 16 bytes each, lie in different banks

// 16 lanes read 8 rows of 16 bytes in LDS, `stride` apart, turned: lane i gets the bytes i of the rows, row 0 first. at: of the first row.
__device__ inline u32x2 turned_bytes8(uint8_t* at, int stride)
{
    int const i = threadIdx.x & 15;
    return bits_as<u32x2>(__builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2*) (at + (i >> 1) * stride + 8 * (i & 1))));
}

// A page and head, its keys or its values, to W wavefronts, with all new rows in registers between the maximum and the quotients: NV
// chunks of 8 values a lane. One (four pages a workgroup, side by side in the packed layouts, and no barrier) up to 512 chunks, four
// above. Values are turned through LDS: they are written there as they come, and 16 tokens of an element are read from it by
// transposing reads. 16621 tokens of 16 heads of 64 in pages of 32: 22.5 us (102 MB, 4.5 TB/s; vector instructions 55 % of the cycles); a
// workgroup a page, values turned byte by byte, 48. Pages of 64 x 128 to one wavefront each 19.7, to four 16.6. One token 3.6, a launch.
template <int NV, bool FP8, int W>
__global__ __launch_bounds__(kThreads) void kv_cache_write_kernel(CopyArgs const a)
{
    extern __shared__ __attribute__((aligned(16))) uint8_t turned[]; // values: [P][d + 16] bytes, W = 1 of two wavefronts
    __shared__ uint32_t tops[4];
    static_assert(W == 1 || W == 4, "four wavefronts a workgroup");
    CacheArgs const& c = a.cache;
    int const wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = W == 1 ? threadIdx.x & 63 : threadIdx.x; // of the unit
    int const unit = W == 1 ? (int) blockIdx.z * 4 + wave : blockIdx.z, b = blockIdx.y, h = unit >> 1, which = unit & 1;
    if (h >= c.heads)
    {
        return; // no barrier follows where wavefronts differ
    }
    constexpr int kLanes = W * kWaveSize;
    int const P = 1 << c.shift, stride = c.d + kRowPad;
    CacheRows const r = cache_rows(c, b);
    int const begin = max(r.begin, 0), end = min(r.begin + r.n, r.len);
    if (begin >= end)
    {
        return; // the whole workgroup: a page that the sequence only reads may be another one's that writes it
    }
    Strided const from = which ? a.kv[1] : a.kv[0];
    uint8_t const* const src = from.p + 2 * (int64_t) h * from.head;
    int const n8 = a.chunks.d;
    uint8_t* const mine = turned + (W == 1 ? wave >> 1 : 0) * P * stride;
    auto const meet = [] {
        if constexpr (W == 1)
        {
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
        else
        {
            __syncthreads();
        }
    };
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
        uint8_t const* const rows = src + 2 * ((int64_t) r.row0 + (first + lo - r.begin)) * from.token;
        f16x8 x[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i)
        {
            uint32_t const at = lane + i * kLanes, row = at / a.chunks, chunk = at - row * n8;
            x[i] = f16x8{};
            if ((int) row < hi - lo)
            {
                x[i] = *reinterpret_cast<f16x8 const*>(rows + 2 * ((int64_t) row * from.token + 8 * chunk));
            }
        }
        u16x2 m = {0, 0};
#pragma unroll
        for (int i = 0; i < NV; ++i)
        {
            m = max_abs(m, bits_as<u32x4>(x[i]));
        }
        uint32_t top = wave_max_bits(m);
        if constexpr (W == 4)
        {
            if ((lane & 63) == 0)
            {
                tops[wave] = top;
            }
            __syncthreads(); // and everybody has read the scale
            top = max(max(tops[0], tops[1]), max(tops[2], tops[3]));
        }
        PageScale const s = page_scale<FP8>(top, old);
        if (lane == 0)
        {
            *scaleAt = s.scale;
        }
#pragma unroll
        for (int i = 0; i < NV; ++i)
        {
            uint32_t const at = lane + i * kLanes, row = at / a.chunks, chunk = at - row * n8;
            u32x2 w = {quantize_codes<FP8>(f16x4{x[i][0], x[i][1], x[i][2], x[i][3]}, s.inverse),
                quantize_codes<FP8>(f16x4{x[i][4], x[i][5], x[i][6], x[i][7]}, s.inverse)};
            w = s.zeros ? u32x2{0, 0} : w; // also of a NaN or an infinity
            if ((int) row < hi - lo)
            {
                uint8_t* const to = which ? mine + (lo + row) * stride : codes + (lo + row) * (uint32_t) c.d;
                *reinterpret_cast<u32x2*>(to + 8 * chunk) = w;
            }
        }
        if (which == 0)
        {
            for (uint32_t at = lane; s.grown && at < (uint32_t) lo * n8; at += kLanes)
            {
                u32x2* const p = reinterpret_cast<u32x2*>(codes) + at;
                *p = u32x2{requantize_codes<FP8>((*p)[0], s.shrink), requantize_codes<FP8>((*p)[1], s.shrink)};
            }
            if constexpr (W == 4)
            {
                __syncthreads(); // tops
            }
            continue;
        }
        meet();
        // Elements 16 e .. + 15 of 16 tokens, four such blocks at a time, side by side in the page. The page and head are this
        // wavefront's, so bytes on either side of the new ones are as well.
        int const from16 = (s.grown ? 0 : lo) >> 4, to16 = (hi + 15) >> 4, groups = to16 - from16;
        for (int at = lane >> 4; at < groups * (c.d >> 4); at += 4 * W)
        {
            int const e = at / groups, group = from16 + at - e * groups;
            uint8_t* const block16 = mine + 16 * group * stride + 16 * e;
            u32x2 const t0 = turned_bytes8(block16, stride), t1 = turned_bytes8(block16 + 8 * stride, stride);
            u32x4* const p = reinterpret_cast<u32x4*>(codes + (uint32_t) (16 * e + (lane & 15)) * P + 16 * group);
            u32x4 w = {t0[0], t0[1], t1[0], t1[1]};
            int const l = min(max(lo - 16 * group, 0), 16), u = min(hi - 16 * group, 16);
            if (l > 0 || u < 16)
            {
                uint32_t const isNew = l < u ? (1u << u) - (1u << l) : 0u;
                u32x4 const was = *p;
#pragma unroll
                for (int k = 0; k < 4; ++k)
                {
                    // behind the new ones nothing is held: whatever lies there stays
                    uint32_t held = was[k];
                    if (s.grown)
                    {
                        held = merge_bytes(requantize_codes<FP8>(held, s.shrink), held, ((1u << l) - 1u) >> (4 * k));
                    }
                    w[k] = merge_bytes(w[k], held, isNew >> (4 * k));
                }
            }
            *p = w;
        }
        meet();
    }
}

template <bool FP8>
__device__ inline f16x4 scaled_codes(uint32_t w, float scale)
{
    f32x4 y;
    if constexpr (FP8)
    {
        auto const lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
        y = {lo[0], lo[1], hi[0], hi[1]};
    }
    else
    {
        y = {i8_to_f32(w, 0), i8_to_f32(w, 1), i8_to_f32(w, 2), i8_to_f32(w, 3)};
    }
    y *= scale;
    f16x2 const lo = __builtin_convertvector(f32x2{y[0], y[1]}, f16x2), hi = __builtin_convertvector(f32x2{y[2], y[3]}, f16x2);
    return {lo[0], lo[1], hi[0], hi[1]};
}

template <bool FP8>
__device__ inline void store_scaled(uint8_t* to, u32x4 const& w, float scale)
{
    f16x4 y[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
    {
        y[k] = scaled_codes<FP8>(w[k], scale);
    }
#pragma unroll
    for (int k = 0; k < 4; k += 2)
    {
        *reinterpret_cast<f16x8*>(to + 8 * k) = __builtin_shufflevector(y[k], y[k + 1], 0, 1, 2, 3, 4, 5, 6, 7);
    }
}

// The way back: 4 KB of a page and head a wavefront, tokens of its keys as they lie, or elements of its values, turned through LDS. Four of
// them a workgroup. The same 16621 tokens 20.7 us (4.9 TB/s); a workgroup a page 45.
constexpr int kReadBytes = 4096;

struct ReadArgs
{
    CopyArgs copy;
    int elements; // of a part of the values: a multiple of 16
    FastDiv parts;
    int tokens; // of a part of the keys
    FastDiv pieces; // d / 16
};

template <bool FP8>
__global__ __launch_bounds__(kThreads) void kv_cache_read_kernel(ReadArgs const ra)
{
    constexpr int NV = kReadBytes / 16 / kWaveSize;
    extern __shared__ __attribute__((aligned(16))) uint8_t turned[]; // four wavefronts' values: [elements][P + 16] bytes each
    CopyArgs const& a = ra.copy;
    CacheArgs const& c = a.cache;
    int const lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int const unit = (int) blockIdx.z * 4 + wave, b = blockIdx.y; // key head, keys or values, part
    int const pair = (int) ((uint32_t) unit / ra.parts), part = unit - pair * (int) ra.parts.d, h = pair >> 1, which = pair & 1;
    if (h >= c.heads)
    {
        return; // no barrier follows
    }
    int const P = 1 << c.shift, stride = P + kRowPad, n16 = ra.pieces.d;
    CacheRows const r = cache_rows(c, b);
    Strided const into = which ? a.kv[1] : a.kv[0];
    uint8_t* const out = into.p + 2 * (int64_t) h * into.head;
    uint8_t* const mine = turned + wave * ra.elements * stride;
    // by position, so that rows without a place in the table get their zeros as well
    int64_t const begin = r.begin, end = begin + r.n;
    for (int64_t block = (begin >> c.shift) + blockIdx.x; block * P < end; block += gridDim.x)
    {
        int const page = block >= 0 && block < c.maxPages ? c.table[(int64_t) b * c.maxPages + block] : -1;
        int64_t const first = block * P;
        int lo = (int) max(begin - first, (int64_t) 0), hi = (int) min(end - first, (int64_t) P);
        bool const there = (uint32_t) page < (uint32_t) c.pages;
        int const sound = there ? page : 0;
        float const scale = there ? (which ? c.vScale : c.kScale)[(size_t) sound * c.heads + h] : 0.f;
        uint8_t const* codes = (which ? c.v : c.k) + page_offset(c, sound, h);
        uint8_t* const rows = out + 2 * (r.row0 + (first - begin)) * into.token; // of the page's first token, which may not be one of the call's
        if (which == 0 || !there)
        {
            lo = max(lo, part * ra.tokens);
            hi = min(hi, (part + 1) * ra.tokens);
            for (int from = lo * n16; from < hi * n16; from += NV * kWaveSize)
            {
                u32x4 w[NV];
#pragma unroll
                for (int i = 0; i < NV; ++i)
                {
                    int const at = from + lane + i * kWaveSize;
                    w[i] = u32x4{0, 0, 0, 0};
                    if (there && at < hi * n16)
                    {
                        w[i] = reinterpret_cast<u32x4 const*>(codes)[at];
                    }
                }
#pragma unroll
                for (int i = 0; i < NV; ++i)
                {
                    int const at = from + lane + i * kWaveSize, token = (int) ((uint32_t) at / ra.pieces), piece = at - token * n16;
                    if (at < hi * n16)
                    {
                        store_scaled<FP8>(rows + 2 * ((int64_t) token * into.token + 16 * piece), w[i], scale);
                    }
                }
            }
            continue;
        }
        int const groups = P >> 4, from16 = lo >> 4, to16 = (hi + 15) >> 4;
        int const e0 = part * ra.elements, elements = min(ra.elements, c.d - e0);
        codes += (uint32_t) e0 * P;
        u32x4 w[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i)
        {
            int const at = lane + i * kWaveSize, group = at & (groups - 1);
            w[i] = u32x4{0, 0, 0, 0};
            if (at < elements * groups && group >= from16 && group < to16)
            {
                w[i] = reinterpret_cast<u32x4 const*>(codes)[at];
            }
        }
#pragma unroll
        for (int i = 0; i < NV; ++i)
        {
            int const at = lane + i * kWaveSize;
            if (at < elements * groups)
            {
                *reinterpret_cast<u32x4*>(mine + (at >> (c.shift - 4)) * stride + 16 * (at & (groups - 1))) = w[i];
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        // elements 16 e .. + 15 of 16 tokens, four such blocks at a time, side by side in the rows
        int const blocks = elements >> 4;
        int e = lane >> 4, token16 = from16;
        while (e >= blocks)
        {
            e -= blocks;
            ++token16;
        }
        while (token16 < to16)
        {
            int const token = 16 * token16 + (lane & 15);
            uint8_t* const block16 = mine + 16 * e * stride + 16 * token16;
            u32x2 const t0 = turned_bytes8(block16, stride), t1 = turned_bytes8(block16 + 8 * stride, stride);
            if (token >= lo && token < hi)
            {
                store_scaled<FP8>(rows + 2 * ((int64_t) token * into.token + e0 + 16 * e), u32x4{t0[0], t0[1], t1[0], t1[1]}, scale);
            }
            e += 4;
            while (e >= blocks)
            {
                e -= blocks;
                ++token16;
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
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
    if (no_tokens(c))
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

} // namespace

int cache_sizes_check(char const* what, trtamd_kv_cache const& c)
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
    if (no_tokens(c))
    {
        return TRTAMD_STATUS_SUCCESS;
    }
    if (c.max_pages == 0 || c.pages == 0)
    {
        return set_error(TRTAMD_STATUS_BAD_PARAM, "%s: max_pages=%d pages=%d", what, c.max_pages, c.pages);
    }
    if (c.B > 65535 || c.kv_heads > 16383)
    {
        return set_error(TRTAMD_STATUS_NOT_SUPPORTED, "%s: B=%d kv_heads=%d (at most 65535 and 16383)", what, c.B, c.kv_heads);
    }
    if ((int64_t) c.max_pages * c.page_tokens > (int64_t) 1 << 30)
    {
        return set_error(TRTAMD_STATUS_NOT_SUPPORTED, "%s: max_pages * page_tokens of more than 2^30", what);
    }
    if ((int64_t) c.pages * c.kv_heads >= (int64_t) 1 << 31)
    {
        return set_error(TRTAMD_STATUS_NOT_SUPPORTED, "%s: pages * kv_heads of 2^31 or more", what);
    }
    return TRTAMD_STATUS_SUCCESS;
}

int cache_check(char const* what, trtamd_kv_cache const& c)
{
    int const st = cache_sizes_check(what, c);
    if (st || no_tokens(c)) // a call without a token: its tensors may have no address
    {
        return st;
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
    if (no_tokens(c))
    {
        return TRTAMD_STATUS_SUCCESS;
    }
    CopyArgs const a = {cache_args(c),
        {{reinterpret_cast<uint8_t*>(const_cast<trtamd_half_t*>(p.k)), p.k_token_stride, p.k_head_stride},
            {reinterpret_cast<uint8_t*>(const_cast<trtamd_half_t*>(p.v)), p.v_token_stride, p.v_head_stride}},
        fast_div((uint32_t) c.d / 8)};
    // of a page at most
    int const chunks = std::min(c.page_tokens, std::min(c.max_tokens, c.T)) * c.d / 8;
    dim3 const pages = copy_grid(c);
    size_t const lds = (size_t) c.page_tokens * (c.d + kRowPad); // values of a page
    auto const run = [&](auto kernel, int wavefronts) {
        bool const one = wavefronts == 1;
        hipLaunchKernelGGL(kernel, dim3(pages.x, pages.y, one ? ceil_div(pages.z, 4u) : pages.z), dim3(kThreads), one ? 2 * lds : lds, as_stream(stream), a);
        return check_launch("kv_cache_write_kernel");
    };
    auto const by_size = [&](auto type) {
        constexpr bool F = decltype(type)::value;
        if (chunks > 8 * kWaveSize || 2 * lds > 65536)
        {
            return chunks <= 16 * kWaveSize ? run(kv_cache_write_kernel<4, F, 4>, 4)
                : chunks <= 32 * kWaveSize  ? run(kv_cache_write_kernel<8, F, 4>, 4)
                                            : run(kv_cache_write_kernel<16, F, 4>, 4);
        }
        return chunks <= 1 * kWaveSize ? run(kv_cache_write_kernel<1, F, 1>, 1)
            : chunks <= 2 * kWaveSize  ? run(kv_cache_write_kernel<2, F, 1>, 1)
            : chunks <= 4 * kWaveSize  ? run(kv_cache_write_kernel<4, F, 1>, 1)
                                       : run(kv_cache_write_kernel<8, F, 1>, 1);
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
    if (no_tokens(c))
    {
        return TRTAMD_STATUS_SUCCESS;
    }
    CopyArgs const a = {cache_args(c),
        {{reinterpret_cast<uint8_t*>(p.k), p.k_token_stride, p.k_head_stride},
            {reinterpret_cast<uint8_t*>(p.v), p.v_token_stride, p.v_head_stride}},
        fast_div((uint32_t) c.d / 8)};
    int const elements = std::min(c.d, kReadBytes / c.page_tokens), parts = ceil_div(c.d, elements);
    ReadArgs const ra = {a, elements, fast_div((uint32_t) parts), ceil_div(c.page_tokens, parts), fast_div((uint32_t) c.d / 16)};
    dim3 const pages = copy_grid(c);
    auto const run = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(pages.x, pages.y, (unsigned) ceil_div((int64_t) pages.z * parts, (int64_t) 4)), dim3(kThreads),
            4 * (size_t) elements * (c.page_tokens + kRowPad), as_stream(stream), ra);
        return check_launch("kv_cache_read_kernel");
    };
    return c.data_type == kCacheFp8 ? run(kv_cache_read_kernel<true>) : run(kv_cache_read_kernel<false>);
}
