// What the kernels of the 8-bit cache share: the cache as a launch's argument, the place of a sequence's tokens in it, and its two
// kinds of bytes.
#pragma once

#include "device_utils.hpp"
#include "trtamd_encoder_ops.h"

#include <type_traits>

namespace trtamd
{

constexpr int kCacheInt8 = 2, kCacheFp8 = 6; // nvinfer1::DataType

struct CacheArgs
{
    uint8_t* k;
    uint8_t* v;
    float* kScale;
    float* vScale;
    int32_t const* table;
    int32_t const* lengths;
    int32_t const* cu;
    int32_t pages, shift /* log2(page_tokens) */, heads, d, maxPages, maxTokens, T;
};

// A call with nothing to do.
inline bool no_tokens(trtamd_kv_cache const& c)
{
    return c.B == 0 || c.T == 0 || c.max_tokens == 0;
}

// Refuses what no call takes; 0 where it is sound. Of the sizes alone, and of everything.
int cache_sizes_check(char const* what, trtamd_kv_cache const& c);
int cache_check(char const* what, trtamd_kv_cache const& c);
CacheArgs cache_args(trtamd_kv_cache const& c);

// The rows of a sequence in the call: rows row0 .. row0 + n - 1 are its tokens begin .. begin + n - 1, of which those from 0 to
// len - 1 have a place in the table.
struct CacheRows
{
    int32_t row0, n, begin, len;
};

__device__ inline CacheRows cache_rows(CacheArgs const& c, int b)
{
    int const lo = min(max(c.cu[b], 0), c.T), next = max(c.cu[b + 1], lo), hi = min(next, c.T);
    int const all = next - lo, length = max(c.lengths[b], 0);
    CacheRows r;
    r.row0 = lo;
    r.n = min(hi - lo, c.maxTokens);
    r.begin = length - all;
    r.len = min(length, c.maxPages << c.shift);
    return r;
}

// Bytes of a page and head in k or v.
__device__ inline uint32_t page_bytes(CacheArgs const& c)
{
    return (uint32_t) c.d << c.shift;
}

// Where head h of a page begins; pages * heads is less than 2^32.
__device__ inline uint64_t page_offset(CacheArgs const& c, int page, int h)
{
    return (uint64_t) ((uint32_t) page * (uint32_t) c.heads + (uint32_t) h) * page_bytes(c);
}

// ---- bytes to binary16, exactly: every INT8 and every E4M3 value is one -----------------------------------------------

// A byte moved by 128 behind 0x64 is 1024 + 128 + its value: one subtraction a pair.
__device__ inline f16x4 codes_to_f16(uint32_t w, std::integral_constant<bool, false>)
{
    uint32_t const moved = w ^ 0x80808080u;
    f16x2 const base = {(f16) 1152.f, (f16) 1152.f};
    f16x2 const lo = bits_as<f16x2>(__builtin_amdgcn_perm(0x64646464u, moved, 0x04010400u)) - base;
    f16x2 const hi = bits_as<f16x2>(__builtin_amdgcn_perm(0x64646464u, moved, 0x04030402u)) - base;
    return {lo[0], lo[1], hi[0], hi[1]};
}

__device__ inline f16x4 codes_to_f16(uint32_t w, std::integral_constant<bool, true>)
{
    auto const lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, false);
    auto const hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, true);
    return {(f16) lo[0], (f16) lo[1], (f16) hi[0], (f16) hi[1]};
}

template <bool FP8>
__device__ inline f16x4 code_values(uint32_t w)
{
    return codes_to_f16(w, std::integral_constant<bool, FP8>{});
}

template <bool FP8>
__device__ inline f16x8 code_values8(uint32_t a, uint32_t b)
{
    return __builtin_shufflevector(code_values<FP8>(a), code_values<FP8>(b), 0, 1, 2, 3, 4, 5, 6, 7);
}

} // namespace trtamd
