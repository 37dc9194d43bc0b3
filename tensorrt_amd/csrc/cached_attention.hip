// Attention of a call's rows over their sequences in the 8-bit cache.
//
//   s_j = scale * q k_j,   o = sum_j 2^(c s_j - m) v_j / sum_j 2^(c s_j - m),   c = log2(e)
//
// Bytes become binary16 exactly, so the products' operands are the bytes' values and the scales go elsewhere: a page's key scale into
// the multiplication that brings its scores to powers of 2, its value scale into the exponent, s + log2(value scale), where it costs
// nothing: the weights P' = p * value scale are what the second product wants, and p = P' / value scale is summed by one multiply-add.
// The running maximum is that of the weights P', so that they fill binary16's range whatever the scales are.
//
// Rows of one key head, (token, query head) with the heads of a group side by side, share the keys. Up to 16 of them (decoding, a few
// drafted tokens) go to `cached_few_kernel`, which is bound by reading the cache; more to `cached_many_kernel`, bound by the matrix
// and vector instructions.
#include "attention_rows.hpp"
#include "host_utils.hpp"
#include "kv_cache.hpp"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace trtamd
{
namespace
{

constexpr int kThreads = 256, kWaves = kThreads / kWaveSize;
constexpr int kFewRows = 16;
constexpr int kTileRows = 128; // of cached_many_kernel

struct AttentionArgs
{
    uint8_t const* q; // FP16
    uint8_t* out;
    int64_t qToken, qHead, outToken, outHead; // elements
    float* partial;   // [row][slot][d], the sums that parts of a row's keys have, and behind them [row][slot][2]
    float* stats;
    FastDiv group;    // query heads of a key head
    int32_t qHeads;
    int32_t window, sinks;
    int32_t slots;    // of a row in partial
    int32_t fewSpan, manySpan; // chunks of 64 keys that a workgroup takes
    int32_t fewLimit; // sequences of up to so many rows are cached_few_kernel's
    float scale;      // in powers of 2
};

// Of the tokens that see the least and the most (i0 <= i1) of some rows.
__device__ inline Chunks chunks_of_tokens(CacheRows const& r, int i0, int i1, AttentionArgs const& a)
{
    int const at0 = max(r.begin + i0, -1), at1 = r.begin + i1;
    return chunks_of(a.window ? max(at0 - a.window + 1, 0) : 0, min(r.len, at1 + 1), a.sinks);
}

__device__ inline Seen seen_by(CacheRows const& r, int i, AttentionArgs const& a)
{
    int const at = max(r.begin + i, -1);
    return {a.window ? max(at - a.window + 1, 0) : 0, min(r.len, at + 1), a.sinks};
}

__device__ inline bool sees_all(Seen const& least, Seen const& most, int key0)
{
    return key0 + kChunkKeys <= least.hi && (key0 >= most.lo || key0 + kChunkKeys <= least.sinks);
}

// What a page's scales are to its scores and weights. No values of 0 or below 2^-126 (a scale of 0 times a score of -infinity is no
// number), but what is a NaN stays one.
struct PageFactors
{
    float score, log2Value, inverse;
};

__device__ inline PageFactors page_factors(float kScale, float vScale, float scale)
{
    PageFactors f;
    float const s = kScale * scale;
    f.score = s < 0x1p-126f ? 0x1p-126f : s;
    // the values of a scale of 0 are zeros: any scale does, and the least one leaves the maximum to the others
    f.log2Value = vScale == 0.f ? -32.f : __builtin_amdgcn_logf(vScale);
    f.inverse = vScale > 0.f ? 1.f / vScale : 0x1p32f;
    return f;
}

__device__ inline float sum_of(float a, float b)
{
    return a + b;
}

// A byte mask of 16: ones below n.
__device__ inline u32x4 bytes_below(int n)
{
    u32x4 m;
#pragma unroll
    for (int e = 0; e < 4; ++e)
    {
        int const k = min(max(n - 4 * e, 0), 4);
        m[e] = k == 4 ? 0xffffffffu : (1u << (8 * k)) - 1u;
    }
    return m;
}

// ------------------------------------------------------------------------------------------
// Up to 16 rows of a key head: v_mfma_f32_16x16x32_f16, S^T = K Q^T and O^T = V^T P^T again. Each wavefront takes chunks of 64 keys
// on its own, from global memory to the operands' registers: lane (g, m) loads 16 bytes of the key 16 (m / 4) + 4 t + m % 4 for tile
// t, so that its scores are those of the keys 16 g .. 16 g + 15 of row m, and 16 bytes of the same keys of element 16 i + m of the
// values. 16 keys lie in one page, so a lane has one page for the keys and one for the values and the factors of a chunk.
// The wavefronts meet in LDS at the end, workgroups that share a row's keys in memory.
// ------------------------------------------------------------------------------------------
template <int KS /* 16 of the head's values */, bool FP8>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(KS <= 4 ? 3 : KS <= 8 ? 2 : 1))) void cached_few_kernel(
    CacheArgs const c, AttentionArgs const a)
{
    constexpr int NT = KS, DC = (KS + 3) / 4;
    __shared__ f32x4 meet[2][NT][kWaveSize];
    __shared__ float stats[kWaves][2][kFewRows];
    int const h = blockIdx.x, b = blockIdx.y, split = blockIdx.z;
    CacheRows const r = cache_rows(c, b);
    int const group = a.group.d;
    if (r.n == 0 || (int64_t) r.n * group > a.fewLimit)
    {
        return;
    }
    int const rows = r.n * group;
    Chunks const chunks = chunks_of_tokens(r, 0, r.n - 1, a);
    int const used = max((chunks.total + a.fewSpan - 1) / a.fewSpan, 1);
    if (split >= used)
    {
        return;
    }
    int const cEnd = min(chunks.total, (split + 1) * a.fewSpan);
    int const lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int const m = lane & 15, g = lane >> 4;
    int const row = min(m, rows - 1);
    int const token = (int) ((uint32_t) row / a.group), head = h * group + row - token * group;
    Seen const seen = seen_by(r, token, a), least = seen_by(r, 0, a), most = seen_by(r, r.n - 1, a);
    int const P = 1 << c.shift;

    f16x8 q[DC][2];
    {
        uint8_t const* const from = a.q + 2 * ((int64_t) (r.row0 + token) * a.qToken + (int64_t) head * a.qHead);
#pragma unroll
        for (int k = 0; k < DC; ++k)
        {
            int const e = 64 * k + 16 * g;
#pragma unroll
            for (int j = 0; j < 2; ++j)
            {
                q[k][j] = f16x8{};
                if (e < c.d)
                {
                    q[k][j] = *reinterpret_cast<f16x8 const*>(from + 2 * (e + 8 * j));
                }
            }
        }
    }

    // pages of a chunk: those of the lane's keys and of its values
    struct Pages
    {
        int k, v;
    };
    int32_t const* const table = c.table + (int64_t) b * c.maxPages;
    auto pages_of = [&](int i) {
        int const key0 = chunks.key0(i);
        return Pages{table[min((key0 + 16 * (m >> 2)) >> c.shift, c.maxPages - 1)], table[min((key0 + 16 * g) >> c.shift, c.maxPages - 1)]};
    };
    u32x4 kr[4][DC], vr[NT];
    float kScale, vScale;
    auto load_keys = [&](int i, Pages const& p) {
        int const key = chunks.key0(i) + 16 * (m >> 2) + (m & 3);
        int const page = (uint32_t) p.k < (uint32_t) c.pages ? p.k : 0;
        uint8_t const* const from = c.k + page_offset(c, page, h) + (uint32_t) (key & (P - 1)) * c.d;
#pragma unroll
        for (int t = 0; t < 4; ++t)
        {
#pragma unroll
            for (int k = 0; k < DC; ++k)
            {
                // lanes behind the head's end read its last values, times a query of zeros
                kr[t][k] = *reinterpret_cast<u32x4 const*>(from + 4 * t * c.d + min(64 * k + 16 * g, c.d - 16));
            }
        }
    };
    auto load_values = [&](int i, Pages const& p) {
        int const key = chunks.key0(i) + 16 * g;
        int const page = (uint32_t) p.v < (uint32_t) c.pages ? p.v : 0;
        size_t const scaleAt = (size_t) page * c.heads + h;
        kScale = c.kScale[scaleAt];
        vScale = c.vScale[scaleAt];
        uint8_t const* const from = c.v + page_offset(c, page, h) + m * P + (key & (P - 1));
#pragma unroll
        for (int t = 0; t < NT; ++t)
        {
            vr[t] = *reinterpret_cast<u32x4 const*>(from + (16 * t < c.d ? 16 * t * P : 0)); // elements behind the head's end are not written
        }
    };

    f32x4 o[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
    {
        o[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    float negMax = kNothingSeen, sum = 0.f;
    int i = split * a.fewSpan + wave;
    Pages now{}, next{};
    if (i < cEnd)
    {
        now = pages_of(i);
        next = pages_of(min(i + kWaves, cEnd - 1));
        load_keys(i, now);
        load_values(i, now);
    }
    for (; i < cEnd; i += kWaves)
    {
        int const key0 = chunks.key0(i);
        f32x4 s[4];
#pragma unroll
        for (int t = 0; t < 4; ++t)
        {
            s[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < DC; ++k)
            {
                s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(code_values8<FP8>(kr[t][k][0], kr[t][k][1]), q[k][0], s[t], 0, 0, 0);
                s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(code_values8<FP8>(kr[t][k][2], kr[t][k][3]), q[k][1], s[t], 0, 0, 0);
            }
        }
        bool const more = i + kWaves < cEnd;
        Pages const after = pages_of(min(i + 2 * kWaves, cEnd - 1));
        if (more)
        {
            load_keys(i + kWaves, next);
        }
        PageFactors const f = page_factors(kScale, vScale, a.scale);
        // keys of this lane that are there at all
        int const there = (uint32_t) now.v < (uint32_t) c.pages ? min(max(r.len - key0 - 16 * g, 0), 16) : 0;
        bool const whole = sees_all(least, most, key0) && __ballot(there < 16) == 0;
        float mx = -__builtin_inff();
#pragma unroll
        for (int t = 0; t < 4; ++t)
        {
#pragma unroll
            for (int e = 0; e < 4; ++e)
            {
                s[t][e] = fmaf(s[t][e], f.score, f.log2Value);
            }
        }
        if (!whole)
        {
#pragma unroll
            for (int t = 0; t < 4; ++t)
            {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                {
                    s[t][e] = 4 * t + e < there && seen(key0 + 16 * g + 4 * t + e) ? s[t][e] : -__builtin_inff();
                }
            }
            u32x4 const keep = bytes_below(there);
#pragma unroll
            for (int t = 0; t < NT; ++t)
            {
                vr[t] &= keep; // what was never written may be anything, and 0 times it not 0
            }
        }
#pragma unroll
        for (int t = 0; t < 4; ++t)
        {
            mx = fmaxf(mx, fmaxf(fmaxf(s[t][0], s[t][1]), fmaxf(s[t][2], s[t][3])));
        }
        mx = reduce_step<32>(reduce_step<16>(mx, max_of), max_of);
        float const negNew = fminf(-mx, kNothingSeen);
        if (__ballot(negNew < negMax - 8.f) != 0)
        {
            float const to = fminf(negNew, negMax), by = __builtin_amdgcn_exp2f(to - negMax);
#pragma unroll
            for (int t = 0; t < NT; ++t)
            {
                o[t] *= by;
            }
            sum *= by;
            negMax = to;
        }
        f16x8 p[2];
#pragma unroll
        for (int j = 0; j < 2; ++j)
        {
            float w[8];
#pragma unroll
            for (int e = 0; e < 8; ++e)
            {
                w[e] = __builtin_amdgcn_exp2f(s[2 * j + (e >> 2)][e & 3] + negMax);
                sum = fmaf(w[e], f.inverse, sum);
            }
            p[j] = weights_f16(w);
        }
#pragma unroll
        for (int t = 0; t < NT; ++t)
        {
            o[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(code_values8<FP8>(vr[t][0], vr[t][1]), p[0], o[t], 0, 0, 0);
            o[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(code_values8<FP8>(vr[t][2], vr[t][3]), p[1], o[t], 0, 0, 0);
        }
        if (more)
        {
            load_values(i + kWaves, next);
        }
        now = next;
        next = after;
    }

    // ---- the wavefronts' sums
    sum = reduce_step<32>(reduce_step<16>(sum, sum_of), sum_of);
    if (g == 0)
    {
        stats[wave][0][m] = negMax;
        stats[wave][1][m] = sum;
    }
    __syncthreads();
    float least4 = kNothingSeen, total = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w)
    {
        least4 = fminf(least4, stats[w][0][m]);
    }
#pragma unroll
    for (int w = 0; w < kWaves; ++w)
    {
        total = fmaf(stats[w][1][m], __builtin_amdgcn_exp2f(least4 - stats[w][0][m]), total);
    }
    float const by = __builtin_amdgcn_exp2f(least4 - negMax);
#pragma unroll
    for (int t = 0; t < NT; ++t)
    {
        o[t] *= by;
    }
#pragma unroll
    for (int half = kWaves / 2; half > 0; half /= 2)
    {
        if (wave >= half && wave < 2 * half)
        {
#pragma unroll
            for (int t = 0; t < NT; ++t)
            {
                meet[wave - half][t][lane] = o[t];
            }
        }
        __syncthreads();
        if (wave < half)
        {
#pragma unroll
            for (int t = 0; t < NT; ++t)
            {
                o[t] += meet[wave][t][lane];
            }
        }
        __syncthreads();
    }
    if (wave != 0 || m >= rows)
    {
        return;
    }
    size_t const outRow = (size_t) (r.row0 + token);
    if (used > 1)
    {
        size_t const slot = (outRow * a.qHeads + head) * a.slots + split;
#pragma unroll
        for (int t = 0; t < NT; ++t)
        {
            if (16 * t < c.d)
            {
                *reinterpret_cast<f32x4*>(a.partial + slot * c.d + 16 * t + 4 * g) = o[t];
            }
        }
        if (g == 0)
        {
            *reinterpret_cast<f32x2*>(a.stats + 2 * slot) = f32x2{least4, total};
        }
        return;
    }
    float const inverse = total == 0.f ? 0.f : 1.f / total; // a row that sees nothing is zeros; a NaN stays one
    uint8_t* const to = a.out + 2 * (outRow * a.outToken + (int64_t) head * a.outHead);
#pragma unroll
    for (int t = 0; t < NT; ++t)
    {
        if (16 * t < c.d)
        {
            f16x4 y;
#pragma unroll
            for (int e = 0; e < 4; ++e)
            {
                y[e] = (f16) (o[t][e] * inverse);
            }
            *reinterpret_cast<f16x4*>(to + 2 * (16 * t + 4 * g)) = y;
        }
    }
}

// ------------------------------------------------------------------------------------------
// More rows: 128 a workgroup, 32 a wavefront (attention_rows.hpp). Chunks of 64 keys become binary16 on their way into LDS, in two
// slots: the next chunk's bytes are requested before this one's products and converted behind them. Values come [d][key], so both
// operands are read as they lie, 16 bytes a lane.
// ------------------------------------------------------------------------------------------
template <int DP>
struct ManyLds
{
    static constexpr int kKeys = kChunkKeys * DP * 2, kValues = DP * kChunkKeys * 2;
    static constexpr int kSlot = kKeys + kValues;
    static constexpr int kFactors = 4 * 16; // of four pages: score, log2Value, inverse, keys that are there
    static constexpr int kTotal = 2 * (kSlot + kFactors);
};

template <int KS /* 16 of the head's values */, bool FP8>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(KS <= 8 ? 2 : 1))) void cached_many_kernel(
    CacheArgs const c, AttentionArgs const a, FastDiv const heads)
{
    constexpr int DP = padded_head(KS);
    using Lds = ManyLds<DP>;
    constexpr int kPieces = DP / 16;                     // of 16 bytes in a key
    constexpr int NL = kChunkKeys * kPieces / kThreads;  // loads a thread of keys, and of values
    constexpr int DV = (KS + 1) / 2;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    // tiles of a head are a multiple of the heads apart, so that where those divide by 8 they share an XCD's L2
    int const fromEnd = (int) (blockIdx.x / heads), h = (int) (blockIdx.x - fromEnd * heads.d), b = blockIdx.y, split = blockIdx.z;
    CacheRows const r = cache_rows(c, b);
    int const group = a.group.d;
    int64_t const rows64 = (int64_t) r.n * group;
    int64_t const tiles = (rows64 + kTileRows - 1) / kTileRows;
    if (rows64 <= a.fewLimit || fromEnd >= tiles)
    {
        return;
    }
    int const rows = (int) rows64;
    int const row0 = (int) (tiles - 1 - fromEnd) * kTileRows, rowEnd = min(row0 + kTileRows, rows); // those that see the most first
    int const i0 = (int) ((uint32_t) row0 / a.group), i1 = (int) ((uint32_t) (rowEnd - 1) / a.group);
    Chunks const chunks = chunks_of_tokens(r, i0, i1, a);
    int const used = max((chunks.total + a.manySpan - 1) / a.manySpan, 1);
    if (split >= used)
    {
        return;
    }
    int const cBegin = split * a.manySpan, cEnd = min(chunks.total, cBegin + a.manySpan);
    int const tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int const lq = lane & 31, half = lane >> 5;
    int const P = 1 << c.shift;
    int const wRow = row0 + 32 * wave;
    bool const active = wRow < rowEnd;
    int const row = min(wRow + lq, rowEnd - 1);
    int const token = (int) ((uint32_t) row / a.group), head = h * group + row - token * group;
    Seen const seen = seen_by(r, token, a);
    Seen const least = seen_by(r, (int) ((uint32_t) min(wRow, rowEnd - 1) / a.group), a);
    Seen const most = seen_by(r, (int) ((uint32_t) min(wRow + 31, rowEnd - 1) / a.group), a);

    f16x8 q[KS]; // row lq, elements 16 s + 8 half .. + 7
    {
        uint8_t const* const from = a.q + 2 * ((int64_t) (r.row0 + token) * a.qToken + (int64_t) head * a.qHead);
#pragma unroll
        for (int s = 0; s < KS; ++s)
        {
            q[s] = f16x8{};
            if (16 * s < c.d)
            {
                q[s] = *reinterpret_cast<f16x8 const*>(from + 2 * (16 * s + 8 * half));
            }
        }
    }

    // this thread's pieces of a chunk: 16 bytes of key (tid + 256 i) / kPieces, 16 keys of value row (tid + 256 i) / 4
    int32_t const* const table = c.table + (int64_t) b * c.maxPages;
    int const piece = tid & (kPieces - 1), vGroup = tid & 3;
    auto page_at = [&](int key) { return table[min(key >> c.shift, c.maxPages - 1)]; };
    auto sound = [&](int page) { return (uint32_t) page < (uint32_t) c.pages ? page : 0; };
    struct Pages
    {
        int k[NL], v;
    };
    auto pages_of = [&](int i) {
        Pages p;
        int const key0 = chunks.key0(i);
#pragma unroll
        for (int l = 0; l < NL; ++l)
        {
            p.k[l] = page_at(key0 + (tid + kThreads * l) / kPieces);
        }
        p.v = page_at(key0 + 16 * vGroup);
        return p;
    };
    u32x4 kr[NL], vr[NL];
    float kScale = 0.f, vScale = 0.f;
    auto request = [&](int i, Pages const& p) {
        int const key0 = chunks.key0(i);
        size_t const vPage = page_offset(c, sound(p.v), h);
#pragma unroll
        for (int l = 0; l < NL; ++l)
        {
            int const key = key0 + (tid + kThreads * l) / kPieces, vRow = (tid + kThreads * l) >> 2;
            kr[l] = u32x4{0, 0, 0, 0};
            vr[l] = u32x4{0, 0, 0, 0};
            if (16 * piece < c.d)
            {
                kr[l] = *reinterpret_cast<u32x4 const*>(c.k + page_offset(c, sound(p.k[l]), h) + (uint32_t) (key & (P - 1)) * c.d + 16 * piece);
            }
            if (vRow < c.d)
            {
                vr[l] = *reinterpret_cast<u32x4 const*>(c.v + vPage + (uint32_t) vRow * P + ((key0 + 16 * vGroup) & (P - 1)));
            }
        }
        if (tid < 4)
        {
            size_t const at = (size_t) sound(p.v) * c.heads + h;
            kScale = c.kScale[at];
            vScale = c.vScale[at];
        }
    };
    auto deliver = [&](int i, Pages const& p, int slot) {
        uint8_t* const keys = lds + slot * Lds::kSlot;
        uint8_t* const values = keys + Lds::kKeys;
        int const there = (uint32_t) p.v < (uint32_t) c.pages ? min(max(r.len - chunks.key0(i) - 16 * vGroup, 0), 16) : 0;
        u32x4 const keep = bytes_below(there);
#pragma unroll
        for (int l = 0; l < NL; ++l)
        {
            int const key = (tid + kThreads * l) / kPieces, vRow = (tid + kThreads * l) >> 2;
            int const kRow = (key & 32) + row_of_key(key & 31);
            uint8_t* const k0 = keys + kRow * DP * 2;
            *reinterpret_cast<f16x8*>(k0 + 16 * swizzled(kRow, 2 * piece)) = code_values8<FP8>(kr[l][0], kr[l][1]);
            *reinterpret_cast<f16x8*>(k0 + 16 * swizzled(kRow, 2 * piece + 1)) = code_values8<FP8>(kr[l][2], kr[l][3]);
            u32x4 const v = vr[l] & keep; // what was never written may be anything, and 0 times it not 0
            uint8_t* const v0 = values + vRow * kChunkKeys * 2;
            *reinterpret_cast<f16x8*>(v0 + 16 * swizzled(vRow, 2 * vGroup)) = code_values8<FP8>(v[0], v[1]);
            *reinterpret_cast<f16x8*>(v0 + 16 * swizzled(vRow, 2 * vGroup + 1)) = code_values8<FP8>(v[2], v[3]);
        }
        if (tid < 4)
        {
            PageFactors const f = page_factors(kScale, vScale, a.scale);
            *reinterpret_cast<f32x4*>(lds + 2 * Lds::kSlot + slot * Lds::kFactors + 16 * tid)
                = f32x4{f.score, f.log2Value, f.inverse, (float) there};
        }
    };

    RowSums<DV> sums;
    sums.clear();
    if (cBegin < cEnd)
    {
        Pages now = pages_of(cBegin), next = pages_of(min(cBegin + 1, cEnd - 1));
        request(cBegin, now);
        deliver(cBegin, now, 0);
        for (int i = cBegin; i < cEnd; ++i)
        {
            __syncthreads(); // chunk i is there, and everybody has read chunk i - 1
            int const slot = (i - cBegin) & 1;
            bool const more = i + 1 < cEnd;
            if (more)
            {
                request(i + 1, next);
            }
            Pages const after = pages_of(min(i + 2, cEnd - 1));
            int const key0 = chunks.key0(i);
            if (active && key0 < most.hi && (key0 + kChunkKeys > least.lo || key0 < a.sinks))
            {
                uint8_t const* const keys = lds + slot * Lds::kSlot;
                uint8_t const* const values = keys + Lds::kKeys;
                f32x4 f[2];
                int there[2];
#pragma unroll
                for (int t = 0; t < 2; ++t)
                {
                    f[t] = *reinterpret_cast<f32x4 const*>(lds + 2 * Lds::kSlot + slot * Lds::kFactors + 16 * (2 * t + half));
                    there[t] = (int) f[t][3];
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
                        int const kRow = 32 * t + lq;
                        f16x8 const k = *reinterpret_cast<f16x8 const*>(keys + kRow * DP * 2 + 16 * swizzled(kRow, 2 * e + half));
                        s[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, q[e], s[t], 0, 0, 0);
                    }
                }
                bool const whole = sees_all(least, most, key0) && __ballot(there[0] < 16 || there[1] < 16) == 0;
#pragma unroll
                for (int t = 0; t < 2; ++t)
                {
#pragma unroll
                    for (int v = 0; v < 16; ++v)
                    {
                        s[t][v] = fmaf(s[t][v], f[t][0], f[t][1]);
                    }
                }
                if (!whole)
                {
                    hide(s, seen, key0 + 16 * half);
#pragma unroll
                    for (int t = 0; t < 2; ++t)
                    {
                        if (__ballot(there[t] < 16) != 0)
                        {
#pragma unroll
                            for (int v = 0; v < 16; ++v)
                            {
                                s[t][v] = v < there[t] ? s[t][v] : -__builtin_inff();
                            }
                        }
                    }
                }
                float mx = -__builtin_inff();
#pragma unroll
                for (int v = 0; v < 32; ++v)
                {
                    mx = fmaxf(mx, s[v >> 4][v & 15]);
                }
                sums.move(reduce_step<32>(mx, max_of));
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
                            p[e] = __builtin_amdgcn_exp2f(s[t][8 * w + e] + sums.negMax);
                            sums.sum = fmaf(p[e], f[t][2], sums.sum);
                        }
                        f16x8 const weights = weights_f16(p);
#pragma unroll
                        for (int d = 0; d < DV; ++d)
                        {
                            int const vRow = 32 * d + lq;
                            f16x8 const v = *reinterpret_cast<f16x8 const*>(
                                values + vRow * kChunkKeys * 2 + 16 * swizzled(vRow, 4 * t + 2 * half + w));
                            sums.out[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, weights, sums.out[d], 0, 0, 0);
                        }
                    }
                }
            }
            if (more)
            {
                deliver(i + 1, next, slot ^ 1);
            }
            next = after;
        }
    }
    if (wRow + lq >= rowEnd)
    {
        return;
    }
    float const total = reduce_step<32>(sums.sum, sum_of);
    size_t const outRow = (size_t) (r.row0 + token);
    size_t const slotAt = (outRow * a.qHeads + head) * a.slots + split;
    float const inverse = total == 0.f ? 0.f : 1.f / total;
    uint8_t* const to = a.out + 2 * (outRow * a.outToken + (int64_t) head * a.outHead);
#pragma unroll
    for (int d = 0; d < DV; ++d)
    {
#pragma unroll
        for (int v = 0; v < 16; v += 4)
        {
            int const e = 32 * d + 2 * v + 4 * half;
            if (e < c.d)
            {
                f32x4 const y = {sums.out[d][v], sums.out[d][v + 1], sums.out[d][v + 2], sums.out[d][v + 3]};
                if (used > 1)
                {
                    *reinterpret_cast<f32x4*>(a.partial + slotAt * c.d + e) = y;
                }
                else
                {
                    *reinterpret_cast<f16x4*>(to + 2 * e)
                        = f16x4{(f16) (y[0] * inverse), (f16) (y[1] * inverse), (f16) (y[2] * inverse), (f16) (y[3] * inverse)};
                }
            }
        }
    }
    if (used > 1 && half == 0)
    {
        *reinterpret_cast<f32x2*>(a.stats + 2 * slotAt) = f32x2{sums.negMax, total};
    }
}

// ------------------------------------------------------------------------------------------
// The parts of a row's keys: a workgroup a row, L lanes on a part's values, 256 / L parts at a time. Rows whose keys one workgroup
// had are written already.
// ------------------------------------------------------------------------------------------
template <int L>
__global__ __launch_bounds__(kThreads) void cached_join_kernel(CacheArgs const c, AttentionArgs const a, FastDiv const heads)
{
    constexpr int kGroups = kThreads / L;
    __shared__ f32x4 meet[kGroups][L];
    __shared__ float totals[kGroups];
    int const b = blockIdx.y, lane = threadIdx.x & 63;
    CacheRows const r = cache_rows(c, b);
    int const group = a.group.d;
    int64_t const rows = (int64_t) r.n * group;
    int const unit = blockIdx.x; // token, query head
    if (unit >= (int64_t) r.n * a.qHeads)
    {
        return;
    }
    int const token = (int) ((uint32_t) unit / heads), head = unit - token * (int) heads.d;
    bool const few = rows <= a.fewLimit;
    int const span = few ? a.fewSpan : a.manySpan;
    int i0 = 0, i1 = r.n - 1;
    if (!few)
    {
        int const own = head - (int) ((uint32_t) head / a.group) * group;
        int const row0 = (token * group + own) / kTileRows * kTileRows;
        i0 = (int) ((uint32_t) row0 / a.group);
        i1 = (int) ((uint32_t) (min((int64_t) row0 + kTileRows, rows) - 1) / a.group);
    }
    int const used = (chunks_of_tokens(r, i0, i1, a).total + span - 1) / span;
    if (used <= 1)
    {
        return;
    }
    size_t const outRow = (size_t) (r.row0 + token);
    size_t const slot = (outRow * a.qHeads + head) * a.slots;
    float least = kNothingSeen;
    for (int s = lane; s < used; s += kWaveSize)
    {
        least = fminf(least, a.stats[2 * (slot + s)]);
    }
    least = group_allreduce<kWaveSize>(least, [](float x, float y) { return fminf(x, y); });
    int const part = threadIdx.x / L, e = 4 * (threadIdx.x & (L - 1));
    float total = 0.f;
    f32x4 y = {0.f, 0.f, 0.f, 0.f};
    if (e < c.d)
    {
#pragma unroll 4
        for (int s = part; s < used; s += kGroups)
        {
            f32x2 const st = *reinterpret_cast<f32x2 const*>(a.stats + 2 * (slot + s));
            float const by = __builtin_amdgcn_exp2f(least - st[0]);
            total = fmaf(st[1], by, total);
            y += *reinterpret_cast<f32x4 const*>(a.partial + (slot + s) * c.d + e) * by;
        }
    }
    meet[part][threadIdx.x & (L - 1)] = y;
    if (e == 0)
    {
        totals[part] = total;
    }
    __syncthreads();
    if (threadIdx.x >= L || e >= c.d)
    {
        return;
    }
    total = totals[0];
    y = meet[0][threadIdx.x];
#pragma unroll
    for (int p = 1; p < kGroups; ++p)
    {
        total += totals[p];
        y += meet[p][threadIdx.x];
    }
    float const inverse = total == 0.f ? 0.f : 1.f / total;
    *reinterpret_cast<f16x4*>(a.out + 2 * (outRow * a.outToken + (int64_t) head * a.outHead + e))
        = f16x4{(f16) (y[0] * inverse), (f16) (y[1] * inverse), (f16) (y[2] * inverse), (f16) (y[3] * inverse)};
}

// ------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------

// How a call is shared out, from its sizes alone.
struct Plan
{
    bool few, many;
    int fewSpan, fewSplits, manySpan, manySplits;
    int fewLimit;
    int slots() const
    {
        return std::max(few ? fewSplits : 1, many ? manySplits : 1);
    }
};

// Chunks of `most` that a part takes, and how many parts that are at most.
void share_out(int64_t chunksAPart, int64_t most, int& span, int& splits)
{
    int64_t const s = std::max(chunksAPart, ceil_div(most, (int64_t) 65535)); // a launch's third extent
    span = (int) s;
    splits = (int) ceil_div(most, s);
}

Plan plan_of(trtamd_kv_cache_attention_params const& p)
{
    trtamd_kv_cache const& c = p.cache;
    Plan plan{};
    int const group = p.q_heads / c.kv_heads;
    int64_t const tokens = std::min(c.max_tokens, c.T);
    int64_t const rows = tokens * group;
    plan.few = rows <= kFewRows || c.B > 1;
    plan.many = rows > kFewRows;
    plan.fewLimit = plan.few ? kFewRows : 0;
    // keys that a row sees at most, and about
    int64_t const capacity = (int64_t) c.max_pages * c.page_tokens;
    auto const seen = [&](int64_t length) {
        int64_t const near = p.window ? (int64_t) p.window + tokens : length;
        return std::min(length, p.window ? near + p.sinks : length);
    };
    int64_t const most = ceil_div(seen(capacity), (int64_t) kChunkKeys) + 2;
    int64_t const chunks = ceil_div(seen(p.max_length > 0 ? std::min<int64_t>(p.max_length, capacity) : capacity), (int64_t) kChunkKeys) + (p.window ? 1 : 0);
    int64_t const cus = num_cus(), head = head_steps(c.d);
    // Few rows: one generation of workgroups, and where there are several sequences, whose lengths differ, parts of no more than 16
    // chunks. Four chunks are one a wavefront.
    int64_t const resident = cus * (head <= 4 ? 3 : head <= 8 ? 2 : 1);
    int64_t const even = ceil_div((int64_t) c.B * c.kv_heads * chunks, resident);
    share_out(std::max<int64_t>(c.B > 1 ? std::min<int64_t>(even, 16) : even, 4), most, plan.fewSpan, plan.fewSplits);
    // More rows: whole where there are tiles enough for two a CU.
    int64_t const tiles = ceil_div((int64_t) c.T * group, (int64_t) kTileRows) * c.kv_heads;
    share_out(tiles >= 2 * cus ? most : std::max<int64_t>(ceil_div(tiles * chunks, 2 * cus), 8), most, plan.manySpan, plan.manySplits);
    return plan;
}

size_t workspace_of(trtamd_kv_cache_attention_params const& p, Plan const& plan)
{
    size_t const slots = (size_t) plan.slots();
    return slots <= 1 ? 0 : (size_t) p.cache.T * p.q_heads * slots * (p.cache.d + 2) * sizeof(float);
}

int attention_check(char const* what, trtamd_kv_cache_attention_params const& p)
{
    if (int const st = cache_check(what, p.cache))
    {
        return st;
    }
    if (p.q_heads <= 0 || p.q_heads % p.cache.kv_heads != 0)
    {
        return set_error(TRTAMD_STATUS_BAD_PARAM, "%s: q_heads=%d (a multiple of kv_heads=%d)", what, p.q_heads, p.cache.kv_heads);
    }
    if (!(p.scale >= 0.f) || !std::isfinite(p.scale))
    {
        return set_error(TRTAMD_STATUS_BAD_PARAM, "%s: scale %g (finite and not negative)", what, p.scale);
    }
    if (p.window < 0 || p.sinks < 0 || p.max_length < 0)
    {
        return set_error(TRTAMD_STATUS_BAD_PARAM, "%s: window=%d sinks=%d max_length=%d", what, p.window, p.sinks, p.max_length);
    }
    if ((int64_t) p.cache.T * p.q_heads >= (int64_t) 1 << 30) // a launch has 2^32 threads
    {
        return set_error(TRTAMD_STATUS_NOT_SUPPORTED, "%s: T * q_heads of 2^30 or more", what);
    }
    return TRTAMD_STATUS_SUCCESS;
}

bool nothing(trtamd_kv_cache const& c)
{
    return c.B == 0 || c.T == 0 || c.max_tokens == 0;
}

template <int KS, bool FP8>
int launch_many(hipStream_t stream, dim3 grid, CacheArgs const& c, AttentionArgs const& a, FastDiv const& heads)
{
    constexpr int kBytes = ManyLds<padded_head(KS)>::kTotal;
    if constexpr (kBytes > 65536)
    {
        static hipError_t const e = hipFuncSetAttribute(reinterpret_cast<void const*>(cached_many_kernel<KS, FP8>),
            hipFuncAttributeMaxDynamicSharedMemorySize, kBytes);
        if (e != hipSuccess)
        {
            return set_error(TRTAMD_STATUS_FAILURE, "kv_cache_attention: cannot reserve %d bytes of LDS: %s", kBytes, hipGetErrorString(e));
        }
    }
    hipLaunchKernelGGL((cached_many_kernel<KS, FP8>), grid, dim3(kThreads), kBytes, stream, c, a, heads);
    return check_launch("cached_many_kernel");
}

template <bool FP8>
int launch(hipStream_t stream, trtamd_kv_cache_attention_params const& p, Plan const& plan, AttentionArgs const& a)
{
    trtamd_kv_cache const& k = p.cache;
    CacheArgs const c = cache_args(k);
    int const group = p.q_heads / k.kv_heads;
    if (plan.few)
    {
        dim3 const grid((unsigned) k.kv_heads, (unsigned) k.B, (unsigned) plan.fewSplits);
        int const st = by_head(k.d, [&](auto steps) {
            hipLaunchKernelGGL((cached_few_kernel<decltype(steps)::value, FP8>), grid, dim3(kThreads), 0, stream, c, a);
            return check_launch("cached_few_kernel");
        });
        if (st)
        {
            return st;
        }
    }
    if (plan.many)
    {
        int64_t const tiles = ceil_div((int64_t) std::min(k.max_tokens, k.T) * group, (int64_t) kTileRows);
        dim3 const grid((unsigned) (tiles * k.kv_heads), (unsigned) k.B, (unsigned) plan.manySplits);
        FastDiv const heads = fast_div((uint32_t) k.kv_heads);
        int const st = by_head(k.d, [&](auto steps) { return launch_many<decltype(steps)::value, FP8>(stream, grid, c, a, heads); });
        if (st)
        {
            return st;
        }
    }
    if (plan.slots() > 1)
    {
        // where only sequences of few rows are shared between workgroups, theirs alone
        int64_t const tokens = plan.many && plan.manySplits > 1 ? std::min(k.max_tokens, k.T) : std::min(std::min(k.max_tokens, k.T), kFewRows / group);
        dim3 const grid((unsigned) (tokens * p.q_heads), (unsigned) k.B);
        FastDiv const heads = fast_div((uint32_t) p.q_heads);
        auto const run = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, stream, c, a, heads); };
        k.d <= 64 ? run(cached_join_kernel<16>) : k.d <= 128 ? run(cached_join_kernel<32>) : run(cached_join_kernel<64>);
        return check_launch("cached_join_kernel");
    }
    return TRTAMD_STATUS_SUCCESS;
}

} // namespace
} // namespace trtamd

using namespace trtamd;

extern "C" size_t trtamd_kv_cache_attention_workspace_size(trtamd_kv_cache_attention_params const* params)
{
    if (params == nullptr)
    {
        return 0;
    }
    trtamd_kv_cache_attention_params const& p = *params;
    trtamd_kv_cache const& c = p.cache;
    if (c.kv_heads <= 0 || p.q_heads <= 0 || p.q_heads % c.kv_heads != 0 || c.page_tokens <= 0 || c.d <= 0 || c.max_pages <= 0 || c.B <= 0
        || c.T <= 0 || c.max_tokens <= 0 || p.window < 0 || p.sinks < 0 || p.max_length < 0)
    {
        return 0;
    }
    return workspace_of(p, plan_of(p));
}

extern "C" int trtamd_kv_cache_attention(trtamd_stream_t stream, trtamd_kv_cache_attention_params const* params)
{
    if (params == nullptr)
    {
        return set_error(TRTAMD_STATUS_BAD_PARAM, "kv_cache_attention: null params");
    }
    trtamd_kv_cache_attention_params const& p = *params;
    if (int const st = attention_check("kv_cache_attention", p))
    {
        return st;
    }
    for (int64_t s : {p.q_token_stride, p.q_head_stride, p.out_token_stride, p.out_head_stride})
    {
        if (s < 0 || s % 8 != 0)
        {
            return set_error(TRTAMD_STATUS_BAD_PARAM, "kv_cache_attention: strides must be multiples of 8 elements, and not negative");
        }
    }
    if (nothing(p.cache))
    {
        return TRTAMD_STATUS_SUCCESS;
    }
    if (p.q == nullptr || p.out == nullptr)
    {
        return set_error(TRTAMD_STATUS_BAD_PARAM, "kv_cache_attention: null pointer");
    }
    if (!aligned16(p.q) || !aligned16(p.out))
    {
        return set_error(TRTAMD_STATUS_BAD_PARAM, "kv_cache_attention: q and out must be 16-byte aligned");
    }
    Plan const plan = plan_of(p);
    size_t const bytes = workspace_of(p, plan);
    if (bytes > 0 && (p.workspace == nullptr || !aligned16(p.workspace) || p.workspace_bytes < bytes))
    {
        return set_error(TRTAMD_STATUS_BAD_PARAM, "kv_cache_attention: a 16-byte aligned workspace of %zu bytes is needed, %zu are there", bytes,
            p.workspace ? p.workspace_bytes : 0);
    }
    trtamd_kv_cache const& c = p.cache;
    AttentionArgs a{};
    a.q = reinterpret_cast<uint8_t const*>(p.q);
    a.out = reinterpret_cast<uint8_t*>(p.out);
    a.qToken = p.q_token_stride, a.qHead = p.q_head_stride, a.outToken = p.out_token_stride, a.outHead = p.out_head_stride;
    a.partial = static_cast<float*>(p.workspace);
    a.stats = a.partial + (bytes ? (size_t) c.T * p.q_heads * plan.slots() * c.d : 0);
    a.group = fast_div((uint32_t) (p.q_heads / c.kv_heads));
    a.qHeads = p.q_heads, a.window = p.window, a.sinks = p.sinks, a.slots = plan.slots();
    a.fewSpan = plan.fewSpan, a.manySpan = plan.manySpan, a.fewLimit = plan.fewLimit;
    a.scale = p.scale * 1.44269504088896f;
    return c.data_type == kCacheFp8 ? launch<true>(as_stream(stream), p, plan, a) : launch<false>(as_stream(stream), p, plan, a);
}
