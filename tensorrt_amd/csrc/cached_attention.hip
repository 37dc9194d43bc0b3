// Attention of a call's rows over their sequences in the 8-bit cache.
//
//   s_j = scale * q k_j,   o = sum_j 2^(c s_j - m) v_j / sum_j 2^(c s_j - m),   c = log2(e)
//
// Bytes become binary16 exactly, so the products' operands are the bytes' values and the scales go elsewhere: a page's key scale into
// the multiplication that brings its scores to powers of 2, its value scale into the exponent, s + log2(value scale), where it costs
// nothing: the weights P' = p * value scale are what the second product wants, and p = P' / value scale is summed by one multiply-add.
// The running maximum is that of the weights P', so that the largest lies where binary16 has the most digits below it (kWeightsTop) whatever
// the scales are.
//
// Rows of one key head, (token, query head) with the heads of a group side by side, share the keys. Up to 16 of them (decoding, a few
// drafted tokens) go to `cached_few_kernel` or `cached_stretch_kernel`, which are bound by reading the cache; more to
// `cached_many_kernel`, bound by the matrix and vector instructions. A call whose sequences may be of both kinds launches both, and
// each leaves the other's sequences alone.
#include "attention_rows.hpp"
#include "host_utils.hpp"
#include "kv_cache.hpp"
#include "trtamd_test_hooks.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace trtamd
{
namespace
{

constexpr int kThreads = 256;
constexpr int kFewRows = 16;
constexpr int kTileRows = 128; // of cached_many_kernel

struct AttentionArgs
{
    uint8_t const* q; // FP16
    uint8_t* out;
    int64_t qToken, qHead, outToken, outHead; // elements
    float* partial;    // [row][slot][d], the sums that parts of a row's keys have in cached_many_kernel
    float* stats;      // [row][slot][2]: negMax (attention_rows.hpp), sum of the weights
    float* fewPartial; // [stretch][2][16][d]
    float* fewStats;   // [stretch][2][16][2]
    int32_t* fewHeads; // [B][key heads][2]: the first of a head's sums in fewPartial, and how many
    FastDiv group;     // query heads of a key head
    int32_t qHeads;
    int32_t window, sinks;
    int32_t slots;    // of a row in partial
    int32_t manySpan; // chunks of 64 keys that a workgroup takes
    int32_t fewLimit; // sequences of up to so many rows are the other kernels'
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

// What a page's scales are to its scores and weights. No score factor of 0 or below 2^-126 (0 times a score of -infinity is no number), nor
// an infinite one (times a score of 0), but what is a NaN stays one. The inverse is finite whatever the scale is: a weight of 0 is
// multiplied by it where no row sees the page, and scales of pages that were never written may be any.
struct PageFactors
{
    float score, log2Value, inverse;
};

__device__ inline PageFactors page_factors(float kScale, float vScale, float scale)
{
    PageFactors f;
    float const s = kScale * scale;
    f.score = s < 0x1p-126f ? 0x1p-126f : s > kLargest ? kLargest : s;
    // the values of a scale of 0 are zeros: any scale does, and the least one leaves the maximum to the others
    f.log2Value = fabsf(vScale) < 0x1p-126f ? -32.f : __builtin_amdgcn_logf(vScale);
    f.inverse = vScale >= 0x1p-126f ? 1.f / vScale : 0x1p32f;
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
// values. 16 keys lie in one page, so a lane has one page for the keys and one for the values and the factors of a chunk. The next
// chunk's keys are requested as soon as this one's are used, its values likewise: 16 KB a wavefront (heads of 128) are always on
// their way, two wavefronts a SIMD (a third one, at six spilled registers, was 7 % slower). Page sizes and the kind of bytes make no difference.
// ------------------------------------------------------------------------------------------

// A sequence and key head, the same for a wavefront.
struct FewUnit
{
    CacheRows r;
    Chunks chunks;
    int b, h, rows;
    // a row that sees nothing has a chunk all the same, which writes its zeros
    __device__ int count() const
    {
        return max(chunks.total, 1);
    }
};

// Sequences that are not here (more rows, or none) have no rows.
__device__ inline FewUnit few_unit(CacheArgs const& c, AttentionArgs const& a, int b, int h)
{
    FewUnit u;
    u.b = b;
    u.h = h;
    u.r = cache_rows(c, b);
    int64_t const rows = (int64_t) u.r.n * a.group.d;
    u.rows = rows <= kFewRows ? (int) rows : 0;
    u.chunks = chunks_of_tokens(u.r, 0, u.r.n - 1, a);
    return u;
}

// Pages of a chunk: those of the lane's keys and of its values.
struct FewPages
{
    int k, v;
};

template <int KS /* 16 of the head's values */, bool FP8>
struct FewWave
{
    static constexpr int DC = (KS + 3) / 4;
    f16x8 q[DC][2];
    u32x4 kr[4][DC], vr[KS];
    float kScale, vScale;
    f32x4 o[KS];
    float negMax, sum;
    int m, g, token, head;
    Seen seen, least, most;

    __device__ void begin(CacheArgs const& c, AttentionArgs const& a, FewUnit const& u)
    {
        int const lane = threadIdx.x & 63, row = min(lane & 15, u.rows - 1), group = a.group.d;
        m = lane & 15;
        g = lane >> 4;
        token = (int) ((uint32_t) row / a.group);
        head = u.h * group + row - token * group;
        seen = seen_by(u.r, token, a);
        least = seen_by(u.r, 0, a);
        most = seen_by(u.r, u.r.n - 1, a);
        uint8_t const* const from = a.q + 2 * ((int64_t) (u.r.row0 + token) * a.qToken + (int64_t) head * a.qHead);
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
#pragma unroll
        for (int t = 0; t < KS; ++t)
        {
            o[t] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
        negMax = kNothingSeen;
        sum = 0.f;
    }

    __device__ static FewPages pages_of(CacheArgs const& c, FewUnit const& u, int i)
    {
        int const lane = threadIdx.x & 63, key0 = u.chunks.key0(i);
        int32_t const* const table = c.table + (int64_t) u.b * c.maxPages;
        return {table[min((key0 + 4 * (lane & 12)) >> c.shift, c.maxPages - 1)], table[min((key0 + 16 * (lane >> 4)) >> c.shift, c.maxPages - 1)]};
    }

    __device__ void load_keys(CacheArgs const& c, FewUnit const& u, int i, FewPages const& p)
    {
        int const lane = threadIdx.x & 63, key = u.chunks.key0(i) + 4 * (lane & 12) + (lane & 3), P = 1 << c.shift;
        int const page = (uint32_t) p.k < (uint32_t) c.pages ? p.k : 0;
        uint8_t const* const from = c.k + page_offset(c, page, u.h) + (uint32_t) (key & (P - 1)) * c.d;
#pragma unroll
        for (int t = 0; t < 4; ++t)
        {
#pragma unroll
            for (int k = 0; k < DC; ++k)
            {
                // lanes behind the head's end read its last values, times a query of zeros
                kr[t][k] = *reinterpret_cast<u32x4 const*>(from + 4 * t * c.d + min(64 * k + 16 * (lane >> 4), c.d - 16));
            }
        }
    }

    __device__ void load_values(CacheArgs const& c, FewUnit const& u, int i, FewPages const& p)
    {
        int const lane = threadIdx.x & 63, key = u.chunks.key0(i) + 16 * (lane >> 4), P = 1 << c.shift;
        int const page = (uint32_t) p.v < (uint32_t) c.pages ? p.v : 0;
        size_t const scaleAt = (size_t) page * c.heads + u.h;
        kScale = c.kScale[scaleAt];
        vScale = c.vScale[scaleAt];
        uint8_t const* const from = c.v + page_offset(c, page, u.h) + (lane & 15) * P + (key & (P - 1));
#pragma unroll
        for (int t = 0; t < KS; ++t)
        {
            vr[t] = *reinterpret_cast<u32x4 const*>(from + (16 * t < c.d ? 16 * t * P : 0)); // elements behind the head's end are not written
        }
    }

    // The chunk that was loaded; the next one's keys and values are requested by `keys` and `values`.
    template <typename Keys, typename Values>
    __device__ __forceinline__ void step(CacheArgs const& c, AttentionArgs const& a, FewUnit const& u, int i, FewPages const& p, Keys&& keys, Values&& values)
    {
        int const key0 = u.chunks.key0(i);
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
        PageFactors const f = page_factors(kScale, vScale, a.scale);
        keys();
        // keys of this lane that are there at all
        int const there = (uint32_t) p.v < (uint32_t) c.pages ? min(max(u.r.len - key0 - 16 * g, 0), 16) : 0;
        bool const whole = sees_all(least, most, key0) && __ballot(there < 16) == 0;
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
            for (int t = 0; t < KS; ++t)
            {
                vr[t] &= keep; // what was never written may be anything, and 0 times it not 0
            }
        }
        float mx = -__builtin_inff();
#pragma unroll
        for (int t = 0; t < 4; ++t)
        {
            mx = fmaxf(mx, fmaxf(fmaxf(s[t][0], s[t][1]), fmaxf(s[t][2], s[t][3])));
        }
        mx = reduce_step<32>(reduce_step<16>(mx, max_of), max_of);
        float const negNew = fminf(kWeightsTop - mx, kNothingSeen);
        if (__ballot(negNew < negMax - 8.f) != 0)
        {
            float const to = fminf(negNew, negMax), by = __builtin_amdgcn_exp2f(to - negMax);
#pragma unroll
            for (int t = 0; t < KS; ++t)
            {
                o[t] *= by;
            }
            sum *= by;
            negMax = to;
        }
        f16x8 w[2];
#pragma unroll
        for (int j = 0; j < 2; ++j)
        {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e)
            {
                x[e] = __builtin_amdgcn_exp2f(s[2 * j + (e >> 2)][e & 3] + negMax);
                sum = fmaf(x[e], f.inverse, sum);
            }
            w[j] = weights_f16(x);
        }
#pragma unroll
        for (int t = 0; t < KS; ++t)
        {
            o[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(code_values8<FP8>(vr[t][0], vr[t][1]), w[0], o[t], 0, 0, 0);
            o[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(code_values8<FP8>(vr[t][2], vr[t][3]), w[1], o[t], 0, 0, 0);
        }
        values();
    }

    // Over the lanes that share a row.
    __device__ float total() const
    {
        return reduce_step<32>(reduce_step<16>(sum, sum_of), sum_of);
    }

};

// The sums of a workgroup's W wavefronts meet in LDS, as they are; then each thread adds some elements up over the wavefronts and gives
// them to store(tile, sums, negMax, sum of the weights).
template <int KS, bool FP8, int W>
struct FewMeeting
{
    static constexpr int kTiles = KS < 32 / W ? KS : 32 / W; // at a time: 32 KB
    f32x4 sums[W][kTiles][kWaveSize];
    float stats[W][2][kFewRows];

    template <typename Store>
    __device__ __forceinline__ void operator()(FewWave<KS, FP8> const& w, int wave, Store&& store)
    {
        int const lane = threadIdx.x & 63, m = w.m;
        float const own = w.total();
        if (lane < kFewRows)
        {
            stats[wave][0][m] = w.negMax;
            stats[wave][1][m] = own;
        }
        float least = kNothingSeen, total = 0.f, by[W];
#pragma unroll
        for (int t0 = 0; t0 < KS; t0 += kTiles)
        {
            if (t0 > 0)
            {
                __syncthreads();
            }
#pragma unroll
            for (int t = 0; t < kTiles; ++t)
            {
                if (t0 + t < KS)
                {
                    sums[wave][t][lane] = w.o[t0 + t];
                }
            }
            __syncthreads();
            if (t0 == 0)
            {
#pragma unroll
                for (int x = 0; x < W; ++x)
                {
                    by[x] = stats[x][0][m];
                    least = fminf(least, by[x]);
                }
#pragma unroll
                for (int x = 0; x < W; ++x)
                {
                    by[x] = __builtin_amdgcn_exp2f(least - by[x]);
                    total = fmaf(stats[x][1][m], by[x], total);
                }
            }
            for (int t = wave; t < kTiles && t0 + t < KS; t += W)
            {
                f32x4 y = sums[0][t][lane] * by[0];
#pragma unroll
                for (int x = 1; x < W; ++x)
                {
                    y += sums[x][t][lane] * by[x];
                }
                store(t0 + t, y, least, total);
            }
        }
    }
};

// Elements 16 t + 4 g .. + 3 of the lane's row, if there is such a row.
template <int KS, bool FP8>
__device__ inline void write_few(CacheArgs const& c, AttentionArgs const& a, FewUnit const& u, FewWave<KS, FP8> const& w, int t, f32x4 const& y, float total)
{
    float const inverse = total == 0.f ? 0.f : 1.f / total; // a row that sees nothing is zeros; a NaN stays one
    if (16 * t < c.d && w.m < u.rows)
    {
        uint8_t* const to = a.out + 2 * ((int64_t) (u.r.row0 + w.token) * a.outToken + (int64_t) w.head * a.outHead);
        *reinterpret_cast<f16x4*>(to + 2 * (16 * t + 4 * w.g))
            = f16x4{(f16) (y[0] * inverse), (f16) (y[1] * inverse), (f16) (y[2] * inverse), (f16) (y[3] * inverse)};
    }
}

// One workgroup a sequence and key head, its W wavefronts' sums meeting in LDS. 1000 keys of 16 heads of 64: 8.0 us with 8 wavefronts, tables,
// pages and two chunks a wavefront behind each other; with 16 it was 6 % slower.
template <int KS, bool FP8, int W>
__global__ __launch_bounds__(W* kWaveSize) __attribute__((amdgpu_waves_per_eu(KS <= 4 ? 3 : KS <= 8 ? 2 : 1))) void cached_few_kernel(
    CacheArgs const c, AttentionArgs const a)
{
    __shared__ FewMeeting<KS, FP8, W> meet;
    FewUnit const u = few_unit(c, a, blockIdx.y, blockIdx.x);
    if (u.rows == 0)
    {
        return;
    }
    int const wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    FewWave<KS, FP8> w;
    int i = wave, end = u.count();
    FewPages now{}, next{};
    if (i < end)
    {
        now = w.pages_of(c, u, i);
        next = w.pages_of(c, u, min(i + W, end - 1));
    }
    w.begin(c, a, u);
    if (i < end)
    {
        w.load_keys(c, u, i, now);
        w.load_values(c, u, i, now);
    }
    for (; i < end; i += W)
    {
        bool const more = i + W < end;
        FewPages after{};
        w.step(
            c, a, u, i, now,
            [&] {
                if (more)
                {
                    after = w.pages_of(c, u, min(i + 2 * W, end - 1));
                    w.load_keys(c, u, i + W, next);
                }
            },
            [&] {
                if (more)
                {
                    w.load_values(c, u, i + W, next);
                }
            });
        now = next;
        next = after;
    }
    meet(w, wave, [&](int t, f32x4 const& y, float, float total) { write_few(c, a, u, w, t, y, total); });
}

// All chunks of all sequences and key heads in a row, in equal stretches, one a workgroup, whose wavefronts take every fourth chunk:
// sequences of any lengths keep the chip evenly busy to the end, and a wavefront's requests never pause, also from one head to the
// next. A stretch that has all of a head's chunks writes its rows; of the others there is at most one at its beginning and one at its
// end, whose sums go to memory, and the stretch in which a head begins says which those are. Where heads are few (ALIGNED) every stretch
// is of one head: the meeting of the wavefronts and the next head's queries would be paid for twice by some.
// 64 sequences of 400 to 8000 keys, 8 heads of 128, in all: parts of 16 chunks of each head 90 us; stretches 85, with the wavefronts' sums
// met by all of them at once 82.5, with heads that count 3 to 6 chunks more 77.5 (12: 81); 64 sequences of 4000 109 -> 99 to 101, of which 94
// are this kernel (5.6 TB/s). Aligned, 16 sequences of up to 2000 17.5 -> 14.8; 131070 keys of 8 heads of 128 49 us with three sets of inputs, so
// that nothing is still in the last-level cache (268 MB, 5.5 TB/s; a copy moves 5.1), matrix cores 7 %, vector instructions 35 % of the cycles.
constexpr int kStretchWaves = 4;
constexpr int kHeadCost = 4; // chunks that a head counts more, for its queries and the wavefronts' meeting: so many places come before its first

// The sum over the lanes up to this one.
__device__ inline int wave_scan(int v)
{
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false); // from 1, 2, 4 and 8 lanes below, in rows of 16
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false); // the last lane of a row into the next
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false); // lane 31 into the upper half
    return v;
}

struct Stretch
{
    FewUnit u; // that it begins with, at chunk `first`
    int first;
    int start;  // the place of u: chunk i of it is at start + kHeadCost + i of all
    int end;    // of the stretch's places
    int share;  // places of a stretch
    bool none;
};

template <bool ALIGNED>
__device__ inline int unit_places(FewUnit const& u)
{
    return u.rows ? u.count() + (ALIGNED ? 0 : kHeadCost) : 0;
}

// u of lane l.
__device__ inline FewUnit unit_of_lane(FewUnit const& u, int b, int l)
{
    auto const from = [&](int x) { return __builtin_amdgcn_readlane(x, l); };
    FewUnit v;
    v.r = CacheRows{from(u.r.row0), from(u.r.n), from(u.r.begin), from(u.r.len)};
    v.chunks = Chunks{from(u.chunks.sinkChunks), from(u.chunks.first), from(u.chunks.total)};
    v.b = b;
    v.h = 0;
    v.rows = from(u.rows);
    return v;
}

template <bool ALIGNED>
__device__ inline Stretch stretch_of_workgroup(CacheArgs const& c, AttentionArgs const& a, int B)
{
    int const lane = threadIdx.x & 63, wgs = (int) gridDim.x, wg = (int) blockIdx.x;
    auto const unit_at = [&](int b) {
        FewUnit u{};
        if (b < B)
        {
            u = few_unit(c, a, b, 0);
        }
        return u;
    };
    FewUnit u = unit_at(lane);
    int n = unit_places<ALIGNED>(u);
    for (int b0 = kWaveSize; b0 < B; b0 += kWaveSize)
    {
        n += unit_places<ALIGNED>(unit_at(b0 + lane));
    }
    int const total = wave_sum_i32(n) * c.heads;
    Stretch s{};
    s.none = true;
    // A chunk a wavefront at least, behind the places in front of a head's first one: every stretch has a chunk. ALIGNED: so that the
    // stretches' number with one more for each head is no more than the workgroups'.
    s.share = max((total + wgs - 1) / (ALIGNED ? max(wgs - B * c.heads, 1) : wgs), kStretchWaves + (ALIGNED ? 0 : kHeadCost));
    int const target = ALIGNED ? wg : wg * s.share; // stretches, or chunks, before this one
    if (!ALIGNED && target >= total)
    {
        return s;
    }
    int before = 0;
    for (int b0 = 0;;)
    {
        int const of = unit_places<ALIGNED>(u), here = (ALIGNED ? (of + s.share - 1) / s.share : of) * c.heads, scanned = wave_scan(here);
        uint64_t const behind = __ballot(before + scanned > target);
        if (behind != 0)
        {
            int const l = __builtin_ctzll(behind);
            before += __builtin_amdgcn_readlane(scanned, l) - __builtin_amdgcn_readlane(here, l);
            s.u = unit_of_lane(u, b0 + l, l);
            break;
        }
        before += __builtin_amdgcn_readlane(scanned, 63);
        b0 += kWaveSize;
        if (b0 >= B)
        {
            return s; // none is left for this workgroup
        }
        u = unit_at(b0 + lane);
    }
    int const places = unit_places<ALIGNED>(s.u), each = ALIGNED ? (places + s.share - 1) / s.share : places;
    s.u.h = (target - before) / each;
    int const at = target - before - s.u.h * each;
    s.none = false;
    if (ALIGNED)
    {
        s.first = at * s.share;
        s.start = -kHeadCost;
        s.end = s.first + s.share;
    }
    else
    {
        s.first = max(at - kHeadCost, 0);
        s.start = target - at;
        s.end = min(target + s.share, total);
    }
    return s;
}

template <int KS, bool FP8, bool ALIGNED>
__global__ __launch_bounds__(kStretchWaves* kWaveSize) __attribute__((amdgpu_waves_per_eu(KS <= 4 ? 3 : KS <= 8 ? 2 : 1))) void cached_stretch_kernel(
    CacheArgs const c, AttentionArgs const a, int const B)
{
    constexpr int W = kStretchWaves;
    __shared__ FewMeeting<KS, FP8, W> meet;
    Stretch start = stretch_of_workgroup<ALIGNED>(c, a, B);
    // the same in every lane, which the compiler does not see behind the search
    int const head_of_start = start.u.h;
    start.u = unit_of_lane(start.u, __builtin_amdgcn_readfirstlane(start.u.b), 0);
    start.u.h = __builtin_amdgcn_readfirstlane(head_of_start);
    start.first = __builtin_amdgcn_readfirstlane(start.first);
    start.start = __builtin_amdgcn_readfirstlane(start.start);
    start.share = __builtin_amdgcn_readfirstlane(start.share);
    int const stop = __builtin_amdgcn_readfirstlane(start.end);
    if (start.none)
    {
        return;
    }
    int const wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // A chunk of the stretch, or none.
    struct Cursor
    {
        FewUnit u;
        int i, start;
        bool valid;
    };
    // By a number of chunks; only heads that have a place in the stretch are looked at.
    auto const next_head = [&](Cursor& x) {
        x.start += x.u.count() + kHeadCost;
        if (x.u.h + 1 < c.heads)
        {
            ++x.u.h;
            return;
        }
        do
        {
            x.u = few_unit(c, a, x.u.b + 1, 0);
        } while (x.u.rows == 0 && x.u.b + 1 < B);
    };
    auto const advance = [&](Cursor& x, int by) {
        x.i += by;
        while (x.i >= x.u.count())
        {
            bool const another = !ALIGNED && x.start + x.u.count() + 2 * kHeadCost < stop; // its first chunk's place
            x.i -= x.u.count();
            if (another)
            {
                next_head(x);
            }
            if (!another || x.u.rows == 0)
            {
                x.valid = false;
                return;
            }
        }
        x.valid = x.start + kHeadCost + x.i < stop;
    };
    Cursor head = {start.u, start.first, start.start, true}; // the head that the wavefronts are at
    Cursor now = head;
    advance(now, wave);
    Cursor next = now;
    FewWave<KS, FP8> w;
    FewPages nowPages{}, nextPages{};
    if (now.valid)
    {
        nowPages = w.pages_of(c, now.u, now.i);
        advance(next, W);
        if (next.valid)
        {
            nextPages = w.pages_of(c, next.u, next.i);
        }
    }
    w.begin(c, a, head.u);
    if (now.valid)
    {
        w.load_keys(c, now.u, now.i, nowPages);
        w.load_values(c, now.u, now.i, nowPages);
    }
    for (bool begun = false;; begun = true) // begun: the head begins in this stretch, behind another
    {
        while (now.valid && now.start == head.start)
        {
            FewPages afterPages{};
            Cursor after = next;
            w.step(
                c, a, head.u, now.i, nowPages,
                [&] {
                    if (next.valid)
                    {
                        advance(after, W);
                        if (after.valid)
                        {
                            afterPages = w.pages_of(c, after.u, after.i);
                        }
                        w.load_keys(c, next.u, next.i, nextPages);
                    }
                },
                [&] {
                    if (next.valid)
                    {
                        w.load_values(c, next.u, next.i, nextPages);
                    }
                });
            now = next;
            next = after;
            nowPages = nextPages;
            nextPages = afterPages;
        }
        FewUnit const& u = head.u;
        int const count = u.count(), last = min(count, stop - head.start - kHeadCost); // one past the stretch's last chunk of u
        bool const all = head.i == 0 && last == count;
        int const slot = 2 * (int) blockIdx.x + (begun ? 1 : 0);
        size_t const row = (size_t) slot * kFewRows + w.m;
        meet(w, wave, [&](int t, f32x4 const& y, float negMax, float total) {
            if (all)
            {
                write_few(c, a, u, w, t, y, total);
            }
            else if (16 * t < c.d && w.m < u.rows)
            {
                *reinterpret_cast<f32x4*>(a.fewPartial + row * c.d + 16 * t + 4 * w.g) = y;
                if (t == 0 && w.g == 0)
                {
                    *reinterpret_cast<f32x2*>(a.fewStats + 2 * row) = f32x2{negMax, total};
                }
            }
        });
        if (head.i == 0 && threadIdx.x == 0)
        {
            int const used = ALIGNED ? (count + start.share - 1) / start.share
                                     : (head.start + kHeadCost + count - 1) / start.share - (int) blockIdx.x + 1;
            *reinterpret_cast<i32x2*>(a.fewHeads + 2 * ((size_t) u.b * c.heads + u.h)) = i32x2{slot, used};
        }
        head.i = 0;
        advance(head, count);
        if (!head.valid)
        {
            return;
        }
        __syncthreads(); // the meeting's LDS
        w.begin(c, a, head.u);
    }
}

// The sums of a row's stretches: a workgroup a row, L lanes on the values of one, 256 / L of them at a time. Rows that one stretch had are
// written already.
template <int L>
__global__ __launch_bounds__(kThreads) void cached_stretch_join_kernel(CacheArgs const c, AttentionArgs const a)
{
    constexpr int kGroups = kThreads / L;
    __shared__ f32x4 meet[kGroups][L];
    __shared__ float totals[kGroups];
    int const row = blockIdx.x, h = blockIdx.y, b = blockIdx.z, lane = threadIdx.x & 63;
    i32x2 const where = *reinterpret_cast<i32x2 const*>(a.fewHeads + 2 * ((size_t) b * c.heads + h));
    CacheRows const r = cache_rows(c, b);
    int64_t const rows = (int64_t) r.n * a.group.d;
    if (row >= rows || rows > kFewRows || where[1] <= 1)
    {
        return;
    }
    // the first is where the head begins, the others are at the beginning of their stretches
    int const used = where[1], s0 = where[0];
    auto slot_of = [&](int s) { return (size_t) (s == 0 ? s0 : (s0 & ~1) + 2 * s) * kFewRows + row; };
    float least = kNothingSeen;
    for (int s = lane; s < used; s += kWaveSize)
    {
        least = fminf(least, a.fewStats[2 * slot_of(s)]);
    }
    least = group_allreduce<kWaveSize>(least, [](float x, float y) { return fminf(x, y); });
    int const part = threadIdx.x / L, e = 4 * (threadIdx.x & (L - 1));
    float sum = 0.f;
    f32x4 y = {0.f, 0.f, 0.f, 0.f};
    if (e < c.d)
    {
#pragma unroll 4
        for (int s = part; s < used; s += kGroups)
        {
            size_t const slot = slot_of(s);
            f32x2 const st = *reinterpret_cast<f32x2 const*>(a.fewStats + 2 * slot);
            float const by = __builtin_amdgcn_exp2f(least - st[0]);
            sum = fmaf(st[1], by, sum);
            y += *reinterpret_cast<f32x4 const*>(a.fewPartial + slot * c.d + e) * by;
        }
    }
    meet[part][threadIdx.x & (L - 1)] = y;
    if (e == 0)
    {
        totals[part] = sum;
    }
    __syncthreads();
    if (threadIdx.x >= L || e >= c.d)
    {
        return;
    }
    sum = totals[0];
    y = meet[0][threadIdx.x];
#pragma unroll
    for (int p = 1; p < kGroups; ++p)
    {
        sum += totals[p];
        y += meet[p][threadIdx.x];
    }
    float const inverse = sum == 0.f ? 0.f : 1.f / sum;
    int const token = (int) ((uint32_t) row / a.group), head = h * (int) a.group.d + row - token * (int) a.group.d;
    *reinterpret_cast<f16x4*>(a.out + 2 * ((int64_t) (r.row0 + token) * a.outToken + (int64_t) head * a.outHead + e))
        = f16x4{(f16) (y[0] * inverse), (f16) (y[1] * inverse), (f16) (y[2] * inverse), (f16) (y[3] * inverse)};
}

// ------------------------------------------------------------------------------------------
// More rows: 128 a workgroup, 32 a wavefront (attention_rows.hpp). Chunks of 64 keys become binary16 on their way into LDS, in two
// slots: the next chunk's bytes are requested before this one's products and converted behind them. Values come [d][key], so both
// operands are read as they lie, 16 bytes a lane.
// 4 x 1024 rows over 8192 keys before them, 32 heads of 128 on 8: 693 us, 849 TFLOP/s (the library's 8192^3 product 1110 to 1180). Matrix
// cores 37 % of the cycles and vector instructions 44 % (270 a wavefront and chunk: 160 of them the softmax and the conversion), which take
// turns. With branches on the head size between the products 4970: every accumulator was moved at each. Tiles of 256 rows, whose keys are
// converted once for twice the rows, 705; four tiles' worth of parts instead of two 3 to 10 % slower where tiles are few.
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
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(KS <= 4 ? 3 : KS <= 8 ? 2 : 1))) void cached_many_kernel(
    CacheArgs const c, AttentionArgs const a, FastDiv const heads)
{
    constexpr int DP = padded_head(KS);
    using Lds = ManyLds<DP>;
    constexpr int NL = DP / 64; // loads a thread of keys, and of values
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

    // This thread's pieces of a chunk: 16 bytes each of key tid / 4, and 16 keys of value rows tid / 4 + 64 l. A wavefront's 16 keys lie in
    // one page, so its place is scalar arithmetic.
    int32_t const* const table = c.table + (int64_t) b * c.maxPages;
    int const ownKey = 16 * wave + (lane >> 2), piece = lane & 3, vGroup = lane & 3, vRow = tid >> 2;
    // behind the head's end again its last values, times a query of zeros, and rows whose sums are not written
    uint32_t kAt[NL], vAt[NL];
#pragma unroll
    for (int l = 0; l < NL; ++l)
    {
        kAt[l] = (uint32_t) ((lane >> 2) * c.d + min(16 * (piece + 4 * l), c.d - 16));
        vAt[l] = (uint32_t) min(vRow + 64 * l, c.d - 1) * P;
    }
    auto page_at = [&](int key) { return table[min(key >> c.shift, c.maxPages - 1)]; };
    auto sound = [&](int page) { return (uint32_t) page < (uint32_t) c.pages ? page : 0; };
    struct Pages
    {
        int k, v;
    };
    auto pages_of = [&](int i) {
        int const key0 = chunks.key0(i);
        return Pages{__builtin_amdgcn_readfirstlane(page_at(key0 + 16 * wave)), page_at(key0 + 16 * vGroup)};
    };
    u32x4 kr[NL], vr[NL];
    float kScale = 0.f, vScale = 0.f;
    auto request = [&](int i, Pages const& p) {
        int const key0 = chunks.key0(i);
        uint8_t const* const keys = c.k + page_offset(c, sound(p.k), h) + (uint32_t) ((key0 + 16 * wave) & (P - 1)) * c.d;
        uint8_t const* const values = c.v + page_offset(c, sound(p.v), h) + ((key0 + 16 * vGroup) & (P - 1));
#pragma unroll
        for (int l = 0; l < NL; ++l)
        {
            kr[l] = *reinterpret_cast<u32x4 const*>(keys + kAt[l]);
            vr[l] = *reinterpret_cast<u32x4 const*>(values + vAt[l]);
        }
        if (tid < 4)
        {
            size_t const at = (size_t) sound(p.v) * c.heads + h;
            kScale = c.kScale[at];
            vScale = c.vScale[at];
        }
    };
    int const kRowAt = (ownKey & 32) + row_of_key(ownKey & 31);
    auto deliver = [&](int i, Pages const& p, int slot) {
        uint8_t* const keys = lds + slot * Lds::kSlot + kRowAt * DP * 2;
        uint8_t* const values = lds + slot * Lds::kSlot + Lds::kKeys + vRow * kChunkKeys * 2;
        int const there = (uint32_t) p.v < (uint32_t) c.pages ? min(max(r.len - chunks.key0(i) - 16 * vGroup, 0), 16) : 0;
        if (__ballot(there < 16) != 0)
        {
            u32x4 const keep = bytes_below(there);
#pragma unroll
            for (int l = 0; l < NL; ++l)
            {
                vr[l] &= keep; // what was never written may be anything, and 0 times it not 0
            }
        }
#pragma unroll
        for (int l = 0; l < NL; ++l)
        {
            int const at = 2 * (piece + 4 * l);
            *reinterpret_cast<f16x8*>(keys + 16 * swizzled<2 * DP>(kRowAt, at)) = code_values8<FP8>(kr[l][0], kr[l][1]);
            *reinterpret_cast<f16x8*>(keys + 16 * swizzled<2 * DP>(kRowAt, at + 1)) = code_values8<FP8>(kr[l][2], kr[l][3]);
            uint8_t* const v = values + 64 * l * kChunkKeys * 2;
            *reinterpret_cast<f16x8*>(v + 16 * swizzled<2 * kChunkKeys>(vRow, 2 * vGroup)) = code_values8<FP8>(vr[l][0], vr[l][1]);
            *reinterpret_cast<f16x8*>(v + 16 * swizzled<2 * kChunkKeys>(vRow, 2 * vGroup + 1)) = code_values8<FP8>(vr[l][2], vr[l][3]);
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
                        f16x8 const k = *reinterpret_cast<f16x8 const*>(keys + kRow * DP * 2 + 16 * swizzled<2 * DP>(kRow, 2 * e + half));
                        s[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, q[e], s[t], 0, 0, 0);
                    }
                }
                bool const whole = sees_all(least, most, key0) && __ballot(there[0] < 16 || there[1] < 16) == 0;
                // in powers of 2, s * by + add: where all keys are seen and there, by one multiply-add together with the maximum
                float by[2] = {f[0][0], f[1][0]}, add[2] = {f[0][1], f[1][1]};
                if (!whole)
                {
#pragma unroll
                    for (int t = 0; t < 2; ++t)
                    {
#pragma unroll
                        for (int v = 0; v < 16; ++v)
                        {
                            s[t][v] = fmaf(s[t][v], by[t], add[t]);
                        }
                        by[t] = 1.f;
                        add[t] = 0.f;
                    }
                    hide(s, seen, key0 + 16 * half, there[0], there[1]);
                }
                float mx = -__builtin_inff();
#pragma unroll
                for (int t = 0; t < 2; ++t)
                {
                    float own = s[t][0];
#pragma unroll
                    for (int v = 1; v < 16; ++v)
                    {
                        own = fmaxf(own, s[t][v]);
                    }
                    mx = fmaxf(mx, fmaf(own, by[t], add[t]));
                }
                sums.move(reduce_step<32>(mx, max_of));
#pragma unroll
                for (int t = 0; t < 2; ++t)
                {
                    float const base = add[t] + sums.negMax;
#pragma unroll
                    for (int w = 0; w < 2; ++w)
                    {
                        float p[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                        {
                            p[e] = __builtin_amdgcn_exp2f(fmaf(s[t][8 * w + e], by[t], base));
                            sums.sum = fmaf(p[e], f[t][2], sums.sum);
                        }
                        f16x8 const weights = weights_f16(p);
#pragma unroll
                        for (int d = 0; d < DV; ++d)
                        {
                            int const vRow = 32 * d + lq;
                            f16x8 const v = *reinterpret_cast<f16x8 const*>(
                                values + vRow * kChunkKeys * 2 + 16 * swizzled<2 * kChunkKeys>(vRow, 4 * t + 2 * half + w));
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
// had are written already. Three trips to memory: 4.6 us whatever the sizes; a wavefront a row, part after part, took up to 70.
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
    int const own = head - (int) ((uint32_t) head / a.group) * group;
    int const row0 = (token * group + own) / kTileRows * kTileRows;
    int const i0 = (int) ((uint32_t) row0 / a.group), i1 = (int) ((uint32_t) (min((int64_t) row0 + kTileRows, rows) - 1) / a.group);
    int const used = (chunks_of_tokens(r, i0, i1, a).total + a.manySpan - 1) / a.manySpan;
    if (used <= 1 || rows <= a.fewLimit)
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
    int fewLimit;
    int fewWaves;  // of a workgroup a sequence and key head, or
    int stretches; // how many
    bool aligned;  // each of one head
    int manySpan, manySplits;
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
    // Where some sequences may have more rows, few where others may have up to 16: not where the tensors' rows are as many as if all had
    // the most (two launches without work, 9 us), though tensors may be longer than their sequences; the tiles take any then.
    plan.few = rows <= kFewRows || (group <= kFewRows && c.T <= (c.B - 1) * tokens + kFewRows / group);
    plan.many = rows > kFewRows;
    plan.fewLimit = plan.few ? kFewRows : 0;
    // keys that a row sees at most, and about
    int64_t const capacity = (int64_t) c.max_pages * c.page_tokens;
    auto const seen = [&](int64_t length) { return p.window ? std::min(length, p.window + tokens + p.sinks) : length; };
    int64_t const most = ceil_div(seen(capacity), (int64_t) kChunkKeys) + 2;
    int64_t const chunks = ceil_div(seen(p.max_length > 0 ? std::min<int64_t>(p.max_length, capacity) : capacity), (int64_t) kChunkKeys) + (p.window ? 1 : 0);
    int64_t const cus = num_cus(), head = head_steps(c.d);
    int64_t const units = (int64_t) c.B * c.kv_heads;
    if (plan.few)
    {
        int64_t const resident = cus * (head <= 4 ? 3 : head <= 8 ? 2 : 1); // workgroups of four wavefronts
        bool const sums = units * most < (int64_t) 1 << 30;                      // of chunks fit 32 bits
        plan.fewWaves = units <= cus && head <= 8 ? 8 : 4;
        // Above 128 KB of keys and values a head, one workgroup a head is slower than stretches and their joining.
        if (chunks * head > 64 && units < 8 * resident && c.B <= 1024 && sums)
        {
            plan.stretches = (int) resident;
            plan.aligned = 4 * units <= resident;
        }
    }
    // More rows: whole keys where there are tiles enough for two a CU, otherwise parts of 8 chunks or more that make as many; of keys past
    // max_length no more than four times as many, since their sums have a place each in the workspace.
    int64_t const tiles = ceil_div((int64_t) c.T * group, (int64_t) kTileRows) * c.kv_heads, parts = ceil_div(2 * cus, std::max<int64_t>(tiles, 1));
    int64_t const span = std::max(std::max<int64_t>(ceil_div(tiles * chunks, 2 * cus), 8), ceil_div(most, 4 * parts));
    share_out(tiles >= 2 * cus ? most : span, most, plan.manySpan, plan.manySplits);
    return plan;
}

// Sums that go to memory, in floats: those of stretches, and of more rows' parts.
size_t few_floats(trtamd_kv_cache_attention_params const& p, Plan const& plan)
{
    return plan.stretches ? (size_t) plan.stretches * 2 * kFewRows * (p.cache.d + 2) + (((size_t) p.cache.B * p.cache.kv_heads * 2 + 3) & ~(size_t) 3) : 0;
}

size_t many_floats(trtamd_kv_cache_attention_params const& p, Plan const& plan)
{
    return plan.many && plan.manySplits > 1 ? (size_t) p.cache.T * p.q_heads * plan.manySplits * (p.cache.d + 2) : 0;
}

size_t workspace_of(trtamd_kv_cache_attention_params const& p, Plan const& plan)
{
    return (few_floats(p, plan) + many_floats(p, plan)) * sizeof(float);
}

// What plan_of relies on, and the size query: no pointer is looked at.
int attention_sizes_check(char const* what, trtamd_kv_cache_attention_params const& p)
{
    if (int const st = cache_sizes_check(what, p.cache))
    {
        return st;
    }
    if (p.q_heads <= 0 || p.q_heads % p.cache.kv_heads != 0)
    {
        return set_error(TRTAMD_STATUS_BAD_PARAM, "%s: q_heads=%d (a multiple of kv_heads=%d)", what, p.q_heads, p.cache.kv_heads);
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

int attention_check(char const* what, trtamd_kv_cache_attention_params const& p)
{
    int st = attention_sizes_check(what, p);
    st = st ? st : cache_check(what, p.cache);
    if (st)
    {
        return st;
    }
    if (!(p.scale >= 0.f) || !std::isfinite(p.scale))
    {
        return set_error(TRTAMD_STATUS_BAD_PARAM, "%s: scale %g (finite and not negative)", what, p.scale);
    }
    return TRTAMD_STATUS_SUCCESS;
}

template <int KS, bool FP8>
int launch_many(hipStream_t stream, dim3 grid, CacheArgs const& c, AttentionArgs const& a, FastDiv const& heads)
{
    constexpr int kBytes = ManyLds<padded_head(KS)>::kTotal;
    if constexpr (kBytes > 65536)
    {
        if (int const st = reserve_lds<cached_many_kernel<KS, FP8>>("kv_cache_attention", kBytes))
        {
            return st;
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
        int const st = by_head(k.d, [&](auto steps) {
            constexpr int S = decltype(steps)::value;
            if (plan.stretches)
            {
                dim3 const grid((unsigned) plan.stretches), block(kStretchWaves * kWaveSize);
                if (plan.aligned)
                {
                    hipLaunchKernelGGL((cached_stretch_kernel<S, FP8, true>), grid, block, 0, stream, c, a, k.B);
                }
                else
                {
                    hipLaunchKernelGGL((cached_stretch_kernel<S, FP8, false>), grid, block, 0, stream, c, a, k.B);
                }
                return check_launch("cached_stretch_kernel");
            }
            dim3 const grid((unsigned) k.kv_heads, (unsigned) k.B);
            if constexpr (S <= 8)
            {
                if (plan.fewWaves == 8)
                {
                    hipLaunchKernelGGL((cached_few_kernel<S, FP8, 8>), grid, dim3(8 * kWaveSize), 0, stream, c, a);
                    return check_launch("cached_few_kernel");
                }
            }
            hipLaunchKernelGGL((cached_few_kernel<S, FP8, 4>), grid, dim3(4 * kWaveSize), 0, stream, c, a);
            return check_launch("cached_few_kernel");
        });
        if (st)
        {
            return st;
        }
        if (plan.stretches)
        {
            dim3 const grid((unsigned) std::min<int64_t>(kFewRows, (int64_t) std::min(k.max_tokens, k.T) * group), (unsigned) k.kv_heads, (unsigned) k.B);
            auto const run = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, stream, c, a); };
            k.d <= 64 ? run(cached_stretch_join_kernel<16>) : k.d <= 128 ? run(cached_stretch_join_kernel<32>) : run(cached_stretch_join_kernel<64>);
            if (int const joined = check_launch("cached_stretch_join_kernel"))
            {
                return joined;
            }
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
    if (plan.many && plan.manySplits > 1)
    {
        dim3 const grid((unsigned) (std::min(k.max_tokens, k.T) * p.q_heads), (unsigned) k.B);
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
    if (params == nullptr || attention_sizes_check("kv_cache_attention_workspace_size", *params) || no_tokens(params->cache))
    {
        return 0;
    }
    return workspace_of(*params, plan_of(*params));
}

extern "C" int64_t trtamd_test_kv_cache_attention_route(trtamd_kv_cache_attention_params const* params)
{
    if (params == nullptr || attention_sizes_check("kv_cache_attention_route", *params) || no_tokens(params->cache))
    {
        return -1;
    }
    Plan const p = plan_of(*params);
    return (p.few && !p.stretches ? p.fewWaves : 0) | (p.stretches ? 16 : 0) | (p.stretches && p.aligned ? 32 : 0) | (p.many ? 64 : 0)
        | (int64_t) (p.many ? p.manySplits : 0) << 8;
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
    if (no_tokens(p.cache))
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
    a.fewPartial = static_cast<float*>(p.workspace);
    a.fewStats = a.fewPartial + (size_t) plan.stretches * 2 * kFewRows * c.d;
    a.fewHeads = reinterpret_cast<int32_t*>(a.fewStats + (size_t) plan.stretches * 2 * kFewRows * 2);
    a.partial = a.fewPartial + few_floats(p, plan);
    a.stats = a.partial + (plan.manySplits > 1 ? (size_t) c.T * p.q_heads * plan.manySplits * c.d : 0);
    a.group = fast_div((uint32_t) (p.q_heads / c.kv_heads));
    a.qHeads = p.q_heads, a.window = p.window, a.sinks = p.sinks, a.slots = plan.manySplits;
    a.manySpan = plan.manySpan, a.fewLimit = plan.fewLimit;
    a.scale = std::min(p.scale * 1.44269504088896f, kLargest);
    return c.data_type == kCacheFp8 ? launch<true>(as_stream(stream), p, plan, a) : launch<false>(as_stream(stream), p, plan, a);
}
