// What the attention kernels over a cache and in windows share: 32 rows of queries a wavefront, keys in chunks of 64 of which each
// half of the wavefront owns 16 consecutive ones twice, and a softmax kept up from chunk to chunk.
//
// S^T = K Q^T and O^T = V^T P^T with v_mfma_f32_32x32x16_f16. Row 8 b + 4 a + c of a block of 32 keys is key 16 a + 4 b + c, so that
// a lane of half a = lane / 32 gets the scores of keys 16 a .. 16 a + 15 of its query lane % 32, in order, and eight of them side by
// side are the second product's operand as they are: nothing moves between lanes but a row's maximum.
#pragma once

#include "device_utils.hpp"

#include <type_traits>

namespace trtamd
{

constexpr int kChunkKeys = 64;
constexpr float kLargest = 3.402823466e+38f;     // binary32
constexpr float kNothingSeen = kLargest;         // minus the maximum of no scores, finite
// Weights reach the second product in binary16, which has 2^-14 to 65504 with all its digits. The largest is held between 2^7 and 2^15 (a
// maximum moves the sums only where it passes the last one by 2^8), so that one of 2^-21 of it still has them and one of 2^-32 does not
// vanish: many keys that only add up to something behind one loud one. With the largest from 1 on, 8191 keys of 2^-26 each came out as nothing.
constexpr float kWeightsTop = 7.f;

// The key of a block of 32 that LDS row m of the block holds, and the row that holds key k.
__device__ inline int key_of_row(int m)
{
    return 16 * ((m >> 2) & 1) + 4 * (m >> 3) + (m & 3);
}

__device__ inline int row_of_key(int k)
{
    return 8 * ((k >> 2) & 3) + 4 * (k >> 4) + (k & 3);
}

// Which keys a row sees: those below sinks and from lo on, all below hi.
struct Seen
{
    int lo, hi, sinks;
    __device__ bool operator()(int key) const
    {
        return key < hi && (key >= lo || key < sinks);
    }
};

// The chunks that any of some rows sees: `sinkChunks` from 0 on, then those from `first` on.
struct Chunks
{
    int sinkChunks, first, total;
    __device__ int key0(int i) const
    {
        return (i < sinkChunks ? i : first + i - sinkChunks) * kChunkKeys;
    }
};

// lo: the lowest of the rows' lo, hi: the highest of their hi.
__device__ inline Chunks chunks_of(int lo, int hi, int sinks)
{
    Chunks c;
    int const sink = max(min(min(sinks, lo), hi), 0);
    c.sinkChunks = (sink + kChunkKeys - 1) / kChunkKeys;
    c.first = max(c.sinkChunks, lo / kChunkKeys);
    int const last = hi > lo ? (int) (((int64_t) hi + kChunkKeys - 1) / kChunkKeys) : 0;
    c.total = c.sinkChunks + max(last - c.first, 0);
    c.first = c.total > 0 ? c.first : 0; // a place that is there, for rows that see nothing
    return c;
}

typedef __attribute__((address_space(3))) uint8_t lds_u8;

// Where the 16-byte chunk `chunk` of LDS row `row` lies in its row, ROW bytes long, a power of 2 from 128 on. The 64 banks are 256 bytes: 16
// lanes that read the same chunk of 16 rows side by side then have them all (an operand's 16 bytes a lane).
template <int ROW>
__device__ inline int swizzled(int row, int chunk)
{
    return ROW == 128 ? chunk ^ ((row >> 1) & 7) : chunk ^ (row & 15);
}

// The same for transposing reads, whose 32 lanes read 64 bytes of four rows side by side.
template <int ROW>
__device__ inline int swizzled_turned(int row, int chunk)
{
    return ROW == 128 ? chunk ^ (2 * row & 4) : chunk ^ (4 * row & 12);
}

// A wavefront's 32 rows: DV blocks of 32 of the head's values.
template <int DV>
struct RowSums
{
    f32x16 out[DV]; // O^T: elements 32 d + 8 (v / 4) + 4 h + v % 4 of query lane % 32
    float negMax;   // kWeightsTop minus the maximum that the weights are relative to, in powers of 2
    float sum;      // of this lane's keys

    __device__ void clear()
    {
#pragma unroll
        for (int d = 0; d < DV; ++d)
        {
#pragma unroll
            for (int v = 0; v < 16; ++v)
            {
                out[d][v] = 0.f;
            }
        }
        negMax = kNothingSeen;
        sum = 0.f;
    }

    // Brings the sums so far to a new maximum where it passes the old one by more than 2^8, which weights in binary16 hold; mx: of
    // this chunk's scores, of both halves.
    __device__ void move(float mx)
    {
        float const negNew = fminf(kWeightsTop - mx, kNothingSeen);
        if (__ballot(negNew < negMax - 8.f) != 0)
        {
            float const to = fminf(negNew, negMax);
            float const f = __builtin_amdgcn_exp2f(to - negMax);
#pragma unroll
            for (int d = 0; d < DV; ++d)
            {
#pragma unroll
                for (int v = 0; v < 16; ++v)
                {
                    out[d][v] *= f;
                }
            }
            sum *= f;
            negMax = to;
        }
    }
};

__device__ inline float max_of(float a, float b)
{
    return fmaxf(a, b);
}

// Steps of 16 values that a head is rounded up to, one of the numbers that kernels are built for.
inline int head_steps(int d)
{
    int const s = (d + 15) / 16;
    return s <= 2 ? 2 : s <= 4 ? 4 : s <= 6 ? s : s <= 8 ? 8 : 16;
}

// Values of a head in LDS, rows of 128 bytes or a multiple.
constexpr int padded_head(int steps)
{
    return steps <= 4 ? 64 : steps <= 8 ? 128 : 256;
}

// Calls f with the number of steps as a constant.
template <typename F>
int by_head(int d, F&& f)
{
    switch (head_steps(d))
    {
    case 2: return f(std::integral_constant<int, 2>{});
    case 4: return f(std::integral_constant<int, 4>{});
    case 5: return f(std::integral_constant<int, 5>{});
    case 6: return f(std::integral_constant<int, 6>{});
    case 8: return f(std::integral_constant<int, 8>{});
    default: return f(std::integral_constant<int, 16>{});
    }
}

// Ones in the lowest n bits of 16.
__device__ inline uint32_t low_ones(int n)
{
    return (1u << min(max(n, 0), 16)) - 1u;
}

// Scores of keys that a row does not see become -infinity; keys key0 + 32 t + v in s[t][v], of which the first there[t] are there. By bits
// of a mask: two instructions a score and no scalar registers, where comparisons take three and a pair of them each.
__device__ inline void hide(f32x16 (&s)[2], Seen const& seen, int key0, int there0, int there1)
{
#pragma unroll
    for (int t = 0; t < 2; ++t)
    {
        int const from = key0 + 32 * t;
        uint32_t const mask = ((low_ones(seen.hi - from) & ~low_ones(seen.lo - from)) | low_ones(min(seen.sinks, seen.hi) - from)) & low_ones(t ? there1 : there0);
#pragma unroll
        for (int v = 0; v < 16; ++v)
        {
            uint32_t const keep = (uint32_t) __builtin_amdgcn_sbfe((int) mask, v, 1);
            s[t][v] = bits_as<float>((bits_as<uint32_t>(s[t][v]) & keep) | (0xff800000u & ~keep));
        }
    }
}

// Eight weights as the second product's operand, rounded half to even, in pairs (one instruction).
__device__ inline f16x8 weights_f16(float const (&p)[8])
{
    f16x8 r;
#pragma unroll
    for (int j = 0; j < 8; j += 2)
    {
        f16x2 const pair = __builtin_convertvector(f32x2{p[j], p[j + 1]}, f16x2);
        r[j] = pair[0];
        r[j + 1] = pair[1];
    }
    return r;
}

} // namespace trtamd
