// Norms of queries and keys for each head and the rotation of their pairs by position, one pass over Q and K.
//
//   y = x | x / sqrt(mean(x^2) + eps) w | (x - mean) / sqrt(var + eps) w + b        over the d values of a head
//   (a, b) -> (a cos(p f) - b sin(p f), b cos(p f) + a sin(p f))                    for its rotary_dim / 2 pairs
//
// HBM streaming: each value is read and written once.  33289 tokens, 16 and 16 heads of 64 in the packed layout, FP16: 54 us, 5.0 TB/s
// (a copy of 1 GiB reaches 5.2); heads of 128 5.7, in FP32 5.9 TB/s.  A group of a few lanes per head, each with 16 bytes a load, keeps the norm's sums
// within a row of 16 lanes and every load whole; with the angles worked out by every group for itself it took 88 us (their
// binary64 and the sine are 130 instructions a pair), with loads one behind the other 63.
#include "device_utils.hpp"
#include "host_utils.hpp"
#include "trtamd_encoder_ops.h"
#include "trtamd_test_hooks.h"

#include <algorithm>
#include <utility>

namespace trtamd
{
namespace
{

struct Side
{
    void const* in;
    void* out;
    int64_t inToken, inHead, outToken, outHead;
    float const* weight;
    float const* bias;
};

struct RotaryArgs
{
    Side side[2]; // queries, keys
    int T, qHeads, heads, d; // heads: of queries and keys
    int norm;
    float eps, inverseD;
    int half, adjacent; // half: pairs
    float const* frequencies;
    int32_t const* positions;
    int axes, cycled;
    int sections[TRTAMD_ROTARY_MAX_AXES];
    FastDiv headsDiv, halfDiv;
    int pitch; // of the cosines and sines of a token in LDS: pairs in whole chunks
};

__device__ inline int axis_of(RotaryArgs const& p, int pair)
{
    if (p.axes == 1)
    {
        return 0;
    }
    if (p.cycled)
    {
        int const turn = pair / p.axes, axis = pair - turn * p.axes;
        int left = 0;
#pragma unroll
        for (int a = 0; a < TRTAMD_ROTARY_MAX_AXES; ++a)
        {
            left = a == axis ? p.sections[a] : left;
        }
        return turn < left ? axis : 0;
    }
    int axis = 0, end = 0;
#pragma unroll
    for (int a = 0; a + 1 < TRTAMD_ROTARY_MAX_AXES; ++a)
    {
        end += p.sections[a]; // 0 behind the last axis
        axis += a + 1 < p.axes && pair >= end ? 1 : 0;
    }
    return axis;
}

// cos and sin of position * frequency: the angle in turns, reduced to half a turn in binary64 (binary32 has none of the
// fraction left at far positions), then the library's function of that in binary32.
__device__ inline void cos_sin(int32_t position, float frequency, float& c, float& s)
{
    constexpr double kInverseTwoPi = 0.15915494309189533577;
    double const turns = (double) position * (double) frequency * kInverseTwoPi;
    sincospif(2.f * (float) (turns - rint(turns)), &s, &c);
}

template <typename T, int V>
struct Chunk
{
    typedef T type __attribute__((ext_vector_type(V)));
};

template <typename T>
struct Chunk<T, 1>
{
    typedef T type;
};

template <typename T, int V>
using ChunkT = typename Chunk<T, V>::type;

template <int V, typename C>
__device__ __forceinline__ float element(C const& c, int e)
{
    if constexpr (V == 1)
    {
        return (float) c;
    }
    else
    {
        return (float) c[e];
    }
}

// Past the caches or not: see past_caches.
template <int V, bool PAST, typename T>
__device__ __forceinline__ void store_values(T* p, float const (&v)[V])
{
    if constexpr (V == 1)
    {
        *p = (T) v[0];
    }
    else
    {
        // converted in pairs, which is one instruction each
        typedef T Pair __attribute__((ext_vector_type(2)));
        ChunkT<T, V> x;
#pragma unroll
        for (int e = 0; e < V; e += 2)
        {
            Pair const two = __builtin_convertvector((f32x2{v[e], v[e + 1]}), Pair);
            x[e] = two[0];
            x[e + 1] = two[1];
        }
        if constexpr (PAST)
        {
            __builtin_nontemporal_store(x, reinterpret_cast<ChunkT<T, V>*>(p));
        }
        else
        {
            *reinterpret_cast<ChunkT<T, V>*>(p) = x;
        }
    }
}

// Values of a head per lane: one slot, or of narrow chunks as many as make 8.
constexpr int lane_values(int V)
{
    return V == 8 ? 16 : 8;
}

// A slot of a head: two chunks of V values, in such places that neighbouring lanes' first ones, and their second ones, lie side by side.  Pairs of
// distant values are the same places of chunks rotary_dim / 2 apart; adjacent pairs are in one chunk (V = 1: in two one behind the other); what
// is not rotated is cut in halves.
struct Slot
{
    int at[2];   // where the chunks are; at[1] < 0: there is no second one
    int pair[2]; // their first pairs (distant values: of both in pair[0]); those from `half` on are not rotated
};

template <int V, bool ADJACENT>
__device__ inline Slot slot_of(RotaryArgs const& p, int slot)
{
    int first, second, pair, pair2 = p.half;
    if constexpr (ADJACENT)
    {
        int const slots = (p.d + 2 * V - 1) / (2 * V);
        first = slot >= slots ? p.d : V == 1 ? 2 * slot : V * slot;
        second = V == 1 ? first + 1 : first + V * slots;
        pair = V == 1 ? slot : first / 2;
        pair2 = V == 1 ? p.half : second / 2;
    }
    else
    {
        int const pairSlots = p.half / V, n = slot - pairSlots, rest = (p.d - 2 * p.half + 2 * V - 1) / (2 * V);
        first = n < 0 ? slot * V : 2 * p.half + n * V;
        second = n < 0 ? first + p.half : n < rest ? first + rest * V : p.d;
        first = n < rest ? first : p.d;
        pair = n < 0 ? first : p.half;
    }
    return {{first < p.d ? first : -1, second < p.d ? second : -1}, {pair, pair2}};
}

// A workgroup takes 256 / G rows (a row: a head of a token), G lanes each.  Rows are numbered token by token, so its
// rows are heads of few tokens: their cosines and sines are worked out once, a thread each, while the rows are on their way, and
// shared through LDS.
template <typename T, int V, int G, bool ADJACENT, int NORM, bool PAST>
__global__ __launch_bounds__(256) void qk_norm_rotary_kernel(RotaryArgs const p)
{
    constexpr int kRows = 256 / G, NS = lane_values(V) / (2 * V);
    extern __shared__ __attribute__((aligned(16))) float lds[]; // [token][cosines | sines][pairs], pairs padded to whole chunks
    uint32_t const rows = (uint32_t) p.T * (uint32_t) p.heads;
    uint32_t const first = blockIdx.x * (uint32_t) kRows, row = first + threadIdx.x / G;
    uint32_t const live = min(row, rows - 1);
    uint32_t const t0 = first / p.headsDiv, t = live / p.headsDiv;
    // Loads come back in the order in which they are asked for: first what the angles need, which are worked out while the rest
    // is on its way.
    uint32_t const angles = p.half > 0 ? (min(first + (uint32_t) kRows - 1, rows - 1) / p.headsDiv - t0 + 1) * (uint32_t) p.half : 0;
    struct Angle
    {
        uint32_t token;
        int pair;
        int32_t position;
        float frequency;
    };
    auto const load_angle = [&](uint32_t i) {
        Angle a;
        a.token = i / p.halfDiv;
        a.pair = (int) (i - a.token * p.halfDiv.d);
        a.frequency = p.frequencies[a.pair];
        a.position = p.positions[(int64_t) axis_of(p, a.pair) * p.T + (t0 + a.token)];
        return a;
    };
    Angle angle = {};
    if (threadIdx.x < angles)
    {
        angle = load_angle(threadIdx.x);
    }

    int const h = (int) (live - t * p.headsDiv.d);
    bool const isQuery = h < p.qHeads;
    Side const& side = p.side[isQuery ? 0 : 1];
    int const head = isQuery ? h : h - p.qHeads;
    T const* in = static_cast<T const*>(side.in) + (int64_t) t * side.inToken + (int64_t) head * side.inHead;
    Slot slots[NS];
    ChunkT<T, V> raw[NS][2];
    ChunkT<float, V> weight[NS][2], bias[NS][2];
#pragma unroll
    for (int n = 0; n < NS; ++n)
    {
        slots[n] = slot_of<V, ADJACENT>(p, (int) (threadIdx.x % G) + n * G);
#pragma unroll
        for (int c = 0; c < 2; ++c)
        {
            // a lane without a chunk reads the first one instead of waiting behind a branch
            raw[n][c] = *reinterpret_cast<ChunkT<T, V> const*>(in + max(slots[n].at[c], 0));
        }
    }
#pragma unroll
    for (int n = 0; NORM != TRTAMD_QK_NORM_NONE && n < NS; ++n)
    {
#pragma unroll
        for (int c = 0; c < 2; ++c)
        {
            weight[n][c] = *reinterpret_cast<ChunkT<float, V> const*>(side.weight + max(slots[n].at[c], 0));
            if constexpr (NORM == TRTAMD_QK_NORM_LAYER)
            {
                bias[n][c] = *reinterpret_cast<ChunkT<float, V> const*>(side.bias + max(slots[n].at[c], 0));
            }
        }
    }
    if (angles > 0) // uniform
    {
        for (uint32_t i = threadIdx.x; i < angles; i += 256)
        {
            if (i >= 256)
            {
                angle = load_angle(i);
            }
            float c, s;
            cos_sin(angle.position, angle.frequency, c, s);
            float* const to = lds + angle.token * 2 * p.pitch + angle.pair;
            to[0] = c;
            to[p.pitch] = s;
        }
        __syncthreads();
    }

    float x[NS][2][V];
    // f on every value; and the sum of f over those that the lane has, chunk by chunk
    auto const each = [&](auto f) {
#pragma unroll
        for (int n = 0; n < NS; ++n)
        {
#pragma unroll
            for (int c = 0; c < 2; ++c)
            {
#pragma unroll
                for (int e = 0; e < V; ++e)
                {
                    f(x[n][c][e], n, c, e);
                }
            }
        }
    };
    auto const total = [&](auto f) {
        float all = 0.f;
#pragma unroll
        for (int n = 0; n < NS; ++n)
        {
#pragma unroll
            for (int c = 0; c < 2; ++c)
            {
                float chunk = 0.f;
#pragma unroll
                for (int e = 0; e < V; ++e)
                {
                    chunk = f(chunk, x[n][c][e]);
                }
                all += slots[n].at[c] >= 0 ? chunk : 0.f;
            }
        }
        return group_allreduce<G>(all, [](float a, float b) { return a + b; });
    };
    auto const square = [](float sum, float v) { return fmaf(v, v, sum); };
    each([&](float& v, int n, int c, int e) { v = element<V>(raw[n][c], e); });
    if constexpr (NORM == TRTAMD_QK_NORM_RMS)
    {
        float const scale = rsqrtf(fmaf(total(square), p.inverseD, p.eps));
        each([&](float& v, int n, int c, int e) { v = v * element<V>(weight[n][c], e) * scale; });
    }
    if constexpr (NORM == TRTAMD_QK_NORM_LAYER)
    {
        float const mean = total([](float sum, float v) { return sum + v; }) * p.inverseD;
        each([&](float& v, int, int, int) { v -= mean; });
        float const scale = rsqrtf(fmaf(total(square), p.inverseD, p.eps));
        each([&](float& v, int n, int c, int e) { v = fmaf(v * scale, element<V>(weight[n][c], e), element<V>(bias[n][c], e)); });
    }
    float const* const turns = lds + (t - t0) * 2 * p.pitch;
    auto const turn = [](float& a, float& b, float c, float s) {
        float const ra = a * c - b * s, rb = b * c + a * s;
        a = ra;
        b = rb;
    };
#pragma unroll
    for (int k = 0; k < NS; ++k)
    {
        if constexpr (ADJACENT && V > 1)
        {
#pragma unroll
            for (int h = 0; h < 2; ++h)
            {
                int const pair = slots[k].pair[h];
                if (pair < p.half)
                {
                    // chunks begin at multiples of V / 2 pairs; what lies behind the last pair is not used
                    ChunkT<float, V / 2> const c = *reinterpret_cast<ChunkT<float, V / 2> const*>(turns + pair);
                    ChunkT<float, V / 2> const s = *reinterpret_cast<ChunkT<float, V / 2> const*>(turns + p.pitch + pair);
#pragma unroll
                    for (int e = 0; e < V / 2; ++e)
                    {
                        if (pair + e < p.half)
                        {
                            turn(x[k][h][2 * e], x[k][h][2 * e + 1], element<V / 2>(c, e), element<V / 2>(s, e));
                        }
                    }
                }
            }
        }
        else
        {
            int const pair = slots[k].pair[0];
            if (pair < p.half)
            {
                ChunkT<float, V> const c = *reinterpret_cast<ChunkT<float, V> const*>(turns + pair);
                ChunkT<float, V> const s = *reinterpret_cast<ChunkT<float, V> const*>(turns + p.pitch + pair);
#pragma unroll
                for (int e = 0; e < V; ++e)
                {
                    turn(x[k][0][e], x[k][1][e], element<V>(c, e), element<V>(s, e));
                }
            }
        }
    }
    if (row >= rows)
    {
        return;
    }
    T* out = static_cast<T*>(side.out) + (int64_t) t * side.outToken + (int64_t) head * side.outHead;
#pragma unroll
    for (int k = 0; k < NS; ++k)
    {
#pragma unroll
        for (int c = 0; c < 2; ++c)
        {
            if (slots[k].at[c] >= 0)
            {
                store_values<V, PAST>(out + slots[k].at[c], x[k][c]);
            }
        }
    }
}

// The slots of a head (pairs of chunks of V values).
int slots_of(RotaryArgs const& a, int V)
{
    return a.adjacent ? ceil_div(a.d, 2 * V) : a.half / V + ceil_div(a.d - 2 * a.half, 2 * V);
}

// Whether chunks of V values start at multiples of their size everywhere.
template <typename T>
bool fits(RotaryArgs const& a, int V)
{
    auto const aligned = [](void const* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; };
    bool ok = a.d % V == 0 && (a.adjacent || a.half % V == 0);
    for (int i = 0; i < 2; ++i)
    {
        if (i == 0 ? a.qHeads == 0 : a.heads == a.qHeads)
        {
            continue;
        }
        Side const& s = a.side[i];
        ok = ok && aligned(s.in, V * sizeof(T)) && aligned(s.out, V * sizeof(T)) && s.inToken % V == 0 && s.inHead % V == 0
            && s.outToken % V == 0 && s.outHead % V == 0 && aligned(s.weight, 16) && aligned(s.bias, 16);
    }
    return ok;
}

// The kernel of a call: values a load, lanes a head, stores past the caches.
struct Route
{
    int values, lanes;
    bool pastCaches;
};

// The least of what a store instruction writes of a head side by side, in values: the rotated chunks and the others are in places of
// their own, and so are first and second chunks.
int shortest_row(RotaryArgs const& a, int V, int lanes)
{
    int const pairSlots = a.adjacent ? 0 : a.half / V, slots = slots_of(a, V);
    bool const odd = (a.adjacent ? a.d : a.d - 2 * a.half) % (2 * V) != 0; // the last slot has one chunk
    int shortest = a.d;
    for (int from = 0; from < slots; from += lanes)
    {
        int const end = std::min(from + lanes, slots), pairs = std::max(std::min(end, pairSlots) - from, 0), first = end - from - pairs;
        int const second = first - (odd && end == slots ? 1 : 0);
        for (int const chunks : {pairs, first, second})
        {
            shortest = chunks > 0 ? std::min(shortest, chunks * V) : shortest;
        }
    }
    return shortest;
}

// Where each row of values that a store instruction writes side by side is longer than 64 bytes, or of 64 and the outputs no more
// than half of the L2s: what ordinary stores leave there is written back at the kernel's end, while nothing else runs.  us by
// itself, past the caches / ordinary, FP16, halves, heads of Q and of K: 4963 tokens of 12 x 64 7.3 / 7.8, but of 16 x 64 9.2 / 8.6
// (20 MB), 33289 of 16 x 64 55 / 53; images (16 x 80) 23.7 / 25.7, a clip (12 x 128) 45 / 49, 33289 of 16 x 128 95 / 100.  Shorter
// rows reach the memory one by one: 33289 of 16 x 32 45 / 32, of 16 x 64 with 32 rotated 66 / 56, of 16 x 96 with 48 96 / 91 (of 16 x
// 72 with 36 and 16 x 80 with 40 121 / 122 and 87 / 89).  With the attention behind it (in place, 128 keys) the two are the same to 1
// %; what reads the outputs faster than that finds less of them in the last-level cache: with a copy of them behind it, 4963 of 16 x
// 128 take 37 / 32, images 56 / 47, 4963 of 16 x 80 with 40 rotated 34 / 29.
template <typename T>
bool past_caches(RotaryArgs const& a, int V, int lanes)
{
    int const row = shortest_row(a, V, lanes) * (int) sizeof(T);
    return row > 64 || (row == 64 && (int64_t) a.T * a.heads * a.d * (int64_t) sizeof(T) <= (int64_t) 16 << 20);
}

template <typename T>
Route route_of(RotaryArgs const& a)
{
    int V = 16 / (int) sizeof(T);
    while (V > 1 && !fits<T>(a, V))
    {
        V /= 2;
    }
    int const need = ceil_div(slots_of(a, V), lane_values(V) / (2 * V));
    int lanes = V >= 4 ? 2 : 8;
    while (lanes < need)
    {
        lanes *= 2;
    }
    return {V, lanes, V > 1 && past_caches<T>(a, V, lanes)};
}

// One of the kernels for the norms.
template <typename T, int V, int G, bool ADJACENT, bool PAST>
auto kernel_of(int norm)
{
    return norm == TRTAMD_QK_NORM_NONE ? qk_norm_rotary_kernel<T, V, G, ADJACENT, TRTAMD_QK_NORM_NONE, PAST>
        : norm == TRTAMD_QK_NORM_RMS  ? qk_norm_rotary_kernel<T, V, G, ADJACENT, TRTAMD_QK_NORM_RMS, PAST>
                                      : qk_norm_rotary_kernel<T, V, G, ADJACENT, TRTAMD_QK_NORM_LAYER, PAST>;
}

template <typename T, int V, int G>
int launch_group(hipStream_t stream, RotaryArgs a, [[maybe_unused]] bool past)
{
    constexpr int kRows = 256 / G;
    dim3 const grid((unsigned) ceil_div<int64_t>((int64_t) a.T * a.heads, kRows));
    a.pitch = ceil_div(a.half, V < 4 ? 4 : V) * (V < 4 ? 4 : V);
    // the rows of a workgroup are heads of no more tokens than this
    unsigned const lds = (unsigned) (2 * a.pitch * (ceil_div(kRows - 1, a.heads) + 1)) * sizeof(float);
    auto kernel = a.adjacent ? kernel_of<T, V, G, true, false>(a.norm) : kernel_of<T, V, G, false, false>(a.norm);
    if constexpr (V > 1 && G * V * sizeof(T) >= 64) // no row is longer than a head's lanes
    {
        if (past)
        {
            kernel = a.adjacent ? kernel_of<T, V, G, true, true>(a.norm) : kernel_of<T, V, G, false, true>(a.norm);
        }
    }
    hipLaunchKernelGGL(kernel, grid, dim3(256), lds, stream, a);
    return check_launch("qk_norm_rotary_kernel");
}

template <typename T, int V>
int launch_width(hipStream_t stream, RotaryArgs const& a, Route const& r)
{
    static_assert(TRTAMD_ROTARY_MAX_HEAD <= 32 * lane_values(1) && TRTAMD_ROTARY_MAX_HEAD <= 16 * lane_values(8), "lanes enough");
    if constexpr (V >= 4)
    {
        if (r.lanes <= 4)
        {
            return r.lanes == 2 ? launch_group<T, V, 2>(stream, a, r.pastCaches) : launch_group<T, V, 4>(stream, a, r.pastCaches);
        }
    }
    if constexpr (V < 8)
    {
        if (r.lanes == 32)
        {
            return launch_group<T, V, 32>(stream, a, r.pastCaches);
        }
    }
    return r.lanes == 8 ? launch_group<T, V, 8>(stream, a, r.pastCaches) : launch_group<T, V, 16>(stream, a, r.pastCaches);
}

template <typename T>
int launch_type(hipStream_t stream, RotaryArgs const& a)
{
    Route const r = route_of<T>(a);
    if constexpr (sizeof(T) == 2)
    {
        if (r.values == 8)
        {
            return launch_width<T, 8>(stream, a, r);
        }
    }
    return r.values == 4 ? launch_width<T, 4>(stream, a, r)
        : r.values == 2  ? launch_width<T, 2>(stream, a, r)
                         : launch_width<T, 1>(stream, a, r);
}

int bad(char const* what)
{
    return set_error(TRTAMD_STATUS_BAD_PARAM, "qk_norm_rotary: %s", what);
}

// Whether any two of n x m rows of d values, at i * a + j * b, overlap.
bool rows_overlap(int64_t n, int64_t a, int64_t m, int64_t b, int64_t d)
{
    typedef __int128 Wide; // strides are any 64 bits
    auto const size = [](Wide v) { return v < 0 ? -v : v; };
    if (size(a) > size(b))
    {
        std::swap(a, b);
        std::swap(n, m);
    }
    if (size(a) >= d && size(b) >= (n - 1) * size(a) + d)
    {
        return false; // all rows of one kind lie between two of the other
    }
    if (n > m)
    {
        std::swap(a, b);
        std::swap(n, m);
    }
    for (int64_t i = 0; i < n; ++i) // the distance of two rows is i * a + j * b, least where j is next to -i * a / b
    {
        Wide const off = (Wide) i * a, near = b == 0 ? i == 0 : -off / b;
        for (Wide j = near - 1; j <= near + 1; ++j)
        {
            if (size(j) < m && (i != 0 || j != 0) && size(off + j * b) < d)
            {
                return true;
            }
        }
    }
    return false;
}

int check(int32_t type, trtamd_qk_norm_rotary_params const* p)
{
    if (type != 0 && type != 1)
    {
        return set_error(TRTAMD_STATUS_NOT_SUPPORTED, "qk_norm_rotary: data type %d (0 = FP32, 1 = FP16)", type);
    }
    if (p == nullptr)
    {
        return bad("null pointer");
    }
    if (p->T < 0 || p->q_heads < 0 || p->k_heads < 0 || p->d < 1 || p->d > TRTAMD_ROTARY_MAX_HEAD)
    {
        return set_error(TRTAMD_STATUS_BAD_PARAM, "qk_norm_rotary: T=%d q_heads=%d k_heads=%d d=%d (d of 1 to %d)", p->T,
            p->q_heads, p->k_heads, p->d, (int) TRTAMD_ROTARY_MAX_HEAD);
    }
    if (p->norm < TRTAMD_QK_NORM_NONE || p->norm > TRTAMD_QK_NORM_LAYER)
    {
        return set_error(TRTAMD_STATUS_BAD_PARAM, "qk_norm_rotary: unknown norm %d", p->norm);
    }
    if (p->norm != TRTAMD_QK_NORM_NONE && !(p->eps >= 0.f))
    {
        return bad("eps must not be negative");
    }
    if (p->rotary_dim < 0 || p->rotary_dim > p->d || p->rotary_dim % 2 != 0)
    {
        return set_error(TRTAMD_STATUS_BAD_PARAM, "qk_norm_rotary: rotary_dim=%d (even, 0 to d=%d)", p->rotary_dim, p->d);
    }
    bool const rotates = p->rotary_dim > 0, norms = p->norm != TRTAMD_QK_NORM_NONE;
    if (!rotates && !norms)
    {
        return bad("neither a norm nor a rotation");
    }
    bool const many = (int64_t) p->T * ((int64_t) p->q_heads + p->k_heads) >= (int64_t) 1 << 26; // a launch has 2^32 threads
    size_t const size = type == 1 ? 2 : 4;
    for (int i = 0; i < 2; ++i)
    {
        bool const q = i == 0;
        if ((q ? p->q_heads : p->k_heads) == 0 || p->T == 0) // tensors without a token may have no address
        {
            continue;
        }
        void const* const data[2] = {q ? p->q : p->k, q ? p->q_out : p->k_out};
        int const used = p->norm == TRTAMD_QK_NORM_NONE ? 0 : p->norm == TRTAMD_QK_NORM_RMS ? 1 : 2;
        float const* const vectors[2] = {q ? p->q_weight : p->k_weight, q ? p->q_bias : p->k_bias};
        if (data[0] == nullptr || data[1] == nullptr || (used > 0 && vectors[0] == nullptr) || (used > 1 && vectors[1] == nullptr))
        {
            return bad("null pointer");
        }
        bool const sameToken = p->T == 1 || (q ? p->q_token_stride == p->q_out_token_stride : p->k_token_stride == p->k_out_token_stride);
        bool const sameHead = (q ? p->q_heads : p->k_heads) == 1
            || (q ? p->q_head_stride == p->q_out_head_stride : p->k_head_stride == p->k_out_head_stride);
        if (data[0] == data[1] && !(sameToken && sameHead))
        {
            return bad("in place the strides have to be the same");
        }
        if (data[0] == data[1] && !many
            && rows_overlap(p->T, q ? p->q_token_stride : p->k_token_stride, q ? p->q_heads : p->k_heads,
                q ? p->q_head_stride : p->k_head_stride, p->d))
        {
            return bad("in place no two heads may overlap");
        }
        for (int j = 0; j < 2; ++j)
        {
            if (reinterpret_cast<uintptr_t>(data[j]) % size != 0 || (j < used && reinterpret_cast<uintptr_t>(vectors[j]) % 4 != 0))
            {
                return bad("pointers must be aligned to their values");
            }
        }
    }
    if (rotates)
    {
        if (p->T > 0 && (p->frequencies == nullptr || p->positions == nullptr))
        {
            return bad("null pointer");
        }
        if (reinterpret_cast<uintptr_t>(p->frequencies) % 4 != 0 || reinterpret_cast<uintptr_t>(p->positions) % 4 != 0)
        {
            return bad("pointers must be aligned to their values");
        }
        if (p->axes < 1 || p->axes > TRTAMD_ROTARY_MAX_AXES)
        {
            return set_error(TRTAMD_STATUS_BAD_PARAM, "qk_norm_rotary: axes=%d (1 to %d)", p->axes, (int) TRTAMD_ROTARY_MAX_AXES);
        }
        int const pairs = p->rotary_dim / 2;
        int64_t sum = 0;
        for (int i = 0; i < p->axes && p->axes > 1; ++i)
        {
            int const n = p->sections[i];
            sum += n;
            // the last turn of an axis has to be a pair
            if (n < 0 || n > pairs || (p->axes_cycled && i > 0 && n > 0 && (n - 1) * p->axes + i >= pairs))
            {
                return set_error(TRTAMD_STATUS_BAD_PARAM, "qk_norm_rotary: sections[%d]=%d of %d pairs", i, n, pairs);
            }
        }
        if (p->axes > 1 && sum != pairs)
        {
            return set_error(TRTAMD_STATUS_BAD_PARAM, "qk_norm_rotary: sections of %lld pairs, rotary_dim has %d", (long long) sum, pairs);
        }
    }
    if (many)
    {
        return set_error(TRTAMD_STATUS_NOT_SUPPORTED, "qk_norm_rotary: 2^26 heads of tokens or more");
    }
    return TRTAMD_STATUS_SUCCESS;
}

RotaryArgs args_of(trtamd_qk_norm_rotary_params const* p)
{
    RotaryArgs a{};
    bool const norms = p->norm != TRTAMD_QK_NORM_NONE, layer = p->norm == TRTAMD_QK_NORM_LAYER;
    a.side[0] = {p->q, p->q_out, p->q_token_stride, p->q_head_stride, p->q_out_token_stride, p->q_out_head_stride,
        norms ? p->q_weight : nullptr, layer ? p->q_bias : nullptr};
    a.side[1] = {p->k, p->k_out, p->k_token_stride, p->k_head_stride, p->k_out_token_stride, p->k_out_head_stride,
        norms ? p->k_weight : nullptr, layer ? p->k_bias : nullptr};
    a.T = p->T;
    a.qHeads = p->q_heads;
    a.heads = p->q_heads + p->k_heads;
    a.d = p->d;
    a.norm = p->norm;
    a.eps = p->eps;
    a.inverseD = 1.f / (float) p->d;
    a.half = p->rotary_dim / 2;
    a.adjacent = p->adjacent_pairs != 0;
    a.frequencies = p->frequencies;
    a.positions = p->positions;
    a.axes = p->axes;
    a.cycled = p->axes_cycled != 0;
    for (int i = 0; i < p->axes && p->axes > 1 && a.half > 0; ++i)
    {
        a.sections[i] = p->sections[i];
    }
    a.headsDiv = fast_div((uint32_t) a.heads);
    a.halfDiv = fast_div((uint32_t) (a.half > 0 ? a.half : 1));
    return a;
}

} // namespace
} // namespace trtamd

using namespace trtamd;

extern "C" int trtamd_qk_norm_rotary(trtamd_stream_t stream, int32_t data_type, trtamd_qk_norm_rotary_params const* p)
{
    int const st = check(data_type, p);
    if (st != TRTAMD_STATUS_SUCCESS || p->T == 0 || p->q_heads + p->k_heads == 0)
    {
        return st;
    }
    RotaryArgs const a = args_of(p);
    return data_type == 1 ? launch_type<f16>(as_stream(stream), a) : launch_type<float>(as_stream(stream), a);
}

extern "C" int trtamd_test_qk_norm_rotary_route(int32_t data_type, trtamd_qk_norm_rotary_params const* p)
{
    if (check(data_type, p) != TRTAMD_STATUS_SUCCESS || p->T == 0 || p->q_heads + p->k_heads == 0)
    {
        return -1;
    }
    RotaryArgs const a = args_of(p);
    Route const r = data_type == 1 ? route_of<f16>(a) : route_of<float>(a);
    return r.values | r.lanes << 8 | (int) r.pastCaches << 16;
}
