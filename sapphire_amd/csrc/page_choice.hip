// page_choice.hip - the choice of pages: bounds of K per page, and the pages whose bounds promise the largest scores.
//
// With lo <= k <= hi in every dim of a page, q . k <= sum_d max(q_d lo_d, q_d hi_d) for all of its rows, so that pages are
// ranked without reading them. Borders between chosen and left pages are as close as scores come, so that sums run in 64 bits
// and ties go by the page's place in the sequence.
#include <algorithm>
#include <type_traits>

#include "internal.h"
#include "lanes.h"
#include "paged_dev.h"

namespace sapphire {

namespace {

typedef unsigned long long u64;

constexpr int kWave = 64, kThreads = 256, kWaves = kThreads / kWave;

struct BoundsArgs {
    PagedCache c;
    PageTable table;
    const int *from, *lengths;
    int slots;                             // pages of a row that the grid has
    uint16_t *bounds;                      // the layer's: [pages][heads][2][hd]
};

__device__ __forceinline__ float low_of(float a, float b) { return __builtin_elementwise_minimum(a, b); }      // (NaN stays)
__device__ __forceinline__ float high_of(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// fp32 to bf16, rounded up or down.
__device__ __forceinline__ uint32_t outward(float x, bool up) {
    if (x != x) return 0x7fc0u;
    const uint32_t u = __float_as_uint(x);
    return ((u >> 31 != 0) == up ? u : u + 0xffffu) >> 16;
}

// Extremes over a row of 16 lanes: each step, which pairs every lane with one of the other half, halves the values that a lane goes
// on with. Of N of them, lane c ends with N / 16, from c * N / 16 on; of eight, lanes 2i and 2i + 1 with value i.
// (Four steps of all N values in every lane are 512 instructions for 32 of them, of both kinds; the elements of a page of 32
// positions take 192.)
template <int CTRL, int H, int N, class Op>
__device__ __forceinline__ void halve(uint32_t (&v)[N], bool upper, Op op) {
#pragma unroll
    for (int i = 0; i < H; ++i) {
        const uint32_t keep = upper ? v[H + i] : v[i], give = upper ? v[i] : v[H + i];
        v[i] = op(keep, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)give, CTRL, 0xF, 0xF, false));
    }
}
template <int N, class Op>
__device__ __forceinline__ void row_extremes(uint32_t (&v)[N], int c, Op op) {
    static_assert(N == 8 || N % 16 == 0);
    halve<0x140, N / 2>(v, c & 8, op);                 // row_mirror, row_half_mirror, quad_perm [2,3,0,1] and [1,0,3,2]
    halve<0x141, N / 4>(v, c & 4, op);
    halve<0x4E, N / 8>(v, c & 2, op);
    if constexpr (N == 8) v[0] = op(v[0], (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v[0], 0xB1, 0xF, 0xF, false));
    else halve<0xB1, N / 16>(v, c & 1, op);
}

// The dims of a lane (c, m) of 16 positions of K: values e of piece j, and where they are. (The layout is that of the attention's
// operands: a lane has position c, so that bounds are the extremes over c.)
template <int CT, int HD>
struct Part {
    using T = Tile<CT, HD>;
    static constexpr int PARTS = HD > 128 ? 2 : 1;                         // of the dims: the extremes of 128 fit the registers
    static constexpr int W = CT == DT_F32 ? 4 : 8, N = HD / (4 * W) / PARTS;           // values of a piece, pieces
    static constexpr int B = CT == DT_Q4_0 ? 4 * T::G : 16;                // bytes of a load
    static constexpr int L = T::ROW / 4 / B / PARTS, NB = T::NB / PARTS;   // loads, scales
    uint32_t w[L][B / 4];
    float s[T::kQuant ? NB : 1];

    __device__ __forceinline__ void load(const uint8_t *tile, uint32_t ps, uint32_t p0, int part, int c, int m) {
#pragma unroll
        for (int l = 0; l < L; ++l) {
            const uint8_t *p = tile + T::k_code(p0, 0) + (uint32_t)(((part * L + l) * 4 + m) * 16 + c) * B;
            if constexpr (B == 8) *reinterpret_cast<pu2 *>(w[l]) = *reinterpret_cast<const pu2 *>(p);
            else *reinterpret_cast<pu4 *>(w[l]) = *reinterpret_cast<const pu4 *>(p);
        }
        if constexpr (T::kQuant) {
#pragma unroll
            for (int b = 0; b < NB; b += 2) {
                const pf2 v = *reinterpret_cast<const pf2 *>(tile + T::k_scale(ps, p0 + c, part * NB + b));
                s[b] = v.x;
                s[b + 1] = v.y;
            }
        }
    }
    static __device__ __forceinline__ int dim(int j, int m) { return (4 * j + m) * W; }
    __device__ __forceinline__ float at(int j, int e) const {
        if constexpr (CT == DT_F32) return __uint_as_float(w[j][e]);
        else if constexpr (CT == DT_Q8_0) return __fmul_rn((float)(int8_t)(w[j / 2][j % 2 * 2 + e / 4] >> (8 * (e % 4))), s[j]);
        else return __fmul_rn((float)((int)(w[j / T::G][j % T::G] << (28 - 8 * (e % 4) - 4 * (e / 4))) >> 28), s[j]);
    }
};

// A lane's extremes of its dims over the positions that it has seen, and its part of them over all sixteen lanes as bounds.
template <int CT, int HD>
struct Extremes {                          // fp32, Q8_0, Q4_0: as fp32
    using P = Part<CT, HD>;
    static constexpr int N = P::N * P::W, EACH = N / 16;
    uint32_t lo[N], hi[N];

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            lo[i] = __float_as_uint(INFINITY);
            hi[i] = __float_as_uint(-INFINITY);
        }
    }
    __device__ __forceinline__ void add(const P &x) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float v = x.at(i / P::W, i % P::W);
            lo[i] = __float_as_uint(low_of(__uint_as_float(lo[i]), v));
            hi[i] = __float_as_uint(high_of(__uint_as_float(hi[i]), v));
        }
    }
    // out: the low ones of the wave's dims; the high ones are HD further on
    __device__ __forceinline__ void store(uint16_t *out, int c, int m) {
        row_extremes(lo, c, [](uint32_t a, uint32_t b) { return __float_as_uint(low_of(__uint_as_float(a), __uint_as_float(b))); });
        row_extremes(hi, c, [](uint32_t a, uint32_t b) { return __float_as_uint(high_of(__uint_as_float(a), __uint_as_float(b))); });
        uint16_t *at = out + P::dim(c * EACH / P::W, m) + c * EACH % P::W;
        uint32_t a[EACH], z[EACH];
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
            a[e] = outward(__uint_as_float(lo[e]), false);
            z[e] = outward(__uint_as_float(hi[e]), true);
        }
        if constexpr (EACH == 2) {
            *reinterpret_cast<uint32_t *>(at) = a[0] | a[1] << 16;
            *reinterpret_cast<uint32_t *>(at + HD) = z[0] | z[1] << 16;
        } else {
            *at = (uint16_t)a[0];
            at[HD] = (uint16_t)z[0];
        }
    }
};
// 16-bit floats, two at a time as whole numbers: with sign and magnitude, the highest is the largest signed one or, where none is
// positive, the smallest unsigned one; the lowest the largest unsigned one if it is negative, or else the smallest. NaN have
// magnitudes above infinity's.
template <int CT, int HD>
struct Extremes16 {
    using P = Part<CT, HD>;
    typedef short s16x2 __attribute__((ext_vector_type(2)));
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    static constexpr int N = P::N * 4;     // words
    static constexpr uint32_t kInf = CT == DT_F16 ? 0x7c00u : 0x7f80u, kNan = CT == DT_F16 ? 0x7e00u : 0x7fc0u;
    uint32_t top[N], least[N], most[N];    // largest signed, smallest and largest unsigned

    static __device__ __forceinline__ uint32_t signed_max(uint32_t a, uint32_t b) {
        return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(s16x2, a), __builtin_bit_cast(s16x2, b)));
    }
    static __device__ __forceinline__ uint32_t unsigned_min(uint32_t a, uint32_t b) {
        return __builtin_bit_cast(uint32_t, __builtin_elementwise_min(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
    }
    static __device__ __forceinline__ uint32_t unsigned_max(uint32_t a, uint32_t b) {
        return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            top[i] = 0x80008000u;
            least[i] = 0xffffffffu;
            most[i] = 0;
        }
    }
    __device__ __forceinline__ void add(const P &x) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t w = x.w[i / 4][i % 4];
            top[i] = signed_max(top[i], w);
            least[i] = unsigned_min(least[i], w);
            most[i] = unsigned_max(most[i], w);
        }
    }
    __device__ __forceinline__ void store(uint16_t *out, int c, int m) {
        row_extremes(top, c, signed_max);
        row_extremes(least, c, unsigned_min);
        row_extremes(most, c, unsigned_max);
        uint32_t low = 0, high = 0;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const uint32_t t = top[0] >> (16 * e) & 0xffffu, l = least[0] >> (16 * e) & 0xffffu, u = most[0] >> (16 * e) & 0xffffu;
            const bool nan = (t < 0x8000u && t > kInf) || u > (0x8000u | kInf);
            low |= (nan ? kNan : u >= 0x8000u ? u : l) << (16 * e);
            high |= (nan ? kNan : t < 0x8000u ? t : l) << (16 * e);
        }
        const int i = N == 8 ? c >> 1 : c;             // the lane's word
        uint16_t *at = out + P::dim(i / 4, m) + i % 4 * 2;
        if (N == 16 || !(c & 1)) *reinterpret_cast<uint32_t *>(at) = low;
        if (N == 16 || c & 1) *reinterpret_cast<uint32_t *>(at + HD) = high;
    }
};

// A wave per page and K/V head (two for 256 dims): lane (c, m) has position c of every tile and a quarter of the dims. The
// bytes of K bound it: three documents of up to 131072 positions, 8 heads of 128 dims, bf16, pages of 32 (635 MB): 131 us, 4.8 TB/s
// (with the extremes of 16-bit values as fp32, and of all lanes alike: 151; with waves that go on to further pages: 136). In
// Q8_0 108 us and in Q4_0 77, bound by the issue of 6.5e7 and 6.2e7 vector instructions where bf16 has 3.7e7. One position of 16
// sequences: 5.2 us. grid (pages / 4, heads x parts, rows).
template <int CT, int HD>
__global__ __launch_bounds__(kThreads) void paged_bounds_kernel(BoundsArgs g) {
    using P = Part<CT, HD>;
    const int lane = threadIdx.x & (kWave - 1), c = lane & 15, m = lane >> 4;
    const int b = blockIdx.z, hk = blockIdx.y / P::PARTS, part = blockIdx.y % P::PARTS, ps = g.c.page_size;
    const int n = (int)min((int64_t)max(g.lengths[b], 0), (int64_t)g.table.ld * ps);
    const int from = g.from ? min(max(g.from[b], 0), n) : 0;
    if (from >= n) return;
    const int last = (int)page_of(g.c, (uint32_t)(n - 1) >> 4), first = max((int)page_of(g.c, (uint32_t)from >> 4), last - g.slots + 1);
    const int i = first + blockIdx.x * kWaves + (threadIdx.x / kWave);
    if (i > last) return;
    const int page = g.table.pages[(size_t)b * g.table.ld + i];
    if (page < 0 || page >= g.c.pages) return;
    const int here = min(n - i * ps, ps);                      // positions written
    const uint8_t *tile = g.c.k + ((size_t)page * g.c.nkv + hk) * g.c.tile_bytes;
    typename std::conditional<CT == DT_BF16 || CT == DT_F16, Extremes16<CT, HD>, Extremes<CT, HD>>::type all;
    all.clear();
    P k[2];                                                    // two tiles under way
    k[0].load(tile, ps, 0, part, c, m);
    if (16 < here) k[1].load(tile, ps, 16, part, c, m);
#pragma unroll 1
    for (int t = 0; t < here; t += 32) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int at = t + 16 * h;
            if (at + c < here) all.add(k[h]);                  // positions behind the last one do not count
            if (at + 32 < here) k[h].load(tile, ps, at + 32, part, c, m);
        }
    }
    all.store(g.bounds + ((size_t)page * g.c.nkv + hk) * 2 * HD + part * (HD / P::PARTS), c, m);
}

// ---- the choice ----

constexpr int kHeads = 4;                  // query heads of a wave: their q takes 128 registers in 64 bits
constexpr u64 kForced = ~0ull;             // above every score's key

struct SelectArgs {
    PagedCache c;
    PageTable table;
    Rows q;
    bool wide;                             // q's data and strides are multiples of 16 bytes
    const uint16_t *bounds;
    const int *lengths;
    int max_length, max_pages, group, k, first, last;
    u64 *keys;                             // [batch][K/V heads][max_pages]
    int *selected;
};

__device__ __forceinline__ int pages_of(const SelectArgs &g, int b) {
    const int n = min(max(g.lengths[b], 0), g.max_length);
    return n ? (int)page_of(g.c, (uint32_t)(n - 1) >> 4) + 1 : 0;
}
// Larger scores have larger keys, NaN the one of +inf; none is 0.
__device__ __forceinline__ u64 key_of(double s) {
    s = s != s ? INFINITY : s + 0.0;
    const u64 u = (u64)__double_as_longlong(s);
    return u >> 63 ? ~u : u | 1ull << 63;
}

// A double moved by DPP, or between halves of 32 lanes.
template <int CTRL>
__device__ __forceinline__ double moved(double v) {
    const u64 u = (u64)__double_as_longlong(v);
    return __longlong_as_double((long long)lanes::u64_dpp<CTRL>(u));
}
constexpr int kMirror = 0x140, kHalfMirror = 0x141, kXor2 = 0x4E, kXor1 = 0xB1, kOther16 = 0;

// Sums over the LP lanes of a page of four heads' values: each step, which pairs every lane with one of the other half, halves
// the heads that a lane goes on with, then the sums of what it has left. Lane l of a page ends with head (l / (LP / 4)) % 4.
template <int CTRL>
__device__ __forceinline__ double partner(double v) {
    if constexpr (CTRL == kOther16) return __shfl_xor(v, 16, kWave);
    else return moved<CTRL>(v);
}
template <int A, int B>
__device__ __forceinline__ double scatter(const double (&s)[4], bool upper_a, bool upper_b) {
    double t[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) t[i] = (upper_a ? s[2 + i] : s[i]) + partner<A>(upper_a ? s[i] : s[2 + i]);
    return (upper_b ? t[1] : t[0]) + partner<B>(upper_b ? t[0] : t[1]);
}
template <int LP>
__device__ __forceinline__ double page_sums(const double (&s)[4], int l) {
    double t;
    if constexpr (LP == 8) {
        t = scatter<kHalfMirror, kXor2>(s, l & 4, l & 2);
        return t + moved<kXor1>(t);
    } else {
        if constexpr (LP == 16) t = scatter<kMirror, kHalfMirror>(s, l & 8, l & 4);
        else {
            t = scatter<kOther16, kMirror>(s, l & 16, l & 8);
            t += moved<kHalfMirror>(t);
        }
        t += moved<kXor2>(t);
        return t + moved<kXor1>(t);
    }
}
// The largest of the four heads' keys, in every lane of the page.
template <int LP>
__device__ __forceinline__ u64 page_max(u64 k) {
    auto mx = [](u64 a, u64 b) { return a > b ? a : b; };
    if constexpr (LP == 8) {
        k = mx(k, lanes::u64_dpp<kXor2>(k));
        return mx(k, lanes::u64_dpp<kHalfMirror>(k));
    } else if constexpr (LP == 16) {
        k = mx(k, lanes::u64_dpp<kHalfMirror>(k));
        return mx(k, lanes::u64_dpp<kMirror>(k));
    } else {
        k = mx(k, lanes::u64_dpp<kMirror>(k));
        return mx(k, (u64)__shfl_xor((long long)k, 16, kWave));
    }
}

// Eight dims of a page per lane, HD / 8 lanes per page; every page's score, as a key, by four query heads at a time. Pages that
// are taken anyway have the largest key, ones that do not exist 0. Four documents of up to 131072 positions, 32 heads over 8 of
// 128 dims, pages of 32 (41 MB of bounds): 18.7 us, of which 8 are vector instructions (16 fused products in 64 bits
// per eight dims and head), the rest the chain lengths -> page -> bounds and the sums over lanes of the steps in turn. grid
// (pages, K/V heads, sequences).
template <int HD, bool F16>
__global__ __launch_bounds__(kThreads) void paged_scores_kernel(SelectArgs g) {
    constexpr int LP = HD / 8, PW = kWave / LP, STEP = kWaves * PW;        // lanes of a page, pages of a wave and of a workgroup
    const int lane = threadIdx.x & (kWave - 1), wid = threadIdx.x / kWave, l = lane % LP;
    const int b = blockIdx.z, hk = blockIdx.y, np = pages_of(g, b);
    const int i0 = blockIdx.x * STEP + wid * PW + lane / LP;
    if ((int)blockIdx.x * STEP >= np) return;
    const int *row = g.table.pages + (size_t)b * g.table.ld;
    u64 *keys = g.keys + ((size_t)b * g.c.nkv + hk) * g.max_pages;
    const uint16_t *of_head = g.bounds + (size_t)hk * 2 * HD + l * 8;
    const size_t stride = (size_t)g.c.nkv * 2 * HD;
    for (int h0 = 0; h0 < g.group; h0 += kHeads) {
        double up[kHeads][8], down[kHeads][8];                 // q where it is positive, and where it is negative
#pragma unroll
        for (int h = 0; h < kHeads; ++h) {
            Raw8 r;
            float x[8];
            // (heads behind the last one repeat it)
            load8(g.q.dtype, g.wide, g.q.p, (int64_t)b * g.q.ts + (int64_t)(hk * g.group + min(h0 + h, g.group - 1)) * g.q.hs + l * 8, r);
            values8(g.q.dtype, r, x);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                up[h][e] = x[e] > 0.f ? x[e] : x[e] != x[e] ? x[e] : 0.f;
                down[h][e] = x[e] < 0.f ? x[e] : 0.f;
            }
        }
        // a step's bounds are under way during the step before, and its page number during the one before that
        const int step = gridDim.x * STEP;
        pu4 lo, hi;
        int page, number = i0 < np ? row[i0] : -1;
        auto load = [&](int next) {
            page = number;
            number = next < np ? row[next] : -1;
            const uint16_t *p = of_head + (page >= 0 && page < g.c.pages ? (size_t)page : 0) * stride;
            lo = *reinterpret_cast<const pu4 *>(p);
            hi = *reinterpret_cast<const pu4 *>(p + HD);
        };
        load(i0 + step);
#pragma unroll 1
        for (int i = i0; i - lane / LP < np; i += step) {
            const pu4 a = lo, z = hi;
            const bool there = page >= 0 && page < g.c.pages;
            load(i + 2 * step);
            double s[kHeads] = {};
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t wa = e & 1 ? a[e / 2] >> 16 : a[e / 2] & 0xffffu, wz = e & 1 ? z[e / 2] >> 16 : z[e / 2] & 0xffffu;
                const double x = F16 ? from_f16(wa) : from_bf16(wa), y = F16 ? from_f16(wz) : from_bf16(wz);
#pragma unroll
                for (int h = 0; h < kHeads; ++h) s[h] = __builtin_fma(up[h][e], y, __builtin_fma(down[h][e], x, s[h]));
            }
            // (a head behind the last one repeats it)
            u64 key = page_max<LP>(key_of(page_sums<LP>(s, l)));
            if (l == 0 && i < np) {
                if (!there) key = 0;
                else if (i < g.first || i >= np - g.last) key = kForced;
                else if (h0 > 0) key = keys[i] > key ? keys[i] : key;
                keys[i] = key;
            }
        }
    }
}

constexpr int kPick = 1024, kPickWaves = kPick / kWave, kHold = 8, kBins = 1024, kFew = 64;
// Pages that are ranked against each other at once: 250 pages of one list 10.4 us with their scores, by bits 14.6; of 512, 18.
constexpr int kRanked = 256;

// The choice of few pages, as below: how many keys are ahead of each, a quarter of them counted by each of four threads.
__device__ __forceinline__ void rank_pages(const u64 *keys, int np, int k, int *out) {
    constexpr int PARTS = kPick / kRanked, EACH = kRanked / PARTS;
    __shared__ __attribute__((aligned(16))) u64 all[kRanked];
    __shared__ int ahead[PARTS][kRanked], taken[kRanked / kWave];
    const int tid = threadIdx.x, lane = tid & (kWave - 1), page = tid % kRanked, part = tid / kRanked;
    if (tid < kRanked) all[tid] = tid < np ? keys[tid] : 0;
    __syncthreads();
    const u64 mine = all[page];
    int count = 0;
#pragma unroll 8
    for (int j = part * EACH; j < (part + 1) * EACH; ++j) count += all[j] > mine || (all[j] == mine && j < page);
    ahead[part][page] = count;
    __syncthreads();
    int rank = 0;
#pragma unroll
    for (int p = 0; p < PARTS; ++p) rank += ahead[p][page];
    const bool on = mine != 0 && rank < k;
    const u64 mask = __ballot(on);
    if (tid < kRanked && lane == 0) taken[tid / kWave] = __popcll(mask);
    __syncthreads();
    int before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < kRanked / kWave; ++w) {
        before += w < page / kWave ? taken[w] : 0;
        total += taken[w];
    }
    if (tid < kRanked && on) out[before + __popcll(mask & ((1ull << lane) - 1))] = page;
    for (int i = total + tid; i < k; i += kPick) out[i] = -1;
}

// The k largest keys of a sequence's K/V head, equal ones from the first page on, in order of the pages. One workgroup; keys of up
// to 8192 pages stay in its registers. By ten bits at a time from the highest one in which keys differ, until the keys that
// decide are few enough to be ranked against each other. 128 of 4096 pages for 32 lists: 10.7 us, a chain of steps between
// barriers. grid (K/V heads, sequences).
__global__ __launch_bounds__(kPick) void paged_select_kernel(SelectArgs g) {
    __shared__ int bins[kBins], wave_sums[kPickWaves];
    __shared__ uint32_t counts[kHold * kPickWaves], sums[kHold * kPickWaves / kWave];
    __shared__ u64 ors[kPickWaves], ands[kPickWaves], few[kFew], few_key;
    __shared__ int few_count, found[3], few_ties;
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wid = tid / kWave;
    const int hk = blockIdx.x, b = blockIdx.y, np = pages_of(g, b);
    int *out = g.selected + ((size_t)b * g.c.nkv + hk) * g.k;
    const u64 *keys = g.keys + ((size_t)b * g.c.nkv + hk) * g.max_pages;
    if (np <= kRanked) {
        rank_pages(keys, np, g.k, out);
        return;
    }
    const int blocks = (np + kHold * kPick - 1) / (kHold * kPick);
    u64 key[kHold];
    auto load = [&](int blk) {
#pragma unroll
        for (int e = 0; e < kHold; ++e) {
            const int i = (blk * kHold + e) * kPick + tid;
            key[e] = i < np ? keys[i] : 0;
        }
    };
    // pages taken anyway, the others that exist, and the bits in which those differ
    int forced = 0, others = 0;
    u64 any = 0, all = ~0ull;
    for (int blk = 0; blk < blocks; ++blk) {
        load(blk);
#pragma unroll
        for (int e = 0; e < kHold; ++e) {
            const bool other = key[e] != 0 && key[e] != kForced;
            forced += __popcll(__ballot(key[e] == kForced));
            others += __popcll(__ballot(other));
            any |= other ? key[e] : 0;
            all &= other ? key[e] : ~0ull;
        }
    }
#pragma unroll
    for (int off = 1; off < kWave; off *= 2) {
        any |= __shfl_xor(any, off, kWave);
        all &= __shfl_xor(all, off, kWave);
    }
    if (lane == 0) {
        ors[wid] = any;
        ands[wid] = all;
        bins[wid] = forced;
        bins[kPickWaves + wid] = others;
    }
    __syncthreads();
    {
        const int w = lane & (kPickWaves - 1);
        any = ors[w];
        all = ands[w];
        forced = bins[w];
        others = bins[kPickWaves + w];
#pragma unroll
        for (int off = 1; off < kPickWaves; off *= 2) {
            any |= __shfl_xor(any, off, kWave);
            all &= __shfl_xor(all, off, kWave);
            forced += __shfl_xor(forced, off, kWave);
            others += __shfl_xor(others, off, kWave);
        }
    }
    __syncthreads();
    int need = min(max(g.k - forced, 0), others), shift = 0;
    u64 edge = 0;                                              // keys >> shift above it are taken, the first `need` that equal it too
    if (need == others) {
        edge = 0;                                              // (no key is 0)
        need = 0;
    } else if (need == 0) {
        edge = kForced - 1;
    } else {
        // (need < others, so that there is a key that decides)
        int top = any == all ? 0 : 64 - __builtin_clzll(any ^ all);        // keys agree from this bit on
        u64 prefix = top == 64 ? 0 : any >> top;
        edge = prefix;
        shift = top;
        while (top > 0) {
            shift = max(top - 10, 0);
            const uint32_t mask = (1u << (top - shift)) - 1;
            bins[tid] = 0;
            if (tid == 0) few_count = 0;
            __syncthreads();
            for (int blk = 0; blk < blocks; ++blk) {
                if (blocks > 1) load(blk);
#pragma unroll
                for (int e = 0; e < kHold; ++e)
                    if (key[e] != 0 && key[e] != kForced && (top == 64 ? 0 : key[e] >> top) == prefix)
                        atomicAdd(&bins[(uint32_t)(key[e] >> shift) & mask], 1);
            }
            __syncthreads();
            // how many keys are above each bin: thread t has bin 1023 - t
            const int mine = bins[kBins - 1 - tid];
            int upto = mine;
#pragma unroll
            for (int off = 1; off < kWave; off *= 2) {
                const int o = __shfl_up(upto, off, kWave);
                upto += lane >= off ? o : 0;
            }
            if (lane == kWave - 1) wave_sums[wid] = upto;
            __syncthreads();
            for (int w = 0; w < wid; ++w) upto += wave_sums[w];
            if (upto >= need && upto - mine < need) {
                found[0] = kBins - 1 - tid;
                found[1] = need - (upto - mine);
                found[2] = mine;
            }
            __syncthreads();
            prefix = prefix << (top - shift) | (u64)found[0];
            edge = prefix;
            need = found[1];
            top = shift;
            const int count = found[2];
            if (count == need || top == 0) break;
            if (count <= kFew) {
                // the keys that decide, each one's place among them
                for (int blk = 0; blk < blocks; ++blk) {
                    if (blocks > 1) load(blk);
#pragma unroll
                    for (int e = 0; e < kHold; ++e)
                        if (key[e] != 0 && key[e] != kForced && key[e] >> shift == prefix) few[atomicAdd(&few_count, 1)] = key[e];
                }
                __syncthreads();
                if (tid < count) {
                    int above = 0, same = 0;
                    for (int j = 0; j < count; ++j) {
                        above += few[j] > few[tid];
                        same += few[j] == few[tid];
                    }
                    if (above < need && above + same >= need) {            // (all that equal it write the same)
                        few_key = few[tid];
                        few_ties = need - above;
                    }
                }
                __syncthreads();
                edge = few_key;
                need = few_ties;
                shift = 0;
                break;
            }
        }
    }
    // in order of the pages, from how many are taken, and tie, ahead of each wave's of every thousand: both counts of a block
    // in one word
    int taken_before = 0, ties_before = 0;
    for (int blk = 0; blk < blocks; ++blk) {
        if (blocks > 1) load(blk);
        u64 above[kHold], ties[kHold];
#pragma unroll
        for (int e = 0; e < kHold; ++e) {
            const u64 v = key[e] >> shift;
            const bool on = key[e] != 0, is_forced = key[e] == kForced;
            above[e] = __ballot(on && (is_forced || v > edge));
            ties[e] = __ballot(on && !is_forced && v == edge);
            if (lane == 0) counts[e * kPickWaves + wid] = (uint32_t)__popcll(above[e]) | (uint32_t)__popcll(ties[e]) << 16;
        }
        __syncthreads();
        if (wid < kHold * kPickWaves / kWave) {
            const uint32_t mine = counts[tid];
            uint32_t upto = mine;
#pragma unroll
            for (int off = 1; off < kWave; off *= 2) {
                const uint32_t o = __shfl_up(upto, off, kWave);
                upto += lane >= off ? o : 0;
            }
            counts[tid] = upto - mine;
            if (lane == kWave - 1) sums[wid] = upto;
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < kHold; ++e) {
            const int at = e * kPickWaves + wid;
            uint32_t ahead = counts[at];
#pragma unroll
            for (int w = 0; w < kHold * kPickWaves / kWave - 1; ++w) ahead += at >= (w + 1) * kWave ? sums[w] : 0;
            const u64 below = (1ull << lane) - 1;
            const int a = taken_before + (int)(ahead & 0xffffu) + __popcll(above[e] & below), t = ties_before + (int)(ahead >> 16) + __popcll(ties[e] & below);
            const bool is_above = above[e] >> lane & 1, is_tie = (ties[e] >> lane & 1) && t < need;
            if (is_above || is_tie) out[a + min(t, need)] = (blk * kHold + e) * kPick + tid;
        }
        uint32_t whole = 0;
#pragma unroll
        for (int w = 0; w < kHold * kPickWaves / kWave; ++w) whole += sums[w];
        taken_before += whole & 0xffffu;
        ties_before += whole >> 16;
        __syncthreads();
    }
    const int total = taken_before + min(ties_before, need);
    for (int i = total + tid; i < g.k; i += kPick) out[i] = -1;
}

}  // namespace

int launch_paged_bounds(const PagedCache &c, uint16_t *bounds, const PageTable &t, const int *from, const int *lengths, int max_new,
                        hipStream_t s) {
    BoundsArgs g;
    g.c = c;
    g.table = t;
    g.from = from;
    g.lengths = lengths;
    g.slots = std::min((max_new - 1) / c.page_size + 2, t.ld);
    g.bounds = bounds;
    const dim3 grid((g.slots + kWaves - 1) / kWaves, c.nkv * (c.hd > 128 ? 2 : 1), t.rows), block(kThreads);
#define SPH_BOUNDS(CT, HD) \
    if (c.dtype == CT && c.hd == HD) hipLaunchKernelGGL((paged_bounds_kernel<CT, HD>), grid, block, 0, s, g);
#define SPH_BOUNDS_HD(HD) SPH_BOUNDS(DT_F32, HD) SPH_BOUNDS(DT_BF16, HD) SPH_BOUNDS(DT_F16, HD) SPH_BOUNDS(DT_Q8_0, HD) SPH_BOUNDS(DT_Q4_0, HD)
    SPH_BOUNDS_HD(64) SPH_BOUNDS_HD(128) SPH_BOUNDS_HD(256)
    return hip_ok(hipGetLastError(), "paged bounds launch") ? 0 : -1;
}

size_t paged_select_workspace(int nkv, int batch, int max_pages) { return (size_t)batch * nkv * max_pages * sizeof(u64); }

int launch_paged_select(const PagedCache &c, const uint16_t *bounds, const Rows &q, const PageTable &t, const int *lengths, int max_length,
                        int k, int first, int last, int *selected, void *ws, hipStream_t s) {
    SelectArgs g;
    g.c = c;
    g.table = t;
    g.q = q;
    g.wide = rows_wide(q);
    g.bounds = bounds;
    g.lengths = lengths;
    g.max_length = max_length;
    g.max_pages = (max_length + c.page_size - 1) / c.page_size;
    g.group = q.heads / c.nkv;
    g.k = k;
    g.first = first;
    g.last = last;
    g.keys = static_cast<u64 *>(ws);
    g.selected = selected;
    const int step = kWaves * 512 / c.hd;
    // q's 64-bit values are loaded once per workgroup, so that a few steps each pay; four documents of up to 131072 positions, 32
    // heads over 8, in pages of 32: 28.9 us with 1024 workgroups in all (the choice with it), 29.6 with 512, 35.1 with 2048
    const int64_t pairs = (int64_t)q.tokens * c.nkv, steps = (g.max_pages + step - 1) / step;
    const int64_t want = std::max<int64_t>(1, 1024 / pairs);
    const dim3 grid((unsigned)std::min(steps, want), c.nkv, q.tokens);
#define SPH_SCORES(HD, F16) \
    if (c.hd == HD && (c.dtype == DT_F16) == F16) hipLaunchKernelGGL((paged_scores_kernel<HD, F16>), grid, dim3(kThreads), 0, s, g);
    SPH_SCORES(64, false) SPH_SCORES(128, false) SPH_SCORES(256, false) SPH_SCORES(64, true) SPH_SCORES(128, true) SPH_SCORES(256, true)
    hipLaunchKernelGGL(paged_select_kernel, dim3(c.nkv, q.tokens), dim3(kPick), 0, s, g);
    return hip_ok(hipGetLastError(), "paged select launch") ? 0 : -1;
}

}  // namespace sapphire
