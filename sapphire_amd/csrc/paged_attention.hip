// paged_attention.hip - attention of one new token per sequence over the paged cache.
//
// With scores s_p in log2 units, out = sum 2^(s_p - m) v_p / sum 2^(s_p - m) in one pass over K and V: a wave takes a
// tile of 16 positions (or two), forms the scores on the matrix cores with the query heads of a K/V head as columns,
// keeps a running maximum m and sum per column, and adds the weighted V on the matrix cores. Nothing is staged in LDS:
// the cache's tiles are in operand order, so that a wave's loads are whole KiB and land in the registers that the
// products read; the next tile's K is under way during the softmax and V's product, its V during the next scores.
//
// The bytes of K and V bound it, each read once by one workgroup for all heads of its K/V head (sixteen at most, over
// quantized caches eight). A sequence is cut into pieces of a fixed number of positions that workgroups take side by
// side, and a second launch joins their (maximum, sum, O); where whole sequences fill the chip they are not cut and the
// longest go first. The products' forms:
//   float cache, fp32 rows, up to 4 heads   4x4x1 fp32: its four columns are the heads
//   float cache, fp32 rows, more            16x16x4 fp32
//   float cache, 16-bit rows                16x16x32 of their type, the weights in two terms of it
//   quantized cache                         K's codes in 8-bit products with q's digits, V's codes as bf16
//
// Whole calls over 400 MB of K and V, sequences of 2000 positions, head_dim 64 to 256: up to four heads per K/V head
// 73-103 us (3.9-5.5 TB/s; a large copy moves 4.9), eight heads 78-107 us over float caches, 87-118 over Q8_0, 115-154
// over Q4_0. There vector and matrix units take turns at two waves per SIMD: of 91 us (100 sequences of up to 2000, 8 K/V heads
// of 256 dims) 49 are vector issue and 36 matrix cores. Sixteen heads over a quantized cache read and convert K and V twice:
// 137-255 us.
#include <algorithm>
#include <climits>
#include <cmath>

#include "internal.h"
#include "lanes.h"
#include "paged_dev.h"

namespace sapphire {

namespace {

constexpr int kWave = 64, kThreads = 256, kWaves = kThreads / kWave;
constexpr int kCols = 16;                  // query heads of a workgroup
constexpr int kPos = 16;                   // positions of a tile
constexpr int kMaxPieces = 256, kManyPieces = 32;          // of a sequence; that sixteen waves join instead of four
constexpr int kPieceUnit = 64;             // a piece is a multiple of so many positions
constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.693147180559945309f;

struct AttnArgs {
    PagedAttn a;
    int n_heads, group, col_tiles, piece, pieces;
    bool ordered;                          // longest sequences first
    bool wide;                             // out's data and strides are multiples of 16 bytes
    float *part;                           // [pieces][batch][n_heads][hd], unnormalised O
    float2 *ms;                            // [pieces][batch][n_heads]: maximum (log2 units), sum
};

// A lane's part of 16 positions of K (lane (c, m): position c, chunk m of each load) or V (positions 4m ..
// 4m + 3, its dims) as raw 16-byte pieces, and their elements as fp32.
template <int CT, int HD>
struct Raw {
    using T = Tile<CT, HD>;
    static constexpr int DPL = HD / 16;                        // V: dims of a lane
    static constexpr bool kHalf = T::ROW < 64;                 // Q4_0, head_dim 64: 8 bytes per lane
    static constexpr int N = kHalf ? 1 : T::ROW / 64;          // pieces
    static constexpr int W = CT == DT_F32 ? 4 : T::kQuant ? DPL : DPL < 8 ? DPL : 8;   // dims together in a V piece
    static constexpr int KE = CT == DT_F32 ? 4 : 8;            // float K: elements of a piece
    pu4 w[N];
    float s[T::kQuant ? (T::NB > 4 ? T::NB : 4) : 1];          // K: a row's block scales; V: four positions'

    __device__ __forceinline__ void load_k(const uint8_t *tile, uint32_t ps, uint32_t off, int c, int m) {
        if constexpr (kHalf) {
            const pu2 v = *reinterpret_cast<const pu2 *>(tile + T::k_code(off + c, 8 * m));
            w[0] = pu4{v.x, v.y, 0, 0};
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j)
                w[j] = *reinterpret_cast<const pu4 *>(tile + T::k_code(off, 0) + (uint32_t)((j * 4 + m) * 16 + c) * 16);
        }
        if constexpr (T::kQuant) {
#pragma unroll
            for (int b = 0; b < T::NB; b += 2) {
                const float2 v = *reinterpret_cast<const float2 *>(tile + T::k_scale(ps, off + c, b));
                s[b] = v.x;
                s[b + 1] = v.y;
            }
        }
    }
    // Float types: dim of element e of piece j in lane chunk m, and the element.
    static __device__ __forceinline__ int k_dim(int j, int m, int e) {
        return CT == DT_F32 ? 16 * j + 4 * m + e : 32 * j + 8 * m + e;
    }
    __device__ __forceinline__ float k_at(int j, int e) const {
        if constexpr (CT == DT_F32) return __uint_as_float(w[j][e]);
        else if constexpr (CT == DT_BF16) return __uint_as_float(e & 1 ? w[j][e >> 1] & 0xffff0000u : w[j][e >> 1] << 16);
        else return from_f16(e & 1 ? w[j][e >> 1] >> 16 : w[j][e >> 1] & 0xffffu);
    }
    __device__ __forceinline__ void load_v(const uint8_t *tile, uint32_t ps, uint32_t off, int c, int m) {
        if constexpr (kHalf) {
            const pu2 v = *reinterpret_cast<const pu2 *>(tile + T::v_run(off + 4 * m, c));
            w[0] = pu4{v.x, v.y, 0, 0};
        } else if constexpr (T::RUN >= 16) {                   // row-major: piece (r, i) of position 4m + r
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int i = 0; i < N / 4; ++i)
                    w[r * (N / 4) + i] = *reinterpret_cast<const pu4 *>(tile + (off + 4 * m + r) * T::ROW + i * 256 + c * 16);
        } else {                                               // P positions of the run
#pragma unroll
            for (int u = 0; u < N; ++u) w[u] = *reinterpret_cast<const pu4 *>(tile + T::v_run(off + 4 * m + u * T::P, c));
        }
        if constexpr (T::kQuant) {
            // of the blocks that column c of the weighted sum stands for
#pragma unroll
            for (int i = 0; i < (T::NB + 3) / 4; ++i) {
                const pf4 v = *reinterpret_cast<const pf4 *>(tile + T::v_scale(ps, off + 4 * m, 4 * i + (c & 3) % T::NB));
#pragma unroll
                for (int r = 0; r < 4; ++r) s[4 * i + r] = v[r];
            }
        }
    }
    // Quantized types. The score product's operand of block j: its codes (Q4_0: times 16) in element order.
    __device__ __forceinline__ pu2 k_codes(int j) const {
        if constexpr (CT == DT_Q8_0) return pu2{w[j / 2][j % 2 * 2], w[j / 2][j % 2 * 2 + 1]};
        const uint32_t v = w[j / T::G][j % T::G];
        return pu2{v << 4 & 0xf0f0f0f0u, v & 0xf0f0f0f0u};
    }
    // V's codes as signed bytes (Q4_0: times 16), word i: position r's DPL bytes start at byte r * DPL; Q4_0: the low
    // nibbles' bytes of all positions, then the high ones'. Of two sets of four blocks (head_dim 256) a lane has the first
    // set's dims in the first half of its elements and the second's in the other: lanes c < 8, which hold the first set, and
    // c + 8 exchange halves (v_element_dim).
    static constexpr int VW = DPL;
    static constexpr bool kTwoSets = T::NB == 8;
    // a in lanes c < 8 and b of lane c - 8 in the others; or b of lane c + 8 and a (row_ror:8 into half of the banks)
    static __device__ __forceinline__ uint32_t low_own(uint32_t a, uint32_t b) {
        return (uint32_t)__builtin_amdgcn_update_dpp((int)a, (int)b, 0x128, 0xF, 0xC, false);
    }
    static __device__ __forceinline__ uint32_t high_own(uint32_t a, uint32_t b) {
        return (uint32_t)__builtin_amdgcn_update_dpp((int)a, (int)b, 0x128, 0xF, 0x3, false);
    }
    __device__ __forceinline__ void v_bytes(uint32_t (&q)[VW], int c) const {
        if constexpr (CT == DT_Q8_0) {
#pragma unroll
            for (int i = 0; i < VW; ++i) {
                if constexpr (!kTwoSets) q[i] = w[i / 4][i % 4];
                else q[i] = i % 4 < 2 ? low_own(w[i / 4][i % 4], w[i / 4][i % 4 + 2]) : high_own(w[i / 4][i % 4], w[i / 4][i % 4 - 2]);
                asm("" : "+v"(q[i]));
            }
        } else {
            const int up = kTwoSets && c >= 8 ? 0 : 4;
#pragma unroll
            for (int i = 0; i < VW / 2; ++i) {
                const uint32_t v = w[i / 4][i % 4] ^ 0x88888888u;
                if constexpr (!kTwoSets) {
                    q[i] = v << 4 & 0xf0f0f0f0u;
                    q[VW / 2 + i] = v & 0xf0f0f0f0u;
                } else {                               // lanes c < 8 keep and take low nibbles, the others high ones
                    q[i] = low_own(v, v) << up & 0xf0f0f0f0u;
                    q[VW / 2 + i] = high_own(v, v) << up & 0xf0f0f0f0u;
                }
                // (the compiler would rather extract nibbles one by one)
                asm("" : "+v"(q[i]), "+v"(q[VW / 2 + i]));
            }
        }
    }
    // Dim of lane c's element x of them.
    static __device__ __forceinline__ int v_element_dim(int x, int c) {
        if constexpr (kTwoSets) return x / 8 * 128 + (c & 7) * 16 + (c >> 3) * 8 + x % 8;
        else return c * DPL + x;
    }
    // Element x of position 4m + r of them.
    static __device__ __forceinline__ float v_byte(const uint32_t (&q)[VW], int r, int x) {
        const int R = CT == DT_Q8_0 ? DPL : DPL / 2, i = (x / R) * (4 * R) + r * R + x % R;
        return (float)(int8_t)(q[i / 4] >> (8 * (i % 4)));
    }
    // Float types: position 4m + r as it is, or zeros.
    __device__ __forceinline__ void keep_v(int r, bool on) {
#pragma unroll
        for (int i = r * N; i < (r + 1) * N; ++i) w[i / 4][i % 4] = on ? w[i / 4][i % 4] : 0u;     // N words per position
    }
    // 16-bit types: elements x and x + 1 of position 4m + r.
    __device__ __forceinline__ uint32_t v_pair(int r, int x) const {
        const int i = r * (DPL / 2) + x / 2;
        return w[i / 4][i % 4];
    }
    // Dim of a lane's element x, and the element at position 4m + r.
    static __device__ __forceinline__ int v_dim(int x, int c) { return x / W * 16 * W + c * W + x % W; }
    __device__ __forceinline__ float v_at(int r, int x) const {
        if constexpr (CT == DT_F32) return __uint_as_float(w[r * (N / 4) + x / 4][x % 4]);
        // words of two elements: DPL / 2 per position, in order
        const uint32_t v = v_pair(r, x);
        if constexpr (CT == DT_BF16) return __uint_as_float(x & 1 ? v & 0xffff0000u : v << 16);
        else return from_f16(x & 1 ? v >> 16 : v & 0xffffu);
    }
};

template <int N>
__device__ __forceinline__ void load_some(int dtype, const uint8_t *p, int64_t i, float (&x)[N]) {
    if (dtype == DT_F32) {
#pragma unroll
        for (int e = 0; e < N; ++e) x[e] = reinterpret_cast<const float *>(p)[i + e];
    } else {
        uint16_t w[N];
#pragma unroll
        for (int e = 0; e < N; ++e) w[e] = reinterpret_cast<const uint16_t *>(p)[i + e];
#pragma unroll
        for (int e = 0; e < N; ++e) x[e] = from_16(dtype, w[e]);
    }
}
__device__ __forceinline__ void store1(int dtype, uint8_t *p, int64_t i, float v) {
    if (dtype == DT_F32) reinterpret_cast<float *>(p)[i] = v;
    else reinterpret_cast<uint16_t *>(p)[i] = (uint16_t)to_16(dtype, v);
}

// Four elements; `wide`: out's data and strides are multiples of 16 bytes.
__device__ __forceinline__ void store4(int dtype, bool wide, uint8_t *p, int64_t i, pf4 x) {
    if (!wide) {
#pragma unroll
        for (int e = 0; e < 4; ++e) store1(dtype, p, i + e, x[e]);
    } else if (dtype == DT_F32) {
        *reinterpret_cast<pf4 *>(p + i * 4) = x;
    } else {
        *reinterpret_cast<pu2 *>(p + i * 2) = pu2{pack_16(dtype, x[0], x[1]), pack_16(dtype, x[2], x[3])};
    }
}

__device__ __forceinline__ float lse_of(float mx, float sum) { return sum == 0.f ? -INFINITY : (mx + log2f(sum)) * kLn2; }

constexpr float kLazy = 8.0f;              // log2 units that a score may exceed the running maximum by

typedef __bf16 pb8 __attribute__((ext_vector_type(8)));
typedef _Float16 ph8 __attribute__((ext_vector_type(8)));
typedef int pi4 __attribute__((ext_vector_type(4)));

template <int CT>
__device__ __forceinline__ pf4 mfma16(pu4 a, pu4 b, pf4 c) {
    if constexpr (CT == DT_F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(ph8, a), __builtin_bit_cast(ph8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(pb8, a), __builtin_bit_cast(pb8, b), c, 0, 0, 0);
}

// The same over 16 positions: two words a lane.
typedef short ps4 __attribute__((ext_vector_type(4)));
typedef _Float16 ph4 __attribute__((ext_vector_type(4)));
template <int CT>
__device__ __forceinline__ pf4 mfma8(pu2 a, pu2 b, pf4 c) {
    if constexpr (CT == DT_F16) return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(ph4, a), __builtin_bit_cast(ph4, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(ps4, a), __builtin_bit_cast(ps4, b), c, 0, 0, 0);
}

// The sequence that workgroups z take when the longest go first, by eighths of max_length (in order within one): where
// whole sequences are a workgroup's work, a long one started late would run alone at the end. The same in every
// workgroup. masks: 64 words of LDS per 512 sequences.
constexpr int kOrdered = 1024, kClasses = 8;
__device__ __forceinline__ int nth_longest(const int *__restrict__ lengths, int batch, int max_length, int z,
                                           unsigned long long *masks) {
    const int lane = threadIdx.x & (kWave - 1), wid = threadIdx.x / kWave, chunks = (batch + kWave - 1) / kWave;
    const float scale = (float)kClasses / (float)max_length;
    for (int q = wid; q < chunks; q += kWaves) {
        const int b = q * kWave + lane, n = b < batch ? min(max(lengths[b], 0), max_length) : 0;
        const int cls = b < batch ? kClasses - 1 - min(kClasses - 1, (int)((float)n * scale)) : -1;
#pragma unroll
        for (int k = 0; k < kClasses; ++k) {
            const unsigned long long mask = __ballot(cls == k);
            if (lane == 0) masks[k * chunks + q] = mask;
        }
    }
    __syncthreads();
    // entries in order, 64 at a time: the one whose running count passes z
    for (int e0 = 0; e0 < kClasses * chunks; e0 += kWave) {
        const unsigned long long mask = e0 + lane < kClasses * chunks ? masks[e0 + lane] : 0;
        const int mine = __popcll(mask);
        int upto = mine;
#pragma unroll
        for (int off = 1; off < kWave; off *= 2) {
            const int below = __shfl_up(upto, off, kWave);
            upto += lane >= off ? below : 0;
        }
        const unsigned long long past = __ballot(upto > z);
        if (past) {
            const int e = __builtin_ctzll(past), left = z - __shfl(upto - mine, e, kWave);
            const unsigned long long m = lanes::u64_lane(mask, e);
            const unsigned long long at = __ballot((m >> lane & 1) && __popcll(m & ((1ull << lane) - 1)) == left);
            return (e0 + e) % chunks * kWave + __builtin_ctzll(at);
        }
        z -= __shfl(upto, kWave - 1, kWave);
    }
    return 0;                                          // (not reached: every sequence is in a class)
}

// A workgroup's part of the call: a piece of one sequence, for one K/V head's query heads h0 .. h0 + heads - 1,
// and its walk over the pages, HALVES tiles of 16 positions at a time.
template <int HALVES>
struct Walk {
    int b, hk, h0, heads, ps, start, lo, hi, last;
    size_t slot0, head_at, page_bytes;
    const __attribute__((address_space(4))) int *row;          // constant: page numbers come by scalar loads
    size_t at[HALVES];                     // a tile's page: its bytes' start
    uint32_t off[HALVES];                  // and its position in it
    bool there[HALVES];

    __device__ __forceinline__ Walk(const AttnArgs &g, int per_group) {
        const PagedAttn &a = g.a;
        b = blockIdx.z;
        if (g.ordered) {
            __shared__ unsigned long long masks[kOrdered / kWave * kClasses];
            b = __builtin_amdgcn_readfirstlane(nth_longest(a.lengths, gridDim.z, a.max_length, b, masks));
        }
        hk = blockIdx.y / g.col_tiles;
        const int ct = blockIdx.y - hk * g.col_tiles;
        h0 = hk * g.group + ct * per_group;
        heads = min(per_group, g.group - ct * per_group);
        ps = a.c.page_size;
        const int n = min(max(a.lengths[b], 0), a.max_length);
        start = a.window > 0 && n > a.window ? n - a.window : 0;
        lo = (start & ~(kPos - 1)) + blockIdx.x * g.piece;
        hi = min(n, lo + g.piece);
        last = hi > lo ? (hi - 1) & ~(kPos - 1) : 0;           // the piece's last tile
        slot0 = ((size_t)blockIdx.x * gridDim.z + b) * g.n_heads + h0;
        head_at = (size_t)hk * a.c.tile_bytes;
        page_bytes = (size_t)a.c.nkv * a.c.tile_bytes;
        row = (const __attribute__((address_space(4))) int *)(a.table.pages + (size_t)b * a.table.ld);
    }
    // nothing to do: the first piece says so to the join
    __device__ __forceinline__ bool empty(const AttnArgs &g) const {
        if (lo < hi || g.pieces == 1) return false;
        if (blockIdx.x == 0 && (int)threadIdx.x < heads) g.ms[slot0 + threadIdx.x] = make_float2(-INFINITY, 0.f);
        return true;
    }
    // tiles t and on; past the end: the last one again
    __device__ __forceinline__ void seek(const AttnArgs &g, int t) {
#pragma unroll
        for (int u = 0; u < HALVES; ++u) {
            const uint32_t t16 = (uint32_t)min(t + u * kPos, last) / kPos, i = page_of(g.a.c, t16);
            off[u] = t16 * kPos - i * (uint32_t)ps;
            const int page = row[__builtin_amdgcn_readfirstlane((int)i)];
            there[u] = page >= 0 && page < g.a.c.pages;
            at[u] = (there[u] ? (size_t)page : 0) * page_bytes + head_at;
        }
    }
    __device__ __forceinline__ bool whole(int t) const {       // every position of the step counts
        bool all = t >= start && t + HALVES * kPos <= hi;
#pragma unroll
        for (int u = 0; u < HALVES; ++u) all &= there[u];
        return all;
    }
};

__device__ __forceinline__ float capped(float x, float cap) { return __fmul_rn(cap, tanhf(__fdiv_rn(x, cap))); }

// The waves' O ([wave][head][HD + 4], unnormalised) and (maximum, sum) of each head: to out, or to the piece's part. A
// thread takes four dims.
template <int HD, int HEADS>
__device__ __forceinline__ void finish(const AttnArgs &g, int b, int h0, int heads, size_t slot0, const float *o,
                                       const float (&wm)[kWaves][HEADS], const float (&wsum)[kWaves][HEADS]) {
    constexpr int LD = HD + 4;
    const PagedAttn &a = g.a;
    __syncthreads();
    for (int i = threadIdx.x; i < heads * (HD / 4); i += kThreads) {
        const int r = i / (HD / 4), d = (i - r * (HD / 4)) * 4;
        float top = wm[0][r], tot = 0.f;
        pf4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 1; w < kWaves; ++w) top = fmaxf(top, wm[w][r]);
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            // a wave without positions, or with scores of -inf only, has sum 0; its factor must not be NaN
            const float s = wsum[w][r], f = s == 0.f ? 0.f : __builtin_amdgcn_exp2f(wm[w][r] - top);
            const pf4 ow = *reinterpret_cast<const pf4 *>(o + (w * HEADS + r) * LD + d);
            tot = __builtin_fmaf(s, f, tot);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = __builtin_fmaf(ow[e], f, x[e]);
        }
        if (g.pieces == 1) {
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = tot == 0.f ? 0.f : __fdiv_rn(x[e], tot);
            store4(a.out.dtype, g.wide, a.out.p, (int64_t)b * a.out.ts + (int64_t)(h0 + r) * a.out.hs + d, x);
            if (a.lse && d == 0) a.lse[(size_t)b * g.n_heads + h0 + r] = lse_of(top, tot);
        } else {
            *reinterpret_cast<pf4 *>(g.part + (slot0 + r) * HD + d) = x;
            if (d == 0) g.ms[slot0 + r] = make_float2(top, tot);
        }
    }
}

// Thread (r, i), r = tid / 16: q's elements HD / 16 * i and on of head h0 + r, zeros past the heads.
template <int N>
__device__ __forceinline__ void load_q(const Rows &q, int b, int h0, int heads, float (&x)[N]) {
    const int r = threadIdx.x >> 4;
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = 0.f;
    if (r < heads) load_some<N>(q.dtype, q.p, (int64_t)b * q.ts + (int64_t)(h0 + r) * q.hs + (threadIdx.x & 15) * N, x);
}

// fp32 rows over a float cache, at most four query heads of a K/V head. v_mfma_f32_4x4x1_16b_f32 is sixteen products of
// four rows and four columns: block (m, c / 4) multiplies the positions 4 (c / 4) .. + 3 of dim chunk m with the heads,
// and for the weighted sum the dims of lanes 4 (c / 4) .. + 3 at position 4m + r. Every column is used, where
// 16x16x4 would leave twelve of sixteen idle: a quarter of its cycles. (Eight heads as two sets of four gained 1 to 4 %
// over 16x16x4: not kept.) One sequence of 1024 positions, window 512, 4 heads of 256 dims, fp32: 6.2 us in nine pieces,
// bound by the chain length -> page -> K -> scores -> sum.
template <int CT, int HD>
__global__ __launch_bounds__(kThreads, HD == 64 ? 4 : HD == 128 ? 3 : 2) void paged_attn_few_kernel(AttnArgs g) {
    using R = Raw<CT, HD>;
    constexpr int LD = HD + 4, DPL = R::DPL, HEADS = 4, STEP = kWaves * kPos;
    __shared__ __attribute__((aligned(16))) float buf[kWaves * HEADS * LD];    // q, later the waves' O
    __shared__ float wm[kWaves][HEADS], wsum[kWaves][HEADS];
    const PagedAttn &a = g.a;
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wid = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int c = lane & 15, m = lane >> 4;
    Walk<1> at(g, HEADS);
    if (at.empty(g)) return;
    float qx[DPL];
    load_q<DPL>(a.q, at.b, at.h0, at.heads, qx);
    R k, v;
    int tb = at.lo + wid * kPos;
    if (tb < at.hi) {
        at.seek(g, tb);
        k.load_k(a.c.k + at.at[0], at.ps, at.off[0], c, m);
        v.load_v(a.c.v + at.at[0], at.ps, at.off[0], c, m);
    }
    if (tid < 16 * HEADS) {
#pragma unroll
        for (int e = 0; e < DPL; e += 4) *reinterpret_cast<pf4 *>(buf + (tid >> 4) * LD + (tid & 15) * DPL + e) = pf4{qx[e], qx[e + 1], qx[e + 2], qx[e + 3]};
    }
    __syncthreads();
    pf4 o[DPL];                                        // o[x][i]: dim v_dim(x, 4 (c / 4) + i) of head c % 4, positions of m only
#pragma unroll
    for (int x = 0; x < DPL; ++x) o[x] = pf4{0.f, 0.f, 0.f, 0.f};
    // scores in log2 units: without a cap in one product
    const float cap = a.softcap, sl2 = cap > 0.f ? a.scale : __fmul_rn(a.scale, kLog2e);
    float mx = -INFINITY, sum = 0.f;                   // sum: this lane's positions only
    // A swap puts two words' lower halves (rows of 16 lanes: even rows) into one and their upper halves into the other:
    // both words' sums over two m, each left in its half of the lanes.
    auto halves = [](float x, float y) {
        const auto w = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(y), false, false);
        return __fadd_rn(__uint_as_float(w[0]), __uint_as_float(w[1]));
    };
    auto rows = [](float x, float y) {
        const auto w = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(y), false, false);
        return __fadd_rn(__uint_as_float(w[0]), __uint_as_float(w[1]));
    };
    for (; tb < at.hi; tb += STEP) {
        const bool all = at.whole(tb), here = at.there[0];
        pf4 st[4] = {};
#pragma unroll
        for (int j = 0; j < R::N; ++j)
#pragma unroll
            for (int e0 = 0; e0 < R::KE; e0 += 4) {
                const pf4 qv = *reinterpret_cast<const pf4 *>(buf + (c & 3) * LD + R::k_dim(j, m, e0));
#pragma unroll
                for (int e = 0; e < 4; ++e) st[e] = __builtin_amdgcn_mfma_f32_4x4x1f32(k.k_at(j, e0 + e), qv[e], st[e], 0, 0, 0);
                if ((j * (R::KE / 4) + e0 / 4) % 4 == 3) __builtin_amdgcn_sched_barrier(0);    // (few words at a time: registers)
            }
        const bool more = tb + STEP < at.hi;           // (with a last tile that loads another one, 7.0 us for the call above)
        if (more) {
            at.seek(g, tb + STEP);
            k.load_k(a.c.k + at.at[0], at.ps, at.off[0], c, m);
        }
        // the four chunks' sums: lane (c, m) is left with position 4 (c / 4) + m of head c % 4
        const pf4 s4 = (st[0] + st[1]) + (st[2] + st[3]);
        float p = __fmul_rn(rows(halves(s4[0], s4[2]), halves(s4[1], s4[3])), sl2);
        if (cap > 0.f) p = __fmul_rn(capped(p, cap), kLog2e);
        if (!all) {                                    // a piece's end, or a page that does not exist
            // [from, to): what counts of the tile
            const int from = here ? at.start - tb : kPos, to = at.hi - tb, pos = (c >> 2) * 4 + m;
            p = pos >= from && pos < to ? p : -INFINITY;
#pragma unroll
            for (int r = 0; r < 4; ++r) v.keep_v(r, 4 * m + r >= from && 4 * m + r < to);      // its weight is 0, and 0 times a NaN there would be NaN
        }
        // The maximum moves, with O and the sums, only for a score far above it: weights up to 2^kLazy do no harm.
        if (__any(p > mx + kLazy)) {
            float ref = p;
#pragma unroll
            for (int off = 4; off < kWave; off *= 2) ref = fmaxf(ref, __shfl_xor(ref, off, kWave));
            const float mn = fmaxf(mx, ref), f = mx == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mx - mn);
            mx = mn;
            sum = __fmul_rn(sum, f);
#pragma unroll
            for (int x = 0; x < DPL; ++x) o[x] *= f;
        }
        const float from = mx == -INFINITY ? 0.f : mx; // nothing above -inf yet: all weights 0
        p = __builtin_amdgcn_exp2f(p - from);
        sum = __fadd_rn(sum, p);
        float w[4];                                    // of position 4m + r
#pragma unroll
        for (int r = 0; r < 4; ++r) w[r] = __shfl(p, (r << 4) | (m << 2) | (c & 3), kWave);
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int x = 0; x < DPL; ++x) o[x] = __builtin_amdgcn_mfma_f32_4x4x1f32(v.v_at(r, x), w[r], o[x], 0, 0, 0);
        if (more) v.load_v(a.c.v + at.at[0], at.ps, at.off[0], c, m);
    }
#pragma unroll
    for (int off = 4; off < kWave; off *= 2) sum += __shfl_xor(sum, off, kWave);
    if (lane < HEADS) {
        wm[wid][lane] = mx;
        wsum[wid][lane] = sum;
    }
    // O's sums over m, each lane left with a quarter of the dims: x = m * DPL / 4 and on
    constexpr int H = DPL / 2, Q = DPL / 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int x = 0; x < H; ++x) o[x][i] = halves(o[x][i], o[x + H][i]);
#pragma unroll
        for (int x = 0; x < Q; ++x) o[x][i] = rows(o[x][i], o[x + Q][i]);
    }
    __syncthreads();                                   // every wave is past its reads of q
#pragma unroll
    for (int x = 0; x < Q; ++x)
#pragma unroll
        for (int i = 0; i < 4; ++i) buf[(wid * HEADS + (c & 3)) * LD + R::v_dim(m * Q + x, (c >> 2) * 4 + i)] = o[x][i];
    finish<HD, HEADS>(g, at.b, at.h0, at.heads, at.slot0, buf, wm, wsum);
}

// Rows over a float cache: S^T = K q^T leaves lane (c, m) head c's scores of positions 4m .. 4m + 3, which is the B operand
// of O^T = V^T P^T. fp32 rows: v_mfma_f32_16x16x4_f32 on the elements as fp32. 16-bit rows (HALF) over a
// cache of their type: 16x16x32 products of the elements as they are, of two tiles for the weighted sum (of one where
// two do not fit the registers, 16x16x16); the weights come in two terms of that type (one
// would be off by as much as the outputs' own rounding), and V's 16-bit words are transposed in pairs on the way.
// 250 sequences of up to 2000 positions, 8 K/V heads of 128 dims, bf16 (1.0 GB): 175 us, 5.7 TB/s; two of three cycles wait
// for memory.
// grid (pieces, K/V heads x column tiles, sequences).
template <int CT, int HD, bool HALF>
__global__ __launch_bounds__(kThreads, HD == 64 ? 4 : HD == 128 ? 3 : 2) void paged_attn_kernel(AttnArgs g) {
    using R = Raw<CT, HD>;
    constexpr int LD = HD + 4, DPL = R::DPL;
    // fp16 weights: mx is held this much below the maximum, so that weights of down to 2^-21 of the largest stay normal
    // (2^(kLift + kLazy) is in range)
    constexpr float kLift = HALF && CT == DT_F16 ? 7.0f : 0.0f;
    constexpr int HALVES = HALF && HD < 256 ? 2 : 1, STEP = kWaves * HALVES * kPos;
    __shared__ __attribute__((aligned(16))) float buf[kWaves * kCols * LD];        // q, later the waves' O
    __shared__ float wm[kWaves][kCols], wsum[kWaves][kCols];
    const PagedAttn &a = g.a;
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wid = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int c = lane & 15, m = lane >> 4;
    Walk<HALVES> at(g, kCols);
    if (at.empty(g)) return;
    float qx[DPL];
    load_q<DPL>(a.q, at.b, at.h0, at.heads, qx);
    R k[HALVES], v[HALVES];
    auto load_k = [&]() {
#pragma unroll
        for (int u = 0; u < HALVES; ++u) k[u].load_k(a.c.k + at.at[u], at.ps, at.off[u], c, m);
    };
    auto load_v = [&]() {
#pragma unroll
        for (int u = 0; u < HALVES; ++u) v[u].load_v(a.c.v + at.at[u], at.ps, at.off[u], c, m);
    };
    int tb = at.lo + wid * HALVES * kPos;
    if (tb < at.hi) {
        at.seek(g, tb);
        load_k();
        load_v();
    }
    pu4 qh[HALF ? HD / 32 : 1];
    {
        const int r = tid >> 4, e0 = (tid & 15) * DPL;
        if constexpr (!HALF) {
#pragma unroll
            for (int e = 0; e < DPL; e += 4) *reinterpret_cast<pf4 *>(buf + r * LD + e0 + e) = pf4{qx[e], qx[e + 1], qx[e + 2], qx[e + 3]};
            __syncthreads();
        } else {
            constexpr int QL = HD + 8;
            uint16_t *qs = reinterpret_cast<uint16_t *>(buf);
#pragma unroll
            for (int e = 0; e < DPL; e += 4)           // (they were of that type: nothing is rounded)
                *reinterpret_cast<pu2 *>(qs + r * QL + e0 + e) =
                    pu2{pack_16(CT, qx[e], qx[e + 1]), pack_16(CT, qx[e + 2], qx[e + 3])};
            __syncthreads();
#pragma unroll
            for (int j = 0; j < HD / 32; ++j) qh[j] = *reinterpret_cast<const pu4 *>(qs + c * QL + 32 * j + 8 * m);
        }
    }
    pf4 o[DPL];                                        // o[x][r']: dim v_dim(x, 4m + r') of column c
#pragma unroll
    for (int x = 0; x < DPL; ++x) o[x] = pf4{0.f, 0.f, 0.f, 0.f};
    // scores in log2 units: without a cap in one product
    const float cap = a.softcap, sl2 = cap > 0.f ? a.scale : __fmul_rn(a.scale, kLog2e);
    float mx = -INFINITY, sum = 0.f;                   // sum: this lane's positions only
    for (; tb < at.hi; tb += STEP) {
        const bool all = at.whole(tb);
        bool here[HALVES];
#pragma unroll
        for (int u = 0; u < HALVES; ++u) here[u] = at.there[u];
        pf4 s4[HALVES];
        if constexpr (!HALF) {
            pf4 st[4] = {};
#pragma unroll
            for (int j = 0; j < R::N; ++j)
#pragma unroll
                for (int e0 = 0; e0 < R::KE; e0 += 4) {
                    const pf4 qv = *reinterpret_cast<const pf4 *>(buf + c * LD + R::k_dim(j, m, e0));
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        st[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[0].k_at(j, e0 + e), qv[e], st[e], 0, 0, 0);
                    if ((j * (R::KE / 4) + e0 / 4) % 4 == 3) __builtin_amdgcn_sched_barrier(0);    // (few words at a time: registers)
                }
            s4[0] = (st[0] + st[1]) + (st[2] + st[3]);
        } else {
#pragma unroll
            for (int u = 0; u < HALVES; ++u) {
                s4[u] = pf4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < HD / 32; ++j) s4[u] = mfma16<CT>(k[u].w[j], qh[j], s4[u]);
            }
        }
        at.seek(g, tb + STEP);
        load_k();
        float p[HALVES][4], ref = -INFINITY;
#pragma unroll
        for (int u = 0; u < HALVES; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                p[u][r] = __fmul_rn(s4[u][r], sl2);
                if (cap > 0.f) p[u][r] = __fmul_rn(capped(p[u][r], cap), kLog2e);
            }
        if (!all) {                                    // a piece's end, or a page that does not exist
#pragma unroll
            for (int u = 0; u < HALVES; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int t = tb + u * kPos + 4 * m + r;
                    const bool on = here[u] && t >= at.start && t < at.hi;
                    p[u][r] = on ? p[u][r] : -INFINITY;
                    v[u].keep_v(r, on);                // its weight is 0, and 0 times a NaN there would be NaN
                }
        }
#pragma unroll
        for (int u = 0; u < HALVES; ++u) ref = fmaxf(ref, fmaxf(fmaxf(p[u][0], p[u][1]), fmaxf(p[u][2], p[u][3])));
        // The maximum moves, with O and the sums, only for a score far above it: weights up to 2^kLazy do no harm.
        if (__any(ref > mx + kLift + kLazy)) {
            ref = fmaxf(ref, __shfl_xor(ref, 16, kWave));
            ref = fmaxf(ref, __shfl_xor(ref, 32, kWave));
            const float mn = fmaxf(mx, ref - kLift), f = mx == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mx - mn);
            mx = mn;
            sum = __fmul_rn(sum, f);
#pragma unroll
            for (int x = 0; x < DPL; ++x) o[x] *= f;
        }
        const float from = mx == -INFINITY ? 0.f : mx; // nothing above -inf yet: all weights 0
#pragma unroll
        for (int u = 0; u < HALVES; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                p[u][r] = __builtin_amdgcn_exp2f(p[u][r] - from);
                sum = __fadd_rn(sum, p[u][r]);
            }
        if constexpr (HALF) {
            // contraction index 4 HALVES m + 4u + r is position 4m + r of half u
            uint32_t pw[2 * HALVES], rest[2 * HALVES]; // the weights in that type, and what that leaves of them
#pragma unroll
            for (int u = 0; u < HALVES; ++u)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float p0 = p[u][2 * i], p1 = p[u][2 * i + 1];
                    const uint32_t w = pack_16(CT, p0, p1);
                    pw[2 * u + i] = w;
                    rest[2 * u + i] = pack_16(CT, __fsub_rn(p0, from_16(CT, w & 0xffffu)), __fsub_rn(p1, from_16(CT, w >> 16)));
                }
#pragma unroll
            for (int x = 0; x < DPL; x += 2) {
                uint32_t even[2 * HALVES], odd[2 * HALVES];
#pragma unroll
                for (int u = 0; u < HALVES; ++u)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint32_t w0 = v[u].v_pair(2 * i, x), w1 = v[u].v_pair(2 * i + 1, x);
                        even[2 * u + i] = __builtin_amdgcn_perm(w1, w0, 0x05040100u);
                        odd[2 * u + i] = __builtin_amdgcn_perm(w1, w0, 0x07060302u);
                    }
                auto product = [](const uint32_t (&a)[2 * HALVES], const uint32_t (&b)[2 * HALVES], pf4 c) {
                    if constexpr (HALVES == 2) return mfma16<CT>(pu4{a[0], a[1], a[2], a[3]}, pu4{b[0], b[1], b[2], b[3]}, c);
                    else return mfma8<CT>(pu2{a[0], a[1]}, pu2{b[0], b[1]}, c);
                };
                o[x] = product(even, pw, o[x]);
                o[x + 1] = product(odd, pw, o[x + 1]);
                o[x] = product(even, rest, o[x]);
                o[x + 1] = product(odd, rest, o[x + 1]);
                if (HD == 256 && x % 4 == 2) __builtin_amdgcn_sched_barrier(0);        // (few words at a time: registers)
            }
        } else {
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int x = 0; x < DPL; ++x) o[x] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[0].v_at(r, x), p[0][r], o[x], 0, 0, 0);
        }
        load_v();
    }
    sum += __shfl_xor(sum, 16, kWave);
    sum += __shfl_xor(sum, 32, kWave);
    if constexpr (HALF) {
        // An infinity in V times a term of 0, or times terms of both signs, is NaN. Where O is NaN and the weights are not, the
        // wave goes over its positions again, with the weights as they are (mx is the last one) on fp32 products.
        bool odd = false;
#pragma unroll
        for (int x = 0; x < DPL; ++x)
#pragma unroll
            for (int r = 0; r < 4; ++r) odd |= o[x][r] != o[x][r];
        if (__any(odd && sum == sum && c < at.heads)) {
#pragma unroll
            for (int x = 0; x < DPL; ++x) o[x] = pf4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
            for (int t0 = at.lo + wid * HALVES * kPos; t0 < at.hi; t0 += STEP)
#pragma unroll 1
                for (int t = t0; t < min(t0 + HALVES * kPos, at.hi); t += kPos) {
                    at.seek(g, t);
                    k[0].load_k(a.c.k + at.at[0], at.ps, at.off[0], c, m);
                    v[0].load_v(a.c.v + at.at[0], at.ps, at.off[0], c, m);
                    pf4 s4 = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int j = 0; j < HD / 32; ++j) s4 = mfma16<CT>(k[0].w[j], qh[j], s4);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        float p = __fmul_rn(s4[r], sl2);
                        if (cap > 0.f) p = __fmul_rn(capped(p, cap), kLog2e);
                        const bool on = at.there[0] && t + 4 * m + r >= at.start && t + 4 * m + r < at.hi;
                        v[0].keep_v(r, on);
                        p = on ? __builtin_amdgcn_exp2f(p - (mx == -INFINITY ? 0.f : mx)) : 0.f;
#pragma unroll
                        for (int x = 0; x < DPL; ++x) o[x] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[0].v_at(r, x), p, o[x], 0, 0, 0);
                    }
                }
        }
    }
    if (m == 0) {
        wm[wid][c] = mx;
        wsum[wid][c] = sum;
    }
    __syncthreads();                                   // every wave is past its reads of q
    if (c < at.heads) {
#pragma unroll
        for (int x = 0; x < DPL; ++x)
#pragma unroll
            for (int r = 0; r < 4; ++r) buf[(wid * kCols + c) * LD + R::v_dim(x, 4 * m + r)] = o[x][r];
    }
    finish<HD, kCols>(g, at.b, at.h0, at.heads, at.slot0, buf, wm, wsum);
}

// Rows over a quantized cache, 4 NT query heads. K's codes meet q as they are: q is rounded to 2^-31 of its head's
// largest element and split into four signed 8-bit digits, a head's digits are four rows of the 16x16x32 product, and
// a lane's four sums, exact in 32 bits, are one head's digits of one position: put together and times the block's
// scale one fma. The weights go through LDS to the other operand's order. There a column stands for a head and one
// of four blocks of V, and carries weight times that block's scale, so that V's codes come in as small bf16 integers; of the
// sums only those of a column's own block are meant. (head_dim 256 has two sets of four blocks, each with products of its own:
// in one, zeros would stand beside the other set's weights, and 0 times the scale NaN of a block is NaN in another; 100
// sequences of up to 2000 positions, 64 heads over 8, Q4_0: 91 us, and 95 with the zeros.) TERMS: bf16 terms of that product, 3 for all its 24 bits;
// 2 where rows are bf16 (its rounding is then 2^-7 of the outputs').
// Three sequences of up to 131072 positions, 32 heads over 8 of 128 dims, Q4_0, fp32 rows (374 MB): 77-83 us, 4.5-4.9 TB/s,
// of which the vector units are busy for 41 and the matrix cores for 15; sixteen of up to 2048, 4 heads over one of 256, Q8_0
// (9.7 MB): 8.5 us, a chain as above.
template <int CT, int HD, int NT, int TERMS>
__global__ __launch_bounds__(kThreads, HD == 256 ? 2 : HD == 64 || (NT == 1 && CT == DT_Q4_0) ? 4 : NT == 1 ? 3 : 2) void paged_attn_digits_kernel(AttnArgs g) {
    using R = Raw<CT, HD>;
    using T = Tile<CT, HD>;
    constexpr int LD = HD + 4, DPL = R::DPL, HEADS = 4 * NT, SETS = (T::NB + 3) / 4, HALVES = 2 / SETS, STEP = kWaves * HALVES * kPos;
    constexpr int kQ = NT * T::NB * kWave * 8, kP = kWaves * HALVES * NT * kWave * 4, kO = kWaves * HEADS * LD * 4;
    __shared__ __attribute__((aligned(16))) uint8_t lds[kQ + kP > kO ? kQ + kP : kO];   // digits, weights; later the waves' O
    __shared__ float wm[kWaves][HEADS], wsum[kWaves][HEADS];
    __shared__ int shift[kCols];                       // q * 2^shift are the digits' integers
    const PagedAttn &a = g.a;
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wid = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int c = lane & 15, m = lane >> 4;
    Walk<HALVES> at(g, HEADS);
    if (at.empty(g)) return;
    float x[DPL];
    load_q<DPL>(a.q, at.b, at.h0, at.heads, x);
    R k[HALVES], v[HALVES];
    auto load_k = [&]() {
#pragma unroll
        for (int u = 0; u < HALVES; ++u) k[u].load_k(a.c.k + at.at[u], at.ps, at.off[u], c, m);
    };
    auto load_v = [&]() {
#pragma unroll
        for (int u = 0; u < HALVES; ++u) v[u].load_v(a.c.v + at.at[u], at.ps, at.off[u], c, m);
    };
    int tb = at.lo + wid * HALVES * kPos;
    if (tb < at.hi) {
        at.seek(g, tb);
        load_k();
        load_v();
    }
    {
        // sixteen threads per head, HD / 16 elements each: the largest magnitude, then the digits, eight
        // elements (or four) at a time, to where the lanes read them: [set][block][lane][8]
        const int r = tid >> 4, e0 = (tid & 15) * DPL;
        constexpr int W = DPL < 8 ? DPL : 8;
        float top = 0.f;
        bool odd = false;
#pragma unroll
        for (int e = 0; e < DPL; ++e) {
            odd |= !(fabsf(x[e]) < INFINITY);
            top = fmaxf(top, fabsf(x[e]));
        }
        top = lanes::row16_max(odd ? INFINITY : top);
        int ex;
        (void)frexpf(top, &ex);                        // top < 2^ex
        const int sh = top > 0.f && top < INFINITY ? 30 - ex : 0;
        if ((tid & 15) == 0) shift[r] = top < INFINITY ? sh : INT_MAX;
        if (r < HEADS) {
#pragma unroll
            for (int w0 = 0; w0 < DPL; w0 += W) {
                const int d = e0 + w0, blk = d >> 5, mm = (d >> 3) & 3;
                uint32_t dig[4][2] = {};
#pragma unroll
                for (int e = 0; e < W; ++e) {
                    int X = top < INFINITY ? (int)rintf(ldexpf(x[w0 + e], sh)) : 0;
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const int dg = (int8_t)X;
                        dig[q][e >> 2] |= (uint32_t)(dg & 255) << (8 * (e & 3));
                        X = (X - dg) >> 8;
                    }
                }
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    uint8_t *o = lds + (((r >> 2) * T::NB + blk) * kWave + mm * 16 + 4 * (r & 3) + q) * 8 + (d & 7);
                    if constexpr (W == 8) *reinterpret_cast<pu2 *>(o) = pu2{dig[q][0], dig[q][1]};
                    else *reinterpret_cast<uint32_t *>(o) = dig[q][0];
                }
            }
        }
    }
    __syncthreads();
    // the digits in registers, or where O takes most of those, read from LDS as they are used
    constexpr bool kHold = NT == 1 || HD == 64;
    pu2 held[kHold ? NT : 1][kHold ? T::NB : 1];
    auto digits = [&](int t, int j) { return *reinterpret_cast<const pu2 *>(lds + ((t * T::NB + j) * kWave + lane) * 8); };
    if constexpr (kHold) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int j = 0; j < T::NB; ++j) held[t][j] = digits(t, j);
    }
    // from the digits' integers to scores in log2 units (or to what the cap takes); lane (c, m): head 4t + m
    const float cap = a.softcap;
    float unit[NT], mx[NT], sum[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int s = shift[4 * t + m];
        unit[t] = s == INT_MAX ? NAN : ldexpf(cap > 0.f ? a.scale : __fmul_rn(a.scale, kLog2e), -s - (CT == DT_Q4_0 ? 4 : 0));
        mx[t] = -INFINITY;
        sum[t] = 0.f;                                  // this lane's position of every tile
    }
    pf4 o[NT][DPL];                                    // o[t][x][r']: dim v_element_dim(x, 4m + r'), column c
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int x = 0; x < DPL; ++x) o[t][x] = pf4{0.f, 0.f, 0.f, 0.f};
    float *pw = reinterpret_cast<float *>(lds + kQ) + wid * HALVES * NT * kWave;
    for (; tb < at.hi; tb += STEP) {
        const bool all = at.whole(tb);
        bool here[HALVES];
#pragma unroll
        for (int u = 0; u < HALVES; ++u) here[u] = at.there[u];
        float sc[HALVES][NT] = {};
#pragma unroll
        for (int j = 0; j < T::NB; ++j) {
#pragma unroll
            for (int u = 0; u < HALVES; ++u) {
                const pu2 kb = k[u].k_codes(j);
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    pu2 qd;
                    if constexpr (kHold) qd = held[t][j];
                    else qd = digits(t, j);
                    const pi4 d = __builtin_amdgcn_mfma_i32_16x16x32_i8(__builtin_bit_cast(long, qd), __builtin_bit_cast(long, kb),
                                                                        pi4{0, 0, 0, 0}, 0, 0, 0);
                    // below 2^28: 32 products of 2^14, times 2^8
                    const float low = (float)(d[1] * 256 + d[0]), high = (float)(d[3] * 256 + d[2]);
                    sc[u][t] = __builtin_fmaf(__builtin_fmaf(high, 65536.0f, low), k[u].s[j], sc[u][t]);
                }
            }
            // (the sums of a few blocks at a time: all of them at once would not fit the registers)
            if (j % 2 == 1) __builtin_amdgcn_sched_barrier(0);
        }
        at.seek(g, tb + STEP);
        load_k();
        float ref[NT];
        bool far = false;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
#pragma unroll
            for (int u = 0; u < HALVES; ++u) {
                sc[u][t] = __fmul_rn(sc[u][t], unit[t]);
                if (cap > 0.f) sc[u][t] = __fmul_rn(capped(sc[u][t], cap), kLog2e);
            }
        }
        if (!all) {                                    // a piece's end, or a page that does not exist
#pragma unroll
            for (int u = 0; u < HALVES; ++u) {
                // [from, to): what counts of the tile
                const int from = here[u] ? at.start - tb - u * kPos : kPos, to = at.hi - tb - u * kPos;
#pragma unroll
                for (int t = 0; t < NT; ++t) sc[u][t] = c >= from && c < to ? sc[u][t] : -INFINITY;
#pragma unroll
                for (int i = 0; i < 4 * SETS; ++i) {   // a weight of 0 times a scale of NaN there would be NaN
                    const int at_r = 4 * m + i % 4;
                    v[u].s[i] = at_r >= from && at_r < to ? v[u].s[i] : 0.f;
                }
            }
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            ref[t] = fmaxf(sc[0][t], sc[HALVES - 1][t]);
            far |= ref[t] > mx[t] + kLazy;
        }
        // The maximum moves, with O and the sums, only for a score far above it: weights up to 2^kLazy do no harm.
        if (__any(far)) {
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const float mn = fmaxf(mx[t], lanes::row16_max(ref[t])), f = mx[t] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mx[t] - mn);
                mx[t] = mn;
                sum[t] = __fmul_rn(sum[t], f);
                const float fc = __shfl(f, (c >> 2) * 16, kWave);          // of the column's head
#pragma unroll
                for (int x = 0; x < DPL; ++x) o[t][x] *= fc;
            }
        }
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const float from = mx[t] == -INFINITY ? 0.f : mx[t];           // nothing above -inf yet: all weights 0
#pragma unroll
            for (int u = 0; u < HALVES; ++u) {
                const float p = __builtin_amdgcn_exp2f(sc[u][t] - from);
                sum[t] = __fadd_rn(sum[t], p);
                pw[(u * NT + t) * kWave + lane] = p;
            }
        }
        // a wave's LDS accesses stay in order; the compiler is told
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        // contraction index 8m + 4i + r is position 4m + r of tile i; of one tile and two sets, words 2i and 2i + 1 are set i's
        pu4 w[NT][TERMS];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int u = 0; u < HALVES; ++u) {
                const pf4 p = *reinterpret_cast<const pf4 *>(pw + (u * NT + t) * kWave + (c >> 2) * 16 + 4 * m);
#pragma unroll
                for (int s = 0; s < SETS; ++s) {
                    float x[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) x[r] = __fmul_rn(p[r], v[u].s[4 * s + r]);
#pragma unroll
                    for (int q = 0; q < TERMS; ++q)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            float &x0 = x[2 * i], &x1 = x[2 * i + 1];
                            // the upper half of the word, and what it leaves
                            w[t][q][2 * (u + s) + i] = __builtin_amdgcn_perm(__float_as_uint(x1), __float_as_uint(x0), 0x07060302u);
                            x0 = __fsub_rn(x0, __uint_as_float(__float_as_uint(x0) & 0xffff0000u));
                            x1 = __fsub_rn(x1, __uint_as_float(__float_as_uint(x1) & 0xffff0000u));
                        }
                }
            }
        uint32_t vb[HALVES][R::VW];
#pragma unroll
        for (int u = 0; u < HALVES; ++u) v[u].v_bytes(vb[u], c);
#pragma unroll
        for (int x0 = 0; x0 < DPL; x0 += 2) {
            pu4 code[2];                               // exact in bf16 (of one tile: two words)
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int u = 0; u < HALVES; ++u)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        code[e][2 * u + i] = __builtin_amdgcn_perm(__float_as_uint(R::v_byte(vb[u], 2 * i + 1, x0 + e)),
                                                                   __float_as_uint(R::v_byte(vb[u], 2 * i, x0 + e)), 0x07060302u);
                    }
#pragma unroll
            for (int q = 0; q < TERMS; ++q)
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        if constexpr (SETS == 1) {
                            o[t][x0 + e] = mfma16<DT_BF16>(code[e], w[t][q], o[t][x0 + e]);
                        } else {
                            const int set = x0 / 8;
                            o[t][x0 + e] = mfma8<DT_BF16>(pu2{code[e][0], code[e][1]}, pu2{w[t][q][2 * set], w[t][q][2 * set + 1]}, o[t][x0 + e]);
                        }
                    }
            // (two dims' codes at a time: all of them at once would not fit the registers)
            __builtin_amdgcn_sched_barrier(0);
        }
        load_v();
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        sum[t] = lanes::row16_sum(sum[t]);
        if (c == 0) {
            wm[wid][4 * t + m] = mx[t];
            wsum[wid][4 * t + m] = sum[t];
        }
    }
    __syncthreads();                                   // every wave is past its digits and weights
    float *buf = reinterpret_cast<float *>(lds);       // the waves' O: [wave][head][LD]
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            // rows 4m + r of the column's own block (of both sets)
            if (R::v_element_dim(0, 4 * m + r) / 32 != (c & 3)) continue;
#pragma unroll
            for (int x = 0; x < DPL; ++x)
                buf[(wid * HEADS + 4 * t + (c >> 2)) * LD + R::v_element_dim(x, 4 * m + r)] = __fmul_rn(o[t][x][r], CT == DT_Q4_0 ? 0.0625f : 1.0f);
        }
    finish<HD, HEADS>(g, at.b, at.h0, at.heads, at.slot0, buf, wm, wsum);
}

// grid (heads, sequences): the pieces of one head. Every wave has all pieces' weights, one or more per lane, and adds
// every W-th piece, HD / 64 dims per lane. Up to 32 pieces, one trip of four waves: nine pieces of 256 dims 2.7 us (sixteen waves
// 3.5), 32 of 64 heads 3.6 (4.3); 128 pieces of 96 heads of 128 dims 7.1 with sixteen waves (four 9.5). All first loads start
// before the length is known: the slots of all pieces are in the workspace.
template <int HD, int W>
__global__ __launch_bounds__(W *kWave) void paged_join_kernel(AttnArgs g) {
    constexpr int D = HD / kWave, U = 8, Q = kMaxPieces / kWave;       // U: loads in flight
    __shared__ float part[W][HD];
    const PagedAttn &a = g.a;
    const int h = blockIdx.x, b = blockIdx.y, lane = threadIdx.x & (kWave - 1), wid = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const size_t stride = (size_t)gridDim.y * g.n_heads, slot = (size_t)b * g.n_heads + h;
    float2 ms[Q];
    ms[0] = g.ms[slot + min(lane, g.pieces - 1) * stride];
    float v[U][D];
    auto load = [&](int i0, int last) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int d = 0; d < D; ++d) v[u][d] = g.part[(slot + min(i0 + u * W, last) * stride) * HD + lane * D + d];
    };
    load(wid, g.pieces - 1);
    const int n = min(max(a.lengths[b], 0), a.max_length);
    const int start = a.window > 0 && n > a.window ? n - a.window : 0;
    const int used = max(1, (n - (start & ~(kPos - 1)) + g.piece - 1) / g.piece);
    float top = lane < used ? ms[0].x : -INFINITY;
#pragma unroll
    for (int q = 1; q < Q; ++q) {
        if (q * kWave >= used) break;
        ms[q] = g.ms[slot + min(lane + q * kWave, used - 1) * stride];
        top = fmaxf(top, ms[q].x);
    }
    top = lanes::wave_max(top);
    float f[Q], tot = 0.f;
    unsigned long long mask[Q];                        // pieces with an O (a sequence of length 0 has none)
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        f[q] = 0.f;
        mask[q] = 0;
        if (q * kWave >= used) continue;
        // a sum of NaN has a weight of NaN, whatever its maximum; one of 0 the weight 0 (its O may be NaN)
        const bool on = lane + q * kWave < used && n > 0;
        f[q] = !on || ms[q].y == 0.f ? 0.f : ms[q].y != ms[q].y ? ms[q].y : __builtin_amdgcn_exp2f(ms[q].x - top);
        tot = __builtin_fmaf(on ? ms[q].y : 0.f, f[q], tot);
        mask[q] = __ballot(on);
    }
    tot = lanes::wave_sum(tot);
    float o[D] = {};
    for (int i0 = wid; i0 < used;) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u * W;
            if (i >= used) break;
            float fi = 0.f;
            bool on = false;
#pragma unroll
            for (int q = 0; q < Q; ++q)
                if (i / kWave == q) {
                    fi = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(f[q]), i % kWave));
                    on = mask[q] >> i % kWave & 1;
                }
            if (!on) continue;
#pragma unroll
            for (int d = 0; d < D; ++d) o[d] = __builtin_fmaf(fi, v[u][d], o[d]);
        }
        i0 += W * U;
        if (i0 < used) load(i0, used - 1);
    }
#pragma unroll
    for (int d = 0; d < D; ++d) part[wid][lane * D + d] = o[d];
    __syncthreads();
    const int t = threadIdx.x;
    if (t >= HD) return;
    float x = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) x += part[w][t];
    store1(a.out.dtype, a.out.p, (int64_t)b * a.out.ts + (int64_t)h * a.out.hs + t, tot == 0.f ? 0.f : __fdiv_rn(x, tot));
    if (a.lse && t == 0) a.lse[slot] = lse_of(top, tot);
}

// A piece is a fixed number of positions, so that sequences of different lengths make equal work. Sequences of many
// (sequence, K/V head) pairs are not cut: each start costs about 2 us and the join 2 to 7, and the longest, first to go,
// end in time where a single workgroup reaches a good part of what its share of the memory's rate is. That takes fewer pairs
// where it does little but load (16-bit rows over their own type, up to four fp32 heads over fp32) than where it converts;
// likewise the pieces of others are larger. In us, for pairs x positions, and at a copy's rate for the bytes:
//   bf16, 4 heads of 128 dims        256 x 2774 (35): whole 39, in 2 to 16 pieces 41-50;    128 x 5548 (38): 42; 41-49
//   fp32 over Q4_0, 4 x 128          256 x 8877 (35): whole 85, in 4 to 16 pieces 45-65;    512 x 6658 (53): 72; 69-81
//   fp32 over fp16, 8 x 128          256 x 2774 (35): whole 88, 51-73;                      512 x 2080 (53): 79; 72-102
// Pieces of 160 KiB and 768 KiB, and fewer than that of long sequences, take 0.92 of the time, in the mean over 64 ragged
// batches of 60 to 1000 MB, that as many pieces as make 2048 workgroups take.
struct Wanted {
    int whole, bytes;                      // pairs from which on sequences are not cut; a piece's bytes of K and V
};
constexpr Wanted kLoads = {256, 768 << 10}, kConverts = {512, 160 << 10};
constexpr int kFill = 512;                 // workgroups that smaller pieces are made for
constexpr int64_t kJoined = 48;            // pieces from which on their number grows as the root of the bytes: the join counts
int pieces_by_bytes(Wanted w, int64_t len, int row) {
    const int64_t n = (len * row + w.bytes - 1) / w.bytes;
    return (int)std::min<int64_t>(kMaxPieces, n <= kJoined ? n : (int64_t)std::sqrt((double)(kJoined * n)));
}
int pieces_wanted(Wanted w, int64_t groups, int64_t len, int row) {
    if (groups >= w.whole) return 1;
    return (int)std::min<int64_t>(kMaxPieces, std::max<int64_t>(pieces_by_bytes(w, len, row), (kFill + groups - 1) / groups));
}
int row_bytes_kv(int dtype, int hd) { return 2 * (dtype == DT_F32 ? 4 * hd : dtype == DT_Q8_0 ? hd * 9 / 8 : dtype == DT_Q4_0 ? hd * 5 / 8 : 2 * hd); }
struct Plan {
    int col_heads, col_tiles, piece, pieces;
    int64_t groups;
};
Plan plan_of(int dtype, bool half, int nkv, int hd, int batch, int n_heads, int max_length, int window) {
    Plan p;
    const int group = n_heads / nkv;
    // quantized caches: four or eight heads a workgroup; float caches: four for fp32 rows of no more, or sixteen
    p.col_heads = is_quant(dtype) ? (group <= 4 ? 4 : 8) : !half && group <= 4 ? 4 : kCols;
    p.col_tiles = (group + p.col_heads - 1) / p.col_heads;
    p.groups = (int64_t)batch * nkv * p.col_tiles;
    const bool loads = !is_quant(dtype) && (half || (dtype == DT_F32 && p.col_heads == 4));
    const int row = row_bytes_kv(dtype, hd);
    const int64_t len = (window > 0 && window < max_length - kPos ? window + kPos : max_length);
    const int64_t want = pieces_wanted(loads ? kLoads : kConverts, p.groups, len, row);
    p.piece = (int)(((len + want - 1) / want + kPieceUnit - 1) / kPieceUnit * kPieceUnit);
    p.pieces = (int)((len + p.piece - 1) / p.piece);
    return p;
}

size_t part_bytes(int hd, int batch, int n_heads, int pieces) { return (size_t)pieces * batch * n_heads * hd * sizeof(float); }

}  // namespace

// Enough for every call of at most `batch` sequences of at most max_length, whatever its window and type of rows: b
// sequences that are cut, b k < kConverts.whole, have no more pieces than max(by bytes, kFill / (b k) + 1), all bounds grow
// with the length, and b times that is at most what the largest such b makes of either term.
size_t paged_attention_workspace(int dtype, int nkv, int hd, int batch, int n_heads, int max_length) {
    const int64_t k = plan_of(dtype, false, nkv, hd, 1, n_heads, max_length, 0).groups;
    const int64_t b = std::min<int64_t>(batch, (kConverts.whole - 1) / k);
    const int64_t most = std::min<int64_t>(kMaxPieces, ((int64_t)max_length + kPieceUnit - 1) / kPieceUnit);
    if (b == 0 || most == 1) return 0;
    const int64_t bytes = pieces_by_bytes(kConverts, max_length, row_bytes_kv(dtype, hd));
    const int64_t slots = std::max(b * std::min(most, bytes), std::min(b * most, kFill / k + b));
    return (size_t)slots * n_heads * (hd * sizeof(float) + sizeof(float2));
}

int launch_paged_attention(const PagedAttn &a, hipStream_t s) {
    AttnArgs g;
    g.a = a;
    g.n_heads = a.q.heads;
    g.group = g.n_heads / a.c.nkv;
    const bool half = a.q.dtype != DT_F32;
    const Plan p = plan_of(a.c.dtype, half, a.c.nkv, a.c.hd, a.q.tokens, g.n_heads, a.max_length, a.window);
    g.col_tiles = p.col_tiles;
    g.piece = p.piece;
    g.pieces = p.pieces;
    g.wide = rows_wide(a.out);
    g.ordered = p.pieces == 1 && a.q.tokens > 1 && a.q.tokens <= kOrdered && p.groups >= kLoads.whole;
    g.part = reinterpret_cast<float *>(a.ws);
    g.ms = reinterpret_cast<float2 *>(a.ws + part_bytes(a.c.hd, a.q.tokens, g.n_heads, p.pieces));
    const dim3 grid(p.pieces, a.c.nkv * p.col_tiles, a.q.tokens), block(kThreads);
    const bool short_terms = a.q.dtype == DT_BF16;
#define SPH_FLOAT(CT, HD, HALF)                                                                    \
    if (a.c.dtype == CT && a.c.hd == HD && half == HALF && p.col_heads == kCols)                  \
        hipLaunchKernelGGL((paged_attn_kernel<CT, HD, HALF>), grid, block, 0, s, g);
#define SPH_FEW(CT, HD) \
    if (a.c.dtype == CT && a.c.hd == HD && p.col_heads == 4) hipLaunchKernelGGL((paged_attn_few_kernel<CT, HD>), grid, block, 0, s, g);
#define SPH_DIGITS(CT, HD, NT, TERMS)                                                             \
    if (a.c.dtype == CT && a.c.hd == HD && p.col_heads == 4 * NT && short_terms == (TERMS == 2))  \
        hipLaunchKernelGGL((paged_attn_digits_kernel<CT, HD, NT, TERMS>), grid, block, 0, s, g);
#define SPH_QUANT(CT, HD) SPH_DIGITS(CT, HD, 1, 2) SPH_DIGITS(CT, HD, 1, 3) SPH_DIGITS(CT, HD, 2, 2) SPH_DIGITS(CT, HD, 2, 3)
#define SPH_ATTN_HD(HD)                                                                           \
    SPH_FEW(DT_F32, HD) SPH_FEW(DT_BF16, HD) SPH_FEW(DT_F16, HD)                                  \
    SPH_FLOAT(DT_F32, HD, false) SPH_FLOAT(DT_BF16, HD, false) SPH_FLOAT(DT_BF16, HD, true)       \
    SPH_FLOAT(DT_F16, HD, false) SPH_FLOAT(DT_F16, HD, true) SPH_QUANT(DT_Q8_0, HD) SPH_QUANT(DT_Q4_0, HD)
    SPH_ATTN_HD(64) SPH_ATTN_HD(128) SPH_ATTN_HD(256)
    if (!hip_ok(hipGetLastError(), "paged attention launch")) return -1;
    if (p.pieces > 1) {
        const dim3 jg(g.n_heads, a.q.tokens);
#define SPH_JOIN(HD, W) \
    if (a.c.hd == HD && (p.pieces > kManyPieces) == (W == 16)) hipLaunchKernelGGL((paged_join_kernel<HD, W>), jg, dim3(W * kWave), 0, s, g);
#define SPH_JOIN_HD(HD) SPH_JOIN(HD, 4) SPH_JOIN(HD, 16)
        SPH_JOIN_HD(64) SPH_JOIN_HD(128) SPH_JOIN_HD(256)
        if (!hip_ok(hipGetLastError(), "paged attention join launch")) return -1;
    }
    return 0;
}

}  // namespace sapphire
