// paged_attention.hip - attention of one new token per sequence over the paged cache.
//
// Scores and the weighted sum run on the fp32 matrix cores as in the prompt's attention
// (prefill.hip): S^T = K q^T with the query heads of a K/V head as columns leaves lane (c, m) head c's
// scores of positions 4m .. 4m + 3, which is the B operand of O^T = V^T P^T. One pass over K and V with
// a running maximum and sum per column; a sequence's positions are cut into pieces that workgroups take
// side by side, and a second launch joins the pieces' (maximum, sum, O).
#include <algorithm>
#include <climits>

#include "internal.h"
#include "lanes.h"
#include "paged_dev.h"

namespace sapphire {

namespace {

constexpr int kWave = 64, kThreads = 256, kWaves = kThreads / kWave;
constexpr int kCols = 16;                  // query heads of a workgroup
constexpr int kPos = 16;                   // positions of a tile
constexpr int kMaxPieces = 256;
constexpr int kPieceUnit = 64;             // a piece is a multiple of so many positions
constexpr int kWantGroups = 1024;          // workgroups that fill the chip (four per CU)
constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.693147180559945309f;

struct AttnArgs {
    PagedAttn a;
    int n_heads, group, col_tiles, piece, pieces;
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
            // of position 4m + c % 4: the score product leaves a lane positions 4m .. 4m + 3, its quad has their scales
#pragma unroll
            for (int b = 0; b < T::NB; b += 2) {
                const float2 v = *reinterpret_cast<const float2 *>(tile + T::k_scale(ps, off + 4 * m + (c & 3), b));
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
            const pf4 v = *reinterpret_cast<const pf4 *>(tile + T::v_scale(ps, off + 4 * m, c * DPL / 32));
#pragma unroll
            for (int r = 0; r < 4; ++r) s[r] = v[r];
        }
    }
    // The operand of block j: its codes (Q4_0: times 16) in element order.
    __device__ __forceinline__ pu2 k_codes(int j) const {
        if constexpr (CT == DT_Q8_0) return pu2{w[j / 2][j % 2 * 2], w[j / 2][j % 2 * 2 + 1]};
        const uint32_t v = w[j / T::G][j % T::G];
        return pu2{v << 4 & 0xf0f0f0f0u, v & 0xf0f0f0f0u};
    }
    // Position 4m + r without effect: zeros, or a scale of 0.
    __device__ __forceinline__ void clear_v(int r) {
        if constexpr (T::kQuant) {
            s[r] = 0.f;
        } else {
#pragma unroll
            for (int i = r * N; i < (r + 1) * N; ++i) w[i / 4][i % 4] = 0;     // N words per position
        }
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
        else if constexpr (!T::kQuant) {
            // words of two elements: DPL / 2 per position, in order
            const int i = r * (DPL / 2) + x / 2;
            const uint32_t v = w[i / 4][i % 4];
            if constexpr (CT == DT_BF16) return __uint_as_float(x & 1 ? v & 0xffff0000u : v << 16);
            else return from_f16(x & 1 ? v >> 16 : v & 0xffffu);
        } else if constexpr (CT == DT_Q8_0) {
            const int i = r * (DPL / 4) + x / 4;
            return __fmul_rn((float)(int8_t)(w[i / 4][i % 4] >> (8 * (x & 3))), s[r]);
        } else {
            const int R = DPL / 2, byte = r * R + x % R;       // R bytes per position
            const uint32_t q = w[byte / 16][byte / 4 % 4] >> (8 * (byte % 4) + (x / R) * 4) & 15u;
            return __fmul_rn((float)((int)q - 8), s[r]);
        }
    }
};

__device__ __forceinline__ float load1(int dtype, const uint8_t *p, int64_t i) {
    return dtype == DT_F32 ? reinterpret_cast<const float *>(p)[i] : from_16(dtype, reinterpret_cast<const uint16_t *>(p)[i]);
}
__device__ __forceinline__ void store1(int dtype, uint8_t *p, int64_t i, float v) {
    if (dtype == DT_F32) reinterpret_cast<float *>(p)[i] = v;
    else reinterpret_cast<uint16_t *>(p)[i] = (uint16_t)to_16(dtype, v);
}

__device__ __forceinline__ float lse_of(float mx, float sum) { return sum == 0.f ? -INFINITY : (mx + log2f(sum)) * kLn2; }

// How scores and weighted sums are formed.
//   kExact  fp32 rows over a float cache: v_mfma_f32_16x16x4_f32 on the elements as fp32.
//   kHalf   16-bit rows over a cache of their type: 16x16x32 products of the elements as they are; the
//           weights are rounded to that type, and V's 16-bit words are transposed in pairs on the way.
//   kDigits a quantized cache: the codes as they are against q in four signed 8-bit digits (q rounded to
//           2^-31 of the head's largest element), exact 32-bit sums per block, one fma with the block's
//           scale. A head takes four columns, one per digit; NT sets of columns share the codes. The
//           weighted sum is kExact's, codes times scale as fp32.
enum Path { kExact = 0, kHalf = 1, kDigits = 2 };
constexpr float kLazy = 8.0f;              // log2 units that a score may exceed the running maximum by

typedef short ps8 __attribute__((ext_vector_type(8)));
typedef __bf16 pb8 __attribute__((ext_vector_type(8)));
typedef _Float16 ph8 __attribute__((ext_vector_type(8)));
typedef int pi4 __attribute__((ext_vector_type(4)));

template <int CT>
__device__ __forceinline__ pf4 mfma16(pu4 a, pu4 b, pf4 c) {
    if constexpr (CT == DT_BF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(pb8, a), __builtin_bit_cast(pb8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(ph8, a), __builtin_bit_cast(ph8, b), c, 0, 0, 0);
}

// Sum over each quad of lanes, in every lane of it.
__device__ __forceinline__ float quad_sum(float v) {
    v += lanes::dpp_mov<0xB1>(v);
    return v + lanes::dpp_mov<0x4E>(v);
}
// Lane R of each quad, in every lane of it.
template <int R>
__device__ __forceinline__ float quad_lane(float v) {
    return lanes::dpp_mov<R * 0x55>(v);
}

// grid (pieces, K/V heads x column tiles, sequences).
template <int CT, int HD, int PATH, int NT>
__global__ __launch_bounds__(kThreads, HD == 64 ? 4 : HD == 128 ? 3 : 2) void paged_attn_kernel(AttnArgs g) {
    using R = Raw<CT, HD>;
    using T = Tile<CT, HD>;
    constexpr int LD = HD + 4, DPL = R::DPL;
    constexpr int HEADS = PATH == kDigits ? 4 * NT : kCols;    // of a workgroup
    constexpr int HALVES = PATH == kHalf ? 2 : 1;              // 16-position tiles of a step
    constexpr int STEP = kWaves * HALVES * kPos;
    __shared__ __attribute__((aligned(16))) float buf[2 * kCols * LD];     // q, later the waves' O
    __shared__ float wm[kWaves][kCols], wsum[kWaves][kCols];
    __shared__ int shift[kCols];                               // kDigits: q * 2^shift are the digits' integers
    const PagedAttn &a = g.a;
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wid = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int c = lane & 15, m = lane >> 4;
    const int b = blockIdx.z, hk = blockIdx.y / g.col_tiles, ct = blockIdx.y - hk * g.col_tiles;
    const int h0 = hk * g.group + ct * HEADS, heads = min(HEADS, g.group - ct * HEADS);
    // the head of column c (kDigits: of the four lanes of a head's digits the first NT take a set's each)
    const int hc = PATH == kDigits ? (c >> 2) * NT + min(c & 3, NT - 1) : c;
    const bool owner = hc < heads && (PATH != kDigits || (c & 3) < NT);
    const int ps = a.c.page_size;
    const int n = min(max(a.lengths[b], 0), a.max_length);
    const int start = a.window > 0 && n > a.window ? n - a.window : 0;
    const int lo = (start & ~(kPos - 1)) + blockIdx.x * g.piece, hi = min(n, lo + g.piece);
    const size_t slot0 = ((size_t)blockIdx.x * gridDim.z + b) * g.n_heads + h0;
    if (lo >= hi && g.pieces > 1) {
        if (blockIdx.x == 0 && tid < heads) g.ms[slot0 + tid] = make_float2(-INFINITY, 0.f);
        return;
    }
    // A step's tiles: page and offset run along with the position.
    const int *row = a.table.pages + (size_t)b * a.table.ld;
    const size_t head_at = (size_t)hk * a.c.tile_bytes, page_bytes = (size_t)a.c.nkv * a.c.tile_bytes;
    const int last = hi > lo ? (hi - 1) & ~(kPos - 1) : 0;     // the piece's last tile
    auto place = [&](int tb, bool &there) -> size_t {          // of a tile: its bytes' start, less the offset's
        const int page = __builtin_amdgcn_readfirstlane(row[tb / ps]);
        there = page >= 0 && page < a.c.pages;
        return (there ? (size_t)page : 0) * page_bytes + head_at;
    };
    R k[HALVES], v[HALVES];
    int tb = lo + wid * HALVES * kPos;
    size_t at[HALVES];
    bool there[HALVES];
    auto seek = [&](int t) {
#pragma unroll
        for (int u = 0; u < HALVES; ++u) at[u] = place(min(t + u * kPos, last), there[u]);
    };
    auto load_k = [&](int t) {
#pragma unroll
        for (int u = 0; u < HALVES; ++u) k[u].load_k(a.c.k + at[u], ps, min(t + u * kPos, last) % ps, c, m);
    };
    auto load_v = [&](int t) {
#pragma unroll
        for (int u = 0; u < HALVES; ++u) v[u].load_v(a.c.v + at[u], ps, min(t + u * kPos, last) % ps, c, m);
    };
    if (tb < hi) {
        seek(tb);
        load_k(tb);
        load_v(tb);
    }
    // q
    uint8_t *qb = reinterpret_cast<uint8_t *>(buf);
    pu4 qh[PATH == kHalf ? HD / 32 : 1];
    pu2 qd[PATH == kDigits ? NT : 1][PATH == kDigits ? T::NB : 1];
    const int64_t q_at = (int64_t)b * a.q.ts + (int64_t)h0 * a.q.hs;
    if constexpr (PATH == kExact) {
        for (int i = tid; i < kCols * HD; i += kThreads) {
            const int r = i / HD, d = i - r * HD;
            buf[r * LD + d] = r < heads ? load1(a.q.dtype, a.q.p, q_at + (int64_t)r * a.q.hs + d) : 0.f;
        }
        __syncthreads();
    } else if constexpr (PATH == kHalf) {
        constexpr int QL = HD + 8;
        uint16_t *qs = reinterpret_cast<uint16_t *>(buf);
        for (int i = tid; i < kCols * HD; i += kThreads) {
            const int r = i / HD, d = i - r * HD;
            qs[r * QL + d] = r < heads ? reinterpret_cast<const uint16_t *>(a.q.p)[q_at + (int64_t)r * a.q.hs + d] : 0;
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < HD / 32; ++j) qh[j] = *reinterpret_cast<const pu4 *>(qs + c * QL + 32 * j + 8 * m);
    } else {
        // sixteen threads per head, HD / 16 elements each: the largest magnitude, then the digits, eight
        // elements (or four) at a time, to where the lanes read them: [set][block][lane][8]
        const int r = tid >> 4, e0 = (tid & 15) * DPL;
        constexpr int W = DPL < 8 ? DPL : 8;
        float x[DPL], top = 0.f;
        bool odd = false;
#pragma unroll
        for (int e = 0; e < DPL; ++e) {
            x[e] = r < heads ? load1(a.q.dtype, a.q.p, q_at + (int64_t)r * a.q.hs + e0 + e) : 0.f;
            odd |= !(fabsf(x[e]) < INFINITY);
            top = fmaxf(top, fabsf(x[e]));
        }
        top = lanes::row16_max(odd ? INFINITY : top);
        int ex;
        (void)frexpf(top, &ex);                                // top < 2^ex
        const int sh = top > 0.f && top < INFINITY ? 30 - ex : 0;
        if ((tid & 15) == 0) shift[r] = top < INFINITY ? sh : INT_MAX;
        if (r < HEADS) {
            const int i = r / NT, t = r - i * NT;
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
                    uint8_t *o = qb + (((size_t)t * T::NB + blk) * kWave + mm * 16 + 4 * i + q) * 8 + (d & 7);
                    if constexpr (W == 8) *reinterpret_cast<pu2 *>(o) = pu2{dig[q][0], dig[q][1]};
                    else *reinterpret_cast<uint32_t *>(o) = dig[q][0];
                }
            }
        }
        __syncthreads();
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int j = 0; j < T::NB; ++j) qd[t][j] = *reinterpret_cast<const pu2 *>(qb + ((size_t)(t * T::NB + j) * kWave + lane) * 8);
    }
    pf4 o[DPL];                                        // o[x][r']: dim v_dim(x, 4m + r') of column c
#pragma unroll
    for (int x = 0; x < DPL; ++x) o[x] = pf4{0.f, 0.f, 0.f, 0.f};
    // scores in log2 units: without a cap in one product
    const float cap = a.softcap, sl2 = cap > 0.f ? a.scale : __fmul_rn(a.scale, kLog2e);
    float digits[PATH == kDigits ? NT : 1];
    if constexpr (PATH == kDigits) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int s = shift[(c >> 2) * NT + t];
            digits[t] = s == INT_MAX ? NAN : ldexpf(CT == DT_Q4_0 ? 0.0625f : 1.0f, 8 * (c & 3) - s);
        }
    }
    float mx = -INFINITY, sum = 0.f;                   // sum: this lane's positions only
    for (; tb < hi; tb += STEP) {
        const int tn = tb + STEP;
        bool here[HALVES];
#pragma unroll
        for (int u = 0; u < HALVES; ++u) here[u] = there[u];
        pf4 s4[HALVES];
        if constexpr (PATH == kExact) {
            pf4 st[4] = {};
#pragma unroll
            for (int j = 0; j < R::N; ++j)
#pragma unroll
                for (int e0 = 0; e0 < R::KE; e0 += 4) {
                    const pf4 qv = *reinterpret_cast<const pf4 *>(buf + c * LD + R::k_dim(j, m, e0));
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        st[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[0].k_at(j, e0 + e), qv[e], st[e], 0, 0, 0);
                }
            s4[0] = (st[0] + st[1]) + (st[2] + st[3]);
        } else if constexpr (PATH == kHalf) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                s4[u] = pf4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < HD / 32; ++j) s4[u] = mfma16<CT>(k[u].w[j], qh[j], s4[u]);
            }
        } else {
            pf4 st[NT] = {};
#pragma unroll
            for (int j = 0; j < T::NB; ++j) {
                pu2 kb = k[0].k_codes(j);
                const float sc[4] = {quad_lane<0>(k[0].s[j]), quad_lane<1>(k[0].s[j]), quad_lane<2>(k[0].s[j]), quad_lane<3>(k[0].s[j])};
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const pi4 d = __builtin_amdgcn_mfma_i32_16x16x32_i8(__builtin_bit_cast(long, kb), __builtin_bit_cast(long, qd[t][j]),
                                                                        pi4{0, 0, 0, 0}, 0, 0, 0);
#pragma unroll
                    for (int r = 0; r < 4; ++r) st[t][r] = __builtin_fmaf((float)d[r], sc[r], st[t][r]);
                }
            }
            // the digits of a head lie in a quad; each lane keeps its own head's score
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                float own = quad_sum(__fmul_rn(st[0][r], digits[0]));
#pragma unroll
                for (int t = 1; t < NT; ++t) {
                    const float other = quad_sum(__fmul_rn(st[t][r], digits[t]));
                    own = (c & 3) >= t ? other : own;
                }
                s4[0][r] = own;
            }
        }
        seek(tn);                                      // past the end: the last tile again
        load_k(tn);
        float p[HALVES][4], ref = -INFINITY;
#pragma unroll
        for (int u = 0; u < HALVES; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                float x = __fmul_rn(s4[u][r], sl2);
                if (cap > 0.f) x = __fmul_rn(__fmul_rn(cap, tanhf(__fdiv_rn(x, cap))), kLog2e);
                p[u][r] = x;
            }
        // the piece's first and last tiles, and pages that do not exist: positions that do not count
        bool all = tb >= start && tb + HALVES * kPos <= hi;
#pragma unroll
        for (int u = 0; u < HALVES; ++u) all &= here[u];
        if (!all) {
#pragma unroll
            for (int u = 0; u < HALVES; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int t = tb + u * kPos + 4 * m + r;
                    if (!here[u] || t < start || t >= hi) {
                        p[u][r] = -INFINITY;
                        // its weight is 0, and 0 times a NaN there would be NaN
                        v[u].clear_v(r);
                    }
                }
        }
#pragma unroll
        for (int u = 0; u < HALVES; ++u) ref = fmaxf(ref, fmaxf(fmaxf(p[u][0], p[u][1]), fmaxf(p[u][2], p[u][3])));
        // The maximum moves, with O and the sums, only for a score far above it: weights up to 2^kLazy do no harm.
        if (__any(ref > mx + kLazy)) {
            ref = fmaxf(ref, __shfl_xor(ref, 16, kWave));
            ref = fmaxf(ref, __shfl_xor(ref, 32, kWave));
            const float mn = fmaxf(mx, ref), f = mx == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mx - mn);
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
        if constexpr (PATH == kHalf) {
            // contraction index 8m + 4u + r is position 4m + r of half u
            pu4 pw;
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < 2; ++i) pw[2 * u + i] = to_16(CT, p[u][2 * i]) | to_16(CT, p[u][2 * i + 1]) << 16;
#pragma unroll
            for (int x = 0; x < DPL; x += 2) {
                pu4 even, odd;
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint32_t w0 = v[u].v_pair(2 * i, x), w1 = v[u].v_pair(2 * i + 1, x);
                        even[2 * u + i] = __builtin_amdgcn_perm(w1, w0, 0x05040100u);
                        odd[2 * u + i] = __builtin_amdgcn_perm(w1, w0, 0x07060302u);
                    }
                o[x] = mfma16<CT>(even, pw, o[x]);
                o[x + 1] = mfma16<CT>(odd, pw, o[x + 1]);
            }
        } else {
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int x = 0; x < DPL; ++x) o[x] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[0].v_at(r, x), p[0][r], o[x], 0, 0, 0);
        }
        load_v(tn);
    }
    sum += __shfl_xor(sum, 16, kWave);
    sum += __shfl_xor(sum, 32, kWave);
    if (m == 0) {
        wm[wid][c] = mx;
        wsum[wid][c] = sum;
    }
    __syncthreads();                                   // every wave is past its reads of q
    float top = wm[0][c];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) top = fmaxf(top, wm[w][c]);
    // a wave without positions, or with scores of -inf only, has sum 0; its factor must not be NaN
    const float fw = sum == 0.f ? 0.f : __builtin_amdgcn_exp2f(mx - top);
    float tot = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w)
        if (wsum[w][c] != 0.f) tot += __fmul_rn(wsum[w][c], __builtin_amdgcn_exp2f(wm[w][c] - top));
#pragma unroll
    for (int x = 0; x < DPL; ++x)
#pragma unroll
        for (int r = 0; r < 4; ++r) o[x][r] = sum == 0.f ? 0.f : __fmul_rn(o[x][r], fw);
    // two waves at a time leave their O, the two before add theirs to it
#pragma unroll
    for (int half = 2; half >= 1; half /= 2) {
        float *mine = buf + ((wid & (half - 1)) * kCols + c) * LD;
        if (wid >= half && wid < 2 * half && owner) {
#pragma unroll
            for (int x = 0; x < DPL; ++x)
#pragma unroll
                for (int r = 0; r < 4; ++r) mine[R::v_dim(x, 4 * m + r)] = o[x][r];
        }
        __syncthreads();
        if (wid < half && owner) {
#pragma unroll
            for (int x = 0; x < DPL; ++x)
#pragma unroll
                for (int r = 0; r < 4; ++r) o[x][r] = __fadd_rn(o[x][r], mine[R::v_dim(x, 4 * m + r)]);
        }
        __syncthreads();
    }
    if (wid != 0 || !owner) return;
    if (g.pieces == 1) {
        const float inv = tot == 0.f ? 0.f : __fdiv_rn(1.0f, tot);
        const int64_t out_at = (int64_t)b * a.out.ts + (int64_t)(h0 + hc) * a.out.hs;
#pragma unroll
        for (int x = 0; x < DPL; ++x)
#pragma unroll
            for (int r = 0; r < 4; ++r) store1(a.out.dtype, a.out.p, out_at + R::v_dim(x, 4 * m + r), __fmul_rn(o[x][r], inv));
        if (a.lse && m == 0) a.lse[(size_t)b * g.n_heads + h0 + hc] = lse_of(top, tot);
    } else {
#pragma unroll
        for (int x = 0; x < DPL; ++x)
#pragma unroll
            for (int r = 0; r < 4; ++r) g.part[(slot0 + hc) * HD + R::v_dim(x, 4 * m + r)] = o[x][r];
        if (m == 0) g.ms[slot0 + hc] = make_float2(top, tot);
    }
}

// grid (heads, sequences): the pieces of one head. A wave takes every fourth piece, HD / 64 dims per lane.
template <int HD>
__global__ __launch_bounds__(kThreads) void paged_join_kernel(AttnArgs g) {
    constexpr int D = HD / kWave, U = 8;               // U: loads in flight
    __shared__ float part[kWaves][HD], ws[kWaves];
    const PagedAttn &a = g.a;
    const int h = blockIdx.x, b = blockIdx.y, lane = threadIdx.x & (kWave - 1), wid = threadIdx.x / kWave;
    const size_t stride = (size_t)gridDim.y * g.n_heads, slot = (size_t)b * g.n_heads + h;
    const int n = min(max(a.lengths[b], 0), a.max_length);
    const int start = a.window > 0 && n > a.window ? n - a.window : 0;
    const int used = max(1, (n - (start & ~(kPos - 1)) + g.piece - 1) / g.piece);
    // every wave finds the maximum, then adds its own pieces
    float top = -INFINITY;
    for (int i = lane; i < used; i += kWave) top = fmaxf(top, g.ms[slot + i * stride].x);
    top = lanes::wave_max(top);
    float o[D] = {}, sum = 0.f;
    for (int i0 = wid; i0 < used; i0 += kWaves * U) {
        float2 ms[U];
        float v[U][D];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const size_t at = slot + (size_t)min(i0 + u * kWaves, used - 1) * stride;
            ms[u] = g.ms[at];
#pragma unroll
            for (int d = 0; d < D; ++d) v[u][d] = g.part[at * HD + lane * D + d];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            // an empty piece has written no O; a sum of NaN has a weight of NaN, whatever its maximum
            if (i0 + u * kWaves >= used || ms[u].y == 0.f) continue;
            const float f = ms[u].y != ms[u].y ? ms[u].y : __builtin_amdgcn_exp2f(ms[u].x - top);
            sum = __builtin_fmaf(f, ms[u].y, sum);
#pragma unroll
            for (int d = 0; d < D; ++d) o[d] = __builtin_fmaf(f, v[u][d], o[d]);
        }
    }
#pragma unroll
    for (int d = 0; d < D; ++d) part[wid][lane * D + d] = o[d];
    if (lane == 0) ws[wid] = sum;
    __syncthreads();
    const int t = threadIdx.x;
    if (t >= HD) return;
    float x = 0.f, tot = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        x += part[w][t];
        tot += ws[w];
    }
    store1(a.out.dtype, a.out.p, (int64_t)b * a.out.ts + (int64_t)h * a.out.hs + t, tot == 0.f ? 0.f : __fdiv_rn(x, tot));
    if (a.lse && t == 0) a.lse[slot] = lse_of(top, tot);
}

// A piece is a fixed number of positions, so that sequences of different lengths make equal work: as
// many as give kWantGroups workgroups if all sequences were max_length long, a stride of the waves
// at least.
struct Plan {
    int col_heads, col_tiles, want, piece, pieces;
};
Plan plan_of(int dtype, int nkv, int batch, int n_heads, int max_length, int window) {
    Plan p;
    const int group = n_heads / nkv;
    p.col_heads = !is_quant(dtype) ? kCols : group <= 4 ? 4 : group <= 8 ? 8 : 16;
    p.col_tiles = (group + p.col_heads - 1) / p.col_heads;
    const int64_t groups = (int64_t)batch * nkv * p.col_tiles;
    const int64_t len = (window > 0 && window < max_length - kPos ? window + kPos : max_length);
    p.want = (int)std::max<int64_t>(1, std::min<int64_t>(kMaxPieces, kWantGroups / groups));
    p.piece = (int)(((len + p.want - 1) / p.want + kPieceUnit - 1) / kPieceUnit * kPieceUnit);
    p.pieces = (int)((len + p.piece - 1) / p.piece);
    return p;
}

size_t part_bytes(int hd, int batch, int n_heads, int pieces) { return (size_t)pieces * batch * n_heads * hd * sizeof(float); }

}  // namespace

// For any window: a plan has at most as many pieces as it may want, and as the positions have units.
size_t paged_attention_workspace(int dtype, int nkv, int hd, int batch, int n_heads, int max_length) {
    const int pieces = std::min(plan_of(dtype, nkv, batch, n_heads, max_length, 0).want, (max_length + kPieceUnit - 1) / kPieceUnit);
    return pieces == 1 ? 0 : part_bytes(hd, batch, n_heads, pieces) + (size_t)pieces * batch * n_heads * sizeof(float2);
}

int launch_paged_attention(const PagedAttn &a, hipStream_t s) {
    AttnArgs g;
    g.a = a;
    g.n_heads = a.q.heads;
    g.group = g.n_heads / a.c.nkv;
    const Plan p = plan_of(a.c.dtype, a.c.nkv, a.q.tokens, g.n_heads, a.max_length, a.window);
    g.col_tiles = p.col_tiles;
    g.piece = p.piece;
    g.pieces = p.pieces;
    g.part = reinterpret_cast<float *>(a.ws);
    g.ms = reinterpret_cast<float2 *>(a.ws + part_bytes(a.c.hd, a.q.tokens, g.n_heads, p.pieces));
    const dim3 grid(p.pieces, a.c.nkv * p.col_tiles, a.q.tokens), block(kThreads);
    const bool half = a.q.dtype != DT_F32;
#define SPH_ATTN(COND, CT, HD, PATH, NT) \
    if (a.c.dtype == CT && a.c.hd == HD && (COND)) hipLaunchKernelGGL((paged_attn_kernel<CT, HD, PATH, NT>), grid, block, 0, s, g);
#define SPH_ATTN_16(CT, HD) SPH_ATTN(!half, CT, HD, kExact, 1) SPH_ATTN(half, CT, HD, kHalf, 1)
#define SPH_ATTN_Q(CT, HD)                                                          \
    SPH_ATTN(p.col_heads == 4, CT, HD, kDigits, 1) SPH_ATTN(p.col_heads == 8, CT, HD, kDigits, 2) \
    SPH_ATTN(p.col_heads == 16, CT, HD, kDigits, 4)
#define SPH_ATTN_HD(HD) \
    SPH_ATTN(true, DT_F32, HD, kExact, 1) SPH_ATTN_16(DT_BF16, HD) SPH_ATTN_16(DT_F16, HD) SPH_ATTN_Q(DT_Q8_0, HD) SPH_ATTN_Q(DT_Q4_0, HD)
    SPH_ATTN_HD(64) SPH_ATTN_HD(128) SPH_ATTN_HD(256)
    if (!hip_ok(hipGetLastError(), "paged attention launch")) return -1;
    if (p.pieces > 1) {
        const dim3 jg(g.n_heads, a.q.tokens);
        if (a.c.hd == 64) hipLaunchKernelGGL((paged_join_kernel<64>), jg, block, 0, s, g);
        else if (a.c.hd == 128) hipLaunchKernelGGL((paged_join_kernel<128>), jg, block, 0, s, g);
        else hipLaunchKernelGGL((paged_join_kernel<256>), jg, block, 0, s, g);
        if (!hip_ok(hipGetLastError(), "paged attention join launch")) return -1;
    }
    return 0;
}

}  // namespace sapphire
