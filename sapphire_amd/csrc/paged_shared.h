// paged_shared.h - attention of the rows of a group over the positions that they share (not installed): the kernel, for the
// sources that build it for float and for quantized caches.
#pragma once

#include <type_traits>

#include "paged_attention.h"

namespace sapphire {

namespace {

// What a workgroup of the shared positions needs beside AttnArgs: columns are the query heads of one K/V head of all rows of a
// group, a tile of them is a workgroup's.
struct SharedPlan {
    int cols, col_tiles, pieces, total;    // total: (piece, K/V head, group) triples
    int cs, nw;                            // of Columns
    bool wide;                             // q's data and strides are multiples of 16 bytes
};

// The products' operands, by the cache's type and the rows'. q comes in TQ terms of the type that K's products run in:
//   F32                 16x16x4 fp32
//   16-bit, its rows    as they are
//   BF16, fp32 rows     three bf16 terms, exact
//   F16, fp32 rows      two fp16 terms of q times a power of two: 2^-23 of an element, or 2^-39 of the largest
//   quantized           the same of any rows (one term of 16-bit ones) against K's codes, whole numbers; a block's sum times
//                       its scale in fp32
// and the weights in TP terms against V in TV of them (16-bit caches: V as it is; quantized: its values in bf16 terms).
template <int CT, bool HALF, bool SHORT>
struct Form {
    static constexpr bool kQuant = CT == DT_Q8_0 || CT == DT_Q4_0, kF32 = CT == DT_F32;
    static constexpr int QT = kQuant ? DT_F16 : CT, VT = kQuant ? DT_BF16 : CT;        // types of the two products
    static constexpr int TQ = HALF || kF32 ? 1 : CT == DT_BF16 ? 3 : 2;
    static constexpr int TV = kQuant ? (SHORT ? 2 : 3) : 1;
    static constexpr int TP = kQuant ? TV : HALF || CT == DT_F16 ? 2 : 3;
    static constexpr bool kScaled = QT == DT_F16 && !(HALF && CT == DT_F16);           // q is brought into fp16's range
    static constexpr float kLift = VT == DT_F16 ? 7.0f : 0.0f;             // as in paged_attn_kernel
    static __device__ __forceinline__ constexpr bool meets(int v, int p) { return v + p < (TV > TP ? TV : TP); }
};

// Two values' term of 16 bits in one word, and what it leaves of them. Rounded to nearest: of a number in [1, 2) two bf16 terms
// leave 2^-17 (cut off: 2^-15, always of the number's sign), at as many instructions. CUT: for three terms that hold
// all bits either way, of numbers up to fp32's largest, which rounded up would be an infinity.
template <int T, bool CUT = false>
__device__ __forceinline__ uint32_t take_term(float &a, float &b) {
    if constexpr (T == DT_BF16) {
        const uint32_t w = CUT ? __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u) : pack_16(DT_BF16, a, b);
        a = __fsub_rn(a, __uint_as_float(CUT ? __float_as_uint(a) & 0xffff0000u : w << 16));
        b = __fsub_rn(b, __uint_as_float((CUT ? __float_as_uint(b) : w) & 0xffff0000u));
        return w;
    } else {
        const uint32_t w = pack_16(DT_F16, a, b);
        a = __fsub_rn(a, from_f16(w & 0xffffu));
        b = __fsub_rn(b, from_f16(w >> 16));
        return w;
    }
}

// Eight signed bytes (Q4_0: codes times 16) as fp16: a byte in 1024's last bits is 1024 plus it.
__device__ __forceinline__ pu4 codes_f16(pu2 q) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    pu4 o;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t b = (i < 2 ? q.x : q.y) ^ 0x80808080u;
        const uint32_t w = __builtin_amdgcn_perm(0x64646464u, b, i & 1 ? 0x04030402u : 0x04010400u);
        o[i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, w) - h2{1152, 1152});
    }
    return o;
}

// A group's columns for one K/V head: column j is query head j % group of it, of row j / group.
struct SharedColumns {
    int r0, group, hk;
    __device__ __forceinline__ int row(int j) const { return r0 + j / group; }
    __device__ __forceinline__ int head(int j) const { return hk * group + j % group; }
};

// A column's q as the score product's operand, and what its sums are multiplied by to be scores in log2 units (or what the cap
// takes): never negative, q has the sign.
template <int CT, int HD, bool HALF, bool SHORT>
struct SharedQuery {
    using F = Form<CT, HALF, SHORT>;
    static constexpr int QW = F::kF32 ? HD / 16 : HD / 32;     // words of 16 bytes of a term
    pu4 w[F::TQ][QW];
    float unit;

    __device__ __forceinline__ void load(const PagedAttn &a, bool wide, const SharedColumns &col, int j, int cols, int m) {
        constexpr int E = F::kF32 ? 4 : 8;
        const bool there = j < cols;
        const int64_t at = there ? (int64_t)col.row(j) * a.q.ts + (int64_t)col.head(j) * a.q.hs : 0;
        const float sl2 = a.softcap > 0.f ? a.scale : __fmul_rn(a.scale, kLog2e);
        float x[QW][E], top = 0.f;
        bool odd = false;
#pragma unroll
        for (int i = 0; i < QW; ++i) {
            if constexpr (F::kF32) {
                load_some<4>(DT_F32, a.q.p, at + 16 * i + 4 * m, x[i]);
            } else {
                Raw8 r;
                load8(a.q.dtype, wide, a.q.p, at + 32 * i + 8 * m, r);
                values8(a.q.dtype, r, x[i]);
            }
#pragma unroll
            for (int e = 0; e < E; ++e) {
                x[i][e] = !there ? 0.f : sl2 < 0.f ? -x[i][e] : x[i][e];
                odd |= !(fabsf(x[i][e]) < INFINITY);
                top = fmaxf(top, fabsf(x[i][e]));
            }
        }
        // (never 0: the mask's -inf times it is -inf, and a score of it is as good as 0)
        constexpr float kLeast = 0x1p-149f;
        unit = fmaxf(fabsf(sl2), kLeast);
        int sh = 0;
        if constexpr (F::kScaled) {
            top = odd ? INFINITY : top;
            top = fmaxf(top, __shfl_xor(top, 16, kWave));
            top = fmaxf(top, __shfl_xor(top, 32, kWave));
            int ex;
            (void)frexpf(top, &ex);                    // top < 2^ex
            sh = top > 0.f && top < INFINITY ? 15 - ex : 0;
            unit = top < INFINITY ? fmaxf(ldexpf(unit, -sh - (CT == DT_Q4_0 ? 4 : 0)), kLeast) : NAN;
        }
#pragma unroll
        for (int i = 0; i < QW; ++i) {
            if constexpr (F::kF32) {
                w[0][i] = pu4{__float_as_uint(x[i][0]), __float_as_uint(x[i][1]), __float_as_uint(x[i][2]), __float_as_uint(x[i][3])};
            } else {
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    float y0 = F::kScaled ? ldexpf(x[i][e], sh) : x[i][e], y1 = F::kScaled ? ldexpf(x[i][e + 1], sh) : x[i][e + 1];
                    if constexpr (HALF && !F::kScaled) {
                        w[0][i][e / 2] = pack_16(F::QT, y0, y1);           // (they were of that type: nothing is rounded)
                    } else {
#pragma unroll
                        for (int t = 0; t < F::TQ; ++t) w[t][i][e / 2] = take_term<F::QT, true>(y0, y1);
                    }
                }
            }
        }
    }
};

// A lane's part of 16 positions of K as the score product's operand.
template <int CT, int HD>
struct KeyTile {
    using R = Raw<CT, HD>;
    using T = Tile<CT, HD>;
    static constexpr bool kQuant = T::kQuant;
    R raw;
    pf4 s[kQuant ? T::NB : 1];             // quantized: s[j][r], the scale of block j of position 4m + r

    __device__ __forceinline__ void load(const uint8_t *tile, uint32_t ps, uint32_t off, int c, int m) {
        if constexpr (!kQuant) {
            raw.load_k(tile, ps, off, c, m);
        } else {
            if constexpr (R::kHalf) {
                const pu2 v = *reinterpret_cast<const pu2 *>(tile + T::k_code(off + c, 8 * m));
                raw.w[0] = pu4{v.x, v.y, 0, 0};
            } else {
#pragma unroll
                for (int j = 0; j < R::N; ++j)
                    raw.w[j] = *reinterpret_cast<const pu4 *>(tile + T::k_code(off, 0) + (uint32_t)((j * 4 + m) * 16 + c) * 16);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int b = 0; b < T::NB; b += 2) {
                    const pf2 v = *reinterpret_cast<const pf2 *>(tile + T::k_scale(ps, off + 4 * m + r, b));
                    s[b][r] = v.x;
                    s[b + 1][r] = v.y;
                }
        }
    }
    // Quantized: the eight codes of block j.
    __device__ __forceinline__ pu4 codes(int j) const { return codes_f16(raw.k_codes(j)); }
};

// A lane's part of 16 positions of V: positions 4m .. 4m + 3, the DPL dims of column c.
template <int CT, int HD>
struct ValueTile {
    using R = Raw<CT, HD>;
    using T = Tile<CT, HD>;
    static constexpr int DPL = R::DPL;
    R raw;
    pf4 s;                                 // quantized: the scales of the four positions' block

    __device__ __forceinline__ void load(const uint8_t *tile, uint32_t ps, uint32_t off, int c, int m) {
        if constexpr (!T::kQuant) {
            raw.load_v(tile, ps, off, c, m);
        } else {
            if constexpr (R::kHalf) {
                const pu2 v = *reinterpret_cast<const pu2 *>(tile + T::v_run(off + 4 * m, c));
                raw.w[0] = pu4{v.x, v.y, 0, 0};
            } else if constexpr (T::RUN >= 16) {
#pragma unroll
                for (int r = 0; r < 4; ++r) raw.w[r] = *reinterpret_cast<const pu4 *>(tile + (off + 4 * m + r) * T::ROW + c * 16);
            } else {
#pragma unroll
                for (int u = 0; u < R::N; ++u) raw.w[u] = *reinterpret_cast<const pu4 *>(tile + T::v_run(off + 4 * m + u * T::P, c));
            }
            s = *reinterpret_cast<const pf4 *>(tile + T::v_scale(ps, off + 4 * m, c * DPL / 32));
        }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < R::N; ++i) raw.w[i] = CT == DT_Q4_0 ? pu4{0x88888888u, 0x88888888u, 0x88888888u, 0x88888888u} : pu4{0, 0, 0, 0};
        s = pf4{0.f, 0.f, 0.f, 0.f};
    }
    // Quantized: element x of position 4m + r.
    __device__ __forceinline__ float at(int r, int x) const {
        if constexpr (CT == DT_Q8_0) {
            const int i = r * DPL + x;
            return __fmul_rn((float)(int8_t)(raw.w[i / 16][i / 4 % 4] >> (8 * (i % 4))), s[r]);
        } else {
            const int i = r * (DPL / 2) + x % (DPL / 2);
            return __fmul_rn((float)((int)(raw.w[i / 16][i / 4 % 4] >> (8 * (i % 4) + 4 * (x / (DPL / 2))) & 15u) - 8), s[r]);
        }
    }
    // Dim of a lane's element x.
    static __device__ __forceinline__ int dim(int x, int c) {
        if constexpr (T::kQuant) return c * DPL + x;
        else return R::v_dim(x, c);
    }
};

// A column's O (lane (c, m): dims V::dim(x, 4m + r)) and (maximum, sum) to its slot.
template <int CT, int HD>
__device__ __forceinline__ void store_sums(const AttnArgs &g, size_t slot, int m, const pf4 (&o)[HD / 16], float mx, float sum) {
    float *out = g.part + slot * HD;
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int x = 0; x < HD / 16; x += 4)
            *reinterpret_cast<pf4 *>(out + ValueTile<CT, HD>::dim(x, 4 * m + r)) = pf4{o[x][r], o[x + 1][r], o[x + 2][r], o[x + 3][r]};
    if (m == 0) g.ms[slot] = make_float2(mx, sum);
}

// The sums O of a column, unnormalised, and its (maximum, sum), of one piece of the shared positions. A wave has CS sets of 16
// columns; WC waves of a workgroup have columns of their own and the same positions, the others other positions.
template <int CT, int HD, bool HALF, bool SHORT, int CS, int WC>
__global__ __launch_bounds__(kThreads, 1) void paged_shared_kernel(AttnArgs g, SharedPlan sp) {
    using F = Form<CT, HALF, SHORT>;
    using K = KeyTile<CT, HD>;
    using V = ValueTile<CT, HD>;
    constexpr int LD = HD + 4, DPL = HD / 16, WP = kWaves / WC, HALVES = F::kF32 || HD == 256 ? 1 : 2;
    constexpr int QW = F::kF32 ? HD / 16 : HD / 32;            // q: words of 16 bytes of a term
    constexpr int kO = WP > 1 ? kWaves * 16 * LD : 1;
    __shared__ __attribute__((aligned(16))) float buf[kO];
    __shared__ float wm[kWaves][16], wsum[kWaves][16];
    const PagedAttn &a = g.a;
    // (piece, K/V head, group) triples go round the dies, the column tiles of one to the same die, after each other
    const int round = blockIdx.x / (8 * sp.col_tiles), in = blockIdx.x - round * 8 * sp.col_tiles;
    const int triple = round * 8 + (in & 7), tile = in >> 3;
    if (triple >= sp.total) return;
    const int piece = triple % sp.pieces, hk = triple / sp.pieces % a.c.nkv, gi = triple / sp.pieces / a.c.nkv;
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wid = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int c = lane & 15, m = lane >> 4, wc = wid % WC, wp = wid / WC;
    const int r0 = gi * a.rows, cols = min(a.rows, a.q.tokens - r0) * g.group, c0 = (tile * WC + wc) * 16 * CS;
    const Group grp = group_of(a, gi);
    const int tiles = grp.shared / kPos, units = (tiles + HALVES - 1) / HALVES;
    const int u0 = (int)((int64_t)units * piece / sp.pieces), u1 = (int)((int64_t)units * (piece + 1) / sp.pieces);
    const SharedColumns col{r0, g.group, hk};
    auto slot_of = [&](int j) { return ((size_t)piece * a.q.tokens + col.row(j)) * g.n_heads + col.head(j); };
    if (u0 == u1) {
        for (int i = tid; i < 16 * CS * WC; i += kThreads) {
            const int j = tile * WC * 16 * CS + i;
            if (j < cols) g.ms[slot_of(j)] = make_float2(-INFINITY, 0.f);
        }
        return;
    }
    const float cap = a.softcap;
    SharedQuery<CT, HD, HALF, SHORT> q[CS];
    float mx[CS], sum[CS];
#pragma unroll
    for (int s = 0; s < CS; ++s) {
        q[s].load(a, sp.wide, col, c0 + 16 * s + c, cols, m);
        mx[s] = -INFINITY;
        sum[s] = 0.f;
    }
    pf4 o[CS][DPL];                                    // o[s][x][r]: dim V::dim(x, 4m + r) of column c
#pragma unroll
    for (int s = 0; s < CS; ++s)
#pragma unroll
        for (int x = 0; x < DPL; ++x) o[s][x] = pf4{0.f, 0.f, 0.f, 0.f};
    const auto *pages = (const __attribute__((address_space(4))) int *)(a.table.pages + (size_t)max(grp.leader, 0) * a.table.ld);
    const size_t page_bytes = (size_t)a.c.nkv * a.c.tile_bytes, head_at = (size_t)hk * a.c.tile_bytes;
    const int ps = a.c.page_size;
    K k[HALVES];
    V v[HALVES];
    size_t at[HALVES];
    uint32_t off[HALVES];
    bool there[HALVES];
    auto seek = [&](int u) {
#pragma unroll
        for (int h = 0; h < HALVES; ++h) {
            const int t = u * HALVES + h;
            const uint32_t t16 = (uint32_t)min(t, tiles - 1), i = page_of(a.c, t16);
            off[h] = t16 * kPos - i * (uint32_t)ps;
            const int page = pages[__builtin_amdgcn_readfirstlane((int)i)];
            there[h] = t < tiles && page >= 0 && page < a.c.pages;
            at[h] = (page >= 0 && page < a.c.pages ? (size_t)page : 0) * page_bytes + head_at;
        }
    };
    auto load_k = [&]() {
#pragma unroll
        for (int h = 0; h < HALVES; ++h) k[h].load(a.c.k + at[h], ps, off[h], c, m);
    };
    auto load_v = [&]() {
#pragma unroll
        for (int h = 0; h < HALVES; ++h) v[h].load(a.c.v + at[h], ps, off[h], c, m);
    };
    int u = c0 < cols ? u0 + wp : u1;                  // (a wave without columns has nothing to do)
    if (u < u1) {
        seek(u);
        load_k();
        load_v();
    }
    for (; u < u1; u += WP) {
        bool here[HALVES], all = true;
#pragma unroll
        for (int h = 0; h < HALVES; ++h) {
            here[h] = there[h];
            all &= here[h];
        }
        pf4 p[CS][HALVES];
        if constexpr (F::kF32) {
#pragma unroll
            for (int s = 0; s < CS; ++s) {
                pf4 st[2] = {};
#pragma unroll
                for (int j = 0; j < QW; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        st[e & 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[0].raw.k_at(j, e), __uint_as_float(q[s].w[0][j][e]), st[e & 1], 0, 0, 0);
                p[s][0] = st[0] + st[1];
            }
        } else if constexpr (F::kQuant) {
#pragma unroll
            for (int h = 0; h < HALVES; ++h)
#pragma unroll
                for (int j = 0; j < QW; ++j) {
                    const pu4 codes = k[h].codes(j);
#pragma unroll
                    for (int s = 0; s < CS; ++s) {
                        pf4 d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int t = 0; t < F::TQ; ++t) d = mfma16<DT_F16>(codes, q[s].w[t][j], d);
                        const pf4 sc = k[h].s[j];
#pragma unroll
                        for (int r = 0; r < 4; ++r) p[s][h][r] = j == 0 ? __fmul_rn(d[r], sc[r]) : __builtin_fmaf(d[r], sc[r], p[s][h][r]);
                    }
                }
        } else {
#pragma unroll
            for (int s = 0; s < CS; ++s)
#pragma unroll
                for (int h = 0; h < HALVES; ++h) {
                    p[s][h] = pf4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int t = F::TQ - 1; t >= 0; --t)
#pragma unroll
                        for (int j = 0; j < QW; ++j) p[s][h] = mfma16<F::QT>(k[h].raw.w[j], q[s].w[t][j], p[s][h]);
                }
        }
        const bool more = u + WP < u1;
        if (more) {
            seek(u + WP);
            load_k();
        }
        if (!all) {
#pragma unroll
            for (int h = 0; h < HALVES; ++h)
                if (!here[h]) v[h].clear();            // its weights are 0, and 0 times a NaN there would be NaN
        }
        uint32_t pw[CS][F::TP][2 * HALVES];            // contraction index 4 HALVES m + 4 h + r: position 4m + r of tile h
#pragma unroll
        for (int s = 0; s < CS; ++s) {
            float ref = -INFINITY;
#pragma unroll
            for (int h = 0; h < HALVES; ++h)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float x = __fmul_rn(p[s][h][r], q[s].unit);
                    if (cap > 0.f) x = __fmul_rn(capped(x, cap), kLog2e);
                    if (!all) x = here[h] ? x : -INFINITY;
                    p[s][h][r] = x;
                    ref = fmaxf(ref, x);
                }
            // the maximum moves, with O and the sums, only for a score far above it (as in paged_attn_kernel)
            if (__any(ref > mx[s] + F::kLift + kLazy)) {
                ref = fmaxf(ref, __shfl_xor(ref, 16, kWave));
                ref = fmaxf(ref, __shfl_xor(ref, 32, kWave));
                const float mn = fmaxf(mx[s], ref - F::kLift), f = mx[s] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mx[s] - mn);
                mx[s] = mn;
                sum[s] = __fmul_rn(sum[s], f);
#pragma unroll
                for (int x = 0; x < DPL; ++x) o[s][x] *= f;
            }
            const float base = mx[s] == -INFINITY ? 0.f : mx[s];
#pragma unroll
            for (int h = 0; h < HALVES; ++h) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    p[s][h][r] = __builtin_amdgcn_exp2f(p[s][h][r] - base);
                    sum[s] = __fadd_rn(sum[s], p[s][h][r]);
                }
                if constexpr (!F::kF32) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float x0 = p[s][h][2 * i], x1 = p[s][h][2 * i + 1];
#pragma unroll
                        for (int t = 0; t < F::TP; ++t) pw[s][t][2 * h + i] = take_term<F::VT>(x0, x1);
                    }
                }
            }
        }
        auto product = [](const uint32_t (&x)[2 * HALVES], const uint32_t (&y)[2 * HALVES], pf4 z) {
            if constexpr (HALVES == 2) return mfma16<F::VT>(pu4{x[0], x[1], x[2], x[3]}, pu4{y[0], y[1], y[2], y[3]}, z);
            else return mfma8<F::VT>(pu2{x[0], x[1]}, pu2{y[0], y[1]}, z);
        };
        if constexpr (F::kF32) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int x = 0; x < DPL; ++x)
#pragma unroll
                    for (int s = 0; s < CS; ++s) o[s][x] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[0].raw.v_at(r, x), p[s][0][r], o[s][x], 0, 0, 0);
        } else if constexpr (F::kQuant) {
#pragma unroll
            for (int x = 0; x < DPL; ++x) {
                uint32_t w[F::TV][2 * HALVES];
#pragma unroll
                for (int h = 0; h < HALVES; ++h)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float x0 = v[h].at(2 * i, x), x1 = v[h].at(2 * i + 1, x);
#pragma unroll
                        for (int t = 0; t < F::TV; ++t) w[t][2 * h + i] = take_term<DT_BF16>(x0, x1);
                    }
#pragma unroll
                for (int t = 0; t < F::TV; ++t)
#pragma unroll
                    for (int y = 0; y < F::TP; ++y)
                        if (F::meets(t, y))
#pragma unroll
                            for (int s = 0; s < CS; ++s) o[s][x] = product(w[t], pw[s][y], o[s][x]);
            }
        } else {
#pragma unroll
            for (int x = 0; x < DPL; x += 2) {
                uint32_t even[2 * HALVES], odd[2 * HALVES];
#pragma unroll
                for (int h = 0; h < HALVES; ++h)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint32_t w0 = v[h].raw.v_pair(2 * i, x), w1 = v[h].raw.v_pair(2 * i + 1, x);
                        even[2 * h + i] = __builtin_amdgcn_perm(w1, w0, 0x05040100u);
                        odd[2 * h + i] = __builtin_amdgcn_perm(w1, w0, 0x07060302u);
                    }
#pragma unroll
                for (int t = 0; t < F::TP; ++t)
#pragma unroll
                    for (int s = 0; s < CS; ++s) {
                        o[s][x] = product(even, pw[s][t], o[s][x]);
                        o[s][x + 1] = product(odd, pw[s][t], o[s][x + 1]);
                    }
            }
        }
        if (more) load_v();
    }
#pragma unroll
    for (int s = 0; s < CS; ++s) {
        sum[s] += __shfl_xor(sum[s], 16, kWave);
        sum[s] += __shfl_xor(sum[s], 32, kWave);
        const int j = c0 + 16 * s + c;
        if constexpr (WP == 1) {
            if (j < cols) store_sums<CT, HD>(g, slot_of(j), m, o[s], mx[s], sum[s]);
        } else {
            __syncthreads();
            if (m == 0) {
                wm[wid][c] = mx[s];
                wsum[wid][c] = sum[s];
            }
#pragma unroll
            for (int x = 0; x < DPL; ++x)
#pragma unroll
                for (int r = 0; r < 4; ++r) buf[(wid * 16 + c) * LD + V::dim(x, 4 * m + r)] = o[s][x][r];
            __syncthreads();
            for (int i = tid; i < WC * 16 * (HD / 4); i += kThreads) {
                const int col = i / (HD / 4), d = (i - col * (HD / 4)) * 4, w0 = col / 16, cc = col & 15;
                const int jj = (tile * WC + w0) * 16 * CS + 16 * s + cc;
                if (jj >= cols) continue;
                float top = -INFINITY, tot = 0.f;
                pf4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int w = 0; w < WP; ++w) top = fmaxf(top, wm[w * WC + w0][cc]);
#pragma unroll
                for (int w = 0; w < WP; ++w) {
                    const int from = w * WC + w0;
                    // a wave without positions, or with scores of -inf only, has sum 0; its factor must not be NaN
                    const float sw = wsum[from][cc], f = sw == 0.f ? 0.f : __builtin_amdgcn_exp2f(wm[from][cc] - top);
                    const pf4 ow = *reinterpret_cast<const pf4 *>(buf + (from * 16 + cc) * LD + d);
                    tot = __builtin_fmaf(sw, f, tot);
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] = __builtin_fmaf(ow[e], f, x[e]);
                }
                *reinterpret_cast<pf4 *>(g.part + slot_of(jj) * HD + d) = x;
                if (d == 0) g.ms[slot_of(jj)] = make_float2(top, tot);
            }
        }
    }
}

// ---- many columns: K and V through LDS ----
//
// The same sums where a workgroup's waves all have columns of their own. They take the same positions at the same time, so each
// loads and converts a part of them, two steps ahead, and writes it to LDS as the products' operands; a step's operands are
// read by all while the next one's are written. Four jobs of a step are V's: the DPL dims (of 256: half of them) of a lane at two
// positions of a tile, a word of every dim's operand; the others copy or convert K, 16 positions of 32 dims each.
//
// A step of eight waves with two sets each, bf16, 128 dims: 3500 cycles of two waves per SIMD, of which the matrix cores are busy
// for 1600. Each wave's are 600 of loads, their addresses and stores, 500 of scores, 400 of the maximum, 700 of weights (an exp2
// takes 8, two terms of a pair 25), 800 of V's product. Measured and left out: 32x32x16 products, four sets in one wave per
// SIMD, LDS reads three products ahead (spills: 233 us for 205).
template <int CT, int HD, bool HALF, bool SHORT>
struct Stage {
    using F = Form<CT, HALF, SHORT>;
    using T = Tile<CT, HD>;
    static constexpr int DPL = HD / 16, HALVES = F::kF32 || HD == 256 ? 1 : 2;
    static constexpr int VX = F::kF32 ? 0 : DPL > 8 ? 8 : DPL;             // dims of a V job
    static constexpr int XP = F::kF32 ? 1 : DPL / VX;
    static constexpr int VB = 8 * HALVES;                                  // bytes of a lane's operand of V, a dim and term
    static constexpr int KC = F::kF32 ? HD / 16 : HALVES * HD / 32;        // K: KiB
    static constexpr int VC = F::kF32 ? HD / 16 : 0;                       // V, fp32: KiB
    static constexpr int kVBytes = F::kF32 ? VC * 1024 : DPL * F::TV * kWave * VB;
    static constexpr int kScales = KC * 1024, kKBytes = kScales + (F::kQuant ? KC * 64 : 0);
};

template <int CT, int HD, bool HALF, bool SHORT, int CS, int NW>
__global__ __launch_bounds__(NW *kWave, 2) void paged_shared_wide_kernel(AttnArgs g, SharedPlan sp) {
    using F = Form<CT, HALF, SHORT>;
    using G = Stage<CT, HD, HALF, SHORT>;
    using T = Tile<CT, HD>;
    constexpr int DPL = G::DPL, HALVES = G::HALVES;
    constexpr int QW = F::kF32 ? HD / 16 : HD / 32;
    // K jobs of a wave (where there are eight waves, of the four that have none of V); fp32: KiB of K, and of V
    constexpr int KJ = F::kF32 ? (G::KC < NW ? 1 : G::KC / NW) : G::KC / 4;
    // Where eight waves fill the compute unit, the upper four form a step's weights while the others multiply, and the other way
    // round: they add V a step later, which needs three steps of V. (64 rows of 32 heads over 8, bf16, behind 16384 positions: 67 us
    // for the call, 69.6 without; Q4_0, 32 rows: 63.4 and 66.)
    constexpr bool SPLIT = NW == 8;
    constexpr int VS = SPLIT ? 3 : 2;
    __shared__ __attribute__((aligned(16))) uint8_t klds[2][G::kKBytes], vlds[VS][G::kVBytes];
    const PagedAttn &a = g.a;
    const int round = blockIdx.x / (8 * sp.col_tiles), in = blockIdx.x - round * 8 * sp.col_tiles;
    const int triple = round * 8 + (in & 7), tile = in >> 3;
    if (triple >= sp.total) return;
    const int piece = triple % sp.pieces, hk = triple / sp.pieces % a.c.nkv, gi = triple / sp.pieces / a.c.nkv;
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wid = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int c = lane & 15, m = lane >> 4;
    const int r0 = gi * a.rows, cols = min(a.rows, a.q.tokens - r0) * g.group, c0 = (tile * NW + wid) * 16 * CS;
    const Group grp = group_of(a, gi);
    const int tiles = grp.shared / kPos, units = (tiles + HALVES - 1) / HALVES;
    const int u0 = (int)((int64_t)units * piece / sp.pieces), u1 = (int)((int64_t)units * (piece + 1) / sp.pieces);
    const SharedColumns col{r0, g.group, hk};
    auto slot_of = [&](int j) { return ((size_t)piece * a.q.tokens + col.row(j)) * g.n_heads + col.head(j); };
    if (u0 == u1) {
        for (int i = tid; i < 16 * CS * NW; i += NW * kWave) {
            const int j = tile * NW * 16 * CS + i;
            if (j < cols) g.ms[slot_of(j)] = make_float2(-INFINITY, 0.f);
        }
        return;
    }
    SharedQuery<CT, HD, HALF, SHORT> q[CS];
    float mx[CS], sum[CS];
    pf4 o[CS][DPL];
#pragma unroll
    for (int s = 0; s < CS; ++s) {
        q[s].load(a, sp.wide, col, c0 + 16 * s + c, cols, m);
        mx[s] = -INFINITY;
        sum[s] = 0.f;
#pragma unroll
        for (int x = 0; x < DPL; ++x) o[s][x] = pf4{0.f, 0.f, 0.f, 0.f};
    }
    const int *pages = a.table.pages + (size_t)max(grp.leader, 0) * a.table.ld;
    const size_t page_bytes = (size_t)a.c.nkv * a.c.tile_bytes, head_at = (size_t)hk * a.c.tile_bytes;
    const int ps = a.c.page_size;
    const float cap = a.softcap;

    // Where a step's tiles are. Page numbers are asked for a step ahead, by vector loads: those come in order with the rows', and
    // a wait for LDS does not wait for them.
    struct Place {
        size_t at[HALVES];
        uint32_t off[HALVES];
        bool on[HALVES];
    };
    int numbers[HALVES];
    auto ask = [&](int u) {
#pragma unroll
        for (int h = 0; h < HALVES; ++h) {
            uint32_t i = page_of(a.c, (uint32_t)min(min(u, u1 - 1) * HALVES + h, tiles - 1));
            asm("" : "+v"(i));
            numbers[h] = pages[i];
        }
    };
    auto seek = [&](int u) {                           // (after ask(u))
        Place w;
#pragma unroll
        for (int h = 0; h < HALVES; ++h) {
            const int t = min(u, u1 - 1) * HALVES + h;
            const uint32_t t16 = (uint32_t)min(t, tiles - 1);
            w.off[h] = t16 * kPos - page_of(a.c, t16) * (uint32_t)ps;
            const int page = __builtin_amdgcn_readfirstlane(numbers[h]);
            const bool there = page >= 0 && page < a.c.pages;
            w.on[h] = there && t < tiles;
            w.at[h] = (there ? (size_t)page : 0) * page_bytes + head_at;
        }
        return w;
    };
    // Raw words from their loads to their conversion: of K of one step, of V of the step before it.
    struct Loaded {
        uint32_t k[KJ][F::kQuant ? (CT == DT_Q8_0 ? 2 : 1) : 4];
        float ks[KJ];
        uint32_t v[F::kF32 ? 4 * KJ : 8];
        float vs[2];
        bool on;                           // V's tile
    };
    const int vjob = wid & 3, vh = vjob / 2 % HALVES, vi = vjob & 1, vx = HALVES == 1 ? vjob >> 1 : 0;    // tile, pair of positions, part
    const int fk = wid * KJ, fv = (NW - 1 - wid) * KJ;         // fp32: the wave's first KiB
    const bool has_v = F::kF32 ? fv < G::VC : wid < 4, has_k = F::kF32 ? fk < G::KC : NW == 4 || wid >= 4;
    auto load_k = [&](const Place &at, Loaded &w) {
        if (!has_k) return;
#pragma unroll
        for (int j = 0; j < KJ; ++j) {
            if constexpr (F::kF32) {
                *reinterpret_cast<pu4 *>(w.k[j]) = *reinterpret_cast<const pu4 *>(a.c.k + at.at[0] + at.off[0] * T::ROW + (fk + j) * 1024 + lane * 16);
            } else {
                const int n = (wid & 3) * KJ + j, h = HALVES == 1 ? 0 : n / (HD / 32), b = n % (HD / 32);
                const uint8_t *t = a.c.k + (h ? at.at[HALVES - 1] : at.at[0]);
                const uint32_t p0 = (h ? at.off[HALVES - 1] : at.off[0]) + c;
                const uint8_t *p = t + T::k_code(p0, 32 * b + 8 * m);
                if constexpr (CT == DT_Q4_0) w.k[j][0] = *reinterpret_cast<const uint32_t *>(p);
                else if constexpr (CT == DT_Q8_0) *reinterpret_cast<pu2 *>(w.k[j]) = *reinterpret_cast<const pu2 *>(p);
                else *reinterpret_cast<pu4 *>(w.k[j]) = *reinterpret_cast<const pu4 *>(p);
                if constexpr (F::kQuant) w.ks[j] = *reinterpret_cast<const float *>(t + T::k_scale(ps, p0, b));
            }
        }
    };
    auto load_v = [&](const Place &at, Loaded &w) {
        if (!has_v) return;
        w.on = vh ? at.on[HALVES - 1] : at.on[0];
        const uint8_t *t = a.c.v + (vh ? at.at[HALVES - 1] : at.at[0]);
        const uint32_t p0 = (vh ? at.off[HALVES - 1] : at.off[0]) + 4 * m + 2 * vi;
        if constexpr (F::kF32) {
#pragma unroll
            for (int j = 0; j < KJ; ++j) *reinterpret_cast<pu4 *>(w.v + 4 * j) = *reinterpret_cast<const pu4 *>(t + at.off[0] * T::ROW + (fv + j) * 1024 + lane * 16);
        } else if constexpr (F::kQuant) {
            // bytes of a position's run in this part: eight (fewer: all of both positions, which are next to each other)
            if constexpr (CT == DT_Q8_0 && HD == 256) {
#pragma unroll
                for (int r = 0; r < 2; ++r) *reinterpret_cast<pu2 *>(w.v + 2 * r) = *reinterpret_cast<const pu2 *>(t + T::v_run(p0 + r, c) + 8 * vx);
            } else if constexpr (T::RUN == 8) {
                *reinterpret_cast<pu4 *>(w.v) = *reinterpret_cast<const pu4 *>(t + T::v_run(p0, c));
            } else if constexpr (T::RUN == 4) {
                *reinterpret_cast<pu2 *>(w.v) = *reinterpret_cast<const pu2 *>(t + T::v_run(p0, c));
            } else {
                w.v[0] = *reinterpret_cast<const uint32_t *>(t + T::v_run(p0, c));
            }
            const pf2 s = *reinterpret_cast<const pf2 *>(t + T::v_scale(ps, p0, c * DPL / 32));
            w.vs[0] = s.x;
            w.vs[1] = s.y;
        } else if constexpr (HD == 64) {               // both positions' runs, next to each other
            *reinterpret_cast<pu4 *>(w.v) = *reinterpret_cast<const pu4 *>(t + T::v_run(p0, c));
        } else {
#pragma unroll
            for (int r = 0; r < 2; ++r) *reinterpret_cast<pu4 *>(w.v + 4 * r) = *reinterpret_cast<const pu4 *>(t + (p0 + r) * T::ROW + vx * 256 + c * 16);
        }
    };
    auto store_k = [&](const Loaded &w, uint8_t *to) {
        if (!has_k) return;
#pragma unroll
        for (int j = 0; j < KJ; ++j) {
            const int n = F::kF32 ? fk + j : (wid & 3) * KJ + j;
            pu4 x;
            if constexpr (F::kQuant) {
                const pu2 bytes = CT == DT_Q8_0 ? pu2{w.k[j][0], w.k[j][CT == DT_Q8_0 ? 1 : 0]} : pu2{w.k[j][0] << 4 & 0xf0f0f0f0u, w.k[j][0] & 0xf0f0f0f0u};
                x = codes_f16(bytes);
                if (m == 0) *reinterpret_cast<float *>(to + G::kScales + (n * 16 + c) * 4) = w.ks[j];
            } else {
                x = *reinterpret_cast<const pu4 *>(w.k[j]);
            }
            *reinterpret_cast<pu4 *>(to + n * 1024 + lane * 16) = x;
        }
    };
    auto store_v = [&](const Loaded &w, uint8_t *to) {
        if (!has_v) return;
        if constexpr (F::kF32) {
#pragma unroll
            for (int j = 0; j < KJ; ++j)
                *reinterpret_cast<pu4 *>(to + (fv + j) * 1024 + lane * 16) = w.on ? *reinterpret_cast<const pu4 *>(w.v + 4 * j) : pu4{0, 0, 0, 0};
        } else {
            uint8_t *at = to + lane * G::VB + (2 * vh + vi) * 4;
            constexpr float kLess = CT == DT_Q8_0 ? -128.0f : -8.0f;
            const float s0 = w.on ? w.vs[0] : 0.f, s1 = w.on ? w.vs[1] : 0.f, less0 = __fmul_rn(kLess, s0), less1 = __fmul_rn(kLess, s1);
#pragma unroll
            for (int e = 0; e < G::VX; e += F::kQuant ? 1 : 2) {
                const int x = vx * G::VX + e;
                if constexpr (F::kQuant) {
                    // bytes of the two positions, as they are above -128 (Q4_0: nibbles above -8); times the scale in one
                    // rounding, as the product of code and scale has
                    constexpr int RB = CT == DT_Q8_0 ? G::VX : T::RUN;
                    const int b0 = CT == DT_Q8_0 || HD == 256 ? e : e % RB, b1 = RB + b0;
                    // (256 dims of Q4_0: a part is the low nibbles of its eight bytes, or the high ones)
                    const int up = CT == DT_Q8_0 ? 0 : HD == 256 ? 4 * vx : 4 * (e / RB);
                    const uint32_t w0 = CT == DT_Q8_0 ? w.v[b0 / 4] ^ 0x80808080u : w.v[b0 / 4] >> up & 0x0f0f0f0fu;
                    const uint32_t w1 = CT == DT_Q8_0 ? w.v[b1 / 4] ^ 0x80808080u : w.v[b1 / 4] >> up & 0x0f0f0f0fu;
                    float x0 = __builtin_fmaf((float)(w0 >> (8 * (b0 % 4)) & 255u), s0, less0), x1 = __builtin_fmaf((float)(w1 >> (8 * (b1 % 4)) & 255u), s1, less1);
#pragma unroll
                    for (int t = 0; t < F::TV; ++t) *reinterpret_cast<uint32_t *>(at + (x * F::TV + t) * kWave * G::VB) = take_term<DT_BF16>(x0, x1);
                } else {
                    const uint32_t w0 = w.on ? w.v[e / 2] : 0u, w1 = w.on ? w.v[G::VX / 2 + e / 2] : 0u;
                    *reinterpret_cast<uint32_t *>(at + x * kWave * G::VB) = __builtin_amdgcn_perm(w1, w0, 0x05040100u);
                    *reinterpret_cast<uint32_t *>(at + (x + 1) * kWave * G::VB) = __builtin_amdgcn_perm(w1, w0, 0x07060302u);
                }
            }
        }
    };
    typedef typename std::conditional<HALVES == 2, pu4, pu2>::type Pair;
    auto product = [](Pair x, Pair y, pf4 z) {
        if constexpr (HALVES == 2) return mfma16<F::VT>(x, y, z);
        else return mfma8<F::VT>(x, y, z);
    };
    // A step's scores, as sums.
    auto scores = [&](const uint8_t *from, pf4 (&p)[CS][HALVES]) {
#pragma unroll
        for (int s = 0; s < CS; ++s)
#pragma unroll
            for (int h = 0; h < HALVES; ++h) p[s][h] = pf4{0.f, 0.f, 0.f, 0.f};
        if constexpr (F::kF32) {
#pragma unroll
            for (int j = 0; j < QW; ++j) {
                const pu4 k = *reinterpret_cast<const pu4 *>(from + j * 1024 + lane * 16);
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int s = 0; s < CS; ++s)
                        p[s][0] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(k[e]), __uint_as_float(q[s].w[0][j][e]), p[s][0], 0, 0, 0);
            }
        } else {
#pragma unroll
            for (int j = 0; j < QW; ++j)
#pragma unroll
                for (int h = 0; h < HALVES; ++h) {
                    const pu4 k = *reinterpret_cast<const pu4 *>(from + (h * QW + j) * 1024 + lane * 16);
                    if constexpr (F::kQuant) {
                        const pf4 sc = *reinterpret_cast<const pf4 *>(from + G::kScales + ((h * QW + j) * 16 + 4 * m) * 4);
#pragma unroll
                        for (int s = 0; s < CS; ++s) {
                            pf4 d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                            for (int t = 0; t < F::TQ; ++t) d = mfma16<DT_F16>(k, q[s].w[t][j], d);
#pragma unroll
                            for (int r = 0; r < 4; ++r) p[s][h][r] = __builtin_fmaf(d[r], sc[r], p[s][h][r]);
                        }
                    } else {
#pragma unroll
                        for (int t = F::TQ - 1; t >= 0; --t)
#pragma unroll
                            for (int s = 0; s < CS; ++s) p[s][h] = mfma16<F::QT>(k, q[s].w[t][j], p[s][h]);
                    }
                }
        }
    };
    // The cap and the mask, and the maximum, which moves, with O and the sums, only for a score far above it (as in
    // paged_attn_kernel).
    auto raise = [&](pf4 (&p)[CS][HALVES], const bool (&on)[HALVES]) {
        bool all = true;
#pragma unroll
        for (int h = 0; h < HALVES; ++h) all &= on[h];
        if (cap > 0.f)
#pragma unroll
            for (int s = 0; s < CS; ++s)
#pragma unroll
                for (int h = 0; h < HALVES; ++h)
#pragma unroll
                    for (int r = 0; r < 4; ++r) p[s][h][r] = __fmul_rn(capped(__fmul_rn(p[s][h][r], q[s].unit), cap), kLog2e);
        if (!all)
#pragma unroll
            for (int s = 0; s < CS; ++s)
#pragma unroll
                for (int h = 0; h < HALVES; ++h)
#pragma unroll
                    for (int r = 0; r < 4; ++r) p[s][h][r] = on[h] ? p[s][h][r] : -INFINITY;
        float ref[CS];
        bool far = false;
#pragma unroll
        for (int s = 0; s < CS; ++s) {
            ref[s] = p[s][0][0];
#pragma unroll
            for (int h = 0; h < HALVES; ++h)
#pragma unroll
                for (int r = h == 0; r < 4; ++r) ref[s] = __builtin_elementwise_maximum(ref[s], p[s][h][r]);
            ref[s] = cap > 0.f ? ref[s] : __fmul_rn(ref[s], q[s].unit);        // (unit >= 0: the largest score is the largest sum's)
            far |= ref[s] > mx[s] + F::kLift + kLazy;
        }
        if (__any(far)) {
#pragma unroll
            for (int s = 0; s < CS; ++s) {
                ref[s] = fmaxf(ref[s], __shfl_xor(ref[s], 16, kWave));
                ref[s] = fmaxf(ref[s], __shfl_xor(ref[s], 32, kWave));
                const float mn = fmaxf(mx[s], ref[s] - F::kLift), f = mx[s] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mx[s] - mn);
                mx[s] = mn;
                sum[s] = __fmul_rn(sum[s], f);
#pragma unroll
                for (int x = 0; x < DPL; ++x) o[s][x] *= f;
            }
        }
    };
    // The weights, in terms, and their sum.
    auto weigh = [&](pf4 (&p)[CS][HALVES], Pair (&pw)[CS][F::TP]) {
#pragma unroll
        for (int s = 0; s < CS; ++s) {
            const float base = mx[s] == -INFINITY ? 0.f : mx[s], unit = cap > 0.f ? 1.0f : q[s].unit;
#pragma unroll
            for (int h = 0; h < HALVES; ++h) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    p[s][h][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(p[s][h][r], unit, -base));
                    sum[s] = __fadd_rn(sum[s], p[s][h][r]);
                }
                if constexpr (!F::kF32) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float x0 = p[s][h][2 * i], x1 = p[s][h][2 * i + 1];
#pragma unroll
                        for (int t = 0; t < F::TP; ++t) pw[s][t][2 * h + i] = take_term<F::VT>(x0, x1);
                    }
                }
            }
        }
    };
    auto add = [&](const uint8_t *from, const pf4 (&p)[CS][HALVES], const Pair (&pw)[CS][F::TP]) {
        if constexpr (F::kF32) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int i = 0; i < DPL / 4; ++i) {
                    const pf4 v = *reinterpret_cast<const pf4 *>(from + (4 * m + r) * T::ROW + i * 256 + c * 16);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
#pragma unroll
                        for (int s = 0; s < CS; ++s) o[s][4 * i + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[e], p[s][0][r], o[s][4 * i + e], 0, 0, 0);
                }
        } else {
#pragma unroll
            for (int x = 0; x < DPL; ++x) {
                Pair v[F::TV];
#pragma unroll
                for (int t = 0; t < F::TV; ++t) v[t] = *reinterpret_cast<const Pair *>(from + (x * F::TV + t) * kWave * G::VB + lane * G::VB);
#pragma unroll
                for (int t = 0; t < F::TV; ++t)
#pragma unroll
                    for (int y = 0; y < F::TP; ++y)
                        if (F::meets(t, y))
#pragma unroll
                            for (int s = 0; s < CS; ++s) o[s][x] = product(v[t], pw[s][y], o[s][x]);
            }
        }
    };
    // Step s: its weights and V's product, and in between the scores of step s + 1, so that the matrix cores have work while the
    // weights are formed; K of step s + 2 and V of s + 1 go to LDS, and those of two steps further are asked for.
    Loaded w[2];
    pf4 p[2][CS][HALVES];
    bool on[2][HALVES];                                // of the step at hand, and the next one
    ask(u0);
    Place at = seek(u0);
    ask(u0 + 1);
    Place next = seek(u0 + 1);
    ask(u0 + 2);
    load_k(at, w[0]);
    load_v(at, w[0]);
    load_k(next, w[1]);
    store_k(w[0], klds[0]);
    store_v(w[0], vlds[0]);
    store_k(w[1], klds[1]);
#pragma unroll
    for (int h = 0; h < HALVES; ++h) {
        on[0][h] = at.on[h];
        on[1][h] = next.on[h];
    }
    at = seek(u0 + 2);
    ask(u0 + 3);
    load_k(at, w[0]);
    load_v(next, w[0]);
    next = seek(u0 + 3);
    ask(u0 + 4);
    load_k(next, w[1]);
    load_v(at, w[1]);
    bool later[2][HALVES];
#pragma unroll
    for (int h = 0; h < HALVES; ++h) {
        later[0][h] = at.on[h];
        later[1][h] = next.on[h];
    }
    __syncthreads();
    scores(klds[0], p[0]);
    __syncthreads();                                   // (the first trip writes there)
    // (Each half of the waves has a loop of its own, with as many barriers.)
    auto run = [&](auto late) {
        constexpr bool LATE = decltype(late)::value;
        Pair pw[CS][F::TP];
        int slot = 0;                                  // of V of step u + d
        for (int u = u0; u < u1; u += 2) {
#pragma unroll
            for (int d = 0; d < 2; ++d) {
                if (u + d < u1) {
                    const int after = slot + 1 == VS ? 0 : slot + 1, before = slot == 0 ? VS - 1 : slot - 1;
                    store_k(w[d], klds[d]);
                    store_v(w[d], vlds[after]);
                    at = seek(u + d + 4);
                    ask(u + d + 5);
                    load_k(at, w[d]);
                    load_v(next, w[d]);
                    next = at;
                    if constexpr (LATE) {
                        if (u + d > u0) add(vlds[before], p[1 - d], pw);
                        scores(klds[1 - d], p[1 - d]);
                        __builtin_amdgcn_sched_barrier(0);
                        raise(p[d], on[0]);
                        weigh(p[d], pw);
                    } else {
                        raise(p[d], on[0]);
                        weigh(p[d], pw);
                        if constexpr (SPLIT) __builtin_amdgcn_sched_barrier(0);
                        scores(klds[1 - d], p[1 - d]);
                        add(vlds[slot], p[d], pw);
                    }
#pragma unroll
                    for (int h = 0; h < HALVES; ++h) {
                        on[0][h] = on[1][h];
                        on[1][h] = later[0][h];
                        later[0][h] = later[1][h];
                        later[1][h] = at.on[h];
                    }
                    slot = after;
                    __syncthreads();
                }
            }
        }
        if constexpr (LATE) {
            if ((u1 - u0) % 2 == 1) add(vlds[slot == 0 ? VS - 1 : slot - 1], p[0], pw);
            else add(vlds[slot == 0 ? VS - 1 : slot - 1], p[1], pw);
        }
    };
    if constexpr (SPLIT) {
        if (wid >= 4) run(std::true_type());
        else run(std::false_type());
    } else {
        run(std::false_type());
    }
#pragma unroll
    for (int s = 0; s < CS; ++s) {
        sum[s] += __shfl_xor(sum[s], 16, kWave);
        sum[s] += __shfl_xor(sum[s], 32, kWave);
        const int j = c0 + 16 * s + c;
        if (j < cols) store_sums<CT, HD>(g, slot_of(j), m, o[s], mx[s], sum[s]);
    }
}

// Columns of a workgroup. Up to 32: as few sets as there are, and the waves take different positions. More: all waves side by
// side, with K and V through LDS. (48 columns behind 16384 positions, Q4_0: 46 us, as few ones in two tiles 56; bf16 35 and 38. 32
// columns, bf16: 28 us, as many ones 32.)
constexpr int kFewColumns = 32;
struct Columns {
    int cs, nw;                            // sets of a wave, waves side by side (0: one, of a workgroup that splits positions)
    int columns() const { return 16 * cs * std::max(nw, 1); }
};
// Sets of a wave at most: two where they are faster over many positions. (32 rows of 32 heads over 8 of 128 dims behind 65536
// positions, bf16 rows over Q4_0: 122 us with one, 144 with two.) They fit the registers of two waves but for fp32 rows over fp16,
// of which eight waves spill 33 registers and four 1, and are still ahead from 48 rows on: 128 rows behind 65536 positions 299 us,
// with one set 323, 64 rows 172 and 176; 24 rows 103 and 97. One set of 256 dims spills too, with fp32 rows: eight waves
// 16 (fp32, Q8_0), 7 (bf16), 5 (Q4_0), four 11 (Q8_0), 1 (Q4_0); 128 rows behind 8192 positions take 335, 214, 149, 207 us with
// eight, 335, 238, 157, 223 with four.
constexpr int wide_sets(int dtype, bool half, int hd) {
    return hd == 64 ? 2 : hd == 128 && (dtype == DT_F16 || (dtype == DT_BF16 && half)) ? 2 : 1;
}
inline Columns columns_of(int sets, int cols, int hd) {
    if (cols <= kFewColumns) return Columns{cols <= 16 || hd == 256 ? 1 : 2, cols > 16 && hd == 256 ? 2 : 0};
    const int cs = cols <= 64 ? 1 : sets;
    return Columns{cs, cols <= 64 * cs ? 4 : 8};
}

template <int CT, int HD, bool HALF, bool SHORT>
void launch_shared_form(const AttnArgs &g, const SharedPlan &sp, hipStream_t s) {
    const dim3 grid((unsigned)((sp.total + 7) / 8 * 8 * sp.col_tiles));
    const bool few = sp.cols <= kFewColumns;
#define SPH_FEW_COLS(CS, WC) \
    if (few && sp.cs == CS && std::max(sp.nw, 1) == WC) hipLaunchKernelGGL((paged_shared_kernel<CT, HD, HALF, SHORT, CS, WC>), grid, dim3(kThreads), 0, s, g, sp);
    SPH_FEW_COLS(1, 1)
    if constexpr (HD == 256) { SPH_FEW_COLS(1, 2) }
    else { SPH_FEW_COLS(2, 1) }
#undef SPH_FEW_COLS
#define SPH_WIDE(CS, NW) \
    if (!few && sp.cs == CS && sp.nw == NW) hipLaunchKernelGGL((paged_shared_wide_kernel<CT, HD, HALF, SHORT, CS, NW>), grid, dim3(NW * kWave), 0, s, g, sp);
    SPH_WIDE(1, 4) SPH_WIDE(1, 8)
    if constexpr (wide_sets(CT, HALF, HD) == 2) { SPH_WIDE(2, 4) SPH_WIDE(2, 8) }
#undef SPH_WIDE
}

}  // namespace

bool launch_shared_quant(const void *args, const void *plan, hipStream_t s);
bool launch_shared_join(const void *args, hipStream_t s);

}  // namespace sapphire
