// paged_shared.h - attention of the rows of a group over the positions that they share (not installed): the kernel, for the
// sources that build it for float and for quantized caches.
#pragma once

#include "paged_attention.h"

namespace sapphire {

namespace {

// What a workgroup of the shared positions needs beside AttnArgs: columns are the query heads of one K/V head of all rows of a
// group, a tile of them is a workgroup's.
struct SharedPlan {
    int cols, col_tiles, pieces, total;    // total: (piece, K/V head, group) triples
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

// Two values' term of 16 bits in one word, and what it leaves of them.
template <int T>
__device__ __forceinline__ uint32_t take_term(float &a, float &b) {
    if constexpr (T == DT_BF16) {          // cut off: exact, and cheaper than rounding
        const uint32_t w = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
        a = __fsub_rn(a, __uint_as_float(__float_as_uint(a) & 0xffff0000u));
        b = __fsub_rn(b, __uint_as_float(__float_as_uint(b) & 0xffff0000u));
        return w;
    } else {
        const uint32_t w = pack_16(DT_F16, a, b);
        a = __fsub_rn(a, from_f16(w & 0xffffu));
        b = __fsub_rn(b, from_f16(w >> 16));
        return w;
    }
}

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
    // Quantized: the eight codes of block j as fp16. A byte below 1024's last bits is 1024 plus it.
    __device__ __forceinline__ pu4 codes(int j) const {
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
        const pu2 q = raw.k_codes(j);      // signed bytes; Q4_0: times 16
        pu4 o;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t b = (i < 2 ? q.x : q.y) ^ 0x80808080u;
            const uint32_t w = __builtin_amdgcn_perm(0x64646464u, b, i & 1 ? 0x04030402u : 0x04010400u);
            o[i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, w) - h2{1152, 1152});
        }
        return o;
    }
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

// The sums O of a column, unnormalised, and its (maximum, sum), of one piece of the shared positions. A wave has CS sets of 16
// columns; WC waves of a workgroup have columns of their own and the same positions, the others other positions.
template <int CT, int HD, bool HALF, bool SHORT, int CS, int WC>
__global__ __launch_bounds__(kThreads, 1) void paged_shared_kernel(AttnArgs g, SharedPlan sp) {
    using F = Form<CT, HALF, SHORT>;
    using K = KeyTile<CT, HD>;
    using V = ValueTile<CT, HD>;
    using R = Raw<CT, HD>;
    using T = Tile<CT, HD>;
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
    auto row_of = [&](int j) { return r0 + j / g.group; };
    auto head_of = [&](int j) { return hk * g.group + j % g.group; };
    auto slot_of = [&](int j) { return ((size_t)piece * a.q.tokens + row_of(j)) * g.n_heads + head_of(j); };
    if (u0 == u1) {
        for (int i = tid; i < 16 * CS * WC; i += kThreads) {
            const int j = tile * WC * 16 * CS + i;
            if (j < cols) g.ms[slot_of(j)] = make_float2(-INFINITY, 0.f);
        }
        return;
    }
    const float cap = a.softcap, sl2 = cap > 0.f ? a.scale : __fmul_rn(a.scale, kLog2e);
    pu4 q[CS][F::TQ][QW];
    float unit[CS], mx[CS], sum[CS];
#pragma unroll
    for (int s = 0; s < CS; ++s) {
        const int j = c0 + 16 * s + c;
        const bool there = j < cols;
        const int64_t at = there ? (int64_t)row_of(j) * a.q.ts + (int64_t)head_of(j) * a.q.hs : 0;
        mx[s] = -INFINITY;
        sum[s] = 0.f;
        unit[s] = sl2;
        if constexpr (F::kF32) {
#pragma unroll
            for (int w = 0; w < QW; ++w) {
                float x[4];
                load_some<4>(DT_F32, a.q.p, at + 16 * w + 4 * m, x);
                q[s][0][w] = there ? pu4{__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3])} : pu4{0, 0, 0, 0};
            }
        } else {
            float x[QW][8], top = 0.f;
            bool odd = false;
#pragma unroll
            for (int w = 0; w < QW; ++w) {
                Raw8 r;
                load8(a.q.dtype, sp.wide, a.q.p, at + 32 * w + 8 * m, r);
                values8(a.q.dtype, r, x[w]);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    x[w][e] = there ? x[w][e] : 0.f;
                    odd |= !(fabsf(x[w][e]) < INFINITY);
                    top = fmaxf(top, fabsf(x[w][e]));
                }
            }
            int sh = 0;
            if constexpr (F::kScaled) {
                top = odd ? INFINITY : top;
                top = fmaxf(top, __shfl_xor(top, 16, kWave));
                top = fmaxf(top, __shfl_xor(top, 32, kWave));
                int ex;
                (void)frexpf(top, &ex);                // top < 2^ex
                sh = top > 0.f && top < INFINITY ? 15 - ex : 0;
                unit[s] = top < INFINITY ? ldexpf(sl2, -sh - (CT == DT_Q4_0 ? 4 : 0)) : NAN;
            }
#pragma unroll
            for (int w = 0; w < QW; ++w)
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    float y0 = F::kScaled ? ldexpf(x[w][e], sh) : x[w][e], y1 = F::kScaled ? ldexpf(x[w][e + 1], sh) : x[w][e + 1];
                    if constexpr (HALF && !F::kScaled) {
                        q[s][0][w][e / 2] = pack_16(F::QT, y0, y1);    // (they were of that type: nothing is rounded)
                    } else {
#pragma unroll
                        for (int t = 0; t < F::TQ; ++t) q[s][t][w][e / 2] = take_term<F::QT>(y0, y1);
                    }
                }
        }
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
                        st[e & 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[0].raw.k_at(j, e), __uint_as_float(q[s][0][j][e]), st[e & 1], 0, 0, 0);
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
                        for (int t = 0; t < F::TQ; ++t) d = mfma16<DT_F16>(codes, q[s][t][j], d);
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
                        for (int j = 0; j < QW; ++j) p[s][h] = mfma16<F::QT>(k[h].raw.w[j], q[s][t][j], p[s][h]);
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
                    float x = __fmul_rn(p[s][h][r], unit[s]);
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
            if (j < cols) {
                float *out = g.part + slot_of(j) * HD;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    constexpr int W = T::kQuant ? (DPL < 4 ? DPL : 4) : 4;
#pragma unroll
                    for (int x = 0; x < DPL; x += W)
                        *reinterpret_cast<pf4 *>(out + V::dim(x, 4 * m + r)) = pf4{o[s][x][r], o[s][x + 1][r], o[s][x + 2][r], o[s][x + 3][r]};
                }
                if (m == 0) g.ms[slot_of(j)] = make_float2(mx[s], sum[s]);
            }
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

// Columns of a workgroup: as few sets and waves side by side as the group's columns need, so that the others take positions.
// (At 256 dims two sets do not fit the registers.)
struct Columns {
    int cs, wc;
};
inline Columns columns_of(int cols, int hd) {
    const int cs = cols <= 16 || hd == 256 ? 1 : 2, sets = (cols + 16 * cs - 1) / (16 * cs);
    return Columns{cs, sets == 1 ? 1 : sets == 2 ? 2 : 4};
}

template <int CT, int HD, bool HALF, bool SHORT>
void launch_shared_form(const AttnArgs &g, const SharedPlan &sp, hipStream_t s) {
    const dim3 grid((unsigned)((sp.total + 7) / 8 * 8 * sp.col_tiles)), block(kThreads);
    const Columns k = columns_of(sp.cols, HD);
    constexpr int MOST = HD == 256 ? 1 : 2;
#define SPH_COLS(CS, WC) \
    if (k.cs == CS && k.wc == WC) hipLaunchKernelGGL((paged_shared_kernel<CT, HD, HALF, SHORT, CS, WC>), grid, block, 0, s, g, sp);
    SPH_COLS(1, 1) SPH_COLS(MOST, 2) SPH_COLS(MOST, 4)
    if constexpr (MOST > 1) { SPH_COLS(MOST, 1) }
#undef SPH_COLS
}

}  // namespace

bool launch_shared_quant(const void *args, const void *plan, hipStream_t s);

}  // namespace sapphire
