// paged_attention.hip - attention of one new token per sequence over the paged cache.
//
// Scores and the weighted sum run on the fp32 matrix cores as in the prompt's attention
// (prefill.hip): S^T = K q^T with the query heads of a K/V head as columns leaves lane (c, m) head c's
// scores of positions 4m .. 4m + 3, which is the B operand of O^T = V^T P^T. One pass over K and V with
// a running maximum and sum per column; a sequence's positions are cut into pieces that workgroups take
// side by side, and a second launch joins the pieces' (maximum, sum, O).
#include <algorithm>

#include "internal.h"
#include "lanes.h"
#include "paged_dev.h"

namespace sapphire {

namespace {

constexpr int kWave = 64, kThreads = 256, kWaves = kThreads / kWave;
constexpr int kCols = 16;                  // query heads of a workgroup
constexpr int kPos = 16;                   // positions of a tile
constexpr int kMaxPieces = 256;
constexpr int kPieceMin = 128;             // positions that a piece has at least
constexpr int kWantGroups = 1024;          // workgroups that fill the chip (four per CU)
constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.693147180559945309f;

struct AttnArgs {
    PagedAttn a;
    int n_heads, group, col_tiles, pieces;
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
    static constexpr int KE = CT == DT_F32 ? 4 : CT == DT_Q8_0 ? 16 : CT == DT_Q4_0 ? 8 * T::G : 8;   // K: elements of a piece
    pu4 w[N];
    float s[T::kQuant ? (T::NB > 4 ? T::NB : 4) : 1];          // K: the row's block scales; V: four positions'

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
    // Dim of element e of piece j in lane chunk m.
    static __device__ __forceinline__ int k_dim(int j, int m, int e) {
        if constexpr (CT == DT_F32) return 16 * j + 4 * m + e;
        else if constexpr (CT == DT_Q8_0) return 64 * j + 32 * (e >> 3) + 8 * m + (e & 7);
        else if constexpr (CT == DT_Q4_0) return 32 * T::G * j + 32 * (e >> 3) + 8 * m + (e & 7);
        else return 32 * j + 8 * m + e;
    }
    __device__ __forceinline__ float k_at(int j, int e) const {
        if constexpr (CT == DT_F32) return __uint_as_float(w[j][e]);
        else if constexpr (CT == DT_BF16) return __uint_as_float(e & 1 ? w[j][e >> 1] & 0xffff0000u : w[j][e >> 1] << 16);
        else if constexpr (CT == DT_F16) return from_f16(e & 1 ? w[j][e >> 1] >> 16 : w[j][e >> 1] & 0xffffu);
        else if constexpr (CT == DT_Q8_0) return __fmul_rn((float)(int8_t)(w[j][e >> 2] >> (8 * (e & 3))), s[2 * j + (e >> 3)]);
        else {
            const uint32_t v = w[j][e >> 3];                   // block e / 8's four bytes
            const int q = (int)(v << (28 - (8 * (e & 3) + (e & 4)))) >> 28;
            return __fmul_rn((float)q, s[T::G * j + (e >> 3)]);
        }
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

// grid (pieces, K/V heads x column tiles, sequences).
template <int CT, int HD>
__global__ __launch_bounds__(kThreads) void paged_attn_kernel(AttnArgs g) {
    using R = Raw<CT, HD>;
    constexpr int LD = HD + 4, DPL = R::DPL;
    __shared__ __attribute__((aligned(16))) float buf[2 * kCols * LD];     // q, later the waves' O
    __shared__ float wm[kWaves][kCols], wsum[kWaves][kCols];
    const PagedAttn &a = g.a;
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wid = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int c = lane & 15, m = lane >> 4;
    const int b = blockIdx.z, hk = blockIdx.y / g.col_tiles, ct = blockIdx.y - hk * g.col_tiles;
    const int h0 = hk * g.group + ct * kCols, cols = min(kCols, g.group - ct * kCols);
    const int ps = a.c.page_size;
    const int n = min(max(a.lengths[b], 0), a.max_length);
    const int start = a.window > 0 && n > a.window ? n - a.window : 0;
    // pieces of whole 64-position strides, from the first tile on
    const int first = start & ~(kPos - 1), unit = kWaves * kPos;
    const int per = ((n - first + g.pieces - 1) / g.pieces + unit - 1) / unit * unit;
    const int lo = first + blockIdx.x * per, hi = min(n, lo + per);
    const size_t slot0 = ((size_t)blockIdx.x * gridDim.z + b) * g.n_heads + h0;
    if (lo >= hi && (g.pieces > 1 || n > 0)) {
        if (tid < cols) g.ms[slot0 + tid] = make_float2(-INFINITY, 0.f);
        return;
    }
    for (int i = tid; i < kCols * HD; i += kThreads) {
        const int r = i / HD, d = i - r * HD;
        buf[r * LD + d] = r < cols ? load1(a.q.dtype, a.q.p, (int64_t)b * a.q.ts + (int64_t)(h0 + r) * a.q.hs + d) : 0.f;
    }
    pf4 o[DPL];                                        // o[x][r']: dim v_dim(x, 4m + r') of column c
#pragma unroll
    for (int x = 0; x < DPL; ++x) o[x] = pf4{0.f, 0.f, 0.f, 0.f};
    float mx = -INFINITY, sum = 0.f;                   // sum: this lane's positions only
    __syncthreads();
    const int *row = a.table.pages + (size_t)b * a.table.ld;
    for (int tb = lo + wid * kPos; tb < hi; tb += kWaves * kPos) {
        const int pi = tb / ps, off = tb - pi * ps;
        const int page = __builtin_amdgcn_readfirstlane(row[pi]);
        if (page < 0 || page >= a.c.pages) continue;
        const size_t at = ((size_t)page * a.c.nkv + hk) * a.c.tile_bytes;
        R k, v;
        k.load_k(a.c.k + at, ps, off, c, m);
        v.load_v(a.c.v + at, ps, off, c, m);
        pf4 st[4] = {};
#pragma unroll
        for (int j = 0; j < R::N; ++j)
#pragma unroll
            for (int e0 = 0; e0 < R::KE; e0 += 4) {
                const pf4 qv = *reinterpret_cast<const pf4 *>(buf + c * LD + R::k_dim(j, m, e0));
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    st[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(k.k_at(j, e0 + e), qv[e], st[e], 0, 0, 0);
            }
        const pf4 s4 = (st[0] + st[1]) + (st[2] + st[3]);
        float sc[4], p[4], mt = -INFINITY;
        bool on[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int t = tb + 4 * m + r;
            on[r] = t >= start && t < hi;
            float x = __fmul_rn(s4[r], a.scale);
            if (a.softcap > 0.f) x = __fmul_rn(a.softcap, tanhf(__fdiv_rn(x, a.softcap)));
            sc[r] = on[r] ? __fmul_rn(x, kLog2e) : -INFINITY;
            mt = fmaxf(mt, sc[r]);
        }
        mt = fmaxf(mt, __shfl_xor(mt, 16, kWave));
        mt = fmaxf(mt, __shfl_xor(mt, 32, kWave));
        const float mn = fmaxf(mx, mt);
        const float f = mx == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mx - mn);
        sum = __fmul_rn(sum, f);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            // masked, or a score of -inf (also where every score so far is, mn included)
            p[r] = sc[r] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(sc[r] - mn);
            sum = __fadd_rn(sum, p[r]);
        }
        mx = mn;
        if (__any(f != 1.0f)) {
#pragma unroll
            for (int x = 0; x < DPL; ++x) o[x] *= f;
        }
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int x = 0; x < DPL; ++x) {
                // a masked position's weight is 0, and 0 times a NaN behind the sequence would be NaN
                const float vv = on[r] ? v.v_at(r, x) : 0.f;
                o[x] = __builtin_amdgcn_mfma_f32_16x16x4f32(vv, p[r], o[x], 0, 0, 0);
            }
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
    // two waves at a time leave their O, the two before add theirs to it
#pragma unroll
    for (int half = 2; half >= 1; half /= 2) {
        if (wid >= half && wid < 2 * half && c < cols) {
            float *mine = buf + (wid - half) * kCols * LD + c * LD;
#pragma unroll
            for (int x = 0; x < DPL; ++x)
#pragma unroll
                for (int r = 0; r < 4; ++r) mine[R::v_dim(x, 4 * m + r)] = half == 2 ? (sum == 0.f ? 0.f : __fmul_rn(o[x][r], fw)) : o[x][r];
        }
        __syncthreads();
        if (wid < half && c < cols) {
            const float *other = buf + wid * kCols * LD + c * LD;
#pragma unroll
            for (int x = 0; x < DPL; ++x)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    o[x][r] = __fadd_rn(half == 2 ? (sum == 0.f ? 0.f : __fmul_rn(o[x][r], fw)) : o[x][r], other[R::v_dim(x, 4 * m + r)]);
        }
        __syncthreads();
    }
    if (wid != 0 || c >= cols) return;
    if (g.pieces == 1) {
        const float inv = tot == 0.f ? 0.f : __fdiv_rn(1.0f, tot);
        const int64_t at = (int64_t)b * a.out.ts + (int64_t)(h0 + c) * a.out.hs;
#pragma unroll
        for (int x = 0; x < DPL; ++x)
#pragma unroll
            for (int r = 0; r < 4; ++r) store1(a.out.dtype, a.out.p, at + R::v_dim(x, 4 * m + r), __fmul_rn(o[x][r], inv));
        if (a.lse && m == 0) a.lse[(size_t)b * g.n_heads + h0 + c] = lse_of(top, tot);
    } else {
#pragma unroll
        for (int x = 0; x < DPL; ++x)
#pragma unroll
            for (int r = 0; r < 4; ++r) g.part[(slot0 + c) * HD + R::v_dim(x, 4 * m + r)] = o[x][r];
        if (m == 0) g.ms[slot0 + c] = make_float2(top, tot);
    }
}

// grid (heads, sequences): the pieces of one head.
template <int HD>
__global__ __launch_bounds__(HD) void paged_join_kernel(AttnArgs g) {
    __shared__ float w[kMaxPieces];
    const PagedAttn &a = g.a;
    const int h = blockIdx.x, b = blockIdx.y, t = threadIdx.x;
    const size_t stride = (size_t)gridDim.y * g.n_heads, slot = (size_t)b * g.n_heads + h;
    float top = -INFINITY;
    for (int i = 0; i < g.pieces; ++i) top = fmaxf(top, g.ms[slot + i * stride].x);
    for (int i = t; i < g.pieces; i += HD) {
        const float2 v = g.ms[slot + i * stride];
        // a sum of NaN has a weight of NaN, whatever its maximum
        w[i] = v.y == 0.f ? 0.f : v.y != v.y ? v.y : __builtin_amdgcn_exp2f(v.x - top);
    }
    __syncthreads();
    float sum = 0.f, o = 0.f;
    for (int i = 0; i < g.pieces; ++i) {
        const float f = w[i];
        if (f == 0.f) continue;                        // an empty piece has written no O
        sum = __builtin_fmaf(f, g.ms[slot + i * stride].y, sum);
        o = __builtin_fmaf(f, g.part[(slot + i * stride) * HD + t], o);
    }
    const float v = sum == 0.f ? 0.f : __fdiv_rn(o, sum);
    store1(a.out.dtype, a.out.p, (int64_t)b * a.out.ts + (int64_t)h * a.out.hs + t, v);
    if (a.lse && t == 0) a.lse[slot] = lse_of(top, sum);
}

struct Plan {
    int col_tiles, pieces;
};
Plan plan_of(int nkv, int batch, int n_heads, int max_length) {
    Plan p;
    p.col_tiles = (n_heads / nkv + kCols - 1) / kCols;
    const int64_t groups = (int64_t)batch * nkv * p.col_tiles;
    const int64_t want = std::max<int64_t>(1, kWantGroups / groups), most = ((int64_t)max_length + kPieceMin - 1) / kPieceMin;
    p.pieces = (int)std::max<int64_t>(1, std::min<int64_t>({want, most, kMaxPieces}));
    return p;
}

size_t part_bytes(int hd, int batch, int n_heads, int pieces) { return (size_t)pieces * batch * n_heads * hd * sizeof(float); }

}  // namespace

size_t paged_attention_workspace(int dtype, int nkv, int hd, int batch, int n_heads, int max_length) {
    const Plan p = plan_of(nkv, batch, n_heads, max_length);
    return p.pieces == 1 ? 0 : part_bytes(hd, batch, n_heads, p.pieces) + (size_t)p.pieces * batch * n_heads * sizeof(float2);
}

int launch_paged_attention(const PagedAttn &a, hipStream_t s) {
    AttnArgs g;
    g.a = a;
    g.n_heads = a.q.heads;
    g.group = g.n_heads / a.c.nkv;
    const Plan p = plan_of(a.c.nkv, a.q.tokens, g.n_heads, a.max_length);
    g.col_tiles = p.col_tiles;
    g.pieces = p.pieces;
    g.part = reinterpret_cast<float *>(a.ws);
    g.ms = reinterpret_cast<float2 *>(a.ws + part_bytes(a.c.hd, a.q.tokens, g.n_heads, p.pieces));
    const dim3 grid(p.pieces, a.c.nkv * p.col_tiles, a.q.tokens);
#define SPH_ATTN(CT, HD) \
    if (a.c.dtype == CT && a.c.hd == HD) hipLaunchKernelGGL((paged_attn_kernel<CT, HD>), grid, dim3(kThreads), 0, s, g);
#define SPH_ATTN_HD(HD) SPH_ATTN(DT_F32, HD) SPH_ATTN(DT_BF16, HD) SPH_ATTN(DT_F16, HD) SPH_ATTN(DT_Q8_0, HD) SPH_ATTN(DT_Q4_0, HD)
    SPH_ATTN_HD(64) SPH_ATTN_HD(128) SPH_ATTN_HD(256)
    if (!hip_ok(hipGetLastError(), "paged attention launch")) return -1;
    if (p.pieces > 1) {
        const dim3 jg(g.n_heads, a.q.tokens);
        if (a.c.hd == 64) hipLaunchKernelGGL((paged_join_kernel<64>), jg, dim3(64), 0, s, g);
        else if (a.c.hd == 128) hipLaunchKernelGGL((paged_join_kernel<128>), jg, dim3(128), 0, s, g);
        else hipLaunchKernelGGL((paged_join_kernel<256>), jg, dim3(256), 0, s, g);
        if (!hip_ok(hipGetLastError(), "paged attention join launch")) return -1;
    }
    return 0;
}

}  // namespace sapphire
