// paged_shared_join.hip - the last launch of the attention of rows that share positions where few are not shared: a row's
// drafted tokens, the end of a page. It forms their weights and sums itself, in fp32, and joins the pieces of the shared ones,
// so that the attention's kernels are left out.
#include "paged_shared.h"

namespace sapphire {

namespace {

// grid (heads, rows). HD / 8 lanes take a position, a workgroup 32 to 128 of them at a time; W waves as in paged_join_kernel.
// Six rows of one sequence of 1018 positions, 4 heads of 256 dims, fp32: 17.0 us for the call, with the attention's kernels for the
// six 19.9; 16 rows of 32 heads over 8 of 128 dims behind 4096 positions, bf16, 8 of their own each: 21.7 and 25.1, 32 each: 23.2 and
// 25.4.
template <int CT, int HD, int W>
__global__ __launch_bounds__(W *kWave) void paged_shared_join_kernel(AttnArgs g, bool wide) {
    constexpr int D = HD / kWave, U = 8, Q = kMaxPieces / 2 / kWave;       // U: loads in flight
    constexpr int LP = HD / 8, PW = kWave / LP, N = W * PW;                // lanes of a position, positions of a wave, at a time
    constexpr int E = (N + kWave - 1) / kWave;
    __shared__ __attribute__((aligned(16))) float part[W][HD], own[N][HD];
    __shared__ float own_m[N], own_s[N], weight[N];
    const PagedAttn &a = g.a;
    const int h = blockIdx.x, b = blockIdx.y, lane = threadIdx.x & (kWave - 1), wid = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int hk = h / g.group, l = lane % LP, sub = wid * PW + lane / LP;
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
    Raw8 r;
    load8(a.q.dtype, wide, a.q.p, (int64_t)b * a.q.ts + (int64_t)h * a.q.hs + l * 8, r);
    const int n = min(max(a.lengths[b], 0), a.max_length), start = min(group_of(a, b / a.rows).shared, n);
    const int *row = a.table.pages + (size_t)b * a.table.ld;
    const float cap = a.softcap, sl2 = cap > 0.f ? a.scale : __fmul_rn(a.scale, kLog2e);
    float q[8], o8[8] = {}, mx = -INFINITY, sum = 0.f;
    values8(a.q.dtype, r, q);
    for (int p0 = start; p0 < n; p0 += N) {
        const int p = p0 + sub;
        const uint32_t i = page_of(a.c, (uint32_t)min(p, n - 1) >> 4);
        const int page = row[i];
        const bool on = p < n && page >= 0 && page < a.c.pages;
        const size_t at = ((on ? (size_t)page : 0) * a.c.nkv + hk) * a.c.tile_bytes;
        const uint32_t off = on ? (uint32_t)p - i * (uint32_t)a.c.page_size : 0;
        float k[8], x[8];
        load_codes<CT, HD, false>(a.c.k + at, a.c.page_size, off, l * 8, k);
        load_codes<CT, HD, true>(a.c.v + at, a.c.page_size, off, l * 8, x);
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) s = __builtin_fmaf(q[e], k[e], s);
        s = __fadd_rn(s, lanes::dpp_mov<0xB1>(s));
        s = __fadd_rn(s, lanes::dpp_mov<0x4E>(s));
        s = __fadd_rn(s, lanes::dpp_mov<0x141>(s));
        if constexpr (LP >= 16) s = __fadd_rn(s, lanes::dpp_mov<0x140>(s));
        if constexpr (LP == 32) s = __fadd_rn(s, __shfl_xor(s, 16, kWave));
        s = __fmul_rn(s, sl2);
        if (cap > 0.f) s = __fmul_rn(capped(s, cap), kLog2e);
        if (!on) s = -INFINITY;
        const float top = fmaxf(mx, s), f = mx == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mx - top);
        const float w = s == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(s - top);
        mx = top;
        sum = __builtin_fmaf(sum, f, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) o8[e] = __builtin_fmaf(w, on ? x[e] : 0.f, __fmul_rn(o8[e], f));
    }
    const int subs = min(n - start, N);                // those that have had a position
    if (sub < subs) {
        *reinterpret_cast<pf4 *>(&own[sub][l * 8]) = pf4{o8[0], o8[1], o8[2], o8[3]};
        *reinterpret_cast<pf4 *>(&own[sub][l * 8 + 4]) = pf4{o8[4], o8[5], o8[6], o8[7]};
    }
    if (l == 0) {
        own_m[sub] = mx;
        own_s[sub] = sum;
    }
    __syncthreads();
    // the largest maximum, and every part's weight against it (a sum of NaN has one of NaN; one of 0 has none)
    const int used = g.pieces;
    float top = lane < used ? ms[0].x : -INFINITY;
#pragma unroll
    for (int i = 1; i < Q; ++i) {
        if (i * kWave >= used) break;
        ms[i] = g.ms[slot + min(lane + i * kWave, used - 1) * stride];
        top = fmaxf(top, ms[i].x);
    }
    float2 es[E];
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const int at = lane + i * kWave;
        es[i] = at < subs ? make_float2(own_m[min(at, N - 1)], own_s[min(at, N - 1)]) : make_float2(-INFINITY, 0.f);
        top = fmaxf(top, es[i].x);
    }
    top = lanes::wave_max(top);
    auto weight_of = [&](float2 x) { return x.y == 0.f ? 0.f : x.y != x.y ? x.y : __builtin_amdgcn_exp2f(x.x - top); };
    float f[Q], tot = 0.f;
    unsigned long long mask[Q];                        // pieces with an O
#pragma unroll
    for (int i = 0; i < Q; ++i) {
        f[i] = 0.f;
        mask[i] = 0;
        if (i * kWave >= used) continue;
        const bool on = lane + i * kWave < used && n > 0 && ms[i].y != 0.f;
        f[i] = on ? weight_of(ms[i]) : 0.f;
        tot = __builtin_fmaf(on ? ms[i].y : 0.f, f[i], tot);
        mask[i] = __ballot(on);
    }
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const float w = weight_of(es[i]);
        tot = __builtin_fmaf(es[i].y, w, tot);
        if (wid == 0 && lane + i * kWave < N) weight[lane + i * kWave] = w;
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
            for (int j = 0; j < Q; ++j)
                if (i / kWave == j) {
                    fi = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(f[j]), i % kWave));
                    on = mask[j] >> i % kWave & 1;
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
    for (int i = 0; i < subs; ++i) x = weight[i] == 0.f ? x : __builtin_fmaf(weight[i], own[i][t], x);
    store1(a.out.dtype, a.out.p, (int64_t)b * a.out.ts + (int64_t)h * a.out.hs + t, tot == 0.f ? 0.f : __fdiv_rn(x, tot));
    if (a.lse && t == 0) a.lse[slot] = lse_of(top, tot);
}

}  // namespace

bool launch_shared_join(const void *args, hipStream_t s) {
    const AttnArgs &g = *static_cast<const AttnArgs *>(args);
    const PagedAttn &a = g.a;
    const bool wide = rows_wide(a.q);
#define SPH_SHARED_JOIN(CT, HD, W)                                                                        \
    if (a.c.dtype == CT && a.c.hd == HD && (g.pieces > kManyPieces) == (W == 16))                  \
        hipLaunchKernelGGL((paged_shared_join_kernel<CT, HD, W>), dim3(g.n_heads, a.q.tokens), dim3(W * kWave), 0, s, g, wide);
#define SPH_SHARED_JOIN_HD(CT)                                                                      \
    SPH_SHARED_JOIN(CT, 64, 4) SPH_SHARED_JOIN(CT, 64, 16) SPH_SHARED_JOIN(CT, 128, 4)             \
    SPH_SHARED_JOIN(CT, 128, 16) SPH_SHARED_JOIN(CT, 256, 4) SPH_SHARED_JOIN(CT, 256, 16)
    SPH_SHARED_JOIN_HD(DT_F32) SPH_SHARED_JOIN_HD(DT_BF16) SPH_SHARED_JOIN_HD(DT_F16) SPH_SHARED_JOIN_HD(DT_Q8_0) SPH_SHARED_JOIN_HD(DT_Q4_0)
    return hip_ok(hipGetLastError(), "shared attention join launch");
}

}  // namespace sapphire
