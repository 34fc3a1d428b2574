// paged_rows.hip - rows into the paged cache and out of it, and the cache's part of a beam step.
//
// Eight dims of a row are one lane's work and four lanes make a quant block, as in the weight
// quantizer (quantize.hip), whose arithmetic this is: Q8_0: d = max|x| / 127, q = roundf(x * (1 / d));
// Q4_0: d = m / -8 with m the first x of largest |x|, q = min(15, trunc(x * (1 / d) + 8.5)); every
// product, sum and quotient rounded on its own. A block with a NaN or an infinity gets the scale NaN.
//
// Bytes bound a prompt's rows, with the vector units close behind: 8192 tokens of 8 heads of 128 dims, bf16 to Q4_0 (K and
// V, 44 MB), are written in 13.4 us and read back in 10.6 (3.3 and 4.2 TB/s; a large copy moves 4.9), 7 and 6 us of that
// being instruction issue: an element written takes 17 vector instructions (conversion, the block's largest of both signs,
// product, sum, minimum, conversion, packing, a share of the loads and addresses), one read 13. A decode step's rows (16
// tokens of a head) are one memory latency after another, position -> page -> row: 3.0 and 2.9 us.
#include <algorithm>
#include <climits>

#include "internal.h"
#include "lanes.h"
#include "paged_dev.h"

namespace sapphire {

namespace {

constexpr int kThreads = 256;

template <int CTRL>
__device__ __forceinline__ uint32_t dpp_u32(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false);
}
// over the four lanes of a quad (quad_perm [1,0,3,2], then [2,3,0,1])
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
    v = max(v, dpp_u32<0xB1>(v));
    return max(v, dpp_u32<0x4E>(v));
}
__device__ __forceinline__ int quad_max(int v) {
    v = max(v, (int)dpp_u32<0xB1>((uint32_t)v));
    return max(v, (int)dpp_u32<0x4E>((uint32_t)v));
}
__device__ __forceinline__ uint32_t quad_min(uint32_t v) {
    v = min(v, dpp_u32<0xB1>(v));
    return min(v, dpp_u32<0x4E>(v));
}

// The quad's block: its scale and this lane's eight codes (Q8_0 -127 .. 127, Q4_0 0 .. 15). As signed integers the
// words' largest is the largest positive element (NaN above infinity), as unsigned ones the negative element of
// largest magnitude.
template <int CT>
__device__ __forceinline__ float quantize8(const float (&x)[8], int lq, int (&q)[8]) {
    int up = INT_MIN;
    uint32_t down = 0;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        up = max(up, max((int)__float_as_uint(x[i]), (int)__float_as_uint(x[i + 1])));
        down = max(down, max(__float_as_uint(x[i]), __float_as_uint(x[i + 1])));
    }
    up = max(quad_max(up), 0);
    down = quad_max(down);
    down = down & 0x80000000u ? down & 0x7fffffffu : 0u;
    const uint32_t top = max((uint32_t)up, down);
    const bool bad = top >= 0x7f800000u;
    float d;
    if constexpr (CT == DT_Q8_0) {
        d = __fdiv_rn(__uint_as_float(top), 127.0f);
    } else {
        bool minus = down > (uint32_t)up;
        if (__any(down == (uint32_t)up)) {             // both signs have that magnitude: the first element's counts
            uint32_t first = ~0u;
#pragma unroll
            for (int i = 7; i >= 0; --i) {
                const uint32_t u = __float_as_uint(x[i]);
                if ((u & 0x7fffffffu) == top) first = (uint32_t)(lq * 8 + i) * 2 + (u >> 31);
            }
            first = quad_min(first);
            minus = first & 1;
        }
        d = __fmul_rn(__uint_as_float(top), minus ? 0.125f : -0.125f);
    }
    const float id = d == 0.0f ? 0.0f : __fdiv_rn(1.0f, d);
    // Adding the float below 1/2 and truncating rounds halves away from zero, the rest to nearest. Magnitudes stay
    // within the codes (Q4_0: but for the one of the other sign, 16).
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float v = __fmul_rn(x[i], id);
        if constexpr (CT == DT_Q8_0) q[i] = (int)__fadd_rn(v, copysignf(0x1.fffffep-2f, v));
        else q[i] = (int)fminf(__fadd_rn(v, 8.5f), 15.0f);
    }
    // a subnormal d has an infinite id: its products saturate, 0 * inf counts as zero
    if (__any(bad || fabsf(id) == INFINITY)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float v = __fmul_rn(x[i], id);
            if constexpr (CT == DT_Q8_0) {
                const float w = v != v ? 0.0f : fminf(fmaxf(v, -127.0f), 127.0f);
                q[i] = bad ? 0 : (int)__fadd_rn(w, copysignf(0x1.fffffep-2f, w));
            } else {
                const float w = __fadd_rn(v, 8.5f);
                q[i] = bad || w != w ? 8 : (int)fminf(fmaxf(w, 0.0f), 15.0f);
            }
        }
        if (bad) d = __uint_as_float(0x7fc00000u);
    }
    return d;
}

// The four low bytes.
__device__ __forceinline__ uint32_t bytes4(int a, int b, int c, int d) {
    const uint32_t lo = __builtin_amdgcn_perm((uint32_t)b, (uint32_t)a, 0x0c0c0400u);
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm((uint32_t)d, (uint32_t)c, 0x0c0c0400u), lo, 0x05040100u);
}

// Dims d .. d + 7 of position p into a tile (V: the V tile). The four lanes of a quad hold one block.
template <int CT, int HD, bool V>
__device__ __forceinline__ void store_codes(uint8_t *tile, uint32_t ps, uint32_t p, uint32_t d, const float (&x)[8]) {
    using T = Tile<CT, HD>;
    if constexpr (!T::kQuant) {
        if constexpr (CT == DT_F32) {
            uint8_t *a = V ? tile + p * T::ROW + d * 4 : tile + T::k_code(p, d);
            uint8_t *b = V ? a + 16 : tile + T::k_code(p, d + 4);
            *reinterpret_cast<pf4 *>(a) = pf4{x[0], x[1], x[2], x[3]};
            *reinterpret_cast<pf4 *>(b) = pf4{x[4], x[5], x[6], x[7]};
        } else {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = pack_16(CT, x[2 * i], x[2 * i + 1]);
            if constexpr (V && HD == 64) {
                *reinterpret_cast<pu2 *>(tile + T::v_run(p, d / 4)) = pu2{w[0], w[1]};
                *reinterpret_cast<pu2 *>(tile + T::v_run(p, d / 4 + 1)) = pu2{w[2], w[3]};
            } else {
                *reinterpret_cast<pu4 *>(tile + (V ? p * T::ROW + d * 2 : T::k_code(p, d))) = pu4{w[0], w[1], w[2], w[3]};
            }
        }
    } else {
        const int lq = (d >> 3) & 3;
        int q[8];
        const float scale = quantize8<CT>(x, lq, q);
        if constexpr (CT == DT_Q8_0) {
            const uint32_t lo = bytes4(q[0], q[1], q[2], q[3]), hi = bytes4(q[4], q[5], q[6], q[7]);
            if constexpr (V && HD == 64) {
                *reinterpret_cast<uint32_t *>(tile + T::v_run(p, d / 4)) = lo;
                *reinterpret_cast<uint32_t *>(tile + T::v_run(p, d / 4 + 1)) = hi;
            } else {
                uint8_t *o = tile + (V ? T::v_run(p, d / T::RUN) + d % T::RUN : T::k_code(p, d));
                *reinterpret_cast<pu2 *>(o) = pu2{lo, hi};
            }
        } else if constexpr (!V) {
            // two's complement nibbles: code - 8 is code ^ 8 in four bits
            *reinterpret_cast<uint32_t *>(tile + T::k_code(p, d)) =
                (bytes4(q[0], q[1], q[2], q[3]) | bytes4(q[4], q[5], q[6], q[7]) << 4) ^ 0x88888888u;
        } else if constexpr (HD == 256) {
            // a run is two lanes' dims: the even lane's in the low nibbles
            const uint32_t a = bytes4(q[0], q[1], q[2], q[3]), b = bytes4(q[4], q[5], q[6], q[7]);
            const uint32_t pa = dpp_u32<0xB1>(a), pb = dpp_u32<0xB1>(b);
            *reinterpret_cast<uint32_t *>(tile + T::v_run(p, d / 16) + (lq & 1) * 4) = lq & 1 ? pb | b << 4 : a | pa << 4;
        } else if constexpr (HD == 128) {
            *reinterpret_cast<uint32_t *>(tile + T::v_run(p, d / 8)) =
                bytes4(q[0], q[1], q[2], q[3]) | bytes4(q[4], q[5], q[6], q[7]) << 4;
        } else {
            *reinterpret_cast<uint16_t *>(tile + T::v_run(p, d / 4)) = (uint16_t)(bytes4(q[0], q[1], 0, 0) | bytes4(q[2], q[3], 0, 0) << 4);
            *reinterpret_cast<uint16_t *>(tile + T::v_run(p, d / 4 + 1)) = (uint16_t)(bytes4(q[4], q[5], 0, 0) | bytes4(q[6], q[7], 0, 0) << 4);
        }
        if (lq == 0) *reinterpret_cast<float *>(tile + (V ? T::v_scale(ps, p, d / 32) : T::k_scale(ps, p, d / 32))) = scale;
    }
}

// A thread's eight dims: the workgroups take the heads' rows sixteen tokens at a time, so that those of a prompt, which go
// to sixteen positions of a tile, leave whole lines to one L2 (an L2 each would write its part of every line).
struct Unit {
    int t, h, d;
};
template <int HD>
__device__ __forceinline__ Unit unit_of(int nkv) {
    constexpr int U = HD / 8, kRows = kThreads / U;            // 32, 16 or 8 rows of a workgroup
    const uint32_t row = blockIdx.x * kRows + threadIdx.x / U, g = __builtin_amdgcn_readfirstlane(row >> 4);     // one per wave
    return Unit{(int)(g / (uint32_t)nkv * 16 + (row & 15)), (int)(g % (uint32_t)nkv), (int)(threadIdx.x % U) * 8};
}
int64_t row_groups(const Rows &r, int nkv, int hd) {
    const int rows = kThreads / (hd / 8);
    return ((int64_t)(r.tokens + 15) / 16 * 16 * nkv + rows - 1) / rows;
}

// grid (row_groups). A thread takes its unit of K and of V: one look at the table, both loads under way together.
template <int CT, int HD>
__global__ __launch_bounds__(kThreads) void paged_write_kernel(PagedCache c, Rows k, Rows v, PageTable tab,
                                                               const int *__restrict__ seqs,
                                                               const int *__restrict__ positions, bool kw, bool vw) {
    const Unit u = unit_of<HD>(c.nkv);
    if (u.t >= k.tokens) return;
    const int row = seqs ? seqs[u.t] : u.t, pos = positions[u.t];
    Raw8 rk, rv;
    load8(k.dtype, kw, k.p, (int64_t)u.t * k.ts + (int64_t)u.h * k.hs + u.d, rk);
    load8(v.dtype, vw, v.p, (int64_t)u.t * v.ts + (int64_t)u.h * v.hs + u.d, rv);
    int page, off;
    if (!paged_place(c, tab, row, pos, page, off)) return;
    const size_t at = ((size_t)page * c.nkv + u.h) * c.tile_bytes;
    float x[8], y[8];
    values8(k.dtype, rk, x);
    store_codes<CT, HD, false>(c.k + at, c.page_size, off, u.d, x);
    values8(v.dtype, rv, y);
    store_codes<CT, HD, true>(c.v + at, c.page_size, off, u.d, y);
}

template <int CT, int HD>
__global__ __launch_bounds__(kThreads) void paged_read_kernel(PagedCache c, Rows k, Rows v, PageTable tab,
                                                              const int *__restrict__ seqs,
                                                              const int *__restrict__ positions, bool kw, bool vw) {
    const Unit u = unit_of<HD>(c.nkv);
    if (u.t >= k.tokens) return;
    int page, off;
    const bool there = paged_place(c, tab, seqs ? seqs[u.t] : u.t, positions[u.t], page, off);
    float x[8] = {}, y[8] = {};
    if (there) {
        const size_t at = ((size_t)page * c.nkv + u.h) * c.tile_bytes;
        load_codes<CT, HD, false>(c.k + at, c.page_size, off, u.d, x);
        load_codes<CT, HD, true>(c.v + at, c.page_size, off, u.d, y);
    }
    store8(k.dtype, kw, k.p, (int64_t)u.t * k.ts + (int64_t)u.h * k.hs + u.d, x);
    store8(v.dtype, vw, v.p, (int64_t)u.t * v.ts + (int64_t)u.h * v.hs + u.d, y);
}

// A copy, at a copy's rate: 16 rows of 26 layers (41 MB read and written) take 9 us.
// grid (rows, 2 * layers * heads): one tile's written part to the spare page; the workgroups of
// blockIdx.y 0 also write their row of the table. code_row, scale_row: bytes of a position's codes
// and scales; both parts of 16 positions are contiguous in K and V tiles alike.
__global__ __launch_bounds__(kThreads) void paged_reorder_kernel(PagedCache c, PageTable tab, const int *__restrict__ parents,
                                                                 const int *__restrict__ lengths,
                                                                 const int *__restrict__ spare, int *__restrict__ table_out,
                                                                 int *__restrict__ lengths_out, int code_row, int scale_row) {
    const int b = blockIdx.x, p = parents[b];
    const bool has = p >= 0 && p < tab.rows;
    const int64_t most = (int64_t)tab.ld * c.page_size;
    const int n = has ? (int)min((int64_t)max(lengths[p], 0), most) : 0;
    const int full = n / c.page_size, rem = n - full * c.page_size;
    const int *from = tab.pages + (size_t)(has ? p : 0) * tab.ld;
    const int dst = rem ? spare[b] : -1, src = rem ? from[full] : -1;
    const bool copy = dst >= 0 && dst < c.pages && src >= 0 && src < c.pages;
    if (blockIdx.y == 0) {
        for (int i = threadIdx.x; i < tab.ld; i += kThreads)
            table_out[(size_t)b * tab.ld + i] = i < full ? from[i] : i == full && copy ? dst : -1;
        if (threadIdx.x == 0) lengths_out[b] = n;
    }
    if (!copy) return;
    const int which = blockIdx.y & 1, lh = blockIdx.y >> 1, layer = lh / c.nkv, h = lh - layer * c.nkv;
    uint8_t *pool = (which ? c.v : c.k) + (size_t)layer * c.layer_bytes;
    const uint8_t *s = pool + ((size_t)src * c.nkv + h) * c.tile_bytes;
    uint8_t *o = pool + ((size_t)dst * c.nkv + h) * c.tile_bytes;
    const int held = (rem + 15) / 16 * 16;
    auto copy16 = [&](uint32_t at, uint32_t bytes) {
        constexpr int U = 4;                           // loads in flight per thread
        const pu4 *sp = reinterpret_cast<const pu4 *>(s + at);
        pu4 *op = reinterpret_cast<pu4 *>(o + at);
        const uint32_t m = bytes / 16;
        for (uint32_t i = threadIdx.x; i < m; i += U * kThreads) {
            pu4 w[U];
#pragma unroll
            for (int u = 0; u < U; ++u) w[u] = sp[min(i + u * kThreads, m - 1)];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (i + u * kThreads < m) op[i + u * kThreads] = w[u];
        }
    };
    copy16(0, (uint32_t)held * code_row);
    if (scale_row) copy16((uint32_t)c.page_size * code_row, (uint32_t)held * scale_row);
}

}  // namespace

#define SPH_PAGED(CALL)                                              \
    switch (c.dtype) {                                               \
        case DT_F32: SPH_PAGED_HD(CALL, DT_F32) break;               \
        case DT_BF16: SPH_PAGED_HD(CALL, DT_BF16) break;             \
        case DT_F16: SPH_PAGED_HD(CALL, DT_F16) break;               \
        case DT_Q8_0: SPH_PAGED_HD(CALL, DT_Q8_0) break;             \
        default: SPH_PAGED_HD(CALL, DT_Q4_0) break;                  \
    }
#define SPH_PAGED_HD(CALL, CT)                                       \
    if (c.hd == 64) CALL(CT, 64);                                    \
    else if (c.hd == 128) CALL(CT, 128);                             \
    else CALL(CT, 256);

int launch_paged_write(const PagedCache &c, const Rows &k, const Rows &v, const PageTable &t, const int *seqs,
                       const int *positions, hipStream_t s) {
    const dim3 grid((unsigned)row_groups(k, c.nkv, c.hd)), block(kThreads);
#define SPH_CALL(CT, HD) \
    hipLaunchKernelGGL((paged_write_kernel<CT, HD>), grid, block, 0, s, c, k, v, t, seqs, positions, rows_wide(k), rows_wide(v))
    SPH_PAGED(SPH_CALL)
#undef SPH_CALL
    return hip_ok(hipGetLastError(), "paged write launch") ? 0 : -1;
}

int launch_paged_read(const PagedCache &c, const Rows &k, const Rows &v, const PageTable &t, const int *seqs,
                      const int *positions, hipStream_t s) {
    const dim3 grid((unsigned)row_groups(k, c.nkv, c.hd)), block(kThreads);
#define SPH_CALL(CT, HD) \
    hipLaunchKernelGGL((paged_read_kernel<CT, HD>), grid, block, 0, s, c, k, v, t, seqs, positions, rows_wide(k), rows_wide(v))
    SPH_PAGED(SPH_CALL)
#undef SPH_CALL
    return hip_ok(hipGetLastError(), "paged read launch") ? 0 : -1;
}

int launch_paged_reorder(const PagedCache &c, const PageTable &t, const int *parents, const int *lengths, const int *spare,
                         int *table_out, int *lengths_out, hipStream_t s) {
    const bool quant = is_quant(c.dtype);
    const int code_row = c.dtype == DT_F32 ? 4 * c.hd : c.dtype == DT_Q8_0 ? c.hd : c.dtype == DT_Q4_0 ? c.hd / 2 : 2 * c.hd;
    hipLaunchKernelGGL(paged_reorder_kernel, dim3(t.rows, 2 * c.layers * c.nkv), dim3(kThreads), 0, s, c, t, parents,
                       lengths, spare, table_out, lengths_out, code_row, quant ? c.hd / 8 : 0);
    return hip_ok(hipGetLastError(), "paged reorder launch") ? 0 : -1;
}

}  // namespace sapphire
