// rope_rows.hip - rotary positions of many rows (rope.c:99-117; in pairs positional_encoding.c:95-99)
// from frequencies instead of tables.
//
// A workgroup takes a few tokens, or some heads of one: it forms the tokens' angles once into LDS (64-bit
// product and reduction to half a turn, then fp32 sine and cosine), and its threads turn 16 bytes of
// each half at a time, two such pieces on their way at once and the first ones while the angles are formed.
//
// Bytes bound it: 8192 tokens of 40 heads of 128 dims, bf16, half of them turned (168 MB read and written) take 36.8 us,
// 4.6 TB/s, a copy's rate; with one piece at a time and none ahead it was 39.5. One token's heads: 2.3 us, a launch.
#include <algorithm>

#include "paged_dev.h"

namespace sapphire {

namespace {

constexpr int kThreads = 256;
constexpr int kAngles = 1024;              // (token, pair) angles of a workgroup at most

struct RopeArgs {
    Rows x, y;
    const int *positions;
    const double *freqs;
    int rot, tok, heads;                   // tokens and heads of a workgroup
    float magnitude;
};

// N elements: 16 bytes, or a single one.
template <int DT, bool WIDE>
struct Piece {
    static constexpr int N = WIDE ? (DT == DT_F32 ? 4 : 8) : 1;
    float v[N];
    __device__ __forceinline__ void load(const uint8_t *p, int64_t at) {
        if constexpr (DT == DT_F32) {
            const float *f = reinterpret_cast<const float *>(p) + at;
            if constexpr (WIDE) {
                const pf4 w = *reinterpret_cast<const pf4 *>(f);
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = w[i];
            } else {
                v[0] = *f;
            }
        } else {
            const uint16_t *f = reinterpret_cast<const uint16_t *>(p) + at;
            if constexpr (WIDE) {
                const pu4 w = *reinterpret_cast<const pu4 *>(f);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    v[2 * i] = from_16(DT, w[i] & 0xffffu);
                    v[2 * i + 1] = from_16(DT, w[i] >> 16);
                }
            } else {
                v[0] = from_16(DT, *f);
            }
        }
    }
    __device__ __forceinline__ void store(uint8_t *p, int64_t at) const {
        if constexpr (DT == DT_F32) {
            float *f = reinterpret_cast<float *>(p) + at;
            if constexpr (WIDE) *reinterpret_cast<pf4 *>(f) = pf4{v[0], v[1], v[2], v[3]};
            else *f = v[0];
        } else {
            uint16_t *f = reinterpret_cast<uint16_t *>(p) + at;
            if constexpr (WIDE) {
                pu4 w;
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = pack_16(DT, v[2 * i], v[2 * i + 1]);
                *reinterpret_cast<pu4 *>(f) = w;
            } else {
                *f = (uint16_t)to_16(DT, v[0]);
            }
        }
    }
};

// y0 = x0 c - x1 s, y1 = x1 c + x0 s
__device__ __forceinline__ void turn(float &a, float &b, float2 cs) {
    const float x0 = a, x1 = b;
    a = __builtin_fmaf(x0, cs.x, -__fmul_rn(x1, cs.y));
    b = __builtin_fmaf(x1, cs.x, __fmul_rn(x0, cs.y));
}

// grid (token groups, head groups)
template <int DT, bool PAIRS, bool WIDE>
__global__ __launch_bounds__(kThreads) void rope_rows_kernel(RopeArgs a) {
    using P = Piece<DT, WIDE>;
    constexpr bool ONE = PAIRS && WIDE;    // a piece holds both of a pair
    constexpr int U = 2;                   // pieces (or pairs of them) of a thread on their way together
    __shared__ float2 cs[kAngles];
    const int half = a.rot / 2, t0 = blockIdx.x * a.tok, nt = min(a.tok, a.x.tokens - t0);
    const int h0 = blockIdx.y * a.heads, nh = min(a.heads, a.x.heads - h0);
    const bool same = a.x.p == a.y.p;      // the remaining dims are there already
    // units of a head: its turning pieces, then the copied ones. A thread keeps its unit and steps over the heads and
    // tokens, `across` at a time.
    const int turning = PAIRS ? (WIDE ? a.rot / P::N : half) : half / P::N;
    const int units = turning + (same ? 0 : (a.x.hd - a.rot) / P::N), across = max(1, kThreads / units);
    const int row = threadIdx.x / units;
    int unit = row < across ? (int)threadIdx.x - row * units : units, t, h;
    int64_t xi, yi;
    P p[U], q[ONE ? 1 : U];
    int of[U];                             // a piece's token, nt where there is none
    int64_t at[U];
    // a unit's first and second dims, and of a pair's second one
    auto dims = [&](int &d0, int &d1) {
        const int d = unit * P::N;
        d0 = unit >= turning ? a.rot + (unit - turning) * P::N : ONE || !PAIRS ? d : 2 * d;
        d1 = PAIRS ? 2 * d + 1 : d + half;
    };
    auto start = [&]() {
        t = 0;
        h = row;
        while (h >= nh) {
            h -= nh;
            ++t;
        }
        xi = (int64_t)(t0 + t) * a.x.ts + (int64_t)(h0 + h) * a.x.hs;
        yi = (int64_t)(t0 + t) * a.y.ts + (int64_t)(h0 + h) * a.y.hs;
    };
    auto fetch = [&]() {
        int d0, d1;
        dims(d0, d1);
#pragma unroll
        for (int i = 0; i < U; ++i) {
            of[i] = min(t, nt);
            at[i] = yi;
            if (t >= nt) continue;
            p[i].load(a.x.p, xi + d0);
            if constexpr (!ONE)
                if (unit < turning) q[i].load(a.x.p, xi + d1);
            h += across;
            xi += across * a.x.hs;
            yi += across * a.y.hs;
            while (h >= nh) {
                h -= nh;
                ++t;
                xi += a.x.ts - nh * a.x.hs;
                yi += a.y.ts - nh * a.y.hs;
            }
        }
    };
    if (unit < units) {
        start();
        fetch();
    }
    for (int i = threadIdx.x; i < nt * half; i += kThreads) {
        const int k = i / half, j = i - k * half;
        const double turns = (double)a.positions[t0 + k] * a.freqs[j] * 0.15915494309189533577;
        const float th = (float)((turns - __builtin_rint(turns)) * 6.2831853071795864769);
        float s, c;
        sincosf(th, &s, &c);
        cs[i] = make_float2(__fmul_rn(c, a.magnitude), __fmul_rn(s, a.magnitude));
    }
    __syncthreads();
    while (unit < units) {
        int d0, d1;
        dims(d0, d1);
#pragma unroll
        for (int i = 0; i < U; ++i) {
            if (of[i] >= nt) continue;
            const float2 *w = cs + of[i] * half;
            if (unit < turning) {
                if constexpr (ONE) {
#pragma unroll
                    for (int e = 0; e < P::N / 2; ++e) turn(p[i].v[2 * e], p[i].v[2 * e + 1], w[d0 / 2 + e]);
                } else {
#pragma unroll
                    for (int e = 0; e < P::N; ++e) turn(p[i].v[e], q[i].v[e], w[unit * P::N + e]);
                    q[i].store(a.y.p, at[i] + d1);
                }
            }
            p[i].store(a.y.p, at[i] + d0);
        }
        if (t >= nt) {                     // the next unit, of heads of more than kThreads
            unit += kThreads;
            if (unit < units) start();
        }
        if (unit < units) fetch();
    }
}

}  // namespace

int launch_rope_rows(const Rows &x, const Rows &y, const int *positions, const double *freqs, int rot, bool interleaved,
                     float magnitude, hipStream_t s) {
    RopeArgs a{x, y, positions, freqs, rot, 1, x.heads, magnitude};
    const int vec = x.dtype == DT_F32 ? 4 : 8;
    const bool wide = rows_wide(x) && rows_wide(y) && x.hd % vec == 0 && (interleaved ? rot : rot / 2) % vec == 0;
    // About four workgroups per CU where the rows suffice, of one to sixteen 16-byte pieces per thread
    // (single elements: as many as the threads take in turn): several tokens, or some heads of one.
    const int64_t units = std::max(1, x.hd / (wide ? 2 * vec : 2)), all = (int64_t)x.tokens * x.heads * units;
    const int64_t want = std::min<int64_t>(16 * kThreads, std::max<int64_t>(kThreads, all / 1024));
    if (x.heads * units >= want) {
        a.heads = (int)std::max<int64_t>(1, want / units);
    } else {
        a.tok = (int)std::max<int64_t>(1, std::min<int64_t>(want / (x.heads * units), kAngles / (rot / 2)));
    }
    const dim3 grid((unsigned)((x.tokens + a.tok - 1) / a.tok), (unsigned)((x.heads + a.heads - 1) / a.heads)), block(kThreads);
#define SPH_ROPE(DT, PAIRS, WIDE) \
    if (x.dtype == DT && interleaved == PAIRS && wide == WIDE) hipLaunchKernelGGL((rope_rows_kernel<DT, PAIRS, WIDE>), grid, block, 0, s, a);
#define SPH_ROPE_DT(DT) SPH_ROPE(DT, false, false) SPH_ROPE(DT, false, true) SPH_ROPE(DT, true, false) SPH_ROPE(DT, true, true)
    SPH_ROPE_DT(DT_F32) SPH_ROPE_DT(DT_BF16) SPH_ROPE_DT(DT_F16)
    return hip_ok(hipGetLastError(), "rope rows launch") ? 0 : -1;
}

}  // namespace sapphire
