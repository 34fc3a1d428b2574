// verify.hip - verification of drafted tokens: which drafts of a request the target model's probabilities keep, and the
// token behind them, from given draws.
//
// With p = softmax(l / T) of a target row and q = softmax(d / T) of a draft row, draft x with draw u stays if
// u q(x) < p(x); the first that does not is replaced by a draw from max(p - q, 0), which gives the tokens the target's own
// distribution. Borders of that draw are as close as 1 / n, so everything behind the logits is in 64 bits:
// weights 2^((l - m) c), c = log2 e / T, and their sums.
//
// Three launches: every row's (maximum, sum of weights) by chunks; the decision, made alike by every workgroup of a request
// from those, and the chunks' sums of max(p - q, 0) of the one row that it ends at; the token, within one chunk.
#include <algorithm>
#include <cmath>

#include "internal.h"
#include "lanes.h"
#include "paged_dev.h"

namespace sapphire {

namespace {

using lanes::u64_lane;
typedef unsigned long long u64;

constexpr int kWave = 64, kThreads = 256, kWaves = kThreads / kWave;
constexpr int kVec = 8;                    // pieces of four logits of a thread
constexpr int kChunk = kThreads * kVec * 4;
constexpr int kPickThreads = 1024, kPickEach = kChunk / kPickThreads;
constexpr int kMaxDrafts = 64;

struct Part {
    float m;                               // a chunk's maximum
    int pad;
    double sum;                            // of weights against it
};
struct VerifyArgs {
    const float *logits, *draft;
    int64_t ld, draft_ld;
    int n, requests, drafts, chunks;
    const int *draft_tokens, *counts;
    const float *draws;
    double c;                              // log2 e / temperature
    int *tokens, *accepted;
    Part *part;                            // [rows][chunks]: the target's rows, then the draft's
    double *rest;                          // [requests][chunks]: sums of max(p - q, 0)
    u64 *key;                              // greedy: [target rows][chunks], in place of part
};

// 2^y for y <= 0 (or NaN, which stays one). 2^f, f in [-1/2, 1/2], by the polynomial through the Chebyshev points of degree 8:
// off by 1.1e-12 relative, far below the 4e-6 between borders of a flat row of 2^18 tokens. (fp64 fused products run at the
// rate of fp32 ones here.)
__device__ __forceinline__ double exp2_64(double y) {
    y = fmax(y, -1100.0);                  // 0, as 2^-1074 is the smallest
    const double n = rint(y), f = y - n;
    double r = 1.3255224887502117e-06;
    r = __builtin_fma(r, f, 1.531007940254368e-05);
    r = __builtin_fma(r, f, 0.0001540345585240991);
    r = __builtin_fma(r, f, 0.0013333450567999414);
    r = __builtin_fma(r, f, 0.009618129159402628);
    r = __builtin_fma(r, f, 0.05550410941205934);
    r = __builtin_fma(r, f, 0.2402265069581299);
    r = __builtin_fma(r, f, 0.6931471805459335);
    r = __builtin_fma(r, f, 1.0);
    return ldexp(r, (int)n);
}
__device__ __forceinline__ float as_logit(float x) { return x != x ? -INFINITY : x; }

// Weights against the maximum m: where that is infinite, the entries that reach it have 1 and the others 0.
struct Weight {
    double c, m64;
    float m;
    bool finite;
    __device__ __forceinline__ Weight(double c, float m) : c(c), m64(m), m(m), finite(fabsf(m) < INFINITY) {}
    __device__ __forceinline__ double operator()(float x) const {
        if (!finite) return x == m ? 1.0 : 0.0;
        // (one fused product less m c would be off by what m c is rounded by)
        return exp2_64(((double)x - m64) * c);
    }
};

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
    for (int off = 1; off < kWave; off *= 2) v += __shfl_xor(v, off, kWave);
    return v;
}
__device__ __forceinline__ double wave_scan64(double v, int lane) {        // inclusive
#pragma unroll
    for (int off = 1; off < kWave; off *= 2) {
        const double b = __shfl_up(v, off, kWave);
        v += lane >= off ? b : 0.0;
    }
    return v;
}

// Four logits from index i of a row (a multiple of four from 16-byte aligned memory where `i` is inside), -inf outside [0, n).
__device__ __forceinline__ pf4 load_logits(const float *row, int i, int n) {
    pf4 x = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
    if (i >= 0 && i + 4 <= n) {
        x = *reinterpret_cast<const pf4 *>(row + i);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (i + e >= 0 && i + e < n) x[e] = row[i + e];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = as_logit(x[e]);
    return x;
}
// Where a row's pieces of four start: 0 to 3 elements ahead of it.
__device__ __forceinline__ int ahead(const float *row) { return (int)(reinterpret_cast<uintptr_t>(row) >> 2 & 3); }

__device__ __forceinline__ int count_of(const VerifyArgs &g, int r) { return g.counts ? min(max(g.counts[r], 0), g.drafts) : g.drafts; }
// The logits of row y of the partials, or null if no draft of the request reaches it.
__device__ __forceinline__ const float *row_of(const VerifyArgs &g, int y) {
    const int targets = g.requests * (g.drafts + 1);
    if (y < targets) {
        const int r = y / (g.drafts + 1);
        return y - r * (g.drafts + 1) <= count_of(g, r) ? g.logits + (size_t)y * g.ld : nullptr;
    }
    y -= targets;
    const int r = y / g.drafts;
    return y - r * g.drafts < count_of(g, r) ? g.draft + (size_t)y * g.draft_ld : nullptr;
}

// Larger logits, then lower indices, have larger keys.
__device__ __forceinline__ u64 key_of(float x, uint32_t i) {
    const uint32_t u = __float_as_uint(x + 0.0f), o = u & 0x80000000u ? ~u : u | 0x80000000u;
    return (u64)o << 32 | (uint32_t)~i;
}

// grid (chunks, rows): the chunk's maximum and sum of weights, or its best key (GREEDY).
template <bool GREEDY>
__global__ __launch_bounds__(kThreads) void verify_rows_kernel(VerifyArgs g) {
    __shared__ double part[kWaves];
    __shared__ float top[kWaves];
    __shared__ u64 best[kWaves];
    const float *row = row_of(g, blockIdx.y);
    if (!row) return;
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wid = tid / kWave;
    const int i0 = blockIdx.x * kChunk - ahead(row);
    pf4 x[kVec];
#pragma unroll
    for (int v = 0; v < kVec; ++v) x[v] = load_logits(row, i0 + (v * kThreads + tid) * 4, g.n);
    if constexpr (GREEDY) {
        u64 k = 0;
#pragma unroll
        for (int v = 0; v < kVec; ++v)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int i = i0 + (v * kThreads + tid) * 4 + e;
                const u64 o = i >= 0 && i < g.n ? key_of(x[v][e], (uint32_t)i) : 0;
                k = o > k ? o : k;
            }
        k = lanes::u64_wave_max(k);
        if (lane == 0) best[wid] = k;
        __syncthreads();
        if (tid == 0) {
#pragma unroll
            for (int w = 1; w < kWaves; ++w) k = best[w] > k ? best[w] : k;
            g.key[(size_t)blockIdx.y * g.chunks + blockIdx.x] = k;
        }
    } else {
        float m = -INFINITY;
#pragma unroll
        for (int v = 0; v < kVec; ++v) m = fmaxf(m, fmaxf(fmaxf(x[v][0], x[v][1]), fmaxf(x[v][2], x[v][3])));
        m = lanes::wave_max(m);
        if (lane == 0) top[wid] = m;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWaves; ++w) m = fmaxf(m, top[w]);
        const Weight weight(g.c, m);
        double s[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
        for (int v = 0; v < kVec; ++v)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int i = i0 + (v * kThreads + tid) * 4 + e;
                // (what lies outside is -inf, which counts where a whole chunk is)
                s[e] += weight.finite || (i >= 0 && i < g.n) ? weight(x[v][e]) : 0.0;
            }
        const double sum = wave_sum64((s[0] + s[1]) + (s[2] + s[3]));
        if (lane == 0) part[wid] = sum;
        __syncthreads();
        if (tid == 0) g.part[(size_t)blockIdx.y * g.chunks + blockIdx.x] = Part{m, 0, (part[0] + part[1]) + (part[2] + part[3])};
    }
}

// A whole row's maximum and sum from its chunks', by one wave; the same in every lane.
__device__ __forceinline__ void row_total(const VerifyArgs &g, int y, float &m, double &sum) {
    const int lane = threadIdx.x & (kWave - 1);
    const Part *p = g.part + (size_t)y * g.chunks;
    m = -INFINITY;
    for (int i = lane; i < g.chunks; i += kWave) m = fmaxf(m, p[i].m);
    m = lanes::wave_max(m);
    const Weight weight(g.c, m);
    double s = 0.0;
    for (int i = lane; i < g.chunks; i += kWave) s += p[i].sum * weight(p[i].m);
    sum = wave_sum64(s);
}

struct Row {
    float m;
    double sum;
};
// The decision of request r by all waves of a workgroup: how many drafts stay, and the rows that the token behind them comes from.
__device__ __forceinline__ int decide(const VerifyArgs &g, int r, Row &p, Row &q) {
    __shared__ Row rows[2 * kMaxDrafts + 1];   // the target's, then the draft's
    __shared__ int stays[kMaxDrafts];
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wid = tid / kWave, waves = blockDim.x / kWave;
    const int count = count_of(g, r), targets = g.requests * (g.drafts + 1);
    const int jobs = count + 1 + (g.draft ? count : 0);
    for (int j = wid; j < jobs; j += waves) {
        Row t;
        row_total(g, j <= count ? r * (g.drafts + 1) + j : targets + r * g.drafts + j - count - 1, t.m, t.sum);
        if (lane == 0) rows[j <= count ? j : kMaxDrafts + 1 + j - count - 1] = t;
    }
    __syncthreads();
    for (int i = tid; i < count; i += blockDim.x) {
        const int x = g.draft_tokens[(size_t)r * g.drafts + i];
        bool ok = false;
        if (x >= 0 && x < g.n) {
            const Row a = rows[i], b = rows[kMaxDrafts + 1 + i];
            const double u = fmin(fmax((double)g.draws[(size_t)r * (g.drafts + 1) + i], 0.0), 1.0);
            const double px = Weight(g.c, a.m)(as_logit(g.logits[((size_t)r * (g.drafts + 1) + i) * g.ld + x]));
            if (!g.draft) ok = u * a.sum < px;
            else ok = u * Weight(g.c, b.m)(as_logit(g.draft[((size_t)r * g.drafts + i) * g.draft_ld + x])) * a.sum < px * b.sum;
        }
        stays[i] = ok;
    }
    __syncthreads();
    int a = 0;
    while (a < count && stays[a]) ++a;
    p = rows[a];
    q = rows[kMaxDrafts + 1 + min(a, kMaxDrafts - 1)];
    return a;
}

// What is left of token i's probability where the drafts end: max(p - q, 0), or p behind the last draft.
struct Rest {
    Weight wp, wq;
    double ip, iq;
    int mode, drafted;                     // mode 0: p; 1: p less q; 2: p but for the drafted token
    __device__ __forceinline__ Rest(const VerifyArgs &g, int r, int a, Row p, Row q)
        : wp(g.c, p.m), wq(g.c, q.m), ip(1.0 / p.sum), iq(1.0 / q.sum), mode(a >= count_of(g, r) ? 0 : g.draft ? 1 : 2), drafted(-1) {
        if (mode == 2) drafted = g.draft_tokens[(size_t)r * g.drafts + a];
    }
    __device__ __forceinline__ double operator()(float lp, float lq, int i) const {
        const double p = wp(lp) * ip;
        if (mode == 1) return fmax(p - wq(lq) * iq, 0.0);
        return mode == 2 && i == drafted ? 0.0 : p;
    }
};

// grid (chunks, requests). Behind the last draft the sums are p's own, which the first launch made.
__global__ __launch_bounds__(kThreads) void verify_rest_kernel(VerifyArgs g) {
    __shared__ double part[kWaves];
    const int r = blockIdx.y, tid = threadIdx.x, lane = tid & (kWave - 1), wid = tid / kWave;
    Row p, q;
    const int a = decide(g, r, p, q);
    const Rest rest(g, r, a, p, q);
    if (rest.mode == 0) return;
    const float *row = g.logits + ((size_t)r * (g.drafts + 1) + a) * g.ld;
    const float *other = rest.mode == 1 ? g.draft + ((size_t)r * g.drafts + a) * g.draft_ld : row;
    const int i0 = blockIdx.x * kChunk - ahead(row);
    double s = 0.0;
#pragma unroll 8
    for (int j = tid; j < kChunk; j += kThreads) {
        const int i = i0 + j;
        if (i >= 0 && i < g.n) s += rest(as_logit(row[i]), as_logit(other[i]), i);
    }
    s = wave_sum64(s);
    if (lane == 0) part[wid] = s;
    __syncthreads();
    if (tid == 0) g.rest[(size_t)r * g.chunks + blockIdx.x] = (part[0] + part[1]) + (part[2] + part[3]);
}

// grid (requests): the token, and the outputs.
__global__ __launch_bounds__(kPickThreads) void verify_pick_kernel(VerifyArgs g) {
    constexpr int kW = kPickThreads / kWave;
    __shared__ double part[kW], left;
    __shared__ int chunk, token, late, whole;
    const int r = blockIdx.x, tid = threadIdx.x, lane = tid & (kWave - 1), wid = tid / kWave;
    Row p, q;
    const int a = decide(g, r, p, q);
    Rest rest(g, r, a, p, q);
    if (wid == 0) {
        // the chunk in which the running sum passes the draw's share of the whole; past the last one by a rounding: the last
        // that has any
        const double *sums = g.rest + (size_t)r * g.chunks;
        const Part *own = g.part + ((size_t)r * (g.drafts + 1) + a) * g.chunks;
        bool of_p = rest.mode == 0;
        auto sum_of = [&](int i) { return i >= g.chunks ? 0.0 : of_p ? own[i].sum * rest.wp(own[i].m) * rest.ip : sums[i]; };
        double all = 0.0;
        auto total = [&]() {
            all = 0.0;
            for (int i0 = 0; i0 < g.chunks; i0 += kWave) all += wave_sum64(sum_of(i0 + lane));
        };
        total();
        if (all == 0.0) {                              // p and q are the same, or all of p is on the drafted token: p itself
            of_p = true;
            total();
        }
        const double u = fmin(fmax((double)g.draws[(size_t)r * (g.drafts + 1) + g.drafts], 0.0), 1.0);
        double run = 0.0;
        int at = -1, last = 0;
        double need = 0.0;
        for (int i0 = 0; i0 < g.chunks && at < 0; i0 += kWave) {
            const double s = sum_of(i0 + lane), upto = run + wave_scan64(s, lane);
            const u64 past = __ballot(i0 + lane < g.chunks && upto > u * all), some = __ballot(s > 0.0);
            if (some) last = i0 + 63 - __builtin_clzll(some);
            if (past) {
                const int l = __builtin_ctzll(past);
                at = i0 + l;
                need = u * all - __shfl(upto - s, l, kWave);
            }
            run = __shfl(upto, kWave - 1, kWave);
        }
        if (lane == 0) {
            chunk = at < 0 ? last : at;
            left = at < 0 ? INFINITY : need;
            token = 1 << 30;
            late = -1;
            whole = of_p;
        }
    }
    __syncthreads();
    if (whole) rest.mode = 0;
    const float *row = g.logits + ((size_t)r * (g.drafts + 1) + a) * g.ld;
    const float *other = rest.mode == 1 ? g.draft + ((size_t)r * g.drafts + a) * g.draft_ld : row;
    const int i0 = chunk * kChunk - ahead(row) + tid * kPickEach;
    double w[kPickEach], sum = 0.0;
#pragma unroll
    for (int j = 0; j < kPickEach; ++j) {
        w[j] = i0 + j >= 0 && i0 + j < g.n ? rest(as_logit(row[i0 + j]), as_logit(other[i0 + j]), i0 + j) : 0.0;
        sum += w[j];
    }
    const double upto = wave_scan64(sum, lane);
    if (lane == kWave - 1) part[wid] = upto;
    __syncthreads();
    double run = upto - sum;
    for (int v = 0; v < wid; ++v) run += part[v];
    int first = 1 << 30, some = -1;
#pragma unroll
    for (int j = 0; j < kPickEach; ++j) {
        run += w[j];
        if (w[j] > 0.0) {
            some = i0 + j;
            if (run > left) first = min(first, i0 + j);
        }
    }
    if (first < 1 << 30) atomicMin(&token, first);
    if (some >= 0) atomicMax(&late, some);
    __syncthreads();
    const int pick = token < 1 << 30 ? token : max(late, 0);
    for (int i = tid; i <= g.drafts; i += kPickThreads)
        g.tokens[(size_t)r * (g.drafts + 1) + i] = i < a ? g.draft_tokens[(size_t)r * g.drafts + i] : i == a ? pick : -1;
    if (tid == 0) g.accepted[r] = a;
}

// grid (requests): drafts stay while they are the target's best tokens.
__global__ __launch_bounds__(kThreads) void verify_greedy_kernel(VerifyArgs g) {
    __shared__ int best[kMaxDrafts + 1];
    const int r = blockIdx.x, tid = threadIdx.x, lane = tid & (kWave - 1), wid = tid / kWave, count = count_of(g, r);
    for (int j = wid; j <= count; j += kWaves) {
        u64 k = 0;
        for (int i = lane; i < g.chunks; i += kWave) {
            const u64 o = g.key[((size_t)r * (g.drafts + 1) + j) * g.chunks + i];
            k = o > k ? o : k;
        }
        k = lanes::u64_wave_max(k);
        if (lane == 0) best[j] = (int)~(uint32_t)k;
    }
    __syncthreads();
    const int *drafted = g.draft_tokens + (size_t)r * g.drafts;
    int a = 0;
    while (a < count && drafted[a] == best[a]) ++a;
    for (int i = tid; i <= g.drafts; i += kThreads) g.tokens[(size_t)r * (g.drafts + 1) + i] = i <= a ? best[i] : -1;
    if (tid == 0) g.accepted[r] = a;
}

// pieces of four start up to three elements ahead of a row
int chunks_of(int n) { return (n + 3 + kChunk - 1) / kChunk; }

}  // namespace

size_t verify_workspace_bytes(int n, int requests, int drafts) {
    const size_t chunks = (size_t)chunks_of(n), rows = (size_t)requests * (2 * drafts + 1);
    return chunks * (rows * sizeof(Part) + (size_t)requests * sizeof(double));
}

int launch_verify(const float *logits, int ld, const float *draft_logits, int draft_ld, int n, int requests, int drafts,
                  const int *draft_tokens, const int *counts, float temperature, const float *draws, int *tokens, int *accepted,
                  void *ws, hipStream_t s) {
    VerifyArgs g;
    g.logits = logits;
    g.draft = draft_logits;
    g.ld = ld;
    g.draft_ld = draft_ld;
    g.n = n;
    g.requests = requests;
    g.drafts = drafts;
    g.chunks = chunks_of(n);
    g.draft_tokens = draft_tokens;
    g.counts = counts;
    g.draws = draws;
    g.c = temperature > 0.0f ? 1.4426950408889634 / (double)temperature : 0.0;
    g.tokens = tokens;
    g.accepted = accepted;
    const int targets = requests * (drafts + 1);
    if (!(temperature > 0.0f)) {
        g.key = static_cast<u64 *>(ws);
        hipLaunchKernelGGL(verify_rows_kernel<true>, dim3(g.chunks, targets), dim3(kThreads), 0, s, g);
        hipLaunchKernelGGL(verify_greedy_kernel, dim3(requests), dim3(kThreads), 0, s, g);
        return hip_ok(hipGetLastError(), "verify launch") ? 0 : -1;
    }
    const int rows = targets + (draft_logits ? requests * drafts : 0);
    g.part = static_cast<Part *>(ws);
    g.rest = reinterpret_cast<double *>(g.part + (size_t)rows * g.chunks);
    hipLaunchKernelGGL(verify_rows_kernel<false>, dim3(g.chunks, rows), dim3(kThreads), 0, s, g);
    hipLaunchKernelGGL(verify_rest_kernel, dim3(g.chunks, requests), dim3(kThreads), 0, s, g);
    hipLaunchKernelGGL(verify_pick_kernel, dim3(requests), dim3(kPickThreads), 0, s, g);
    return hip_ok(hipGetLastError(), "verify launch") ? 0 : -1;
}

}  // namespace sapphire
