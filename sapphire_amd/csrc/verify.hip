// verify.hip - verification of drafted tokens: which drafts of a request the target model's probabilities keep, and the
// token behind them, from given draws.
//
// With p = softmax(l / T) of a target row and q = softmax(d / T) of a draft row, draft x with draw u stays if
// u q(x) < p(x); the first that does not is replaced by a draw from max(p - q, 0), which gives the tokens the target's own
// distribution. Borders of that draw are as close as 1 / n, so everything behind the logits is in 64 bits:
// weights 2^((l - m) c), c = log2 e / T, and their sums.
//
// Two launches: every row's (maximum, sum of weights) by units of 2048 logits; then the decision, made alike by every
// workgroup of a request from those, the units' sums of max(p - q, 0) of the one row that it ends at, and, by the workgroup
// that is the last to write its sums, the token, within one unit.
//
// 16 requests of 5 drafts over 262144 tokens, both models' logits (185 MB): 68 us for a call. The first launch, 39.1 us at 4.7
// TB/s, has as much vector work in 64 bits (16.5 million instructions: 26 us at full clock) as loads, and the two overlap in
// part. The second, 31.9 us, is a chain: the rows' sums from the units', the decision, three steps of logits in turn, the count of
// workgroups, and two scans by the last one. One request of 3 drafts over 4096 tokens: 13.6 us, 4.9 and 8.8 on the GPU.
// Greedy, the target's 100 MB of the first: 22 us, 18.1 and 4.1.
#include <algorithm>
#include <climits>
#include <cmath>

#include "internal.h"
#include "lanes.h"
#include "paged_dev.h"

namespace sapphire {

namespace {

using lanes::u64_lane;
typedef unsigned long long u64;

constexpr int kWave = 64, kThreads = 256, kWaves = kThreads / kWave;
constexpr int kVec = 8;                    // pieces of four logits of a lane
constexpr int kUnit = kWave * kVec * 4;    // a wave's logits
// The second launch: few workgroups, each with a chain of steps, so its waves take a quarter of a unit each.
constexpr int kThreads2 = 512, kWaves2 = kThreads2 / kWave;
constexpr int kQuarters = 4, kUnits2 = kWaves2 / kQuarters, kVec2 = kVec / kQuarters;
constexpr int kEach = kUnit / kThreads2;   // a thread's logits, where a workgroup goes over a unit
constexpr int kMaxDrafts = 64;
constexpr int kPerUnit = 2, kFill = 256 * kPerUnit;    // workgroups of the second launch on a compute unit, and at once

struct Part {
    float m;                               // a unit's maximum
    int pad;
    double sum;                            // of weights against it
};
struct VerifyArgs {
    const float *logits, *draft;
    int64_t ld, draft_ld;
    int n, requests, drafts, units;
    const int *draft_tokens, *counts;
    const float *draws;
    double c;                              // log2 e / temperature
    int *tokens, *accepted;
    Part *part;                            // [rows][units]: the target's rows, then the draft's
    double *rest;                          // [requests][units]: sums of max(p - q, 0)
    unsigned *done;                        // [requests]: workgroups that have written theirs
    u64 *key;                              // greedy: [target rows][units], in place of the three
};

// 2^y for -1000 <= y <= 0. 2^f, f in [-1/2, 1/2], by the polynomial through the Chebyshev points of degree 8: off by 1.1e-12
// relative, far below the 4e-6 between borders of a flat row of 2^18 tokens. The sum with 1.5 * 2^52 leaves y's nearest
// whole number in its low word, and the exponent takes it as it is: rounding, conversion and scaling instructions run at a
// quarter of the fused products' rate.
__device__ __forceinline__ double exp2_64(double y) {
    const double t = y + 6755399441055744.0, f = y - (t - 6755399441055744.0);
    double r = 1.3255224887502117e-06;
    r = __builtin_fma(r, f, 1.531007940254368e-05);
    r = __builtin_fma(r, f, 0.0001540345585240991);
    r = __builtin_fma(r, f, 0.0013333450567999414);
    r = __builtin_fma(r, f, 0.009618129159402628);
    r = __builtin_fma(r, f, 0.05550410941205934);
    r = __builtin_fma(r, f, 0.2402265069581299);
    r = __builtin_fma(r, f, 0.6931471805459335);
    r = __builtin_fma(r, f, 1.0);
    return __hiloint2double(__double2hiint(r) + (__double2loint(t) << 20), __double2loint(r));
}
__device__ __forceinline__ double draw_of(float u) { return fmin(fmax((double)u, 0.0), 1.0); }
__device__ __forceinline__ float as_logit(float x) { return fmaxf(x, -INFINITY); }

// Weights against the maximum m: where that is infinite, the entries that reach it have 1 and the others 0.
struct Weight {
    double c, m64;
    float m;
    bool finite;
    __device__ __forceinline__ Weight(double c, float m) : c(c), m64(m), m(m), finite(fabsf(m) < INFINITY) {}
    // (a fused product less m c would be off by what m c is rounded by)
    __device__ __forceinline__ double log2(float x) const { return ((double)x - m64) * c; }
    // for sums, in which 2^-1000 is nothing
    __device__ __forceinline__ double summand(float x) const { return exp2_64(fmax(log2(x), -1000.0)); }
    __device__ __forceinline__ double of(float x) const {
        const double y = log2(x), w = exp2_64(fmax(y, -1000.0));
        return y < -1000.0 ? 0.0 : w;
    }
    __device__ __forceinline__ double operator()(float x) const { return finite ? of(x) : x == m ? 1.0 : 0.0; }
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
    pf4 x;
    if (i >= 0 && i + 4 <= n) {
        x = *reinterpret_cast<const pf4 *>(row + i);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = row[min(max(i + e, 0), n - 1)];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = i + e >= 0 && i + e < n ? x[e] : -INFINITY;
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

// grid (four units, rows): a unit's maximum and sum of weights, or its best key (GREEDY), by one wave.
template <bool GREEDY>
__global__ __launch_bounds__(kThreads) void verify_rows_kernel(VerifyArgs g) {
    const int lane = threadIdx.x & (kWave - 1), unit = blockIdx.x * kWaves + threadIdx.x / kWave;
    const float *row = row_of(g, blockIdx.y);
    if (!GREEDY && blockIdx.x == 0 && threadIdx.x == 0 && (int)blockIdx.y < g.requests) g.done[blockIdx.y] = 0;
    if (!row || unit >= g.units) return;
    const int i0 = unit * kUnit - ahead(row) + lane * 4;
    pf4 x[kVec];
#pragma unroll
    for (int v = 0; v < kVec; ++v) x[v] = load_logits(row, i0 + v * kWave * 4, g.n);
    if constexpr (GREEDY) {
        u64 k = 0;
#pragma unroll
        for (int v = 0; v < kVec; ++v)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int i = i0 + v * kWave * 4 + e;
                const u64 o = i >= 0 && i < g.n ? key_of(x[v][e], (uint32_t)i) : 0;
                k = o > k ? o : k;
            }
        k = lanes::u64_wave_max(k);
        if (lane == 0) g.key[(size_t)blockIdx.y * g.units + unit] = k;
    } else {
        float m = -INFINITY;
#pragma unroll
        for (int v = 0; v < kVec; ++v) m = fmaxf(m, fmaxf(fmaxf(x[v][0], x[v][1]), fmaxf(x[v][2], x[v][3])));
        m = lanes::wave_max(m);
        const Weight weight(g.c, m);
        double s[4] = {0.0, 0.0, 0.0, 0.0};
        if (weight.finite) {
#pragma unroll
            for (int v = 0; v < kVec; ++v)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[e] += weight.summand(x[v][e]);
        } else {                                       // (what lies outside is -inf, which may be the maximum)
#pragma unroll
            for (int v = 0; v < kVec; ++v)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int i = i0 + v * kWave * 4 + e;
                    s[e] += i >= 0 && i < g.n && x[v][e] == m ? 1.0 : 0.0;
                }
        }
        const double sum = wave_sum64((s[0] + s[1]) + (s[2] + s[3]));
        if (lane == 0) g.part[(size_t)blockIdx.y * g.units + unit] = Part{m, 0, sum};
    }
}

// A whole row's maximum and sum from its units', by sixteen lanes; the same in each. (Ten loads of a lane under way together:
// one trip for rows of up to 2^18.)
__device__ __forceinline__ void row_total(const VerifyArgs &g, int y, float &m, double &sum) {
    constexpr int B = 10;
    const Part *p = g.part + (size_t)y * g.units;
    m = -INFINITY;
    sum = 0.0;
    for (int i0 = threadIdx.x & 15; i0 < g.units; i0 += 16 * B) {
        Part t[B];
#pragma unroll
        for (int b = 0; b < B; ++b) {
            t[b] = p[min(i0 + 16 * b, g.units - 1)];
            if (i0 + 16 * b >= g.units) t[b].sum = 0.0;
        }
        float top = m;
#pragma unroll
        for (int b = 0; b < B; ++b) top = fmaxf(top, t[b].m);
        const Weight weight(g.c, top);
        sum *= weight(m);
#pragma unroll
        for (int b = 0; b < B; ++b) sum += t[b].sum * weight(t[b].m);
        m = top;
    }
    const float top = lanes::row16_max(m);
    sum *= Weight(g.c, top)(m);
    m = top;
#pragma unroll
    for (int off = 1; off < 16; off *= 2) sum += __shfl_xor(sum, off, 16);
}

struct Row {
    float m;
    double sum;
};
// The decision of request r by a workgroup: how many drafts stay, and the rows that the token behind them comes from.
__device__ __forceinline__ int decide(const VerifyArgs &g, int r, Row &p, Row &q) {
    __shared__ Row rows[2 * kMaxDrafts + 1];   // the target's, then the draft's
    __shared__ u64 refused;
    const int tid = threadIdx.x, count = count_of(g, r), targets = g.requests * (g.drafts + 1);
    // (the first wave's lanes: a draft each, its logits under way during the sums)
    const int x = tid < count ? g.draft_tokens[(size_t)r * g.drafts + tid] : -1;
    const bool there = x >= 0 && x < g.n;
    const float u = tid < count ? g.draws[(size_t)r * (g.drafts + 1) + tid] : 0.0f;
    const float lp = there ? g.logits[((size_t)r * (g.drafts + 1) + tid) * g.ld + x] : 0.0f;
    const float lq = there && g.draft ? g.draft[((size_t)r * g.drafts + tid) * g.draft_ld + x] : 0.0f;
    const int jobs = count + 1 + (g.draft ? count : 0);
    for (int j = tid / 16; j < jobs; j += kThreads2 / 16) {
        Row t;
        row_total(g, j <= count ? r * (g.drafts + 1) + j : targets + r * g.drafts + j - count - 1, t.m, t.sum);
        if (tid % 16 == 0) rows[j <= count ? j : kMaxDrafts + j - count] = t;
    }
    __syncthreads();
    if (tid < kWave) {
        bool stays = false;
        if (there) {
            const Row a = rows[tid];
            const double px = Weight(g.c, a.m)(as_logit(lp)), d = draw_of(u);
            if (!g.draft) {
                stays = d * a.sum < px;
            } else {
                const Row b = rows[kMaxDrafts + 1 + tid];
                stays = d * Weight(g.c, b.m)(as_logit(lq)) * a.sum < px * b.sum;
            }
        }
        const u64 mask = __ballot(tid < count && !stays);
        if (tid == 0) refused = mask;
    }
    __syncthreads();
    const int a = refused ? __builtin_ctzll(refused) : count;
    p = rows[a];
    q = rows[kMaxDrafts + 1 + min(a, kMaxDrafts - 1)];
    return a;
}

// What is left of token i's probability where the drafts end: max(p - q, 0), or p behind the last draft. p less q is formed of p
// less 2^-37 of it, 7.3e-12: sums of rows that lie differently in memory differ by up to 4.4e-12 (two factors of 1.1e-12 in each,
// see exp2_64), and where p and q are the same nothing must be left.
struct Rest {
    Weight wp, wq;
    double ip, iq;
    int mode, drafted;                     // mode 0: p; 1: p less q; 2: p but for the drafted token
    __device__ __forceinline__ Rest(const VerifyArgs &g, int r, int a, Row p, Row q)
        : wp(g.c, p.m), wq(g.c, q.m), ip(1.0 / p.sum), iq(1.0 / q.sum), mode(a >= count_of(g, r) ? 0 : g.draft ? 1 : 2), drafted(-1) {
        if (mode == 1) ip *= 1.0 - 0x1p-37;
        if (mode == 2) drafted = g.draft_tokens[(size_t)r * g.drafts + a];
    }
    __device__ __forceinline__ double operator()(float lp, float lq, int i) const {
        const double p = wp(lp) * ip;
        if (mode == 1) return fmax(p - wq(lq) * iq, 0.0);
        return mode == 2 && i == drafted ? 0.0 : p;
    }
    // the same where neither maximum is infinite
    __device__ __forceinline__ bool plain() const { return wp.finite && (mode != 1 || wq.finite); }
    __device__ __forceinline__ double of(float lp, float lq, int i) const {
        const double p = wp.of(lp) * ip;
        if (mode == 1) return fmax(p - wq.of(lq) * iq, 0.0);
        return mode == 2 && i == drafted ? 0.0 : p;
    }
};

// grid (parts of a row, requests): the decision, the units' sums of what is left of the row that it ends at, and, by the last
// workgroup of a request, the token. (Behind the last draft the sums are p's own, which the first launch made.)
__global__ __launch_bounds__(kThreads2, kPerUnit * kWaves2 / 4) void verify_token_kernel(VerifyArgs g) {
    __shared__ double part[kWaves2], needs[kWaves2];
    __shared__ int firsts[kWaves2], lasts[kWaves2];
    __shared__ unsigned arrived;
    const int r = blockIdx.y, tid = threadIdx.x, lane = tid & (kWave - 1), wid = tid / kWave;
    Row p, q;
    const int a = decide(g, r, p, q);
    Rest rest(g, r, a, p, q);
    const bool plain = rest.plain();
    const float *row = g.logits + ((size_t)r * (g.drafts + 1) + a) * g.ld;
    const float *other = rest.mode == 1 ? g.draft + ((size_t)r * g.drafts + a) * g.draft_ld : row;
    double *sums = g.rest + (size_t)r * g.units;
    if (rest.mode == 0) {
        if (blockIdx.x != 0) return;
    } else {
        for (int group = blockIdx.x; group * kUnits2 < g.units; group += gridDim.x) {
            const int i0 = (group * kWaves2 + wid) * (kUnit / kQuarters) - ahead(row) + lane * 4;
            pf4 x[kVec2], y[kVec2];
#pragma unroll
            for (int v = 0; v < kVec2; ++v) {
                const int i = i0 + v * kWave * 4;
                x[v] = load_logits(row, i, g.n);
                if (ahead(row) == ahead(other)) {
                    y[v] = load_logits(other, i, g.n);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) y[v][e] = as_logit(other[min(max(i + e, 0), g.n - 1)]);
                }
            }
            double s[4] = {0.0, 0.0, 0.0, 0.0};
            if (plain) {                               // without branches, so that the chains run side by side (outside: 0)
#pragma unroll
                for (int v = 0; v < kVec2; ++v)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[e] += rest.of(x[v][e], y[v][e], i0 + v * kWave * 4 + e);
            } else {
#pragma unroll
                for (int v = 0; v < kVec2; ++v)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int i = i0 + v * kWave * 4 + e;
                        s[e] += i >= 0 && i < g.n ? rest(x[v][e], y[v][e], i) : 0.0;
                    }
            }
            const double sum = wave_sum64((s[0] + s[1]) + (s[2] + s[3]));
            __syncthreads();                           // the sums before are out of `part`
            if (lane == 0) part[wid] = sum;
            __syncthreads();
            const int mine = group * kUnits2 + tid;
            if (tid < kUnits2 && mine < g.units) {
                const double *u = part + tid * kQuarters;
                __hip_atomic_store(&sums[mine], (u[0] + u[1]) + (u[2] + u[3]), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
        }
        // acknowledged before the workgroup counts itself done
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        if (tid == 0) arrived = __hip_atomic_fetch_add(&g.done[r], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        if (arrived != gridDim.x - 1) return;
    }
    // The unit in which the running sum passes the draw's share of the whole; past the last one by a rounding: the last one that
    // has any. A thread takes `each` units.
    const Part *own = g.part + ((size_t)r * (g.drafts + 1) + a) * g.units;
    const int each = (g.units + kThreads2 - 1) / kThreads2, u0 = tid * each;
    const double draw = draw_of(g.draws[(size_t)r * (g.drafts + 1) + g.drafts]);
    auto sum_of = [&](int i) {
        if (i >= g.units) return 0.0;
        if (rest.mode == 0) return own[i].sum * rest.wp(own[i].m) * rest.ip;
        return __hip_atomic_load(&sums[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    };
    double run, all;
    auto scan = [&](double mine) {                     // run: what the threads ahead have; all: what all have
        const double upto = wave_scan64(mine, lane);
        __syncthreads();
        if (lane == kWave - 1) part[wid] = upto;
        __syncthreads();
        run = upto - mine;
        all = 0.0;
#pragma unroll
        for (int w = 0; w < kWaves2; ++w) {
            run += w < wid ? part[w] : 0.0;
            all += part[w];
        }
    };
    // the first thread's `found` that is not -1, with its `need`, or the last thread's `some` (0: there is none), and no need
    auto choose = [&](int found, int some, double &need) {
        const u64 f = __ballot(found >= 0), l = __ballot(some >= 0);
        const int ff = __shfl(found, f ? __builtin_ctzll(f) : 0, kWave), ll = __shfl(some, l ? 63 - __builtin_clzll(l) : 0, kWave);
        const double nn = __shfl(need, f ? __builtin_ctzll(f) : 0, kWave);
        __syncthreads();
        if (lane == 0) {
            firsts[wid] = f ? ff : -1;
            lasts[wid] = l ? ll : -1;
            needs[wid] = nn;
        }
        __syncthreads();
        int at = -1, last = 0;
        need = INFINITY;
#pragma unroll
        for (int w = 0; w < kWaves2; ++w) {
            if (at < 0 && firsts[w] >= 0) {
                at = firsts[w];
                need = needs[w];
            }
            last = lasts[w] >= 0 ? lasts[w] : last;
        }
        return at >= 0 ? at : last;
    };
    auto total = [&]() {
        double s = 0.0;
        for (int j = 0; j < each; ++j) s += sum_of(u0 + j);
        scan(s);
    };
    total();
    if (all == 0.0 && rest.mode != 0) {                // p and q are the same, or all of p is on the drafted token: p itself
        rest.mode = 0;
        total();
    }
    int found = -1, some = -1;
    double need = INFINITY;
    for (int j = 0; j < each; ++j) {
        const double s = sum_of(u0 + j);
        if (s > 0.0) {
            some = u0 + j;
            if (found < 0 && run + s > draw * all) {
                found = u0 + j;
                need = draw * all - run;
            }
        }
        run += s;
    }
    const int unit = choose(found, some, need);
    const double left = need;
    const int i0 = unit * kUnit - ahead(row) + tid * kEach;
    float x[kEach], y[kEach];
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
        const int at = min(max(i0 + j, 0), g.n - 1);
        x[j] = row[at];
        y[j] = other[at];
    }
    double w[kEach], sum = 0.0;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
        const float lx = as_logit(x[j]), ly = as_logit(y[j]);
        w[j] = rest.plain() ? rest.of(lx, ly, i0 + j) : rest(lx, ly, i0 + j);
    }
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
        w[j] = i0 + j >= 0 && i0 + j < g.n ? w[j] : 0.0;
        sum += w[j];
    }
    scan(sum);
    found = some = -1;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
        run += w[j];
        if (w[j] > 0.0) {
            some = i0 + j;
            if (found < 0 && run > left) found = i0 + j;
        }
    }
    const int pick = choose(found, some, need);
    for (int i = tid; i <= g.drafts; i += kThreads2)
        g.tokens[(size_t)r * (g.drafts + 1) + i] = i < a ? g.draft_tokens[(size_t)r * g.drafts + i] : i == a ? pick : -1;
    if (tid == 0) g.accepted[r] = a;
}

// grid (requests): drafts stay while they are the target's best tokens.
__global__ __launch_bounds__(kThreads) void verify_greedy_kernel(VerifyArgs g) {
    __shared__ int best[kMaxDrafts + 1];
    const int r = blockIdx.x, tid = threadIdx.x, lane = tid & (kWave - 1), wid = tid / kWave, count = count_of(g, r);
    for (int j = wid; j <= count; j += kWaves) {
        u64 k = 0;
        for (int i = lane; i < g.units; i += kWave) {
            const u64 o = g.key[((size_t)r * (g.drafts + 1) + j) * g.units + i];
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
int units_of(int n) { return (n + 3 + kUnit - 1) / kUnit; }

}  // namespace

size_t verify_workspace_bytes(int n, int requests, int drafts) {
    const size_t units = (size_t)units_of(n), rows = (size_t)requests * (2 * drafts + 1);
    return units * (rows * sizeof(Part) + (size_t)requests * sizeof(double)) + (size_t)requests * sizeof(unsigned);
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
    g.units = units_of(n);
    g.draft_tokens = draft_tokens;
    g.counts = counts;
    g.draws = draws;
    g.c = temperature > 0.0f ? 1.4426950408889634 / (double)temperature : 0.0;
    g.tokens = tokens;
    g.accepted = accepted;
    const int targets = requests * (drafts + 1);
    const unsigned groups = (unsigned)((g.units + kWaves - 1) / kWaves);
    if (!(temperature > 0.0f)) {
        g.key = static_cast<u64 *>(ws);
        hipLaunchKernelGGL(verify_rows_kernel<true>, dim3(groups, targets), dim3(kThreads), 0, s, g);
        hipLaunchKernelGGL(verify_greedy_kernel, dim3(requests), dim3(kThreads), 0, s, g);
        return hip_ok(hipGetLastError(), "verify launch") ? 0 : -1;
    }
    const int rows = targets + (draft_logits ? requests * drafts : 0);
    g.part = static_cast<Part *>(ws);
    g.rest = reinterpret_cast<double *>(g.part + (size_t)rows * g.units);
    g.done = reinterpret_cast<unsigned *>(g.rest + (size_t)requests * g.units);
    hipLaunchKernelGGL(verify_rows_kernel<false>, dim3(groups, rows), dim3(kThreads), 0, s, g);
    // no more workgroups than run at once (a second round would decide everything again), with even shares of a row
    const unsigned steps = (unsigned)((g.units + kUnits2 - 1) / kUnits2), most = std::max(1u, (unsigned)(kFill / requests));
    const unsigned each = (steps + most - 1) / most, parts = (steps + each - 1) / each;
    hipLaunchKernelGGL(verify_token_kernel, dim3(parts, requests), dim3(kThreads2), 0, s, g);
    return hip_ok(hipGetLastError(), "verify launch") ? 0 : -1;
}

}  // namespace sapphire
