// beam.hip - beam search's selection: one pass over the logits, then one workgroup per request.
//
// Within a row the order of the scores is the order of the logits, so the pass needs no normaliser: each
// wave keeps its best W (logit, index) keys, and beside that it sums exp. The rows' lists and normalisers
// meet in the second launch, where the scores of the W x W candidates left are formed and compared in 64 bits.
//
// 64 rows of 262144 logits, a quarter of them ended (50 MB read): the pass 16.3 us (3.1 TB/s), the second launch 5.1. Half
// of the pass is vector issue, 25 instructions per logit of a lane: about seven make its part of the maximum and the sum, a few
// compare it, and most look for keys, since a wave of that size has one batch and must find a value that W of it reach, some
// keys above it and their order for that alone. The rest is the latency of first loads, lists and joins, where a
// copy's rate would be 10 us for the bytes. Four rows of 4096: 4.8 and 2.9 us, launches and latency.
#include <algorithm>

#include "internal.h"
#include "lanes.h"
#include "paged_dev.h"

namespace sapphire {

namespace {

using lanes::u64_lane;
typedef unsigned long long u64;

constexpr int kThreads = 256, kWave = 64, kWaves = kThreads / kWave;
constexpr int kMaxBeams = 16;
constexpr int kStep = 8, kBatch = 4;       // logits of a lane, two times four consecutive ones; times as many at once
constexpr int kChunkMin = 2048;            // logits of a workgroup at least
constexpr int kWantGroups = 2048;

// Larger logits, then lower indices, have larger keys; NaN counts as -inf, -0 as 0. Never 0.
__device__ __forceinline__ u64 key_of(float x, uint32_t i) {
    x = x != x ? -INFINITY : x + 0.0f;
    const uint32_t u = __float_as_uint(x), o = u & 0x80000000u ? ~u : u | 0x80000000u;
    return (u64)o << 32 | (uint32_t)~i;
}
__device__ __forceinline__ float key_value(u64 k) {
    const uint32_t o = (uint32_t)(k >> 32);
    return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ uint32_t key_index(u64 k) { return ~(uint32_t)k; }

// How many of the first `n` keys of `list` (16-byte aligned, zeros up to the next multiple of eight) are larger than k.
// All lanes read the same words, which costs the LDS one read each.
__device__ __forceinline__ int larger_than(u64 k, const u64 *list, int n) {
    typedef u64 two __attribute__((ext_vector_type(2)));
    int c = 0;
    for (int j = 0; j < n; j += 8) {
        two o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = *reinterpret_cast<const two *>(list + j + 2 * i);
#pragma unroll
        for (int i = 0; i < 4; ++i) c += (o[i].x > k) + (o[i].y > k);
    }
    return c;
}

// The `w` largest keys that a wave has seen. Keys above the w-th (`last`) gather in 64 words of LDS; when they would
// not fit, and at the end, each one's place is the number of larger ones, and the first w stay.
struct Best {
    u64 *buf;
    int w, count = 0;
    u64 last = 0;                          // 0: fewer than w so far

    __device__ __forceinline__ Best(u64 *lds, int beams) : buf(lds), w(beams) {}
    // a wave's LDS accesses stay in order; the compiler is told
    static __device__ __forceinline__ void handover() {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    __device__ __forceinline__ void sort() {
        const int lane = threadIdx.x & (kWave - 1);
        handover();
        const u64 k = lane < count ? buf[lane] : 0;
        if (lane >= count) buf[lane] = 0;
        handover();
        const int place = larger_than(k, buf, count);
        handover();
        if (lane < count && place < w) buf[place] = k;
        count = min(count, w);
        const u64 mask = __ballot(k != 0 && place == w - 1);
        last = mask ? u64_lane(k, __builtin_ctzll(mask)) : 0;
        handover();
    }
    // every lane offers one key (0: none)
    __device__ __forceinline__ void offer(u64 k) {
        u64 mask = __ballot(k > last);
        if (count + __popcll(mask) > kWave) {
            sort();
            mask = __ballot(k > last);
            if (count + __popcll(mask) > kWave) {      // up to w held and 64 offered: in two halves
                const bool low = (threadIdx.x & (kWave - 1)) < kWave / 2;
                put(low ? k : 0, __ballot(low && k > last));
                sort();
                k = low ? 0 : k;
                mask = __ballot(k > last);
            }
        }
        put(k, mask);
    }
    __device__ __forceinline__ void put(u64 k, u64 mask) {
        const int lane = threadIdx.x & (kWave - 1);
        if (mask >> lane & 1) buf[count + __popcll(mask & ((1ull << lane) - 1))] = k;
        count += __popcll(mask);
    }
};

// Over the wave, the same in every lane: rows of 16 lanes, then the four rows.
template <int CTRL>
__device__ __forceinline__ double dpp_f64(double v) {
    const u64 u = __builtin_bit_cast(u64, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, 0xF, 0xF, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, 0xF, 0xF, false);
    return __builtin_bit_cast(double, (u64)hi << 32 | lo);
}
__device__ __forceinline__ double wave_sum(double s) {
    s += dpp_f64<0xB1>(s);
    s += dpp_f64<0x4E>(s);
    s += dpp_f64<0x141>(s);
    s += dpp_f64<0x140>(s);
    const u64 u = __builtin_bit_cast(u64, s);
    auto of = [&](int l) { return __builtin_bit_cast(double, u64_lane(u, l)); };
    return (of(0) + of(16)) + (of(32) + of(48));
}

// Part of a row's normaliser: its largest logit and the sum of exp(x - max).
struct Norm {
    double sum;
    float max;
};

// exp(x - m) for x <= m, m above -inf; 0 for a NaN x, and for every x where m is +inf. The difference is taken first: next to
// an m of 2^32 and more, m - 150 is m. log2 e in two floats: the rounding of one would be off the same way in every term,
// where the others' roundings even out over a row.
__device__ __forceinline__ float exp_of(float x, float m) {
    constexpr float hi = 0x1.715476p+0f, lo = 0x1.4ae0cp-26f;
    const float d = fmaxf(__fsub_rn(x, m), -150.0f);
    return __builtin_amdgcn_exp2f(__builtin_fmaf(d, hi, __fmul_rn(d, lo)));
}

// A value that at least w of the wave's 64 reach: the least of the maxima of (at least) w groups of lanes.
__device__ __forceinline__ float reached_by(float t, int w) {
    t = fmaxf(t, lanes::dpp_mov<0xB1>(t));
    t = fmaxf(t, lanes::dpp_mov<0x4E>(t));             // of four lanes
    if (w <= 8) t = fmaxf(t, lanes::dpp_mov<0x141>(t));
    if (w <= 4) t = fmaxf(t, lanes::dpp_mov<0x140>(t));
    return -lanes::wave_max(-t);
}

// grid (chunks, rows): keys[row][place][chunk], norm[row][chunk]. Rows that have ended, and dead ones, need neither.
// A wave holds BATCH x 512 logits in its registers, eight of 512 in a lane, and has as many more on their way (BATCH
// 1 for chunks of no more than that per wave: a quarter of the code to fetch). Only those that reach a value that W of
// them do are looked at as keys.
template <int BATCH>
__global__ __launch_bounds__(kThreads, 4) void beam_rows_kernel(const float *__restrict__ logits, int ld, int n, int beams,
                                                             const float *__restrict__ scores, const int *__restrict__ done,
                                                             int chunk, u64 *__restrict__ keys, Norm *__restrict__ norm) {
    __shared__ __attribute__((aligned(16))) u64 lists[kWaves][kWave], all[kWave];
    __shared__ Norm part[kWaves];
    const int row = blockIdx.y, lane = threadIdx.x & (kWave - 1), wid = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    if ((done && done[row] != 0) || !(fabsf(scores[row]) < INFINITY)) return;
    const float *x = logits + (size_t)row * ld;
    const int lo = blockIdx.x * chunk, hi = min(n, lo + chunk);
    Best best(lists[wid], beams);
    float mx = -INFINITY;
    double sum = 0.0;
    constexpr int kSpan = kStep * kWave, kAll = kWaves * BATCH * kSpan;
    auto spot = [](int u) { return (u >> 2) * (4 * kWave) + (u & 3); };       // of a lane's u-th logit, from its first
    auto load = [&](float (&v)[BATCH][kStep], int i0) {
#pragma unroll
        for (int g = 0; g < BATCH; ++g) {
            const int first = i0 + g * kWaves * kSpan, at = first + lane * 4;
            if (first + kSpan <= hi) {                                 // rows start anywhere
                __builtin_memcpy(v[g], x + at, 16);
                __builtin_memcpy(v[g] + 4, x + at + 4 * kWave, 16);
            } else if (first < hi) {
#pragma unroll
                for (int u = 0; u < kStep; ++u) v[g][u] = x[min(at + spot(u), hi - 1)];
            }
        }
    };
    float v[BATCH][kStep];
    int i0 = lo + wid * kSpan;
    if (i0 < hi) load(v, i0);
    while (i0 < hi) {
        float next[BATCH][kStep];                                      // on its way during this batch's work
        if (i0 + kAll < hi) load(next, i0 + kAll);
        float most[BATCH], top = -INFINITY;                            // (a maximum with a NaN is the other one)
#pragma unroll
        for (int g = 0; g < BATCH; ++g) {
            const int first = i0 + g * kWaves * kSpan, at = first + lane * 4;
            if (first + kSpan > hi) {
#pragma unroll
                for (int u = 0; u < kStep; ++u) v[g][u] = at + spot(u) < hi ? v[g][u] : -INFINITY;
            }
            most[g] = -INFINITY;
#pragma unroll
            for (int u = 0; u < kStep; u += 2) most[g] = fmaxf(most[g], fmaxf(v[g][u], v[g][u + 1]));
            top = fmaxf(top, most[g]);
        }
        const float m = fmaxf(mx, top), from = m > -INFINITY ? m : 0.f;
        sum *= (double)exp_of(mx, from);                               // 0 before the first
        mx = m;
        float floor = key_value(best.last);
        if (best.last == 0) floor = reached_by(top, beams);
        uint32_t reach = 0;                                            // bit 8 g + u
#pragma unroll
        for (int g = 0; g < BATCH; ++g) {
            const int first = i0 + g * kWaves * kSpan;
            if (first >= hi) continue;
            float e[kStep];
#pragma unroll
            for (int u = 0; u < kStep; ++u) e[u] = exp_of(v[g][u], from);
            sum += (double)(((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7])));
            if (__any(most[g] >= floor)) {
                uint32_t byte = 0;
#pragma unroll
                for (int u = 0; u < kStep; ++u) byte |= v[g][u] < floor ? 0u : 1u << u;
                reach |= byte << (g * kStep);
            }
        }
        if (i0 + kAll > hi) {                          // past the end: no keys
#pragma unroll 1
            for (int g = 0; g < BATCH; ++g) {
                const int left = hi - (i0 + g * kWaves * kSpan + lane * 4);
                const uint32_t one = (1u << min(max(left, 0), 4)) - 1, two = (1u << min(max(left - 4 * kWave, 0), 4)) - 1;
                reach &= ~((~(one | two << 4) & 255u) << (g * kStep));
            }
        }
        while (__any(reach != 0)) {
            const int bit = reach ? __builtin_ctz(reach) : 0, at = i0 + bit / kStep * kWaves * kSpan + lane * 4 + spot(bit % kStep);
            float pick[BATCH * kStep];                                 // v[bit], a bit of its number at a time
#pragma unroll
            for (int i = 0; i < BATCH * kStep; ++i) pick[i] = v[i / kStep][i % kStep];
#pragma unroll
            for (int b = 0; (1 << b) < BATCH * kStep; ++b)
#pragma unroll
                for (int i = 0; i < (BATCH * kStep) >> (b + 1); ++i) pick[i] = bit >> b & 1 ? pick[2 * i + 1] : pick[2 * i];
            best.offer(reach ? key_of(pick[0], (uint32_t)at) : 0);
            reach &= reach - 1;
        }
        best.sort();
        i0 += kAll;
#pragma unroll
        for (int g = 0; g < BATCH; ++g)
#pragma unroll
            for (int u = 0; u < kStep; ++u) v[g][u] = next[g][u];
    }
    const float wm = lanes::wave_max(mx);
    const double ws = wave_sum(mx > -INFINITY ? sum * (double)exp_of(mx, wm) : 0.0);
    // the waves' lists one behind the other, zeros where there are fewer and up to a multiple of eight
    if (lane < beams) all[wid * beams + lane] = lane < best.count ? lists[wid][lane] : 0;
    if (wid == kWaves - 1 && kWaves * beams + lane < (kWaves * beams + 7) / 8 * 8) all[kWaves * beams + lane] = 0;
    if (lane == 0) part[wid] = Norm{ws, wm};
    __syncthreads();
    if (wid != 0) return;
    const u64 k = lane < kWaves * beams ? all[lane] : 0;
    const int place = larger_than(k, all, kWaves * beams), held = __popcll(__ballot(k != 0));
    u64 *out = keys + (size_t)row * beams * gridDim.x + blockIdx.x;
    if (k != 0 && place < beams) out[(size_t)place * gridDim.x] = k;
    if (lane >= held && lane < beams) out[(size_t)lane * gridDim.x] = 0;
    if (lane == 0) {
        float m = -INFINITY;
        double s = 0.0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) m = fmaxf(m, part[w].max);
#pragma unroll
        for (int w = 0; w < kWaves; ++w)
            if (part[w].max > -INFINITY) s += part[w].sum * (double)exp_of(part[w].max, m);
        norm[(size_t)row * gridDim.x + blockIdx.x] = Norm{s, m};
    }
}

// grid (requests), a wave per beam
__global__ __launch_bounds__(kMaxBeams *kWave) void beam_pick_kernel(int n, int beams, int chunks, const float *scores,
                                                                     const int *done, int end_token,
                                                                     const u64 *__restrict__ keys,
                                                                     const Norm *__restrict__ norm, float *scores_out,
                                                                     int *__restrict__ tokens, int *__restrict__ parents,
                                                                     int *done_out) {
    __shared__ __attribute__((aligned(16))) u64 lists[kMaxBeams][kWave];
    __shared__ double score[kMaxBeams * kMaxBeams];
    __shared__ int token[kMaxBeams * kMaxBeams], ended[kMaxBeams];
    const int r0 = blockIdx.x * beams, lane = threadIdx.x & (kWave - 1), b = threadIdx.x / kWave, row = r0 + b;
    const float cum = scores[row];
    const bool over = done && done[row] != 0;
    bool dead = !(fabsf(cum) < INFINITY) || (over && (end_token < 0 || end_token >= n));
    Best best(lists[b], beams);
    u64 mine = 0;
    double lse = 0.0;
    if (!dead && !over) {
        const u64 *kr = keys + (size_t)row * chunks * beams;
        const Norm *nr = norm + (size_t)row * chunks;
        const Norm first = nr[min(lane, chunks - 1)];          // (on its way beside the keys)
        for (int i0 = 0; i0 < chunks * beams; i0 += 4 * kWave) {
            u64 k[4];                                  // (on their way together)
#pragma unroll
            for (int j = 0; j < 4; ++j) k[j] = kr[min(i0 + j * kWave + lane, chunks * beams - 1)];
            for (int j = 0; j < 4; ++j) {
                const u64 mine = j == 0 ? k[0] : j == 1 ? k[1] : j == 2 ? k[2] : k[3];
                best.offer(i0 + j * kWave + lane < chunks * beams ? mine : 0);
            }
        }
        best.sort();
        mine = lane < beams ? lists[b][lane] : 0;
        const float m = key_value(u64_lane(mine, 0));  // the largest logit
        double s = lane < chunks && first.max > -INFINITY ? first.sum * (double)exp_of(first.max, m) : 0.0;
        for (int i = lane + kWave; i < chunks; i += kWave)
            if (nr[i].max > -INFINITY) s += nr[i].sum * (double)exp_of(nr[i].max, m);
        lse = (double)m + log(wave_sum(s));
        dead = !(fabs(lse) < (double)INFINITY);        // a logit of +inf (inf + log 0), or none above -inf
    }
    if (lane < beams) {
        double sc = -(double)INFINITY;
        int tok = lane;                                // what a row of -inf offers
        if (!dead && over) {
            tok = lane == 0 ? end_token : lane - 1 + (lane - 1 >= end_token);
            if (lane == 0) sc = (double)cum;
        } else if (!dead) {
            sc = (double)cum + ((double)key_value(mine) - lse);
            tok = (int)key_index(mine);
        }
        score[b * beams + lane] = sc;
        token[b * beams + lane] = tok;
        if (lane == 0) ended[b] = over;
    }
    __syncthreads();
    // Each candidate's place is the number of better ones; of equal scores the lower row, then the row's own order,
    // goes first. Four threads count for one candidate (64 beams threads are at least 4 beams^2).
    const int i = threadIdx.x >> 2, all = beams * beams;
    if (i >= all) return;
    const double sc = score[i];
    int place = 0;
#pragma unroll 4
    for (int j = threadIdx.x & 3; j < all; j += 4) place += score[j] > sc || (score[j] == sc && j < i);
    place += __builtin_amdgcn_update_dpp(0, place, 0xB1, 0xF, 0xF, false);
    place += __builtin_amdgcn_update_dpp(0, place, 0x4E, 0xF, 0xF, false);
    if (place >= beams || (threadIdx.x & 3) != 0) return;
    const int from = i / beams;
    scores_out[r0 + place] = (float)sc;
    tokens[r0 + place] = token[i];
    parents[r0 + place] = r0 + from;
    if (done_out) done_out[r0 + place] = ended[from] || token[i] == end_token;
}

int chunks_of(int n, int rows) {
    const int want = std::max(1, kWantGroups / std::max(1, rows));
    return std::min(want, (n + kChunkMin - 1) / kChunkMin);
}
int chunk_of(int n, int chunks) { return (n + chunks - 1) / chunks; }

}  // namespace

// Enough for calls of fewer rows too, which have more chunks: rows times chunks is at most kWantGroups, or one chunk each.
size_t beam_workspace_bytes(int n, int rows, int beams) {
    const size_t slots = std::min((size_t)rows * ((n + kChunkMin - 1) / kChunkMin), (size_t)std::max(kWantGroups, rows));
    return slots * (beams * sizeof(u64) + sizeof(Norm));
}

int launch_beam_select(const float *logits, int ld, int n, int requests, int beams, const float *scores, const int *done,
                       int end_token, float *scores_out, int *tokens, int *parents, int *done_out, void *ws,
                       hipStream_t s) {
    const int rows = requests * beams, chunks = chunks_of(n, rows);
    u64 *keys = static_cast<u64 *>(ws);
    Norm *norm = reinterpret_cast<Norm *>(keys + (size_t)rows * chunks * beams);
    const int chunk = chunk_of(n, chunks);
    if (chunk <= kWaves * kStep * kWave)
        hipLaunchKernelGGL((beam_rows_kernel<1>), dim3(chunks, rows), dim3(kThreads), 0, s, logits, ld, n, beams, scores, done, chunk, keys, norm);
    else
        hipLaunchKernelGGL((beam_rows_kernel<kBatch>), dim3(chunks, rows), dim3(kThreads), 0, s, logits, ld, n, beams, scores, done, chunk, keys, norm);
    if (!hip_ok(hipGetLastError(), "beam rows launch")) return -1;
    hipLaunchKernelGGL(beam_pick_kernel, dim3(requests), dim3(beams * kWave), 0, s, n, beams, chunks, scores, done, end_token,
                       keys, norm, scores_out, tokens, parents, done_out);
    return hip_ok(hipGetLastError(), "beam pick launch") ? 0 : -1;
}

}  // namespace sapphire
