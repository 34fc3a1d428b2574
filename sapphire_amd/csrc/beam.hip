// beam.hip - beam search's selection: one pass over the logits, then one workgroup per request.
//
// Within a row the order of the scores is the order of the logits, so the pass needs no normaliser: each
// wave keeps its best W (logit, index) keys in its first lanes, sorted, and only elements above the W-th
// touch them; beside that it sums exp. The rows' lists and normalisers meet in the second launch, where
// the scores of the W x W candidates left are formed and compared in 64 bits.
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
constexpr int kStep = 8;                   // loads in flight per lane
constexpr int kChunkMin = 2048;            // logits of a workgroup at least
constexpr int kWantGroups = 1024;

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

// The `w` largest keys seen by a wave, in its lanes 0 .. w - 1, largest first (0: none yet).
struct Best {
    u64 key = 0, last = 0;                 // this lane's, the w-th
    // every lane offers one key (0: none)
    __device__ __forceinline__ void offer(u64 k, int w) {
        const int lane = threadIdx.x & (kWave - 1);
        u64 mask = __ballot(k > last);
        while (mask) {
            const u64 top = u64_lane(k, __builtin_ctzll(mask));
            const int at = __popcll(__ballot(lane < w && key > top));
            const u64 up = __shfl_up(key, 1, kWave);
            key = lane < at ? key : lane == at ? top : up;
            last = u64_lane(key, w - 1);
            mask &= mask - 1;
            mask &= __ballot(k > last);
        }
    }
};

// grid (chunks, rows): keys[row][chunk][beams] largest first, norm[row][chunk] = (max, sum exp(x - max)).
// Rows that have ended, and dead ones, need neither.
__global__ __launch_bounds__(kThreads) void beam_rows_kernel(const float *__restrict__ logits, int ld, int n, int beams,
                                                             const float *__restrict__ scores, const int *__restrict__ done,
                                                             int chunk, u64 *__restrict__ keys, float2 *__restrict__ norm) {
    __shared__ u64 all[kWaves * kMaxBeams];
    __shared__ float2 part[kWaves];
    const int row = blockIdx.y, lane = threadIdx.x & (kWave - 1), wid = threadIdx.x / kWave;
    if ((done && done[row] != 0) || !(fabsf(scores[row]) < INFINITY)) return;
    const float *x = logits + (size_t)row * ld;
    const int lo = blockIdx.x * chunk, hi = min(n, lo + chunk);
    Best best;
    float mx = -INFINITY, sum = 0.f;
    for (int i0 = lo + wid * kStep * kWave; i0 < hi; i0 += kWaves * kStep * kWave) {
        float v[kStep];
#pragma unroll
        for (int u = 0; u < kStep; ++u) v[u] = x[min(i0 + u * kWave + lane, hi - 1)];
        float top = -INFINITY;
#pragma unroll
        for (int u = 0; u < kStep; ++u) {
            if (i0 + u * kWave + lane >= hi || v[u] != v[u]) v[u] = -INFINITY;
            top = fmaxf(top, v[u]);
        }
        const float m = fmaxf(mx, top);
        if (m > -INFINITY) {
            sum *= __expf(mx - m);
#pragma unroll
            for (int u = 0; u < kStep; ++u) sum += __expf(v[u] - m);
            mx = m;
        }
#pragma unroll
        for (int u = 0; u < kStep; ++u) {
            const int i = i0 + u * kWave + lane;
            best.offer(i < hi ? key_of(v[u], (uint32_t)i) : 0, beams);
        }
    }
    const float wm = lanes::wave_max(mx);
    const float ws = lanes::wave_sum(mx > -INFINITY ? sum * __expf(mx - wm) : 0.f);
    if (lane < beams) all[wid * beams + lane] = best.key;
    if (lane == 0) part[wid] = make_float2(wm, ws);
    __syncthreads();
    if (wid != 0) return;
    Best merged;                                       // of the waves' lists, a key per lane
    merged.offer(lane < kWaves * beams ? all[lane] : 0, beams);
    if (lane < beams) keys[((size_t)row * gridDim.x + blockIdx.x) * beams + lane] = merged.key;
    if (lane == 0) {
        float m = -INFINITY, s = 0.f;
        for (int w = 0; w < kWaves; ++w) m = fmaxf(m, part[w].x);
        for (int w = 0; w < kWaves; ++w)
            if (part[w].x > -INFINITY) s += part[w].y * __expf(part[w].x - m);
        norm[(size_t)row * gridDim.x + blockIdx.x] = make_float2(m, s);
    }
}

// grid (requests)
__global__ __launch_bounds__(kThreads) void beam_pick_kernel(int n, int beams, int chunks, const float *scores,
                                                             const int *done, int end_token,
                                                             const u64 *__restrict__ keys, const float2 *__restrict__ norm,
                                                             float *scores_out, int *__restrict__ tokens,
                                                             int *__restrict__ parents, int *done_out) {
    __shared__ double score[kMaxBeams * kMaxBeams];
    __shared__ int token[kMaxBeams * kMaxBeams], ended[kMaxBeams];
    const int r0 = blockIdx.x * beams, lane = threadIdx.x & (kWave - 1), wid = threadIdx.x / kWave;
    for (int b = wid; b < beams; b += kWaves) {
        const int row = r0 + b;
        const float cum = scores[row];
        const bool over = done && done[row] != 0;
        bool dead = !(fabsf(cum) < INFINITY) || (over && (end_token < 0 || end_token >= n));
        Best best;
        double lse = 0.0;
        if (!dead && !over) {
            const float2 *nr = norm + (size_t)row * chunks;
            float m = -INFINITY;
            for (int i = lane; i < chunks; i += kWave) m = fmaxf(m, nr[i].x);
            m = lanes::wave_max(m);
            double s = 0.0;
            for (int i = lane; i < chunks; i += kWave)
                if (nr[i].x > -INFINITY) s += (double)nr[i].y * (double)__expf(nr[i].x - m);
#pragma unroll
            for (int off = kWave / 2; off > 0; off >>= 1) s += __shfl_xor(s, off, kWave);
            lse = (double)m + log(s);
            dead = !(fabs(lse) < (double)INFINITY);    // a logit of +inf, or none above -inf
            const u64 *kr = keys + (size_t)row * chunks * beams;
            for (int i0 = 0; i0 < chunks * beams; i0 += kWave) best.offer(i0 + lane < chunks * beams ? kr[i0 + lane] : 0, beams);
        }
        if (lane < beams) {
            double sc = -(double)INFINITY;
            int tok = lane;                            // what a row of -inf offers
            if (!dead && over) {
                tok = lane == 0 ? end_token : lane - 1 + (lane - 1 >= end_token);
                if (lane == 0) sc = (double)cum;
            } else if (!dead) {
                sc = (double)cum + ((double)key_value(best.key) - lse);
                tok = (int)key_index(best.key);
            }
            score[b * beams + lane] = sc;
            token[b * beams + lane] = tok;
            if (lane == 0) ended[b] = over;
        }
    }
    __syncthreads();
    // each candidate's place is the number of better ones; of equal scores the lower row, then the
    // row's own order, goes first
    const int i = threadIdx.x, all = beams * beams;
    if (i >= all) return;
    const double sc = score[i];
    int place = 0;
    for (int j = 0; j < all; ++j) place += score[j] > sc || (score[j] == sc && j < i);
    if (place >= beams) return;
    const int b = i / beams;
    scores_out[r0 + place] = (float)sc;
    tokens[r0 + place] = token[i];
    parents[r0 + place] = r0 + b;
    if (done_out) done_out[r0 + place] = ended[b] || token[i] == end_token;
}

int chunks_of(int n, int rows) {
    const int want = std::max(1, kWantGroups / std::max(1, rows));
    return std::min(want, (n + kChunkMin - 1) / kChunkMin);
}
int chunk_of(int n, int chunks) { return (n + chunks - 1) / chunks; }

}  // namespace

size_t beam_workspace_bytes(int n, int rows, int beams) {
    return (size_t)rows * chunks_of(n, rows) * (beams * sizeof(u64) + sizeof(float2));
}

int launch_beam_select(const float *logits, int ld, int n, int requests, int beams, const float *scores, const int *done,
                       int end_token, float *scores_out, int *tokens, int *parents, int *done_out, void *ws,
                       hipStream_t s) {
    const int rows = requests * beams, chunks = chunks_of(n, rows);
    u64 *keys = static_cast<u64 *>(ws);
    float2 *norm = reinterpret_cast<float2 *>(keys + (size_t)rows * chunks * beams);
    hipLaunchKernelGGL(beam_rows_kernel, dim3(chunks, rows), dim3(kThreads), 0, s, logits, ld, n, beams, scores, done,
                       chunk_of(n, chunks), keys, norm);
    if (!hip_ok(hipGetLastError(), "beam rows launch")) return -1;
    hipLaunchKernelGGL(beam_pick_kernel, dim3(requests), dim3(kThreads), 0, s, n, beams, chunks, scores, done, end_token,
                       keys, norm, scores_out, tokens, parents, done_out);
    return hip_ok(hipGetLastError(), "beam pick launch") ? 0 : -1;
}

}  // namespace sapphire
