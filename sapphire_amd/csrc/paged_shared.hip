// paged_shared.hip - attention of one new token per row where groups of rows share their first positions: the requests behind
// one prompt, beams, the drafted tokens of a sequence.
//
// The query heads of a K/V head of all rows of a group are columns of one product: K and V of the shared positions are read
// once for all of them, and what would be one row's share of memory becomes work for the matrix cores. The positions are cut
// into pieces; each row's own positions, behind the shared ones, are the attention's kernels' (paged_attention.h), or, where they
// are few, the last launch's (paged_shared_join.hip); that joins the pieces of both. Only positions that all rows of a group
// have count as shared, in whole tiles, so that no score is masked for one row and not for another.
//
// Few columns are bound by memory and, where positions are few, by the chain page -> K -> scores -> sum: 8 rows of 32 heads over 8
// of 128 dims behind 131072 positions, bf16 (537 MB): 110 us for the call. Many are bound by the issue of vector and matrix
// instructions, which take turns: 128 rows behind 32768 positions with up to 1000 of their own, bf16: 183 us, of which the shared
// positions take about 120 (their products 41 us of matrix cores, with the weights in two terms, and 45 of vector instructions at
// full clock; it falls to 1.9 GHz), the own ones and the join the rest (each kernel alone under a profiler: 137, 56 and 12). 16
// rows of each of two documents of 65536 positions, Q4_0, fp32 rows: 156 to 161 us, nearly all of it for the shared positions (168
// alone under a profiler, the others 19): 71 are vector instructions, most of them V's codes becoming three bf16 terms, 46 matrix
// cores.
#include "paged_shared.h"

namespace sapphire {

namespace {

// Pieces: a piece more shortens every workgroup's walk, and adds a slot of each column that is written and joined. As many as
// fill the chip (two waves per SIMD; of few columns, whose waves have no barriers, one: 8 rows of 32 heads over 8, bf16, behind
// 16384 positions 28 us, with two 35; behind 131072 109 and 115), of eight steps of a wide workgroup (32 rows behind 4096
// positions 33 us, of four 40) or one of each wave of few columns; but half of the compute
// units get a workgroup in any case (six drafted rows of 4 heads behind 1018 positions, fp32: 19.6 us in 32 pieces, 21.8 in 16, both with three launches).
constexpr int kSharedFill = 2048, kFewFill = 1024;         // waves of the shared positions at once
constexpr int kSharedUnit = 32, kFewUnit = 128, kWideSteps = 8;
constexpr int kUnits = 256;               // compute units
// Positions of a piece from which on two sets a wave pay: they read K and V half as often, but twice as many pieces of half as
// many workgroups are joined (bf16, 64 rows of 32 heads over 8: behind 16384 positions 69 us with two sets, 62 with one; behind
// 65536 141 and 162).
constexpr int kTwoSets = 768;
constexpr int kOwnJoined = 32;            // positions of a row behind the shared ones that the join takes along
constexpr int kMostCols = 256;             // columns of a workgroup at most
struct Both {
    Plan own;
    SharedPlan shared;
};
SharedPlan shared_plan(int dtype, int sets, int nkv, int hd, int groups, int cols, int max_length) {
    SharedPlan p;
    p.cols = cols;
    const Columns k = columns_of(sets, cols, hd);
    p.cs = k.cs;
    p.nw = k.nw;
    p.col_tiles = (cols + k.columns() - 1) / k.columns();
    const bool few = cols <= kFewColumns;
    const int64_t wgs = (int64_t)groups * nkv * p.col_tiles;
    const int64_t full = (few ? kFewFill : kSharedFill) / (wgs * (k.nw == 8 ? 8 : 4)), one = kUnits / wgs;
    const int unit = few ? kFewUnit : kWideSteps * (dtype == DT_F32 || hd == 256 ? 16 : 32);
    int64_t pieces = std::max(std::min<int64_t>(one / 2, (max_length + kSharedUnit - 1) / kSharedUnit),
                              std::min<int64_t>(full, max_length / unit));
    // (few compute units with two workgroups would keep the others waiting: 12 rows over 4 K/V heads, fp32, behind 8192 positions
    // 31 us in 64 pieces, 37.5 in 65)
    if (pieces > one && 2 * pieces < 3 * one) pieces = one;
    p.pieces = (int)std::min<int64_t>(std::max<int64_t>(1, pieces), kMaxPieces / 2);
    p.total = p.pieces * nkv * groups;
    return p;
}
Both both_of(int dtype, bool half, int nkv, int hd, int batch, int n_heads, int max_length, int rows, int max_own) {
    Both b;
    const int groups = (batch + rows - 1) / rows, cols = std::min(rows, batch) * (n_heads / nkv);
    // (not known: as many as there may be. Pieces that stay empty cost the join a little; few pieces of thousands of positions are
    // walked by a few compute units: four rows of 32 bf16 heads over 8 with 4000 of their own 44 us in one piece, 27 so. The dearest call found that does not say it has
    // few: 16 rows of two Q4_0 documents of 32768 positions, 300 own ones each, 124 us, 108 if it does.)
    b.own = plan_of(dtype, half, nkv, hd, batch, n_heads, max_own > 0 ? std::min(max_length, max_own) : max_length, 0);
    b.own.pieces = std::min(b.own.pieces, kMaxPieces / 2);
    b.shared = shared_plan(dtype, wide_sets(dtype, half, hd), nkv, hd, groups, cols, max_length);
    if (b.shared.cs == 2 && cols > kFewColumns && max_length < (int64_t)kTwoSets * b.shared.pieces)
        b.shared = shared_plan(dtype, 1, nkv, hd, groups, cols, max_length);
    return b;
}

}  // namespace

// Enough for every call of at most `batch` rows of at most max_length, whatever its groups. A row's query head has one slot of
// shared pieces, or as many as make kSharedFill workgroups, of up to kMostCols columns each; and the attention's own.
size_t paged_shared_workspace(int dtype, int nkv, int hd, int batch, int n_heads, int max_length) {
    const int64_t heads = (int64_t)batch * n_heads, most = std::min<int64_t>(kMaxPieces / 2, ((int64_t)max_length + kSharedUnit - 1) / kSharedUnit);
    const size_t slot = hd * sizeof(float) + sizeof(float2);
    return (size_t)(heads + std::min<int64_t>(kSharedFill / 8 * kMostCols, heads * most)) * slot +
           std::max((size_t)heads * slot, paged_attention_workspace(dtype, nkv, hd, batch, n_heads, max_length));
}

int launch_paged_shared_attention(const PagedAttn &a, hipStream_t s) {
    AttnArgs g;
    g.a = a;
    g.n_heads = a.q.heads;
    g.group = g.n_heads / a.c.nkv;
    const bool half = a.q.dtype != DT_F32;
    Both b = both_of(a.c.dtype, half, a.c.nkv, a.c.hd, a.q.tokens, g.n_heads, a.max_length, a.rows, a.max_own);
    const int total = b.shared.pieces + b.own.pieces;
    g.longest = a.max_length;
    g.col_tiles = b.own.col_tiles;
    g.piece = 0;
    g.pieces = b.own.pieces;
    g.first_piece = b.shared.pieces;
    g.wide = rows_wide(a.out);
    g.ordered = false;
    g.part = reinterpret_cast<float *>(a.ws);
    g.ms = reinterpret_cast<float2 *>(a.ws + part_bytes(a.c.hd, a.q.tokens, g.n_heads, total));
    b.shared.wide = rows_wide(a.q);
    if (is_quant(a.c.dtype)) {
        if (!launch_shared_quant(&g, &b.shared, s)) return -1;
    } else {
#define SPH_FORM(CT, HD, HALF) if (a.c.dtype == CT && a.c.hd == HD && half == HALF) launch_shared_form<CT, HD, HALF, false>(g, b.shared, s);
#define SPH_FORM_HD(HD) SPH_FORM(DT_F32, HD, false) SPH_FORM(DT_BF16, HD, false) SPH_FORM(DT_BF16, HD, true) SPH_FORM(DT_F16, HD, false) SPH_FORM(DT_F16, HD, true)
        SPH_FORM_HD(64) SPH_FORM_HD(128) SPH_FORM_HD(256)
        if (!hip_ok(hipGetLastError(), "shared attention launch")) return -1;
    }
    if (a.max_own > 0 && a.max_own <= kOwnJoined) {
        g.pieces = b.shared.pieces;
        return launch_shared_join(&g, s) ? 0 : -1;
    }
    if (!launch_pieces<BEHIND>(g, b.own, half, s)) return -1;
    g.pieces = total;
    return launch_join<BEHIND>(g, s) ? 0 : -1;
}

}  // namespace sapphire
