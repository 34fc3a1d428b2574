// paged_shared.hip - attention of one new token per row where groups of rows share their first positions: the requests behind
// one prompt, beams, the drafted tokens of a sequence.
//
// The query heads of a K/V head of all rows of a group are columns of one product: K and V of the shared positions are read
// once for all of them, and what would be one row's share of memory becomes work for the matrix cores. The positions are cut
// into pieces; each row's own positions, behind the shared ones, are the attention's kernels' (paged_attention.h); a last launch
// joins the pieces of both. Only positions that all rows of a group have count as shared, in whole tiles, so that no score is
// masked for one row and not for another.
#include "paged_shared.h"

namespace sapphire {

namespace {

constexpr int kSharedFill = 2048;          // waves of the shared positions: two per SIMD
constexpr int kSharedUnit = 32;            // positions of a piece at least
constexpr int kMostCols = 256;             // columns of a workgroup at most
struct Both {
    Plan own;
    SharedPlan shared;
};
Both both_of(int dtype, bool half, int nkv, int hd, int batch, int n_heads, int max_length, int rows, int max_own) {
    Both b;
    const int group = n_heads / nkv, groups = (batch + rows - 1) / rows;
    b.own = plan_of(dtype, half, nkv, hd, batch, n_heads, std::min(max_length, std::max(max_own, 1)), 0);
    b.own.pieces = std::min(b.own.pieces, kMaxPieces / 2);
    b.shared.cols = std::min(rows, batch) * group;
    const Columns k = columns_of(dtype, half, b.shared.cols, hd);
    b.shared.col_tiles = (b.shared.cols + k.columns() - 1) / k.columns();
    const int64_t wgs = (int64_t)groups * nkv * b.shared.col_tiles;
    const int64_t want = std::max<int64_t>(1, kSharedFill / (wgs * (k.nw == 8 ? 8 : 4)));
    b.shared.pieces = (int)std::min<int64_t>({want, (max_length + kSharedUnit - 1) / kSharedUnit, kMaxPieces / 2});
    b.shared.total = b.shared.pieces * nkv * groups;
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
    if (!launch_pieces<BEHIND>(g, b.own, half, s)) return -1;
    g.pieces = total;
    return launch_join<BEHIND>(g, s) ? 0 : -1;
}

}  // namespace sapphire
