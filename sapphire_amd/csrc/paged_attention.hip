// paged_attention.hip - attention of one new token per sequence over the paged cache.
//
// With scores s_p in log2 units, out = sum 2^(s_p - m) v_p / sum 2^(s_p - m) in one pass over K and V: a wave takes a
// tile of 16 positions (or two), forms the scores on the matrix cores with the query heads of a K/V head as columns,
// keeps a running maximum m and sum per column, and adds the weighted V on the matrix cores. Nothing is staged in LDS:
// the cache's tiles are in operand order, so that a wave's loads are whole KiB and land in the registers that the
// products read; the next tile's K is under way during the softmax and V's product, its V during the next scores.
//
// The bytes of K and V bound it, each read once by one workgroup for all heads of its K/V head (sixteen at most, over
// quantized caches eight). A sequence is cut into pieces of a fixed number of positions that workgroups take side by
// side, and a second launch joins their (maximum, sum, O); where whole sequences fill the chip they are not cut and the
// longest go first. The products' forms:
//   float cache, fp32 rows, up to 4 heads   4x4x1 fp32: its four columns are the heads
//   float cache, fp32 rows, more            16x16x4 fp32
//   float cache, 16-bit rows                16x16x32 of their type, the weights in two terms of it
//   quantized cache                         K's codes in 8-bit products with q's digits, V's codes as bf16
//
// Whole calls over 400 MB of K and V, sequences of 2000 positions, head_dim 64 to 256: up to four heads per K/V head
// 73-103 us (3.9-5.5 TB/s; a large copy moves 4.9), eight heads 78-107 us over float caches, 87-118 over Q8_0, 115-154
// over Q4_0. There vector and matrix units take turns at two waves per SIMD: of 91 us (100 sequences of up to 2000, 8 K/V heads
// of 256 dims) 49 are vector issue and 36 matrix cores. Sixteen heads over a quantized cache read and convert K and V twice:
// 137-255 us.
#include "paged_attention.h"

namespace sapphire {

// Enough for every call of at most `batch` sequences of at most max_length, whatever its window and type of rows: b
// sequences that are cut, b k < kConverts.whole, have no more pieces than max(by bytes, kFill / (b k) + 1), all bounds grow
// with the length, and b times that is at most what the largest such b makes of either term.
size_t paged_attention_workspace(int dtype, int nkv, int hd, int batch, int n_heads, int max_length) {
    const int64_t k = plan_of(dtype, false, nkv, hd, 1, n_heads, max_length, 0).groups;
    const int64_t b = std::min<int64_t>(batch, (kConverts.whole - 1) / k);
    const int64_t most = std::min<int64_t>(kMaxPieces, ((int64_t)max_length + kPieceUnit - 1) / kPieceUnit);
    if (b == 0 || most == 1) return 0;
    const int64_t bytes = pieces_by_bytes(kConverts, max_length, row_bytes_kv(dtype, hd));
    const int64_t slots = std::max(b * std::min(most, bytes), std::min(b * most, kFill / k + b));
    return (size_t)slots * n_heads * (hd * sizeof(float) + sizeof(float2));
}

int launch_paged_attention(const PagedAttn &a, hipStream_t s) { return launch_attention<WHOLE>(a, s); }

}  // namespace sapphire
