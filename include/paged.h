/*
 * paged.h - a paged key-value cache on one MI355X and the operators that serve from it.
 *
 * The cache keeps the K and V rows of every layer in pages of page_size positions, shared by any
 * number of sequences: a page table gives each sequence its pages, in any order. Rows are held as
 * F32, BF16, F16, or quantized when they are written to Q8_0 / Q4_0 blocks of 32 dims with fp32
 * scales (the arithmetic of quantize.h). All calls take device pointers of the current device,
 * only enqueue work on `stream` (NULL = the null stream), allocate nothing, can be captured into a
 * HIP graph, and return 0, or -1 with sapphire_last_error() and nothing enqueued.
 *
 * The reference has one fp32 cache per session (src/memory/kv_cache.c) and attends from it in
 * attention.c:93-163; these entry points have no counterpart there.
 *
 * A decode step of a batch: sapphire_rope_rows_dev (sapphire_hip.h) on the q and k heads of the
 * fused projection, sapphire_paged_write_dev of k and v at the sequences' next positions,
 * sapphire_paged_attention_dev; for beam search sapphire_beam_select_dev on the logits and
 * sapphire_paged_reorder_dev.
 */
#ifndef SAPPHIRE_HIP_PAGED_H
#define SAPPHIRE_HIP_PAGED_H

#include "sapphire_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* k and v: two buffers of sapphire_paged_cache_bytes() each, 16-byte aligned, that the caller
 * allocates (no initialisation needed: only positions that were written count). dtype: SAPPHIRE_F32,
 * _BF16, _F16, _Q8_0 or _Q4_0. page_size: a multiple of 16, at most 1024. head_dim: 64, 128 or 256. */
typedef struct {
    void *k, *v;
    int dtype;
    int layers, pages, page_size, n_kv_heads, head_dim;
} sapphire_paged_cache_t;

/* Bytes of k (and of v); 0, with sapphire_last_error(), for a shape the cache does not take (k and
 * v are not looked at). Position p of sequence s lies in page pages[s * ld + p / page_size].
 *
 * The bytes are in the order in which the matrix cores take them, so rows go in and out by the
 * calls below; for a program that moves caches itself: [layers][pages][n_kv_heads][tile], and in a
 * tile, with hd = head_dim, es the bytes of an element, nb = hd / 32,
 *   K  F32, BF16, F16  [page_size/16][hd*es/16][16 positions][16 bytes]
 *      Q8_0            [page_size/16][nb/2][4][16 positions][2 blocks][8 codes], code e of [..][m][..][b] is
 *                      element 8m + e of block b
 *      Q4_0            [page_size/16][nb/g][4][16 positions][g blocks][4 bytes], g = min(4, nb): byte i holds
 *                      element 8m + i (low nibble) and 8m + 4 + i (high) as 4-bit two's complement
 *      then            fp32 scales [page_size][nb]
 *   V  all types       [page_size/P][16][P positions][hd/16 dims], P = 16 / (bytes of hd/16 dims), between 1 and 4
 *      Q4_0            byte i of hd/16 dims: dim i (low nibble), dim hd/32 + i (high), value + 8
 *      then            fp32 scales [page_size/4][nb][4 positions]. */
size_t sapphire_paged_cache_bytes(const sapphire_paged_cache_t *cache);

/* The page table: pages[row * ld + i] is the page of row's positions i * page_size and on (device
 * memory, int32). An entry outside [0, cache->pages) is no page: nothing is written there, reads
 * give zeros, attention leaves its positions out. */
typedef struct {
    const int *pages;
    int rows, ld;
} sapphire_page_table_t;

/* Token t's K row (k: tokens x n_kv_heads x head_dim, see sapphire_rows_t) and V row into `layer`
 * at position positions[t] of table row seqs[t] (seqs NULL: row t). Rows are F32, BF16 or F16, both
 * of one type; a cache of another float type takes them rounded to nearest even, Q8_0 / Q4_0
 * quantized per 32 dims as quantize.h does. A block that has a NaN or an infinity reads back as NaN.
 * Tokens whose position is negative or past the table, or whose row or page does not exist, are left
 * out (padding). The tokens of one call go to different places: of two at the same place, what is
 * kept is unspecified. */
int sapphire_paged_write_dev(const sapphire_paged_cache_t *cache, int layer, const sapphire_rows_t *k,
                             const sapphire_rows_t *v, const sapphire_page_table_t *table, const int *seqs,
                             const int *positions, void *stream);

/* The reverse: the rows at those places, as the values they stand for, rounded to the type of k and
 * v. Places that do not exist give zero rows. k and v share no element: they lie apart, or are slices
 * of one buffer, of the same strides (rows between each other with other strides are refused). */
int sapphire_paged_read_dev(const sapphire_paged_cache_t *cache, int layer, const sapphire_rows_t *k,
                            const sapphire_rows_t *v, const sapphire_page_table_t *table, const int *seqs,
                            const int *positions, void *stream);

/* Attention of one new token per sequence. For sequence b (row b of the table; q->tokens rows) and
 * query head h, over the positions p with max(0, n - window) <= p < n, n = lengths[b]:
 *   s_p = scale * q . k_p;  softcap > 0: s_p = softcap * tanh(s_p / softcap)
 *   out = sum exp(s_p - max s) v_p / sum exp(s_p - max s);   lse = log sum exp(s_p)
 * in fp32 or more (attention.c:93-163 with a window and a cap). The new token's own row is written
 * first and counted in n. Query head h reads K/V head h / (n_heads / n_kv_heads). window <= 0: all
 * positions. lengths outside [0, max_length] are taken as its nearest end; max_length is at most
 * table->ld * page_size. A sequence of length 0 gets out = 0 and lse = -inf, and so does one whose
 * scores are all -inf or whose pages do not exist. A NaN or +inf score makes the head's outputs NaN.
 * What lies behind a sequence's last position, NaN included, does not count. A NaN in V makes its dim
 * NaN whatever its weight (over a quantized cache its block's dims), an infinity makes it infinite, or
 * NaN where infinities of both signs meet or one meets a weight that is 0 in fp32. Over a quantized
 * cache a NaN or an infinity in q makes its head's outputs NaN. (Sums are of up to 2^8 times the values
 * before they are scaled: they do not overflow where the largest |V| times the number of positions is
 * below 2^119, over Q4_0 2^115, nor those of the scores over a quantized cache where |K| is below 2^85.)
 * q and out: q->tokens x n_heads x head_dim, both of one type: F32; or BF16 / F16 over a cache of the
 * same type or a quantized one. out is q itself (same data and strides) or shares no element with it,
 * as k and v of a read.
 * out is rounded once, at the end; with 16-bit rows the weights exp(s_p - max s) meet V with 16 bits
 * or more. lse: [tokens][n_heads] fp32, or NULL. Long sequences are cut into pieces that run side by
 * side and are joined by a second launch; the results do not depend on which workgroup runs when, nor
 * on what the other sequences hold.
 * workspace: sapphire_paged_attention_workspace_bytes() bytes, 16-byte aligned (NULL where that is
 * 0), which are enough for calls of fewer and shorter sequences too; calls that share one must be
 * ordered on one stream. */
typedef struct {
    float scale;
    int window;
    float softcap;
} sapphire_attention_t;
size_t sapphire_paged_attention_workspace_bytes(const sapphire_paged_cache_t *cache, int batch, int n_heads,
                                                int max_length);
int sapphire_paged_attention_dev(const sapphire_paged_cache_t *cache, int layer, const sapphire_rows_t *q,
                                 const sapphire_rows_t *out, const sapphire_page_table_t *table, const int *lengths,
                                 int max_length, const sapphire_attention_t *attention, float *lse, void *workspace,
                                 void *stream);

/* After sapphire_beam_select_dev: row b continues row p = parents[b] of `table`, of which lengths[p]
 * positions are written. Row b of table_out gets p's full pages (shared, not copied); a partly
 * filled last page is copied, in every layer and head, to page spare[b], which takes its place: its
 * 16-position tiles that hold written positions, the rest of the spare page stays as it was. Entries
 * behind are -1. lengths_out[b] = lengths[p] (within [0, ld * page_size]). A parent outside the table
 * gives an empty row. table_out has the rows and ld of table; it, lengths_out and their inputs do not
 * overlap. spare[0 .. rows) name different pages that no row of table uses; one that does not
 * exist is left out (-1, nothing copied). */
int sapphire_paged_reorder_dev(const sapphire_paged_cache_t *cache, const sapphire_page_table_t *table,
                               const int *parents, const int *lengths, const int *spare,
                               const sapphire_page_table_t *table_out, int *lengths_out, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* SAPPHIRE_HIP_PAGED_H */
