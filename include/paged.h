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
 * sapphire_paged_reorder_dev. Where rows share their first positions, or are the drafted tokens that
 * sapphire_verify_dev decides about, sapphire_paged_shared_attention_dev reads the shared ones once;
 * of long sequences sapphire_paged_select_dev chooses pages by the bounds that
 * sapphire_paged_bounds_dev keeps, for sapphire_paged_pages_attention_dev.
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

/* The same where rows share their first positions: requests behind one prompt, the beams of a request, the drafted tokens of a
 * sequence (each a row of its own, with the sequence's pages and one position more than the one before). Group g is the
 * `rows` rows from g * rows on (the last one may have fewer), and shared[g] (device memory) says that their first shared[g]
 * positions are the same ones: the same pages, or pages of the same K and V. Those that every row of the group with a length
 * above 0 has, in whole tiles of 16, are read once for the group, by the table row of its first such row; each row's others by
 * its own. lengths, softcap, lse and types as for sapphire_paged_attention_dev, whose results these are but for the order of
 * sums and what products over the shared positions leave out: over an F16 cache with F32 rows q comes in two fp16 terms (off
 * by 2^-23 of an element or 2^-39 of its row's largest) and the weights in two (2^-22); over a quantized one q likewise, and V
 * in bf16 terms as the weights, for BF16 rows two of each (2^-15 of a weight times a value), for others three (2^-24). A
 * shared[g] of 0 or less shares nothing, one beyond the lengths all. A window is refused: what rows share under one starts
 * where the last of their windows does, which differs from row to row and is not formed here; layers with one take
 * sapphire_paged_attention_dev, drafted tokens too, which reads a window's K and V once per row. Over the shared positions a
 * NaN or an infinity in V makes its dim (over a quantized cache its block's dims) NaN or infinite; one in q or K, other than
 * over a cache of the rows' own type, makes its heads' outputs NaN. What is said there of positions behind the last one and of
 * pages that do not exist holds here too. max_own: about how many positions a row has behind the shared ones at most (0: not
 * known); it is for speed only, any value gives the same positions. workspace:
 * sapphire_paged_shared_attention_workspace_bytes() bytes, 16-byte aligned, which are enough for calls of fewer and shorter
 * rows too, whatever their groups; calls that share one must be ordered on one stream. */
typedef struct {
    const int *shared;
    int rows, max_own;
} sapphire_groups_t;
size_t sapphire_paged_shared_attention_workspace_bytes(const sapphire_paged_cache_t *cache, int batch, int n_heads,
                                                       int max_length);
int sapphire_paged_shared_attention_dev(const sapphire_paged_cache_t *cache, int layer, const sapphire_rows_t *q,
                                        const sapphire_rows_t *out, const sapphire_page_table_t *table, const int *lengths,
                                        int max_length, const sapphire_groups_t *groups,
                                        const sapphire_attention_t *attention, float *lse, void *workspace, void *stream);

/* Bounds of K per page, for the choice below: of each dim the lowest and the highest value of the page's written rows, as
 * 16 bits (F16 over an F16 cache, else BF16; values of other types rounded down and up). bounds: a buffer of
 * sapphire_paged_bounds_bytes(), 16-byte aligned, [layers][pages][n_kv_heads][2][head_dim], low ones first. A call makes those
 * of the pages that hold positions start[b] .. lengths[b] - 1 of table row b (every row of the table; start NULL: from 0;
 * both taken into 0 .. ld * page_size), from all their positions below lengths[b]. So a program calls it after each
 * sapphire_paged_write_dev, with start = the first position written, and for a page that sapphire_paged_reorder_dev copied.
 * max_new: at least lengths[b] - start[b]; of more positions the last max_new's pages are made. A NaN in K makes its dim's
 * bounds NaN. Rows that share a page write the same to it if they are of the same length there; else which is unspecified. */
size_t sapphire_paged_bounds_bytes(const sapphire_paged_cache_t *cache);
int sapphire_paged_bounds_dev(const sapphire_paged_cache_t *cache, int layer, void *bounds, const sapphire_page_table_t *table,
                              const int *start, const int *lengths, int max_new, void *stream);

/* The pages of each sequence and K/V head that its new token attends to. With lo and hi the bounds of a page of row b, its
 * score is the largest, over the query heads h of the K/V head, of sum_d max(q_hd lo_d, q_hd hi_d): no q . k of the page is
 * larger (a positive scale is assumed). choice->pages are chosen, all if there are no more: the first `first` and the last
 * `last` of the ceil(lengths[b] / page_size) pages, and the others by score, in 64 bits, of equal ones the first. The sum is
 * formed as max(q_hd, 0) hi_d + min(q_hd, 0) lo_d: an infinite bound that q's sign passes over is 0 times an infinity, as a
 * q_hd of 0 on any, and NaN. A score of NaN, from those or from NaN in q or bounds, counts as +inf. Pages that do not exist
 * are not chosen. selected[b][head][0 .. pages): their places in the sequence (page p / page_size of position p), rising, then
 * -1. q: tokens x n_heads x head_dim as for the attention, of any of the three types. lengths and max_length as there. first +
 * last <= pages <= 2^30 / page_size. workspace: sapphire_paged_select_workspace_bytes() bytes, 16-byte aligned, which are
 * enough for calls of fewer and shorter sequences too; calls that share one must be ordered. */
typedef struct {
    int pages, first, last;
} sapphire_page_choice_t;
size_t sapphire_paged_select_workspace_bytes(const sapphire_paged_cache_t *cache, int batch, int max_length);
int sapphire_paged_select_dev(const sapphire_paged_cache_t *cache, int layer, const void *bounds, const sapphire_rows_t *q,
                              const sapphire_page_table_t *table, const int *lengths, int max_length,
                              const sapphire_page_choice_t *choice, int *selected, void *workspace, void *stream);

/* Attention of one new token per sequence over the pages that selected[b][K/V head][0 .. pages) names (as
 * sapphire_paged_select_dev chooses them): as sapphire_paged_attention_dev, over the positions p of those pages with
 * max(0, n - window) <= p < n, n = lengths[b] (taken into 0 .. ld * page_size). A place that is negative, at or behind the
 * sequence's last page, or whose page does not exist, is left out. A list's places are different ones, its first
 * ceil(n / page_size) count (of a page named twice it is unspecified whether it counts twice), and their order does not matter.
 * A head without a position gets out = 0 and lse = -inf. workspace:
 * sapphire_paged_attention_workspace_bytes(cache, tokens, n_heads, pages * page_size). */
int sapphire_paged_pages_attention_dev(const sapphire_paged_cache_t *cache, int layer, const sapphire_rows_t *q,
                                       const sapphire_rows_t *out, const sapphire_page_table_t *table, const int *lengths,
                                       const int *selected, int pages, const sapphire_attention_t *attention, float *lse,
                                       void *workspace, void *stream);

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
