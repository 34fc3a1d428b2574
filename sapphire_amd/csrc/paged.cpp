// paged.cpp - the entry points of paged.h, and of sapphire_hip.h's rows of heads and beam search: checks of
// what can be checked on the host, then the launches.
#include <algorithm>
#include <cmath>
#include <cstdlib>
#include <numeric>

#include "../../include/paged.h"
#include "paged_dev.h"

using namespace sapphire;

namespace {

constexpr int kMaxPage = 1024;
constexpr int kGridYZ = 65535;
constexpr int64_t kMaxUnits = (int64_t)1 << 31;        // threads of a launch

bool float_dtype(int dt) { return dt == DT_F32 || dt == DT_BF16 || dt == DT_F16; }

int row_bytes(int dt, int hd) {
    const int codes = dt == DT_F32 ? 4 * hd : dt == DT_Q8_0 ? hd : dt == DT_Q4_0 ? hd / 2 : 2 * hd;
    return codes + (is_quant(dt) ? hd / 8 : 0);
}

// Bytes from the first element to behind the last one.
bool rows_span(const sapphire_rows_t *r, uint64_t &bytes) {
    const int es = r->dtype == DT_F32 ? 4 : 2;
    __int128 last = r->head_dim;
    last += (__int128)(r->tokens - 1) * r->token_stride + (__int128)(r->heads - 1) * r->head_stride;
    if (last > ((__int128)1 << 60)) return false;
    bytes = (uint64_t)last * es;
    return true;
}

bool rows_ok(const sapphire_rows_t *r, const char *what, bool written) {
    if (!r || !r->data) { set_error("%s: no rows", what); return false; }
    if (!float_dtype(r->dtype)) { set_error("%s: dtype %d is not F32, BF16 or F16", what, r->dtype); return false; }
    if (r->tokens <= 0 || r->heads <= 0 || r->head_dim <= 0) {
        set_error("%s: bad shape (%d tokens, %d heads, head_dim %d)", what, r->tokens, r->heads, r->head_dim);
        return false;
    }
    if (r->token_stride < 0 || r->head_stride < 0) { set_error("%s: negative stride", what); return false; }
    uint64_t bytes;
    if (!rows_span(r, bytes)) { set_error("%s: strides too large", what); return false; }
    if (reinterpret_cast<uintptr_t>(r->data) % (r->dtype == DT_F32 ? 4 : 2) != 0) {
        set_error("%s: data is not aligned to its elements", what);
        return false;
    }
    if (written) {
        // one of the two dims steps over whole blocks of the other
        const long long hd = r->head_dim, ts = r->token_stride, hs = r->head_stride;
        const bool one_t = r->tokens == 1, one_h = r->heads == 1;
        const bool in = (one_h || hs >= hd) && (one_t || ts >= (long long)(r->heads - 1) * hs + hd);
        const bool out = (one_t || ts >= hd) && (one_h || hs >= (long long)(r->tokens - 1) * ts + hd);
        if (!in && !out) { set_error("%s: rows that are written overlap", what); return false; }
    }
    return true;
}

bool overlap(const void *a, uint64_t na, const void *b, uint64_t nb) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y + nb && y < x + na;
}

// Whether a and b, of one type, share no element, as far as their strides tell: their spans do not meet; or, as slices of one
// buffer, they stay in different parts of a period (modulo the period a stride that is a multiple of it does not move; another
// one adds its whole way to the part); or, of the same strides, no row of b starts within head_dim elements of one of a.
bool apart(const sapphire_rows_t *a, const sapphire_rows_t *b) {
    uint64_t na = 0, nb = 0;
    if (!rows_span(a, na) || !rows_span(b, nb)) return false;
    if (!overlap(a->data, na, b->data, nb)) return true;
    const int64_t off = (reinterpret_cast<intptr_t>(b->data) - reinterpret_cast<intptr_t>(a->data)) / (a->dtype == DT_F32 ? 4 : 2);
    auto differ = [&](int64_t period) {
        if (period <= 0) return false;
        auto part = [&](const sapphire_rows_t *r) {            // (below 2^60: rows_span)
            int64_t n = r->head_dim;
            if (r->tokens > 1 && r->token_stride % period != 0) n += (int64_t)(r->tokens - 1) * r->token_stride;
            if (r->heads > 1 && r->head_stride % period != 0) n += (int64_t)(r->heads - 1) * r->head_stride;
            return n;
        };
        const int64_t o = (off % period + period) % period;
        return part(a) <= o && part(b) <= period - o;
    };
    auto step = [](int n, long long stride) { return n > 1 ? (int64_t)stride : 0; };
    const int64_t ta = step(a->tokens, a->token_stride), tb = step(b->tokens, b->token_stride);
    const int64_t ha = step(a->heads, a->head_stride), hb = step(b->heads, b->head_stride);
    if (differ(std::gcd(std::gcd(ta, tb), std::gcd(ha, hb))) || (ta == tb && differ(ta)) || (ha == hb && differ(ha))) return true;
    if (ta != tb || ha != hb) return false;
    for (int64_t h = 1 - (int64_t)a->heads; h < b->heads; ++h) {       // b's head less a's; t: b's token less a's
        const int64_t at = off + h * ha;
        const int64_t t0 = ta ? -at / ta : 0;                          // (and its neighbours: at + t ta nearest to 0)
        for (int64_t t = t0 - 1; t <= t0 + 1; ++t)
            if (t > -(int64_t)a->tokens && t < b->tokens && std::llabs(at + t * ta) < std::max(a->head_dim, b->head_dim)) return false;
    }
    return true;
}
// The same rows in the same place.
bool identical(const sapphire_rows_t *a, const sapphire_rows_t *b) {
    return a->data == b->data && (a->tokens == 1 || a->token_stride == b->token_stride) &&
           (a->heads == 1 || a->head_stride == b->head_stride);
}

Rows as_rows(const sapphire_rows_t *r) {
    Rows o;
    o.p = static_cast<uint8_t *>(r->data);
    o.dtype = r->dtype;
    o.tokens = r->tokens;
    o.heads = r->heads;
    o.hd = r->head_dim;
    o.ts = r->token_stride;
    o.hs = r->head_stride;
    return o;
}

bool shape_ok(const sapphire_paged_cache_t *c) {
    if (!c) { set_error("paged cache: NULL"); return false; }
    if (!float_dtype(c->dtype) && !is_quant(c->dtype)) { set_error("paged cache: dtype %d", c->dtype); return false; }
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) {
        set_error("paged cache: head_dim %d is not 64, 128 or 256", c->head_dim);
        return false;
    }
    if (c->page_size < 16 || c->page_size > kMaxPage || c->page_size % 16 != 0) {
        set_error("paged cache: page_size %d is not a multiple of 16 up to %d", c->page_size, kMaxPage);
        return false;
    }
    if (c->layers <= 0 || c->pages <= 0 || c->n_kv_heads <= 0 || c->n_kv_heads > kGridYZ) {
        set_error("paged cache: bad shape (%d layers, %d pages, %d heads)", c->layers, c->pages, c->n_kv_heads);
        return false;
    }
    const __int128 bytes = (__int128)c->layers * c->pages * c->n_kv_heads * c->page_size * row_bytes(c->dtype, c->head_dim);
    if (bytes > ((__int128)1 << 60)) { set_error("paged cache: too large"); return false; }
    return true;
}

// The cache with its pools moved to `layer` (-1: all layers).
bool cache_ok(const sapphire_paged_cache_t *c, int layer, PagedCache &o) {
    if (!shape_ok(c)) return false;
    if (!c->k || !c->v || reinterpret_cast<uintptr_t>(c->k) % 16 != 0 || reinterpret_cast<uintptr_t>(c->v) % 16 != 0) {
        set_error("paged cache: k and v must be 16-byte aligned device buffers");
        return false;
    }
    if (layer < -1 || layer >= c->layers) { set_error("paged cache: layer %d of %d", layer, c->layers); return false; }
    o.dtype = c->dtype;
    o.layers = c->layers;
    o.pages = c->pages;
    o.page_size = c->page_size;
    o.nkv = c->n_kv_heads;
    o.hd = c->head_dim;
    set_page_division(o);
    o.tile_bytes = (uint32_t)(c->page_size * row_bytes(c->dtype, c->head_dim));
    o.layer_bytes = (size_t)c->pages * c->n_kv_heads * o.tile_bytes;
    const size_t at = layer > 0 ? (size_t)layer * o.layer_bytes : 0;
    o.k = static_cast<uint8_t *>(c->k) + at;
    o.v = static_cast<uint8_t *>(c->v) + at;
    return true;
}

bool table_ok(const sapphire_page_table_t *t) {
    if (!t || !t->pages || t->rows <= 0 || t->ld <= 0) { set_error("paged cache: bad page table"); return false; }
    return true;
}
PageTable as_table(const sapphire_page_table_t *t) { return PageTable{t->pages, t->rows, t->ld}; }

// What a write and a read check alike.
bool move_ok(const sapphire_paged_cache_t *c, int layer, const sapphire_rows_t *k, const sapphire_rows_t *v,
             const sapphire_page_table_t *t, const int *seqs, const int *positions, bool written, PagedCache &pc) {
    if (layer < 0) { set_error("paged cache: layer %d", layer); return false; }
    if (!cache_ok(c, layer, pc) || !rows_ok(k, "k rows", written) || !rows_ok(v, "v rows", written) || !table_ok(t)) return false;
    if (k->dtype != v->dtype || k->tokens != v->tokens || k->heads != c->n_kv_heads || v->heads != c->n_kv_heads ||
        k->head_dim != c->head_dim || v->head_dim != c->head_dim) {
        set_error("paged cache: k and v rows must be of one type and of the cache's heads and head_dim");
        return false;
    }
    if (!positions) { set_error("paged cache: no positions"); return false; }
    if (!seqs && k->tokens > t->rows) { set_error("paged cache: %d tokens for %d table rows", k->tokens, t->rows); return false; }
    if (((int64_t)k->tokens + 15) * c->n_kv_heads * (c->head_dim / 8) > kMaxUnits) { set_error("paged cache: too many rows in one call"); return false; }
    return true;
}

}  // namespace

extern "C" {

size_t sapphire_paged_cache_bytes(const sapphire_paged_cache_t *c) {
    if (!shape_ok(c)) return 0;
    return (size_t)c->layers * c->pages * c->n_kv_heads * c->page_size * row_bytes(c->dtype, c->head_dim);
}

int sapphire_paged_write_dev(const sapphire_paged_cache_t *c, int layer, const sapphire_rows_t *k, const sapphire_rows_t *v,
                             const sapphire_page_table_t *t, const int *seqs, const int *positions, void *stream) {
    PagedCache pc;
    if (!move_ok(c, layer, k, v, t, seqs, positions, false, pc)) return -1;
    return launch_paged_write(pc, as_rows(k), as_rows(v), as_table(t), seqs, positions, as_stream(stream));
}

int sapphire_paged_read_dev(const sapphire_paged_cache_t *c, int layer, const sapphire_rows_t *k, const sapphire_rows_t *v,
                            const sapphire_page_table_t *t, const int *seqs, const int *positions, void *stream) {
    PagedCache pc;
    if (!move_ok(c, layer, k, v, t, seqs, positions, true, pc)) return -1;
    if (!apart(k, v)) { set_error("paged read: k and v overlap"); return -1; }
    return launch_paged_read(pc, as_rows(k), as_rows(v), as_table(t), seqs, positions, as_stream(stream));
}

size_t sapphire_paged_attention_workspace_bytes(const sapphire_paged_cache_t *c, int batch, int n_heads, int max_length) {
    if (!shape_ok(c) || batch <= 0 || n_heads <= 0 || n_heads % c->n_kv_heads != 0 || max_length <= 0) return 0;
    return paged_attention_workspace(c->dtype, c->n_kv_heads, c->head_dim, batch, n_heads, max_length);
}

// What the attentions check alike; a's fields but the lengths' bound and the workspace.
static bool attend_ok(const sapphire_paged_cache_t *c, int layer, const sapphire_rows_t *q, const sapphire_rows_t *out,
                      const sapphire_page_table_t *t, const int *lengths, const sapphire_attention_t *at, float *lse, PagedAttn &a) {
    if (layer < 0) { set_error("paged attention: layer %d", layer); return false; }
    if (!cache_ok(c, layer, a.c) || !rows_ok(q, "q", false) || !rows_ok(out, "out", true) || !table_ok(t)) return false;
    if (q->dtype != out->dtype || q->tokens != out->tokens || q->heads != out->heads || q->head_dim != c->head_dim ||
        out->head_dim != c->head_dim) {
        set_error("paged attention: q and out must have one type and shape, and the cache's head_dim");
        return false;
    }
    if (q->heads % c->n_kv_heads != 0) { set_error("paged attention: %d heads over %d K/V heads", q->heads, c->n_kv_heads); return false; }
    if (q->dtype != DT_F32 && q->dtype != c->dtype && !is_quant(c->dtype)) {
        set_error("paged attention: 16-bit rows need a cache of their type or a quantized one (rows %d, cache %d)", q->dtype, c->dtype);
        return false;
    }
    if (!lengths || !at) { set_error("paged attention: no lengths or parameters"); return false; }
    if (!(std::fabs(at->scale) < INFINITY) || !(at->softcap >= 0.0f) || !(at->softcap < INFINITY)) {
        set_error("paged attention: scale %g, softcap %g", (double)at->scale, (double)at->softcap);
        return false;
    }
    if (q->tokens > t->rows || q->tokens > kGridYZ || q->heads > kGridYZ) {
        set_error("paged attention: %d sequences, %d heads, %d table rows", q->tokens, q->heads, t->rows);
        return false;
    }
    if (!identical(q, out) && !apart(q, out)) { set_error("paged attention: out overlaps q without being q"); return false; }
    a.q = as_rows(q);
    a.out = as_rows(out);
    a.table = as_table(t);
    a.lengths = lengths;
    a.window = at->window;
    a.scale = at->scale;
    a.softcap = at->softcap;
    a.lse = lse;
    return true;
}

static bool workspace_ok(size_t need, void *workspace, PagedAttn &a) {
    if (need && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16 != 0)) {
        set_error("paged attention: needs a 16-byte aligned workspace of %zu bytes", need);
        return false;
    }
    a.ws = static_cast<uint8_t *>(workspace);
    return true;
}

int sapphire_paged_attention_dev(const sapphire_paged_cache_t *c, int layer, const sapphire_rows_t *q,
                                 const sapphire_rows_t *out, const sapphire_page_table_t *t, const int *lengths,
                                 int max_length, const sapphire_attention_t *at, float *lse, void *workspace,
                                 void *stream) {
    PagedAttn a;
    if (!attend_ok(c, layer, q, out, t, lengths, at, lse, a)) return -1;
    if (max_length <= 0 || max_length > (int64_t)t->ld * c->page_size || max_length > (1 << 30)) {
        set_error("paged attention: max_length %d with %d pages of %d per row", max_length, t->ld, c->page_size);
        return -1;
    }
    a.max_length = max_length;
    if (!workspace_ok(sapphire_paged_attention_workspace_bytes(c, q->tokens, q->heads, max_length), workspace, a)) return -1;
    return launch_paged_attention(a, as_stream(stream));
}

int sapphire_paged_pages_attention_dev(const sapphire_paged_cache_t *c, int layer, const sapphire_rows_t *q,
                                       const sapphire_rows_t *out, const sapphire_page_table_t *t, const int *lengths,
                                       const int *selected, int pages, const sapphire_attention_t *at, float *lse,
                                       void *workspace, void *stream) {
    PagedAttn a;
    if (!attend_ok(c, layer, q, out, t, lengths, at, lse, a)) return -1;
    if (!selected || pages <= 0 || (int64_t)pages * c->page_size > (1 << 30)) {
        set_error("paged attention: lists of %d pages of %d", pages, c->page_size);
        return -1;
    }
    a.selected = selected;
    a.listed = pages;
    a.max_length = (int)std::min<int64_t>((int64_t)t->ld * c->page_size, 1 << 30);
    if (!workspace_ok(sapphire_paged_attention_workspace_bytes(c, q->tokens, q->heads, pages * c->page_size), workspace, a)) return -1;
    return launch_paged_pages_attention(a, as_stream(stream));
}

size_t sapphire_paged_shared_attention_workspace_bytes(const sapphire_paged_cache_t *c, int batch, int n_heads, int max_length) {
    if (!shape_ok(c) || batch <= 0 || n_heads <= 0 || n_heads % c->n_kv_heads != 0 || max_length <= 0) return 0;
    return paged_shared_workspace(c->dtype, c->n_kv_heads, c->head_dim, batch, n_heads, max_length);
}

int sapphire_paged_shared_attention_dev(const sapphire_paged_cache_t *c, int layer, const sapphire_rows_t *q,
                                        const sapphire_rows_t *out, const sapphire_page_table_t *t, const int *lengths,
                                        int max_length, const sapphire_groups_t *groups, const sapphire_attention_t *at,
                                        float *lse, void *workspace, void *stream) {
    PagedAttn a;
    if (!attend_ok(c, layer, q, out, t, lengths, at, lse, a)) return -1;
    if (max_length <= 0 || max_length > (int64_t)t->ld * c->page_size || max_length > (1 << 30)) {
        set_error("shared attention: max_length %d with %d pages of %d per row", max_length, t->ld, c->page_size);
        return -1;
    }
    if (!groups || !groups->shared || groups->rows <= 0 || groups->max_own < 0) { set_error("shared attention: bad groups"); return -1; }
    if (at->window > 0) { set_error("shared attention: a window (%d): what rows share under one is not formed", at->window); return -1; }
    a.max_length = max_length;
    a.shared = groups->shared;
    a.rows = std::min(groups->rows, q->tokens);
    a.max_own = groups->max_own;
    if (!workspace_ok(sapphire_paged_shared_attention_workspace_bytes(c, q->tokens, q->heads, max_length), workspace, a)) return -1;
    return launch_paged_shared_attention(a, as_stream(stream));
}

int sapphire_paged_reorder_dev(const sapphire_paged_cache_t *c, const sapphire_page_table_t *t, const int *parents,
                               const int *lengths, const int *spare, const sapphire_page_table_t *out, int *lengths_out,
                               void *stream) {
    PagedCache pc;
    if (!cache_ok(c, -1, pc) || !table_ok(t) || !table_ok(out)) return -1;
    if (!parents || !lengths || !spare || !lengths_out) { set_error("paged reorder: bad arguments"); return -1; }
    if (out->rows != t->rows || out->ld != t->ld) { set_error("paged reorder: the two tables differ in shape"); return -1; }
    if ((int64_t)2 * c->layers * c->n_kv_heads > kGridYZ) { set_error("paged reorder: %d layers x %d heads", c->layers, c->n_kv_heads); return -1; }
    const uint64_t tb = (uint64_t)t->rows * t->ld * sizeof(int), rb = (uint64_t)t->rows * sizeof(int);
    const void *ins[] = {t->pages, parents, lengths, spare};
    const uint64_t nin[] = {tb, rb, rb, rb};
    for (int i = 0; i < 4; ++i)
        if (overlap(ins[i], nin[i], out->pages, tb) || overlap(ins[i], nin[i], lengths_out, rb)) {
            set_error("paged reorder: outputs overlap inputs");
            return -1;
        }
    if (overlap(out->pages, tb, lengths_out, rb)) { set_error("paged reorder: outputs overlap"); return -1; }
    return launch_paged_reorder(pc, as_table(t), parents, lengths, spare, const_cast<int *>(out->pages), lengths_out, as_stream(stream));
}

size_t sapphire_paged_bounds_bytes(const sapphire_paged_cache_t *c) {
    if (!shape_ok(c)) return 0;
    return (size_t)c->layers * c->pages * c->n_kv_heads * 2 * c->head_dim * sizeof(uint16_t);
}

// The layer's bounds.
static bool bounds_ok(const sapphire_paged_cache_t *c, int layer, const void *bounds, uint16_t *&at) {
    if (!bounds || reinterpret_cast<uintptr_t>(bounds) % 16 != 0) { set_error("paged bounds: must be a 16-byte aligned device buffer"); return false; }
    at = static_cast<uint16_t *>(const_cast<void *>(bounds)) + (size_t)layer * c->pages * c->n_kv_heads * 2 * c->head_dim;
    return true;
}

int sapphire_paged_bounds_dev(const sapphire_paged_cache_t *c, int layer, void *bounds, const sapphire_page_table_t *t, const int *start,
                              const int *lengths, int max_new, void *stream) {
    PagedCache pc;
    uint16_t *at;
    if (layer < 0) { set_error("paged bounds: layer %d", layer); return -1; }
    if (!cache_ok(c, layer, pc) || !table_ok(t) || !bounds_ok(c, layer, bounds, at)) return -1;
    if (!lengths || max_new <= 0 || t->rows > kGridYZ || 2 * c->n_kv_heads > kGridYZ) {
        set_error("paged bounds: no lengths, max_new %d, %d table rows, %d heads", max_new, t->rows, c->n_kv_heads);
        return -1;
    }
    return launch_paged_bounds(pc, at, as_table(t), start, lengths, max_new, as_stream(stream));
}

static bool select_shape_ok(const sapphire_paged_cache_t *c, int batch, int max_length) {
    if (!shape_ok(c)) return false;
    if (batch <= 0 || batch > kGridYZ || max_length <= 0 || max_length > (1 << 30)) {
        set_error("paged select: %d sequences of up to %d positions", batch, max_length);
        return false;
    }
    return true;
}

size_t sapphire_paged_select_workspace_bytes(const sapphire_paged_cache_t *c, int batch, int max_length) {
    if (!select_shape_ok(c, batch, max_length)) return 0;
    return paged_select_workspace(c->n_kv_heads, batch, (max_length + c->page_size - 1) / c->page_size);
}

int sapphire_paged_select_dev(const sapphire_paged_cache_t *c, int layer, const void *bounds, const sapphire_rows_t *q,
                              const sapphire_page_table_t *t, const int *lengths, int max_length, const sapphire_page_choice_t *choice,
                              int *selected, void *workspace, void *stream) {
    PagedCache pc;
    uint16_t *at;
    if (layer < 0) { set_error("paged select: layer %d", layer); return -1; }
    if (!cache_ok(c, layer, pc) || !rows_ok(q, "q", false) || !table_ok(t) || !bounds_ok(c, layer, bounds, at) ||
        !select_shape_ok(c, q->tokens, max_length))
        return -1;
    if (q->heads % c->n_kv_heads != 0) { set_error("paged select: %d heads over %d K/V heads", q->heads, c->n_kv_heads); return -1; }
    if (q->head_dim != c->head_dim || q->tokens > t->rows || max_length > (int64_t)t->ld * c->page_size) {
        set_error("paged select: q of %d rows of head_dim %d, max_length %d, for %d table rows of %d pages", q->tokens, q->head_dim, max_length,
                  t->rows, t->ld);
        return -1;
    }
    if (!lengths || !choice || !selected || !workspace || reinterpret_cast<uintptr_t>(workspace) % 16 != 0) { set_error("bad paged select arguments"); return -1; }
    if (choice->pages <= 0 || (int64_t)choice->pages * c->page_size > (1 << 30) || choice->first < 0 || choice->last < 0 ||
        (int64_t)choice->first + choice->last > choice->pages) {
        set_error("paged select: %d pages with the first %d and the last %d", choice->pages, choice->first, choice->last);
        return -1;
    }
    return launch_paged_select(pc, at, as_rows(q), as_table(t), lengths, max_length, choice->pages, choice->first, choice->last, selected,
                               workspace, as_stream(stream));
}

int sapphire_rope_rows_dev(const sapphire_rows_t *x, const sapphire_rows_t *y, const int *positions,
                           const sapphire_rope_t *rope, void *stream) {
    if (!rows_ok(x, "rope x", false) || !rows_ok(y, "rope y", true)) return -1;
    if (!positions || !rope || !rope->freqs || rope->rotary_dim < 2 || rope->rotary_dim % 2 != 0 ||
        rope->rotary_dim > x->head_dim || x->head_dim > 1024 || x->heads > kGridYZ || !(std::fabs(rope->magnitude) < INFINITY)) {
        set_error("bad rope arguments");
        return -1;
    }
    if (x->dtype != y->dtype || x->tokens != y->tokens || x->heads != y->heads || x->head_dim != y->head_dim) {
        set_error("rope: x and y must have one type and shape");
        return -1;
    }
    if (!identical(x, y) && !apart(x, y)) { set_error("rope: y overlaps x without being x"); return -1; }
    return launch_rope_rows(as_rows(x), as_rows(y), positions, rope->freqs, rope->rotary_dim, rope->interleaved != 0,
                            rope->magnitude, as_stream(stream));
}

int sapphire_rope_frequencies(double *freqs, float *magnitude, int rotary_dim, double base, int scaling, double factor,
                              double trained, double low, double high) {
    if (!freqs || rotary_dim < 2 || rotary_dim % 2 != 0 || !(base > 0.0) || !(base < INFINITY) ||
        scaling < SAPPHIRE_ROPE_PLAIN || scaling > SAPPHIRE_ROPE_PARTS) {
        set_error("bad rope frequency arguments");
        return -1;
    }
    const bool scaled = scaling != SAPPHIRE_ROPE_PLAIN, parts = scaling == SAPPHIRE_ROPE_PARTS;
    if ((scaled && (!(factor >= 1.0) || !(factor < INFINITY))) || (scaling == SAPPHIRE_ROPE_BASE && rotary_dim == 2) ||
        (parts && (!(trained > 0.0) || !(trained < INFINITY) || !(low >= 0.0) || !(low < high) || !(high < INFINITY)))) {
        set_error("rope frequencies: bad scaling arguments");
        return -1;
    }
    if (scaling == SAPPHIRE_ROPE_BASE) base *= std::pow(factor, (double)rotary_dim / (rotary_dim - 2));
    for (int i = 0; i < rotary_dim / 2; ++i) {
        double f = std::pow(base, -2.0 * i / rotary_dim);
        if (scaling == SAPPHIRE_ROPE_LINEAR) f /= factor;
        if (parts) {
            const double turns = trained * f / 6.2831853071795864769;
            const double g = turns <= low ? 0.0 : turns >= high ? 1.0 : (turns - low) / (high - low);
            f *= (1.0 - g) / factor + g;
        }
        freqs[i] = f;
    }
    if (magnitude) *magnitude = parts ? (float)(0.1 * std::log(factor) + 1.0) : 1.0f;
    return 0;
}

static bool beam_shape_ok(int n, int requests, int beams) {
    return beams >= 1 && beams <= 16 && n >= beams && n <= (1 << 21) && requests >= 1 && (int64_t)requests * beams <= kGridYZ;
}

size_t sapphire_beam_workspace_bytes(int n, int requests, int beams) {
    return beam_shape_ok(n, requests, beams) ? beam_workspace_bytes(n, requests * beams, beams) : 0;
}

int sapphire_beam_select_dev(const float *logits, int ld, int n, int requests, int beams, const float *scores,
                             const int *done, int end_token, float *scores_out, int *tokens, int *parents, int *done_out,
                             void *workspace, void *stream) {
    if (!logits || !scores || !scores_out || !tokens || !parents || !workspace || ld < n || (done == nullptr) != (done_out == nullptr)) {
        set_error("bad beam search arguments");
        return -1;
    }
    if (!beam_shape_ok(n, requests, beams)) {
        set_error("beam search: 1..16 beams, beams..2^21 logits per row, up to 65535 rows (n %d, %d requests of %d beams)", n, requests, beams);
        return -1;
    }
    if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0) { set_error("the beam search workspace must be 16-byte aligned"); return -1; }
    return launch_beam_select(logits, ld, n, requests, beams, scores, done, end_token, scores_out, tokens, parents,
                              done_out, workspace, as_stream(stream));
}

static bool verify_shape_ok(int n, int requests, int drafts) {
    return drafts >= 1 && drafts <= 64 && n >= 1 && n <= (1 << 21) && requests >= 1 && (int64_t)requests * (2 * drafts + 1) <= kGridYZ;
}

size_t sapphire_verify_workspace_bytes(int n, int requests, int drafts) {
    return verify_shape_ok(n, requests, drafts) ? verify_workspace_bytes(n, requests, drafts) : 0;
}

int sapphire_verify_dev(const float *logits, int ld, const float *draft_logits, int draft_ld, int n, int requests, int drafts,
                        const int *draft_tokens, const int *counts, float temperature, const float *draws, int *tokens,
                        int *accepted, void *workspace, void *stream) {
    if (!logits || ld < n || (draft_logits && draft_ld < n) || !draft_tokens || !tokens || !accepted || !workspace) {
        set_error("bad verify arguments");
        return -1;
    }
    if (!verify_shape_ok(n, requests, drafts)) {
        set_error("verify: 1..64 drafts, 1..2^21 logits per row, up to 65535 rows (n %d, %d requests of %d drafts)", n, requests, drafts);
        return -1;
    }
    if (!(std::fabs(temperature) < INFINITY) || (temperature > 0.0f && !draws)) {
        set_error("verify: temperature %g%s", (double)temperature, draws ? "" : ", no draws");
        return -1;
    }
    if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0) { set_error("the verify workspace must be 16-byte aligned"); return -1; }
    const uint64_t rb = (uint64_t)requests * sizeof(int), db = rb * drafts, tb = rb * (drafts + 1);
    if (overlap(tokens, tb, accepted, rb) || overlap(tokens, tb, draft_tokens, db) || overlap(accepted, rb, draft_tokens, db) ||
        (counts && (overlap(tokens, tb, counts, rb) || overlap(accepted, rb, counts, rb))) ||
        (draws && (overlap(tokens, tb, draws, tb) || overlap(accepted, rb, draws, tb)))) {
        set_error("verify: outputs overlap inputs or one another");
        return -1;
    }
    return launch_verify(logits, ld, draft_logits, draft_ld, n, requests, drafts, draft_tokens, counts, temperature, draws, tokens,
                         accepted, workspace, as_stream(stream));
}

}  // extern "C"
