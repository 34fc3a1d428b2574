// paged_dev.h - the paged cache's layout and the launchers of its kernels (not installed).
//
// A tile is one page of one K/V head. K tiles keep 16 positions x 16 bytes together, so that a load of
// a wave (lane (c, m): position c, chunk m) is one contiguous KiB and each lane's 16 bytes are its part
// of the score product's operand; V tiles keep the hd/16 dims of a lane together, P positions of
// them where one position has less than 16 bytes, so that lane (c, m)'s four positions 4m .. 4m + 3
// come by 16-byte loads too.
#pragma once

#include "internal.h"

namespace sapphire {

struct PagedCache {
    uint8_t *k = nullptr, *v = nullptr;    // the layer's pools (all layers' for the reorder)
    int dtype = 0, layers = 0, pages = 0, page_size = 0, nkv = 0, hd = 0;
    uint32_t tile_bytes = 0;               // one page of one head
    uint32_t page_mul = 0, page_shift = 0; // see page_of
    size_t layer_bytes = 0;
};
struct Rows {
    uint8_t *p = nullptr;
    int dtype = 0, tokens = 0, heads = 0, hd = 0;
    int64_t ts = 0, hs = 0;                // strides in elements
};
struct PageTable {
    const int *pages = nullptr;
    int rows = 0, ld = 0;
};

// Offsets in a tile, in bytes. CT: the cache's type, HD: head_dim.
template <int CT, int HD>
struct Tile {
    static constexpr bool kQuant = CT == DT_Q8_0 || CT == DT_Q4_0;
    static constexpr int NB = HD / 32;                                         // quant blocks of a row
    static constexpr int ROW = CT == DT_F32 ? 4 * HD : CT == DT_Q8_0 ? HD : CT == DT_Q4_0 ? HD / 2 : 2 * HD;   // code bytes
    static constexpr int RUN = ROW / 16;                                       // V: bytes of hd / 16 dims
    static constexpr int P = RUN >= 16 ? 1 : 16 / RUN > 4 ? 4 : 16 / RUN;      // V: positions together
    static constexpr int G = NB < 4 ? NB : 4;                                  // K, Q4_0: blocks of a chunk
    // K: the bytes of dims d .. d + 7 (d % 8 == 0; F32: of d .. d + 3) of position p
    __host__ __device__ static uint32_t k_code(uint32_t p, uint32_t d) {
        const uint32_t t = p >> 4, c = p & 15, b = d >> 5, m = (d >> 3) & 3;
        if constexpr (CT == DT_F32) return ((t * (HD / 4) + (d >> 2)) * 16 + c) * 16;
        else if constexpr (CT == DT_Q8_0) return (((t * (NB / 2) + (b >> 1)) * 4 + m) * 16 + c) * 16 + (b & 1) * 8;
        else if constexpr (CT == DT_Q4_0) return (((t * (NB / G) + b / G) * 4 + m) * 16 + c) * (4 * G) + b % G * 4;
        else return ((t * (HD / 8) + (d >> 3)) * 16 + c) * 16;
    }
    // V: run r (dims r * hd / 16 and on) of position p
    __host__ __device__ static uint32_t v_run(uint32_t p, uint32_t r) {
        return ((p / P * 16 + r) * P + p % P) * RUN;
    }
    __host__ __device__ static uint32_t k_scale(uint32_t ps, uint32_t p, uint32_t b) { return ps * ROW + (p * NB + b) * 4; }
    __host__ __device__ static uint32_t v_scale(uint32_t ps, uint32_t p, uint32_t b) {
        return ps * ROW + ((p / 4 * NB + b) * 4 + p % 4) * 4;
    }
    static constexpr uint32_t bytes(int ps) { return (uint32_t)ps * (ROW + (kQuant ? NB * 4 : 0)); }
};

// The page of a row that 16 positions belong to, t16 / d with d = page_size / 16 (at most 64) and t16 < 2^27: a power of two
// by a shift, others by the high product with ceil(2^33 / d) < 2^32, which is off by less than 2^6 / 2^33 relative to 1 / d:
// t16 times that is less than 1 / d.
inline void set_page_division(PagedCache &c) {
    const uint32_t d = (uint32_t)c.page_size / 16;
    if ((d & (d - 1)) == 0) {
        c.page_mul = 0;
        c.page_shift = (uint32_t)__builtin_ctz(d);
    } else {
        c.page_mul = (uint32_t)((((uint64_t)1 << 33) + d - 1) / d);
        c.page_shift = 1;
    }
}
__device__ __forceinline__ uint32_t page_of(const PagedCache &c, uint32_t t16) {
    return (c.page_mul ? __umulhi(t16, c.page_mul) : t16) >> c.page_shift;
}

// Where position pos of a table row lies: its page and the position in it, or false.
__device__ __forceinline__ bool paged_place(const PagedCache &c, const PageTable &tab, int row, int pos, int &page, int &off) {
    if (row < 0 || row >= tab.rows || pos < 0) return false;
    const uint32_t i = page_of(c, (uint32_t)pos >> 4);
    if (i >= (uint32_t)tab.ld) return false;
    page = tab.pages[(size_t)row * tab.ld + i];
    off = pos - (int)(i * (uint32_t)c.page_size);
    return page >= 0 && page < c.pages;
}

typedef float pf4 __attribute__((ext_vector_type(4)));
typedef uint32_t pu4 __attribute__((ext_vector_type(4)));
typedef uint32_t pu2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ float from_bf16(uint32_t b) { return __uint_as_float(b << 16); }
__device__ __forceinline__ float from_f16(uint32_t b) { return (float)__builtin_bit_cast(_Float16, (uint16_t)b); }
__device__ __forceinline__ uint32_t to_bf16(float v) {
    const uint32_t u = __float_as_uint(v);
    if ((u & 0x7fffffffu) > 0x7f800000u) return (u >> 16) | 0x40u;             // NaN stays one
    return (u + 0x7fffu + ((u >> 16) & 1u)) >> 16;
}
__device__ __forceinline__ uint32_t to_f16(float v) { return (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v); }
__device__ __forceinline__ uint32_t to_16(int dtype, float v) { return dtype == DT_BF16 ? to_bf16(v) : to_f16(v); }
// two values in one word, the first in its lower half
typedef float pf2 __attribute__((ext_vector_type(2)));
typedef __bf16 pb2 __attribute__((ext_vector_type(2)));
typedef _Float16 ph2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t pack_16(int dtype, float a, float b) {
    const pf2 v = {a, b};
    return dtype == DT_BF16 ? __builtin_bit_cast(uint32_t, __builtin_convertvector(v, pb2)) : __builtin_bit_cast(uint32_t, __builtin_convertvector(v, ph2));
}
__device__ __forceinline__ float from_16(int dtype, uint32_t b) { return dtype == DT_BF16 ? from_bf16(b) : from_f16(b); }

// Eight consecutive elements of a row as they are, and as fp32. `wide`: the rows' data and strides are multiples of 16
// bytes. (Loading and converting are apart, so that several rows' loads are under way together.)
struct Raw8 {
    pu4 a, b;                              // b: fp32's second half
};
__device__ __forceinline__ void load8(int dtype, bool wide, const uint8_t *base, int64_t at, Raw8 &r) {
    if (dtype == DT_F32) {
        const uint32_t *p = reinterpret_cast<const uint32_t *>(base) + at;
        if (wide) {
            r.a = *reinterpret_cast<const pu4 *>(p);
            r.b = *reinterpret_cast<const pu4 *>(p + 4);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                r.a[i] = p[i];
                r.b[i] = p[4 + i];
            }
        }
    } else {
        const uint16_t *p = reinterpret_cast<const uint16_t *>(base) + at;
        if (wide) {
            r.a = *reinterpret_cast<const pu4 *>(p);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) r.a[i] = (uint32_t)p[2 * i] | (uint32_t)p[2 * i + 1] << 16;
        }
    }
}
__device__ __forceinline__ void values8(int dtype, const Raw8 &r, float (&x)[8]) {
    if (dtype == DT_F32) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[i] = __uint_as_float(r.a[i]);
            x[4 + i] = __uint_as_float(r.b[i]);
        }
    } else if (dtype == DT_BF16) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(i & 1 ? r.a[i / 2] & 0xffff0000u : r.a[i / 2] << 16);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = from_f16(i & 1 ? r.a[i / 2] >> 16 : r.a[i / 2] & 0xffffu);
    }
}

__device__ __forceinline__ void store8(int dtype, bool wide, uint8_t *base, int64_t at, const float (&x)[8]) {
    if (dtype == DT_F32) {
        float *p = reinterpret_cast<float *>(base) + at;
        if (wide) {
            *reinterpret_cast<pf4 *>(p) = pf4{x[0], x[1], x[2], x[3]};
            *reinterpret_cast<pf4 *>(p + 4) = pf4{x[4], x[5], x[6], x[7]};
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) p[i] = x[i];
        }
    } else {
        uint16_t *p = reinterpret_cast<uint16_t *>(base) + at;
        pu4 w;
        if (dtype == DT_BF16) {
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = pack_16(DT_BF16, x[2 * i], x[2 * i + 1]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = pack_16(DT_F16, x[2 * i], x[2 * i + 1]);
        }
        if (wide) {
            *reinterpret_cast<pu4 *>(p) = w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) p[i] = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
        }
    }
}

// Elements d .. d + 7 of position p of a tile of K or V.
template <int CT, int HD, bool V>
__device__ __forceinline__ void load_codes(const uint8_t *tile, uint32_t ps, uint32_t p, uint32_t d, float (&x)[8]) {
    using T = Tile<CT, HD>;
    if constexpr (CT == DT_F32) {
        const uint8_t *a = V ? tile + p * T::ROW + d * 4 : tile + T::k_code(p, d);
        const uint8_t *b = V ? a + 16 : tile + T::k_code(p, d + 4);
        const pf4 u = *reinterpret_cast<const pf4 *>(a), w = *reinterpret_cast<const pf4 *>(b);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[i] = u[i];
            x[4 + i] = w[i];
        }
    } else if constexpr (!T::kQuant) {
        pu4 w;
        if constexpr (V && HD == 64) {
            const pu2 a = *reinterpret_cast<const pu2 *>(tile + T::v_run(p, d / 4));
            const pu2 b = *reinterpret_cast<const pu2 *>(tile + T::v_run(p, d / 4 + 1));
            w = pu4{a.x, a.y, b.x, b.y};
        } else {
            w = *reinterpret_cast<const pu4 *>(tile + (V ? p * T::ROW + d * 2 : T::k_code(p, d)));
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = from_16(CT, w[i] & 0xffffu);
            x[2 * i + 1] = from_16(CT, w[i] >> 16);
        }
    } else {
        const float scale = *reinterpret_cast<const float *>(tile + (V ? T::v_scale(ps, p, d / 32) : T::k_scale(ps, p, d / 32)));
        if constexpr (CT == DT_Q8_0) {
            uint32_t lo, hi;
            if constexpr (V && HD == 64) {
                lo = *reinterpret_cast<const uint32_t *>(tile + T::v_run(p, d / 4));
                hi = *reinterpret_cast<const uint32_t *>(tile + T::v_run(p, d / 4 + 1));
            } else {
                const pu2 w = *reinterpret_cast<const pu2 *>(tile + (V ? T::v_run(p, d / T::RUN) + d % T::RUN : T::k_code(p, d)));
                lo = w.x;
                hi = w.y;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[i] = __fmul_rn((float)(int8_t)(lo >> (8 * i)), scale);
                x[4 + i] = __fmul_rn((float)(int8_t)(hi >> (8 * i)), scale);
            }
        } else {
            uint32_t lo, hi;                           // codes 0..3 and 4..7, one nibble per byte
            if constexpr (!V) {
                const uint32_t w = *reinterpret_cast<const uint32_t *>(tile + T::k_code(p, d)) ^ 0x88888888u;
                lo = w & 0x0f0f0f0fu;
                hi = w >> 4 & 0x0f0f0f0fu;
            } else if constexpr (HD == 256) {
                const pu2 w = *reinterpret_cast<const pu2 *>(tile + T::v_run(p, d / 16));
                const uint32_t sh = d & 8 ? 4 : 0;
                lo = w.x >> sh & 0x0f0f0f0fu;
                hi = w.y >> sh & 0x0f0f0f0fu;
            } else if constexpr (HD == 128) {
                const uint32_t w = *reinterpret_cast<const uint32_t *>(tile + T::v_run(p, d / 8));
                lo = w & 0x0f0f0f0fu;
                hi = w >> 4 & 0x0f0f0f0fu;
            } else {
                const uint32_t a = *reinterpret_cast<const uint16_t *>(tile + T::v_run(p, d / 4));
                const uint32_t b = *reinterpret_cast<const uint16_t *>(tile + T::v_run(p, d / 4 + 1));
                lo = (a & 0x0f0fu) | (a >> 4 & 0x0f0fu) << 16;
                hi = (b & 0x0f0fu) | (b >> 4 & 0x0f0fu) << 16;
            }
            asm("" : "+v"(lo), "+v"(hi));              // (the compiler would rather extract nibbles one by one)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[i] = __fmul_rn(__fsub_rn((float)(lo >> (8 * i) & 255u), 8.0f), scale);
                x[4 + i] = __fmul_rn(__fsub_rn((float)(hi >> (8 * i) & 255u), 8.0f), scale);
            }
        }
    }
}

inline int elem_bytes(int dt) { return dt == DT_F32 ? 4 : 2; }
// Data and strides in whole 16-byte pieces.
inline bool rows_wide(const Rows &r) {
    const int es = elem_bytes(r.dtype);
    return reinterpret_cast<uintptr_t>(r.p) % 16 == 0 && (r.tokens == 1 || r.ts * es % 16 == 0) &&
           (r.heads == 1 || r.hs * es % 16 == 0);
}

// ---- launchers (arguments checked by the callers) ----
int launch_rope_rows(const Rows &x, const Rows &y, const int *positions, const double *freqs, int rot, bool interleaved,
                     float magnitude, hipStream_t s);
int launch_paged_write(const PagedCache &c, const Rows &k, const Rows &v, const PageTable &t, const int *seqs,
                       const int *positions, hipStream_t s);
int launch_paged_read(const PagedCache &c, const Rows &k, const Rows &v, const PageTable &t, const int *seqs,
                      const int *positions, hipStream_t s);
int launch_paged_reorder(const PagedCache &c, const PageTable &t, const int *parents, const int *lengths, const int *spare,
                         int *table_out, int *lengths_out, hipStream_t s);
struct PagedAttn {
    PagedCache c;
    Rows q, out;
    PageTable table;
    const int *lengths = nullptr;
    int max_length = 0, window = 0;
    float scale = 1.f, softcap = 0.f;
    float *lse = nullptr;
    uint8_t *ws = nullptr;
    const int *selected = nullptr;         // attention over chosen pages: [batch][K/V heads][listed]
    int listed = 0;
    const int *shared = nullptr;           // attention of groups of rows: their first positions that are the same
    int rows = 1, max_own = 0;             // rows of a group; about how many positions each has behind those
};
size_t paged_attention_workspace(int dtype, int nkv, int hd, int batch, int n_heads, int max_length);
int launch_paged_attention(const PagedAttn &a, hipStream_t s);
int launch_paged_pages_attention(const PagedAttn &a, hipStream_t s);
size_t paged_shared_workspace(int dtype, int nkv, int hd, int batch, int n_heads, int max_length);
int launch_paged_shared_attention(const PagedAttn &a, hipStream_t s);
int launch_paged_bounds(const PagedCache &c, uint16_t *bounds, const PageTable &t, const int *from, const int *lengths, int max_new,
                        hipStream_t s);
size_t paged_select_workspace(int nkv, int batch, int max_pages);
int launch_paged_select(const PagedCache &c, const uint16_t *bounds, const Rows &q, const PageTable &t, const int *lengths, int max_length,
                        int k, int first, int last, int *selected, void *ws, hipStream_t s);
size_t beam_workspace_bytes(int n, int rows, int beams);
int launch_beam_select(const float *logits, int ld, int n, int requests, int beams, const float *scores, const int *done,
                       int end_token, float *scores_out, int *tokens, int *parents, int *done_out, void *ws,
                       hipStream_t s);
size_t verify_workspace_bytes(int n, int requests, int drafts);
int launch_verify(const float *logits, int ld, const float *draft_logits, int draft_ld, int n, int requests, int drafts,
                  const int *draft_tokens, const int *counts, float temperature, const float *draws, int *tokens, int *accepted,
                  void *ws, hipStream_t s);

}  // namespace sapphire
