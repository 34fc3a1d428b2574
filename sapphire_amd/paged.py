"""The paged key-value cache and the operators that serve from it (include/paged.h, and the rows of heads
and beam search of include/sapphire_hip.h). Arrays are device addresses (an int, or an object with
.ptr such as DeviceArray); errors raise."""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import load
from ._lib import AttentionC, PageTableC, PagedCacheC, RopeC, RowsC
from .device import DeviceArray, check

ROPE_PLAIN, ROPE_LINEAR, ROPE_BASE, ROPE_PARTS = range(4)


def _at(a):
    return getattr(a, "ptr", a)


def Rows(data, dtype, tokens, heads, head_dim, token_stride=None, head_stride=None) -> RowsC:
    """Rows of heads, [tokens][heads][head_dim] unless strides (in elements) say otherwise."""
    head_stride = head_dim if head_stride is None else head_stride
    return RowsC(_at(data), dtype, tokens, heads, head_dim, heads * head_stride if token_stride is None else token_stride,
                 head_stride)


def PageTable(pages, rows, ld) -> PageTableC:
    """rows x ld page numbers, int32 in device memory."""
    return PageTableC(_at(pages), rows, ld)


def rope_frequencies(rotary_dim, base, scaling=ROPE_PLAIN, factor=1.0, trained=0.0, low=0.0, high=0.0):
    """(float64 [rotary_dim / 2], magnitude): the frequencies that rope() takes, on the host."""
    out, mag = np.empty(max(rotary_dim // 2, 0), np.float64), C.c_float()
    check(load().sapphire_rope_frequencies(out.ctypes.data, C.byref(mag), rotary_dim, base, scaling, factor, trained, low,
                                           high), "rope frequencies")
    return out, mag.value


def rope(x: RowsC, y: RowsC, positions, freqs, rotary_dim, interleaved=False, magnitude=1.0, stream=None) -> None:
    """y = x with the first rotary_dim dims of every head turned by its token's position; y may be x."""
    r = RopeC(_at(freqs), rotary_dim, int(interleaved), magnitude)
    check(load().sapphire_rope_rows_dev(C.byref(x), C.byref(y), _at(positions), C.byref(r), stream), "rope")


def beam_workspace_bytes(n, requests, beams) -> int:
    return load().sapphire_beam_workspace_bytes(n, requests, beams)


def beam_select(logits, ld, n, requests, beams, scores, scores_out, tokens, parents, workspace, done=None, done_out=None,
                end_token=-1, stream=None) -> None:
    """The best `beams` continuations of each request's beams."""
    check(load().sapphire_beam_select_dev(_at(logits), ld, n, requests, beams, _at(scores), _at(done), end_token,
                                          _at(scores_out), _at(tokens), _at(parents), _at(done_out), _at(workspace), stream),
          "beam select")


class PagedCache:
    """Pages of K and V rows of every layer. k and v: device buffers of `nbytes` each; allocated when not given."""

    def __init__(self, dtype, layers, pages, page_size, n_kv_heads, head_dim, k=None, v=None):
        self.c = PagedCacheC(None, None, dtype, layers, pages, page_size, n_kv_heads, head_dim)
        self.ref = C.byref(self.c)
        self.nbytes = load().sapphire_paged_cache_bytes(self.ref)
        if not self.nbytes:
            raise ValueError(load().sapphire_last_error().decode(errors="replace"))
        self.k = DeviceArray(self.nbytes) if k is None else k
        self.v = DeviceArray(self.nbytes) if v is None else v
        self.c.k, self.c.v = _at(self.k), _at(self.v)

    def write(self, layer, k: RowsC, v: RowsC, table: PageTableC, positions, seqs=None, stream=None) -> None:
        check(load().sapphire_paged_write_dev(self.ref, layer, C.byref(k), C.byref(v), C.byref(table), _at(seqs),
                                              _at(positions), stream), "paged write")

    def read(self, layer, k: RowsC, v: RowsC, table: PageTableC, positions, seqs=None, stream=None) -> None:
        check(load().sapphire_paged_read_dev(self.ref, layer, C.byref(k), C.byref(v), C.byref(table), _at(seqs),
                                             _at(positions), stream), "paged read")

    def attention_workspace_bytes(self, batch, n_heads, max_length) -> int:
        return load().sapphire_paged_attention_workspace_bytes(self.ref, batch, n_heads, max_length)

    def attention(self, layer, q: RowsC, out: RowsC, table: PageTableC, lengths, max_length, scale, window=0, softcap=0.0,
                  lse=None, workspace=None, stream=None) -> None:
        """out[b] = attention of q[b] over the lengths[b] positions of table row b."""
        a = AttentionC(scale, window, softcap)
        check(load().sapphire_paged_attention_dev(self.ref, layer, C.byref(q), C.byref(out), C.byref(table), _at(lengths),
                                                  max_length, C.byref(a), _at(lse), _at(workspace), stream), "paged attention")

    def reorder(self, table: PageTableC, parents, lengths, spare, table_out: PageTableC, lengths_out, stream=None) -> None:
        """Row b of table_out continues row parents[b] of table."""
        check(load().sapphire_paged_reorder_dev(self.ref, C.byref(table), _at(parents), _at(lengths), _at(spare),
                                                C.byref(table_out), _at(lengths_out), stream), "paged reorder")
