"""The paged key-value cache and the operators that serve from it (include/paged.h, and the rows of heads
and beam search of include/sapphire_hip.h). Arrays are device addresses (an int, or an object with
.ptr such as DeviceArray); errors raise."""
from __future__ import annotations

import ctypes as C
from ctypes import byref

import numpy as np

from . import load
from ._lib import AttentionC, PageTableC, PagedCacheC, RopeC, RowsC
from .device import DeviceArray, check

ROPE_PLAIN, ROPE_LINEAR, ROPE_BASE, ROPE_PARTS = range(4)


def _at(a):
    return a if a is None or type(a) is int else getattr(a, "ptr", a)


def Rows(data, dtype, tokens, heads, head_dim, token_stride=None, head_stride=None) -> RowsC:
    """Rows of heads, [tokens][heads][head_dim] unless strides (in elements) say otherwise."""
    if head_stride is None:
        head_stride = head_dim
    if token_stride is None:
        token_stride = heads * head_stride
    return RowsC(data if type(data) is int else _at(data), dtype, tokens, heads, head_dim, token_stride, head_stride)


def PageTable(pages, rows, ld) -> PageTableC:
    """rows x ld page numbers, int32 in device memory."""
    return PageTableC(pages if type(pages) is int else _at(pages), rows, ld)


def rope_frequencies(rotary_dim, base, scaling=ROPE_PLAIN, factor=1.0, trained=0.0, low=0.0, high=0.0):
    """(float64 [rotary_dim / 2], magnitude): the frequencies that rope() takes, on the host."""
    out, mag = np.empty(max(rotary_dim // 2, 0), np.float64), C.c_float()
    check(load().sapphire_rope_frequencies(out.ctypes.data, byref(mag), rotary_dim, base, scaling, factor, trained, low,
                                           high), "rope frequencies")
    return out, mag.value


def rope(x: RowsC, y: RowsC, positions, freqs, rotary_dim, interleaved=False, magnitude=1.0, stream=None) -> None:
    """y = x with the first rotary_dim dims of every head turned by its token's position; y may be x."""
    r = RopeC(_at(freqs), rotary_dim, interleaved, magnitude)
    if load().sapphire_rope_rows_dev(byref(x), byref(y), _at(positions), byref(r), stream):
        check(-1, "rope")


def beam_workspace_bytes(n, requests, beams) -> int:
    return load().sapphire_beam_workspace_bytes(n, requests, beams)


def beam_select(logits, ld, n, requests, beams, scores, scores_out, tokens, parents, workspace, done=None, done_out=None,
                end_token=-1, stream=None) -> None:
    """The best `beams` continuations of each request's beams."""
    if load().sapphire_beam_select_dev(_at(logits), ld, n, requests, beams, _at(scores), _at(done), end_token, _at(scores_out),
                                       _at(tokens), _at(parents), _at(done_out), _at(workspace), stream):
        check(-1, "beam select")


class PagedCache:
    """Pages of K and V rows of every layer. k and v: device buffers of `nbytes` each; allocated when not given."""

    def __init__(self, dtype, layers, pages, page_size, n_kv_heads, head_dim, k=None, v=None):
        lib = load()
        self.c = PagedCacheC(None, None, dtype, layers, pages, page_size, n_kv_heads, head_dim)
        self.ref = byref(self.c)
        self.nbytes = lib.sapphire_paged_cache_bytes(self.ref)
        if not self.nbytes:
            raise ValueError(lib.sapphire_last_error().decode(errors="replace"))
        self.k = DeviceArray(self.nbytes) if k is None else k
        self.v = DeviceArray(self.nbytes) if v is None else v
        self.c.k, self.c.v = _at(self.k), _at(self.v)
        self._write, self._read = lib.sapphire_paged_write_dev, lib.sapphire_paged_read_dev
        self._attention, self._reorder = lib.sapphire_paged_attention_dev, lib.sapphire_paged_reorder_dev

    def write(self, layer, k: RowsC, v: RowsC, table: PageTableC, positions, seqs=None, stream=None) -> None:
        """Row t of k and v to position positions[t] of table row seqs[t] (t where seqs is None)."""
        if self._write(self.ref, layer, byref(k), byref(v), byref(table), _at(seqs), _at(positions), stream):
            check(-1, "paged write")

    def read(self, layer, k: RowsC, v: RowsC, table: PageTableC, positions, seqs=None, stream=None) -> None:
        """The reverse of write."""
        if self._read(self.ref, layer, byref(k), byref(v), byref(table), _at(seqs), _at(positions), stream):
            check(-1, "paged read")

    def attention_workspace_bytes(self, batch, n_heads, max_length) -> int:
        return load().sapphire_paged_attention_workspace_bytes(self.ref, batch, n_heads, max_length)

    def attention(self, layer, q: RowsC, out: RowsC, table: PageTableC, lengths, max_length, scale, window=0, softcap=0.0,
                  lse=None, workspace=None, stream=None) -> None:
        """out[b] = attention of q[b] over the lengths[b] positions of table row b."""
        if self._attention(self.ref, layer, byref(q), byref(out), byref(table), _at(lengths), max_length,
                           byref(AttentionC(scale, window, softcap)), _at(lse), _at(workspace), stream):
            check(-1, "paged attention")

    def reorder(self, table: PageTableC, parents, lengths, spare, table_out: PageTableC, lengths_out, stream=None) -> None:
        """Row b of table_out continues row parents[b] of table."""
        if self._reorder(self.ref, byref(table), _at(parents), _at(lengths), _at(spare), byref(table_out), _at(lengths_out), stream):
            check(-1, "paged reorder")
