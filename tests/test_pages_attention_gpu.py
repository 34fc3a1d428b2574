"""Attention over chosen pages on the GPU against plain numpy in 64 bits, with the attention's own error bound; the choice before it
and a decode step through all of it."""
import numpy as np
import pytest

from tests import paged_ref as ref
from tests.paged_ref import BF16, F16, F32, Q4_0, Q8_0
from tests.test_page_choice_gpu import page_bounds, select64, values
from tests.test_paged_gpu import IDS, IO, Cache, Graph, dev, device_rows, sync, tables

pytestmark = pytest.mark.gpu


class Case:
    """A cache of ragged sequences (NaN behind their last positions), q, and outputs between guards."""

    def __init__(self, rng, cache, io, hd, nkv, heads, ps, lens, order="thd", pad=0, peak=2.0):
        from sapphire_amd.paged import PageTable
        self.cache, self.io, self.hd, self.nkv, self.heads, self.ps, self.lens = cache, io, hd, nkv, heads, ps, lens
        self.table, pages = tables(rng, lens, ps)
        self.c = Cache(cache, 1, pages, ps, nkv, hd)
        self.k, self.v, self.scale = [], [], hd**-0.5
        for s, n in enumerate(lens):
            k, v = (rng.normal(size=(n, nkv, hd)).astype(np.float32) for _ in range(2))
            self.c.fill(0, self.table, s, k, v)
            self.k.append(ref.stored(cache, k))
            self.v.append(ref.stored(cache, v))
        self.c.upload()
        self.rq = device_rows((rng.normal(size=(len(lens), heads, hd)) * peak).astype(np.float32), io, order, pad)
        self.ro = device_rows(np.zeros((len(lens), heads, hd), np.float32), io, order, pad)
        self.q = ref.from_type(io, self.rq[3].copy())
        self.dt, self.dn, self.lse = dev(self.table), dev(np.array(lens, np.int32)), dev(np.full((len(lens), heads), 5, np.float32))
        self.pt = PageTable(self.dt, *self.table.shape)
        self.ws = None

    def run(self, sel, window=0, cap=0.0, stream=None):
        from sapphire_amd.device import DeviceArray
        k = sel.shape[2]
        self.ws = self.ws or DeviceArray(max(1, self.c.c.attention_workspace_bytes(len(self.lens), self.heads, k * self.ps)))
        self.sel = dev(sel.astype(np.int32))
        self.c.c.pages_attention(0, self.rq[0], self.ro[0], self.pt, self.dn, self.sel, k, self.scale, window=window, softcap=cap, lse=self.lse,
                                 workspace=self.ws, stream=stream)

    def check(self, sel, window=0, cap=0.0):
        sync()
        raw = self.ro[1].numpy()
        self.ro[2][...] = raw
        got, lse = ref.from_type(self.io, self.ro[3].copy()).astype(np.float64), self.lse.numpy()
        g = self.heads // self.nkv
        for s, n in enumerate(self.lens):
            for h in range(self.nkv):
                keep = np.zeros(max(n, 1), bool)
                for i in sel[s, h]:
                    if i >= 0 and i * self.ps < n and 0 <= self.table[s, i] < self.c.pool["k"].a.shape[1]:
                        keep[i * self.ps:(i + 1) * self.ps] = True
                keep[:max(0, n - window) if window > 0 else 0] = False
                keep = keep[:n]
                q = self.q[s, h * g:(h + 1) * g]
                out, l, size, mean = ref.attention64(q, self.k[s][keep][:, h:h + 1], self.v[s][keep][:, h:h + 1], float(np.float32(self.scale)), 0, cap)
                tol, ltol = ref.attention_bound(self.io, self.io != F32, self.hd, int(keep.sum()), out, l, size, mean, cap)
                at = slice(h * g, (h + 1) * g)
                worst = np.max(np.abs(got[s, at] - out) / tol)
                assert worst <= 1, (s, h, n, worst)
                dead = np.isneginf(l)
                assert np.array_equal(np.isneginf(lse[s, at]), dead) and (got[s, at][dead] == 0).all()
                assert (np.abs(lse[s, at][~dead] - l[~dead]) <= ltol[~dead]).all(), (s, h, n)


def chosen(rng, lens, nkv, ps, k, order=True):
    """Different places per list, short lists padded by -1, which also stand between the places."""
    out = np.full((len(lens), nkv, k), -1)
    for s, n in enumerate(lens):
        for h in range(nkv):
            p = rng.permutation(-(-n // ps))[:k]
            out[s, h, :len(p)] = np.sort(p) if order else p
    return out


LENS = [0, 1, 15, 16, 17, 100, 333, 700]


@pytest.mark.parametrize("cache,io", IO, ids=IDS)
@pytest.mark.parametrize("hd,nkv,heads,ps", [(64, 1, 4, 16), (128, 3, 3, 48), (256, 1, 4, 64), (128, 2, 16, 32), (64, 2, 34, 16), (256, 2, 10, 48)])
def test_pages(hip, cache, io, hd, nkv, heads, ps):
    """Lists of one page, of some, and of more than there are; each K/V head its own."""
    rng = np.random.default_rng(hd + heads)
    c = Case(rng, cache, io, hd, nkv, heads, ps, LENS)
    for k in (1, 5, 60):
        c.ws = None
        sel = chosen(rng, LENS, nkv, ps, k, order=k != 5)
        c.run(sel)
        c.check(sel)


@pytest.mark.parametrize("cache,io", [(F32, F32), (BF16, BF16), (Q8_0, F32), (Q4_0, F16)], ids=["f32", "bf16", "q8_0_f32", "q4_0_f16"])
def test_places_that_do_not_exist(hip, cache, io):
    """Negative places, places behind the end and the table, -1 between places, rows of the table without a page."""
    rng = np.random.default_rng(2)
    c = Case(rng, cache, io, 64, 2, 4, 16, [200, 90, 40], order="htd", pad=5)
    c.table[0, 3] = -1
    c.table[0, 5] = 10**6
    c.dt.upload(c.table)
    for sel in ([[[0, 3, 5, 9, 12, -1], [-1, 3, 12, -5, 2, 1]], [[5, 6, 7, -1, -1, -1], [2**30, 5, 2**31 - 1, 0, -2**31, 3]],
                 [[-1] * 6, [3, 4, 5, 6, 7, 8]]],):
        sel = np.array(sel)
        # of a list, the first ceil(n / page_size) places count
        want = sel.copy()
        for s, n in enumerate(c.lens):
            want[s, :, -(-n // 16):] = -1
        want = np.where(want > 10**6, -1, want)
        c.run(sel)
        c.check(want)


@pytest.mark.parametrize("cache,io", [(F32, F32), (F16, F16), (Q8_0, BF16)], ids=["f32", "f16", "q8_0_bf16"])
@pytest.mark.parametrize("window,cap", [(1, 0.0), (100, 0.0), (333, 30.0), (0, 5.0)])
def test_window_and_cap(hip, cache, io, window, cap):
    rng = np.random.default_rng(window)
    c = Case(rng, cache, io, 128, 1, 6, 48, [1, 99, 100, 101, 700], peak=4.0)
    sel = chosen(rng, c.lens, 1, 48, 12)
    c.run(sel, window, cap)
    c.check(sel, window, cap)


@pytest.mark.parametrize("cache,io", [(BF16, BF16), (Q4_0, F32), (F32, F32)], ids=["bf16", "q4_0_f32", "f32"])
def test_long_lists_and_many_sequences(hip, cache, io):
    """Lists cut into pieces; and enough sequences that they are not cut and the longest go first."""
    rng = np.random.default_rng(9)
    c = Case(rng, cache, io, 64, 1, 4, 64, [5000, 130, 0])
    sel = chosen(rng, c.lens, 1, 64, 70)
    c.run(sel)
    c.check(sel)
    c = Case(rng, cache, io, 64, 4, 8, 16, [int(n) for n in rng.integers(0, 90, 300)])
    sel = chosen(rng, c.lens, 4, 16, 3)
    c.run(sel)
    c.check(sel)


def test_all_pages_are_the_whole_attention(hip):
    """A list of all pages in order: what the attention over all positions gives, bit for bit, as the walk is the same."""
    rng = np.random.default_rng(10)
    for cache, io in ((F32, F32), (BF16, BF16), (Q8_0, F32)):
        c = Case(rng, cache, io, 128, 2, 4, 32, [96, 64, 320, 0])
        sel = np.broadcast_to(np.where(np.arange(10) < np.array([3, 2, 10, 0])[:, None], np.arange(10), -1)[:, None], (4, 2, 10))
        c.run(sel)
        sync()
        a, la = c.ro[1].numpy(), c.lse.numpy()
        c.c.c.attention(0, c.rq[0], c.ro[0], c.pt, c.dn, 320, 128**-0.5, lse=c.lse, workspace=c.ws)
        sync()
        np.testing.assert_array_equal(a, c.ro[1].numpy())
        np.testing.assert_array_equal(la, c.lse.numpy())


@pytest.mark.parametrize("cache,io", [(F32, F32), (BF16, BF16), (Q8_0, F32)], ids=["f32", "bf16", "q8_0"])
def test_step(hip, cache, io):
    """Decode steps as a program takes them, captured and replayed as the sequences grow: the new rows, their pages' bounds, the
    choice, the attention over it."""
    from sapphire_amd.device import DeviceArray
    from sapphire_amd.paged import Rows
    rng = np.random.default_rng(11)
    hd, nkv, heads, ps, batch, k = 64, 2, 6, 16, 3, 6
    lens = np.array([150, 31, 20])
    c = Case(rng, cache, io, hd, nkv, heads, ps, [170, 48, 48])        # room for the steps; rows there are overwritten
    f16 = cache == F16
    bounds, sel = DeviceArray(c.c.c.bounds_bytes), dev(np.zeros((batch, nkv, k), np.int32))
    pages = c.c.pool["k"].a.shape[1]
    top = c.table.shape[1] * ps
    ws = [DeviceArray(n) for n in (c.c.c.select_workspace_bytes(batch, top), max(1, c.c.c.attention_workspace_bytes(batch, heads, k * ps)))]
    new = [dev(np.zeros((batch, nkv, hd), ref.np_type(io))) for _ in range(2)]
    pos, n = dev(lens.astype(np.int32)), dev(lens.astype(np.int32))
    c.c.c.bounds(0, bounds, c.pt, n, 200)

    def step(stream):
        c.c.c.write(0, *(Rows(x, io, batch, nkv, hd) for x in new), c.pt, pos, stream=stream)
        c.c.c.bounds(0, bounds, c.pt, n, 1, start=pos, stream=stream)
        c.c.c.select(0, bounds, c.rq[0], c.pt, n, top, sel, k, first=1, last=2, workspace=ws[0], stream=stream)
        c.c.c.pages_attention(0, c.rq[0], c.ro[0], c.pt, n, sel, k, hd**-0.5, lse=c.lse, workspace=ws[1], stream=stream)

    g = Graph(step)
    for _ in range(14):                                # a page ends on the way
        x = [rng.normal(size=(batch, nkv, hd)).astype(np.float32) for _ in range(2)]
        for d, a, held in zip(new, x, (c.k, c.v)):
            raw = ref.to_type(io, a)
            d.upload(raw)
            for s in range(batch):
                held[s][lens[s]] = ref.stored(cache, ref.from_type(io, raw[s]))
        pos.upload(lens.astype(np.int32))
        lens = lens + 1
        n.upload(lens.astype(np.int32))
        sync()
        g.replay()
        sync()
        b = np.zeros((pages, nkv, 2, hd), np.uint16)
        for s in range(batch):
            for i in range(-(-lens[s] // ps)):
                held = c.k[s][i * ps:min(lens[s], (i + 1) * ps)]
                b[c.table[s, i]] = page_bounds(F32 if cache == Q8_0 else cache, held)
        got = bounds.numpy().view(np.uint16).reshape(b.shape)
        for s in range(batch):
            rows = c.table[s, :-(-lens[s] // ps)]
            np.testing.assert_array_equal(values(got[rows], f16), values(b[rows], f16))
        want = select64(c.q, values(got, f16), c.table, list(lens), ps, k, 1, 2, pages, top)
        np.testing.assert_array_equal(sel.numpy(), want)
        c.lens = list(lens)
        held = c.k, c.v
        c.k, c.v = ([a[s][:lens[s]] for s in range(batch)] for a in held)
        c.check(want)
        c.k, c.v = held
    g.close()


def test_pages_past_four_gigabytes(hip):
    """The same rows in the first pages and in the last ones of pools of more than 2^32 bytes: the same bounds, choice and outputs."""
    from sapphire_amd.device import DeviceArray
    from sapphire_amd.paged import PagedCache, PageTable
    rng = np.random.default_rng(12)
    hd, ps, pages, heads, n, chosen_pages = 256, 64, 70000, 4, 700, 4
    c = PagedCache(F32, 1, pages, ps, 1, hd)
    assert c.nbytes > 2**32
    ld = -(-n // ps)
    k, v = (device_rows(rng.normal(size=(n, 1, hd)).astype(np.float32), F32) for _ in range(2))
    q = device_rows(rng.normal(size=(1, heads, hd)).astype(np.float32), F32)
    at, seqs, lens = dev(np.arange(n, dtype=np.int32)), dev(np.zeros(n, np.int32)), dev(np.array([n], np.int32))
    bounds, got = DeviceArray(c.bounds_bytes), []
    ws = [DeviceArray(max(1, b)) for b in (c.select_workspace_bytes(1, n), c.attention_workspace_bytes(1, heads, chosen_pages * ps))]
    for first in (0, pages - ld):
        t = dev(np.arange(first, first + ld, dtype=np.int32)[None])
        pt = PageTable(t, 1, ld)
        o, sel = device_rows(np.zeros((1, heads, hd), np.float32), F32), dev(np.zeros((1, 1, chosen_pages), np.int32))
        c.write(0, k[0], v[0], pt, at, seqs=seqs)
        c.bounds(0, bounds, pt, lens, n)
        c.select(0, bounds, q[0], pt, lens, n, sel, chosen_pages, workspace=ws[0])
        c.pages_attention(0, q[0], o[0], pt, lens, sel, chosen_pages, hd**-0.5, workspace=ws[1])
        sync()
        b = bounds.numpy().view(np.uint16).reshape(pages, 2, hd)[first:first + ld]
        got.append((b, sel.numpy(), o[1].numpy()))
    for x, y in zip(*got):
        np.testing.assert_array_equal(x, y)
    want = np.stack([page_bounds(F32, k[3][i * ps:(i + 1) * ps])[0] for i in range(ld)])
    np.testing.assert_array_equal(values(got[0][0], False), values(want, False))
    for d in (c.k, c.v):
        d.free()


@pytest.mark.parametrize("cache,io", IO, ids=IDS)
def test_scales(hip, cache, io):
    """Scales below 0 and of 0; lists that end inside a piece."""
    rng = np.random.default_rng(13)
    for scale in (-0.15, 0.0):
        c = Case(rng, cache, io, 64, 2, 6, 16, [200, 33, 5])
        c.scale = scale
        sel = chosen(rng, c.lens, 2, 16, 7)
        c.run(sel)
        c.check(sel)


def test_calls_at_once(hip):
    """Choice and attention under way on two streams, each in workspaces of its own: the same as alone."""
    from tests.test_page_choice_gpu import Select
    rng = np.random.default_rng(14)
    cases = [Case(rng, BF16, BF16, 128, 2, 8, 32, [3000, 500]), Case(rng, Q8_0, F32, 64, 1, 4, 16, [900, 100, 5])]
    chooses = [Select(rng, BF16, BF16, 2, 8, 128, 32, [32 * 9000, 32 * 100]), Select(rng, Q4_0, F32, 1, 3, 64, 16, [16 * 500])]
    lists = [chosen(rng, c.lens, c.nkv, c.ps, 20) for c in cases]
    streams = [hip.sapphire_stream_create() for _ in cases]
    want, keep = [], []
    for c, sel in zip(cases, lists):
        c.run(sel)
        c.check(sel)
        want.append(c.ro[1].numpy())
    for _ in range(4):
        outs = []
        for _ in range(6):
            for c, s, sel, stream in zip(cases, chooses, lists, streams):
                c.run(sel, stream=stream)
                keep.append(c.sel)                     # (the list is read after the call returns)
                outs.append((s, s.run(50, 1, 1, stream=stream)))
        sync()
        for c, w in zip(cases, want):
            np.testing.assert_array_equal(c.ro[1].numpy(), w)
        for s, o in outs[-2:]:
            np.testing.assert_array_equal(o.numpy(), s.want(50, 1, 1))
    for s in streams:
        hip.sapphire_stream_destroy(s)
