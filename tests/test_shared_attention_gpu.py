"""Attention of rows that share their first positions on the GPU against plain numpy in 64 bits, with the attention's own error
bound (its spare roundings cover q's and the weights' terms: 2^-23 of an element of q, 2^-21 of a weight times a value, of
which the bound has 16 and 256 steps of 2^-24); and speculative decoding through it."""
import numpy as np
import pytest

from tests import paged_ref as ref
from tests.paged_ref import BF16, F16, F32, Q4_0, Q8_0
from tests.test_paged_gpu import IDS, IO, Cache, Graph, dev, device_rows, sync

pytestmark = pytest.mark.gpu


class Case:
    """Groups of rows: `common[g]` positions of the group's own pages, whole ones, and what each row has behind them in pages of
    its own; NaN wherever nothing is written. drafts: all rows of a group are one sequence."""

    def __init__(self, rng, cache, io, hd, nkv, heads, ps, rows, common, lens, drafts=False, order="thd", pad=0, peak=2.0, broken=()):
        from sapphire_amd.paged import PageTable
        self.cache, self.io, self.hd, self.heads, self.rows, self.lens, self.nkv = cache, io, hd, heads, rows, list(lens), nkv
        groups = -(-len(lens) // rows)
        need = [-(-max(n, 0) // ps) for n in lens]
        ld = max(1, max(need + [-(-c // ps) for c in common]))
        pages = ld * (groups + (0 if drafts else len(lens))) + 3
        order_of = iter(rng.permutation(pages))
        self.table = np.full((len(lens), ld), -1, np.int32)
        self.c = Cache(cache, 1, pages, ps, nkv, hd)
        self.k, self.v, self.scale = [], [], hd**-0.5
        for g in range(groups):
            mine = range(g * rows, min(len(lens), (g + 1) * rows))
            top = max(lens[r] for r in mine) if drafts else -(-common[g] // ps) * ps
            shared_pages = [next(order_of) for _ in range(-(-top // ps))]
            base = [rng.normal(size=(top, nkv, hd)).astype(np.float32) for _ in range(2)]
            for r in mine:
                n = max(lens[r], 0)
                self.table[r, :len(shared_pages)] = shared_pages
                for i in range(len(shared_pages), need[r]):
                    self.table[r, i] = next(order_of)
                k, v = (np.concatenate([b[:n], rng.normal(size=(max(0, n - top), nkv, hd)).astype(np.float32)]) for b in base)
                if n:
                    self.c.fill(0, self.table, r, k, v)
                self.k.append(ref.stored(cache, k))
                self.v.append(ref.stored(cache, v))
        self.c.upload()
        self.broken = [(r, i) for g, i in broken for r in range(g * rows, min(len(lens), (g + 1) * rows))]
        for r, i in self.broken:
            self.table[r, i] = pages + 3 if i % 2 else -7
        x = (rng.normal(size=(len(lens), heads, hd)) * peak).astype(np.float32)
        self.rq, self.ro = device_rows(x, io, order, pad), device_rows(x * 0 + 3, io, order, pad)
        self.q, self.ps = ref.from_type(io, self.rq[3].copy()), ps
        self.dt, self.dn = dev(self.table), dev(np.array(lens, np.int32))
        self.pt, self.top = PageTable(self.dt, *self.table.shape), max(1, max(lens))
        self.lse = dev(np.full((len(lens) + 1, heads), 5, np.float32))
        self.ws = None

    def run(self, shared, own, cap=0.0, stream=None, lse=True, out=None):
        from sapphire_amd.device import DeviceArray
        self.ws = self.ws or DeviceArray(self.c.c.shared_attention_workspace_bytes(len(self.lens), self.heads, self.top))
        self.shared = dev(np.array(shared, np.int32)) if isinstance(shared, list) else shared
        self.c.c.shared_attention(0, self.rq[0], out or self.ro[0], self.pt, self.dn, self.top, self.rows, self.shared, self.scale, max_own=own,
                                  softcap=cap, lse=self.lse if lse else None, workspace=self.ws, stream=stream)

    def got(self):
        sync()
        raw = self.ro[1].numpy()
        self.ro[2][...] = raw
        got = ref.from_type(self.io, self.ro[3].copy()).astype(np.float64)
        mask = np.ones(raw.shape, bool)
        one = np.ones_like(self.ro[2])
        np.lib.stride_tricks.as_strided(mask, got.shape, tuple(s // one.itemsize for s in self.ro[3].strides))[...] = False
        assert (raw[mask] == 7).all(), "elements between the rows were written"
        return got, self.lse.numpy()

    def check(self, cap=0.0, but=None):
        """but: a (row, head) that is NaN."""
        got, lse = self.got()
        if but:
            assert np.isnan(got[but]).all() and np.isnan(lse[but])
        assert (lse[-1] == 5).all()
        for r, n in enumerate(self.lens):
            n = min(max(n, 0), self.top)
            keep = np.ones(n, bool)
            for rr, i in self.broken:
                if rr == r:
                    keep[i * self.ps:(i + 1) * self.ps] = False
            out, l, size, mean = ref.attention64(self.q[r], self.k[r][:n][keep], self.v[r][:n][keep], float(np.float32(self.scale)), 0, cap)
            tol, ltol = ref.attention_bound(self.io, self.io != F32, self.hd, n, out, l, size, mean, cap)
            if but and but[0] == r:
                got[but], lse[but] = out[but[1]], l[but[1]]
            worst = np.max(np.abs(got[r] - out) / tol)
            assert worst <= 1, (r, n, worst)
            dead = np.isneginf(l)
            assert np.array_equal(np.isneginf(lse[r]), dead) and (got[r][dead] == 0).all()
            assert (np.abs(lse[r][~dead] - l[~dead]) <= ltol[~dead]).all(), (r, n)


SHAPES = [(64, 1, 4, 16), (128, 3, 3, 48), (256, 1, 4, 64), (128, 2, 16, 32), (64, 2, 34, 16), (256, 2, 10, 48)]


@pytest.mark.parametrize("cache,io", IO, ids=IDS)
@pytest.mark.parametrize("hd,nkv,heads,ps", SHAPES)
def test_shared(hip, cache, io, hd, nkv, heads, ps):
    """Three groups, the last with fewer rows; padded rows, the first of a group too; few positions behind the shared ones and many."""
    rng = np.random.default_rng(hd + heads)
    common = [ps * 5, ps * 12, ps]
    lens = [common[0] + n for n in (1, 17, 0, 300, 5)] + [0, common[1] + 2, common[1] + 33, 0, common[1] + 1] + [common[2] + 40, common[2] + 1]
    c = Case(rng, cache, io, hd, nkv, heads, ps, 5, common, lens)
    for own in (300, 20):                              # the attention's kernels take what is not shared, or the join does
        c.run(common, own)
        c.check()


SOME = [(F32, F32), (BF16, BF16), (BF16, F32), (F16, F32), (Q8_0, F32), (Q4_0, BF16)]


@pytest.mark.parametrize("cache,io", SOME, ids=[f"{ref.NAME[a]}-{ref.NAME[b]}" for a, b in SOME])
@pytest.mark.parametrize("rows,heads", [(1, 1), (4, 4), (5, 4), (8, 4), (9, 4), (16, 4), (17, 4), (33, 4), (3, 100)])
def test_columns(hip, cache, io, rows, heads):
    """Around the numbers of columns at which sets, waves and workgroups run out; more pieces than units, and the other way round."""
    rng = np.random.default_rng(rows * heads)
    for hd, n in ((64, 700), (128, 40), (256, 130)):
        c = Case(rng, cache, io, hd, 1, heads, 32, rows, [n // 32 * 32], [n // 32 * 32 + 1 + r % 7 for r in range(rows)])
        for own in (0, 7):
            c.run([n // 32 * 32], own)
            c.check()


@pytest.mark.parametrize("cache,io", IO, ids=IDS)
def test_drafted_tokens(hip, cache, io):
    """Rows that are the next tokens of one sequence: each sees the ones before it. shared says all that is written, some of it, or
    none; it ends inside tiles and pages."""
    rng = np.random.default_rng(3)
    lens = [n + i for n in (1, 15, 16, 60, 250, 1000) for i in range(6)]
    c = Case(rng, cache, io, 64, 2, 8, 48, 6, [0] * 6, lens, drafts=True)
    for shared in ([1, 15, 16, 60, 250, 1000], [10**9] * 6, [0] * 6, [-5, 3, 17, 47, 96, 999]):
        for own in (0, 6, 1000):
            c.run(shared, own)
            c.check()


@pytest.mark.parametrize("cache", [F32, BF16, F16, Q8_0, Q4_0], ids=ref.NAME.get)
def test_pages_that_do_not_exist(hip, cache):
    rng = np.random.default_rng(4)
    c = Case(rng, cache, F32, 64, 1, 4, 16, 4, [320, 64], [400, 321, 330, 350, 70, 65, 80, 0], broken=[(0, 0), (0, 7), (0, 8), (0, 19), (0, 20), (1, 0), (1, 1), (1, 2), (1, 3)])
    for own in (80, 32):
        c.run([320, 64], own)
        c.check()
    c = Case(rng, cache, F32, 128, 1, 2, 16, 2, [64], [64, 64], broken=[(0, i) for i in range(4)])
    c.run([64], 1)
    c.check()


@pytest.mark.parametrize("cache,io", IO, ids=IDS)
def test_cap_peaks_and_strides(hip, cache, io):
    rng = np.random.default_rng(5)
    for cap, peak, order, pad in ((30.0, 4.0, "thd", 0), (5.0, 2.0, "htd", 3), (0.0, 100.0, "thd", 192), (0.0, 0.0, "thd", 8)):
        c = Case(rng, cache, io, 128, 1, 4, 48, 8, [480], [481 + 9 * r for r in range(8)], order=order, pad=pad, peak=peak)
        for own in (64, 32):
            c.run([480], own, cap)
            c.check(cap)


@pytest.mark.parametrize("cache,io", IO, ids=IDS)
@pytest.mark.parametrize("rows", [2, 20], ids=["few", "many"])
def test_scales_and_sizes_of_q(hip, cache, io, rows):
    """Scales below 0 and of 0, and rows of q so small that with the scale they leave fp32's range: behind tiles that do not count (a
    page that does not exist, an odd number of tiles) too."""
    rng = np.random.default_rng(13)
    for size, scale in ((1.0, -0.1), (1.0, 0.0), (1e-30, 0.0), (2.0**-149, 0.125), (2.0**-24, 1e-30), (1e30, 1e-31)):
        c = Case(rng, cache, io, 128, 1, 4, 16, rows, [144], [145 + r for r in range(rows)], broken=[(0, 3)])
        with np.errstate(over="ignore", under="ignore"):
            x = ref.to_type(io, np.minimum(np.abs(c.q) * size, 6e4 if io == F16 else 1e38).astype(np.float32) * np.sign(c.q))
        c.rq[3][...] = x
        c.rq[1].upload(c.rq[2])
        c.q, c.scale = ref.from_type(io, x), scale
        for own in (0, 20):
            c.run([144], own)
            c.check()
    c = Case(rng, cache, io, 128, 1, 4, 16, rows, [144], [145 + r for r in range(rows)], broken=[(0, 3)])
    c.scale = -0.2
    c.run([144], 20, 10.0)
    c.check(10.0)


@pytest.mark.parametrize("cache,io", IO, ids=IDS)
@pytest.mark.parametrize("rows", [3, 20], ids=["few", "many"])
def test_not_finite(hip, cache, io, rows):
    """A NaN and an infinity in V of shared positions: their dim (quantized: the dims of their block) is not finite, the others have
    the same bits as without; a NaN in q: its head is NaN, the others are not touched."""
    rng = np.random.default_rng(14)
    heads, hd = 4, 128
    c = Case(rng, cache, io, hd, 1, heads, 16, rows, [160], [161 + r for r in range(rows)])
    c.run([160], 30)
    want = c.got()[0]
    q = c.rq[3][1, 2, 7].copy()
    c.rq[3][1, 2, 7] = ref.to_type(io, np.full(1, np.nan, np.float32))[0]
    c.rq[1].upload(c.rq[2])
    c.q[1, 2] = 0.0
    for own in (40, 30):
        c.run([160], own)
        c.check(but=(1, 2))
    c.rq[3][1, 2, 7] = q
    c.rq[1].upload(c.rq[2])
    k, v = c.k[0][:160], c.v[0][:160].copy()
    odd = np.zeros((rows, heads, hd), bool)
    for p, dim, x in ((37, 5, np.nan), (100, 41, np.inf)):
        v[p, 0, dim] = x
        if cache in (Q8_0, Q4_0):
            odd[:, :, dim // 32 * 32:dim // 32 * 32 + 32] = True
        else:
            odd[:, :, dim] = True
    with np.errstate(all="ignore"):
        c.c.fill(0, c.table, 0, k, v)
    c.c.upload()
    c.run([160], 30)
    got = c.got()[0]
    assert not np.isfinite(got[odd]).any()
    if cache not in (Q8_0, Q4_0):                      # (written again, the codes may be others)
        np.testing.assert_array_equal(got[~odd], want[~odd])
    assert np.isfinite(got[~odd]).all()


def test_rows_of_a_group_beyond_the_call(hip):
    """A number of rows far above the call's: one group."""
    rng = np.random.default_rng(15)
    c = Case(rng, BF16, BF16, 64, 1, 8, 16, 5, [96], [97, 100, 113, 96, 120])
    for rows in (5, 6, 2**30, 2**31 - 1):
        c.rows = rows
        c.run([96], 24)
        c.check()


def test_calls_at_once(hip):
    """Two calls under way on two streams, each in a workspace of its own, again and again: the same bits as alone."""
    rng = np.random.default_rng(16)
    cases = [Case(rng, BF16, BF16, 128, 2, 16, 32, 8, [960], [961 + r for r in range(8)]), Case(rng, Q8_0, F32, 128, 1, 4, 32, 30, [480], [490 + r for r in range(30)])]
    shared = [dev(np.array([n], np.int32)) for n in (960, 480)]
    streams = [hip.sapphire_stream_create() for _ in cases]
    want = []
    for c, on in zip(cases, shared):
        c.run(on, 40)
        want.append(c.got()[0])
        c.ro[1].upload(c.ro[2] * 0 + 7)
    for _ in range(5):
        for _ in range(8):
            for c, on, s in zip(cases, shared, streams):
                c.run(on, 40, stream=s)
        for c, w in zip(cases, want):
            np.testing.assert_array_equal(c.got()[0], w)
    for s in streams:
        hip.sapphire_stream_destroy(s)


@pytest.mark.parametrize("rows", [4, 12], ids=["few", "many"])
def test_pages_past_four_gigabytes(hip, rows):
    """The same rows in the first pages and in the last ones of pools of more than 2^32 bytes: the same bits."""
    from sapphire_amd.device import DeviceArray
    from sapphire_amd.paged import PagedCache, PageTable
    rng = np.random.default_rng(17)
    hd, ps, pages, heads, n = 256, 64, 140000, 4, 400
    c = PagedCache(BF16, 1, pages, ps, 1, hd)
    assert c.nbytes > 2**32
    ld = -(-n // ps)
    k, v = (device_rows(rng.normal(size=(n, 1, hd)).astype(np.float32), BF16) for _ in range(2))
    q = device_rows(rng.normal(size=(rows, heads, hd)).astype(np.float32), BF16)
    at, lens, shared = dev(np.arange(n, dtype=np.int32)), dev(n - rows + 1 + np.arange(rows, dtype=np.int32)), dev(np.array([n], np.int32))
    ws, got = DeviceArray(c.shared_attention_workspace_bytes(rows, heads, n)), []
    for first in (0, pages - ld):
        table = np.broadcast_to(np.arange(first, first + ld, dtype=np.int32), (rows, ld)).copy()
        t = dev(table)
        o = device_rows(np.zeros((rows, heads, hd), np.float32), BF16)
        c.write(0, k[0], v[0], PageTable(t, rows, ld), at, seqs=dev(np.zeros(n, np.int32)))
        c.shared_attention(0, q[0], o[0], PageTable(t, rows, ld), lens, n, rows, shared, hd**-0.5, max_own=rows, workspace=ws)
        sync()
        got.append(o[1].numpy())
    np.testing.assert_array_equal(got[0], got[1])
    assert (got[0] != 0).mean() > 0.9
    for d in (c.k, c.v):
        d.free()


def test_lengths_are_clamped_and_no_lse(hip):
    rng = np.random.default_rng(6)
    c = Case(rng, BF16, BF16, 64, 1, 4, 16, 3, [160], [170, 200, 200])
    c.lens, c.top = [-5, 10**9, 200], 200
    c.dn.upload(np.array(c.lens, np.int32))
    c.run([160], 40)
    c.check()
    c.lse.upload(np.full((4, 4), 9, np.float32))
    c.run([160], 40, lse=False)
    sync()
    assert (c.lse.numpy() == 9).all()


@pytest.mark.parametrize("cache,io", [(BF16, BF16), (F16, F32), (Q8_0, F32), (Q4_0, BF16), (F32, F32)], ids=["bf16", "f16_f32", "q8_0_f32", "q4_0_bf16", "f32"])
def test_many_pieces(hip, cache, io):
    """Few columns over thousands of positions; many groups."""
    rng = np.random.default_rng(7)
    c = Case(rng, cache, io, 128, 1, 2, 128, 2, [8192], [8193, 9000])
    c.run([8192], 10)
    c.check()
    c = Case(rng, cache, io, 64, 2, 2, 16, 3, [48] * 100, [49 + r % 50 for r in range(299)])
    c.run([48] * 100, 60)
    c.check()


def test_in_place_streams_and_replays(hip):
    """out is q; another stream; a captured call replayed as rows and shared positions grow, in a workspace of the largest call."""
    from sapphire_amd.device import DeviceArray
    rng = np.random.default_rng(8)
    for cache, io, own in ((BF16, BF16, 80), (Q8_0, F32, 80), (BF16, BF16, 30), (Q4_0, F32, 30)):
        c = Case(rng, cache, io, 64, 1, 8, 32, 4, [320, 320], [400] * 8)
        c.run([320, 320], own)
        want = c.got()[0]
        c.run([320, 320], own, out=c.rq[0])
        sync()
        got = ref.from_type(io, c.rq[1].numpy()[:want.size]).reshape(want.shape)
        np.testing.assert_array_equal(got, want)
        c = Case(rng, cache, io, 64, 1, 8, 32, 4, [320, 320], [400] * 8)
        c.ws = DeviceArray(c.c.c.shared_attention_workspace_bytes(50, 16, 100000))
        s = hip.sapphire_stream_create()
        c.run([320, 320], own, stream=s)
        c.check()
        hip.sapphire_stream_destroy(s)
        on = dev(np.array([320, 320], np.int32))
        g = Graph(lambda stream: c.run(on, own, stream=stream))
        k, v = c.k, c.v
        for lens, shared in (([400] * 8, [320, 320]), ([0] * 4 + [330, 0, 321, 399], [5, 319]), ([7, 400, 330, 1, 0, 0, 0, 0], [320, 320]), ([400] * 8, [320, 0])):
            c.lens = lens
            c.dn.upload(np.array(lens, np.int32))
            on.upload(np.array(shared, np.int32))
            g.replay()
            c.check()
        assert k is c.k and v is c.v
        g.close()


def test_groups_do_not_touch_each_other(hip):
    """A group's outputs are the same bits whatever the other groups hold."""
    rng = np.random.default_rng(9)
    c = Case(rng, BF16, BF16, 128, 2, 8, 32, 4, [256, 256, 256], [300, 270, 260, 257] * 3)
    c.run([256] * 3, 50)
    a, _ = c.got()
    q = c.rq[2].copy()
    c.rq[3][:4] = ref.to_type(BF16, np.full((4, 8, 128), np.nan, np.float32))
    c.rq[1].upload(c.rq[2])
    c.dn.upload(np.array([300, 270, 260, 257] + [300, 270, 260, 257] + [300, 0, 0, 5], np.int32))
    c.run([256] * 3, 50)
    b, _ = c.got()
    np.testing.assert_array_equal(a[4:8], b[4:8])
    assert np.isnan(b[:4]).all() and len(q)


@pytest.mark.parametrize("cache,io", [(F32, F32), (BF16, F32), (Q8_0, F32)], ids=["f32", "bf16_f32", "q8_0_f32"])
def test_speculative_decoding(hip, cache, io):
    """The operators together, as a program takes them: the drafted tokens' rows are written, attended to by the group, their logits
    verified. The model is one attention layer over embeddings; with greedy verification the tokens are those of decoding
    one at a time."""
    from sapphire_amd.device import DeviceArray
    from sapphire_amd.paged import PageTable, Rows, verify, verify_workspace_bytes
    from tests.test_paged_gpu import Cache as Held
    rng = np.random.default_rng(12)
    hd, nkv, heads, ps, vocab, requests, drafts = 64, 1, 4, 16, 300, 3, 4
    rows = drafts + 1
    emb = [rng.normal(size=(vocab, n, hd)).astype(np.float32) for n in (heads, nkv, nkv)]
    place = rng.normal(size=(200, 1, hd)).astype(np.float32)
    head = rng.normal(size=(heads * hd, vocab)).astype(np.float32)
    ld, n_pages = 12, requests * 12
    table = rng.permutation(n_pages).reshape(requests, ld).astype(np.int32)
    c = Held(cache, 1, n_pages, ps, nkv, hd)
    scale = hd**-0.5

    def qkv(tokens, pos):
        return [e[tokens] + place[pos] for e in emb]

    def write(tokens, pos, seqs):
        _, k, v = qkv(tokens, pos)
        rk, rv = device_rows(k, io), device_rows(v, io)
        t = dev(table)
        c.c.write(0, rk[0], rv[0], PageTable(t, *table.shape), dev(np.array(pos, np.int32)), seqs=dev(np.array(seqs, np.int32)))
        sync()

    def attend(tokens, pos, seqs, group_rows=None):
        q = device_rows(qkv(tokens, pos)[0], io)
        o = device_rows(np.zeros((len(tokens), heads, hd), np.float32), io)
        t, n = dev(table[seqs]), dev(np.array(pos, np.int32) + 1)
        pt = PageTable(t, len(seqs), ld)
        top = int(max(pos)) + 1
        if group_rows is None:
            ws = DeviceArray(max(1, c.c.attention_workspace_bytes(len(seqs), heads, top)))
            c.c.attention(0, q[0], o[0], pt, n, top, scale, workspace=ws)
        else:
            ws = DeviceArray(c.c.shared_attention_workspace_bytes(len(seqs), heads, top))
            shared = dev((np.array(pos, np.int32) + 1)[::group_rows].copy())
            c.c.shared_attention(0, q[0], o[0], pt, n, top, group_rows, shared, scale, max_own=group_rows, workspace=ws)
        sync()
        x = ref.from_type(io, o[1].numpy()[:len(seqs) * heads * hd]).reshape(len(seqs), heads * hd)
        return (x.astype(np.float64) @ head).astype(np.float32)

    prompt = rng.integers(0, vocab, (requests, 40))
    for r in range(requests):
        write(prompt[r, :-1], np.arange(39), [r] * 39)
    # one token at a time
    want, last = [[] for _ in range(requests)], prompt[:, -1].copy()
    for i in range(24):
        pos = [39 + i] * requests
        write(last, pos, range(requests))
        last = attend(last, pos, list(range(requests))).argmax(1)
        for r in range(requests):
            want[r].append(int(last[r]))
    # drafts: the right tokens, some of them spoilt
    c.upload()
    for r in range(requests):
        write(prompt[r, :-1], np.arange(39), [r] * 39)
    got, last, at = [[] for _ in range(requests)], prompt[:, -1].copy(), np.full(requests, 39)
    ws = DeviceArray(verify_workspace_bytes(vocab, requests, drafts))
    calls, kept_all = 0, []
    while min(map(len, got)) < 20:
        d = np.array([(want[r][len(got[r]):] + [0] * drafts)[:drafts] for r in range(requests)])
        spoil = rng.random(d.shape) < 0.3
        d = np.where(spoil, (d + 1) % vocab, d)
        tokens = np.concatenate([last[:, None], d], 1)
        pos = (at[:, None] + np.arange(rows)).ravel()
        seqs = np.repeat(np.arange(requests), rows)
        write(tokens.ravel(), pos, seqs)
        logits = dev(attend(tokens.ravel(), pos, list(seqs), rows))
        out, kept = dev(np.zeros((requests, rows), np.int32)), dev(np.zeros(requests, np.int32))
        verify(logits, vocab, vocab, requests, drafts, dev(d.astype(np.int32)), None, out, kept, ws, temperature=0.0)
        sync()
        out, kept = out.numpy(), kept.numpy()
        for r in range(requests):
            got[r] += [int(t) for t in out[r, :kept[r] + 1]]
            assert (out[r, kept[r] + 1:] == -1).all()
            last[r] = out[r, kept[r]]
            at[r] += kept[r] + 1
        kept_all += list(kept)
        calls += 1
    assert calls < 20 and len(set(kept_all)) > 2
    for r in range(requests):
        n = min(len(want[r]), len(got[r]))
        assert n >= 20 and got[r][:n] == want[r][:n]


@pytest.mark.parametrize("cache,io", IO, ids=IDS)
def test_positions_that_the_join_takes(hip, cache, io):
    """None to hundreds of positions behind the shared ones, whatever max_own says of them; pieces few and many; a NaN and an
    infinity in their V: the dim (quantized: its block) of the rows that see them."""
    rng = np.random.default_rng(18)
    for hd, n, own in ((64, 64, (0, 1, 15, 16, 63, 64, 65, 300)), (128, 1024, (1, 7, 31, 32, 33, 500)), (256, 4096, (0, 1, 8, 33))):
        c = Case(rng, cache, io, hd, 2, 6, 16, len(own), [n], [n + i for i in own])
        c.run([n], 32)
        c.check()
    r, hd = 2, 128
    c = Case(rng, cache, io, hd, 1, 2, 16, 3, [64], [70, 66, 75])
    k, v = c.k[r], c.v[r].copy()
    v[68, 0, 5], v[70, 0, 40] = np.nan, np.inf
    with np.errstate(all="ignore"):
        c.c.fill(0, c.table, r, k, v)
    c.c.upload()
    c.run([64], 16)
    got = c.got()[0]
    odd = np.zeros((3, 2, hd), bool)
    for dim in (5, 40):
        odd[r, :, slice(dim // 32 * 32, dim // 32 * 32 + 32) if cache in (Q8_0, Q4_0) else dim] = True
    assert not np.isfinite(got[odd]).any() and np.isfinite(got[~odd]).all()
