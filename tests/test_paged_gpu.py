"""The paged cache on the GPU against plain numpy: rows in and out (bytes and values), attention of one new token,
reordering, and a beam-search decode through all of it."""
import ctypes as C

import numpy as np
import pytest

from tests import paged_ref as ref
from tests.paged_ref import BF16, F16, F32, Q4_0, Q8_0

pytestmark = pytest.mark.gpu
CACHES = [F32, BF16, F16, Q8_0, Q4_0]


def dev(a):
    from sapphire_amd.device import DeviceArray
    return DeviceArray.from_numpy(np.ascontiguousarray(a))


def sync():
    from sapphire_amd import load
    assert load().sapphire_synchronize() == 0


class Cache:
    """A cache on the device with its byte-for-byte double on the host."""

    def __init__(self, dtype, layers, pages, ps, nkv, hd, fill=0xff):
        from sapphire_amd.paged import PagedCache
        self.dtype, self.ps, self.nkv, self.hd = dtype, ps, nkv, hd
        self.pool = {w: ref.Pool(w, dtype, layers, pages, ps, nkv, hd, fill) for w in "kv"}
        self.on = {w: dev(self.pool[w].a) for w in "kv"}
        self.c = PagedCache(dtype, layers, pages, ps, nkv, hd, k=self.on["k"].ptr, v=self.on["v"].ptr)
        assert self.c.nbytes == self.pool["k"].a.nbytes

    def upload(self):
        for w in "kv":
            self.on[w].upload(self.pool[w].a)

    def fill(self, layer, table, seq, k, v):
        """Host side only: rows [positions][heads][hd] of sequence `seq`."""
        for p in range(len(k)):
            page = table[seq, p // self.ps]
            if page >= 0:
                self.pool["k"].put(layer, page, p % self.ps, k[p])
                self.pool["v"].put(layer, page, p % self.ps, v[p])


def tables(rng, lens, ps, extra=3, ld_extra=1):
    """A table with its pages in no order, -1 behind each row's, and the number of pages."""
    need = [-(-max(n, 0) // ps) for n in lens]
    order = rng.permutation(sum(need) + extra)
    t, at = np.full((len(lens), max(need) + ld_extra), -1, np.int32), 0
    for r, k in enumerate(need):
        t[r, :k] = order[at:at + k]
        at += k
    return t, len(order)


def device_rows(x, dtype, order="thd", pad=0, shift=0):
    """(rows, buffer, view of a host copy) of fp32 x [tokens][heads][hd] in a layout: tokens or heads outermost, `pad`
    elements between rows of the outer dim, the data `shift` elements into the buffer."""
    from sapphire_amd.paged import Rows
    t, h, hd = x.shape
    ts, hs = (h * hd + pad, hd) if order == "thd" else (hd, t * hd + pad)
    n = shift + (t - 1) * ts + (h - 1) * hs + hd
    host = np.full(n + 5, 7, ref.np_type(dtype))
    view = np.lib.stride_tricks.as_strided(host[shift:], x.shape, tuple(s * host.itemsize for s in (ts, hs, 1)))
    view[...] = ref.to_type(dtype, x)
    d = dev(host)
    return Rows(d.ptr + shift * host.itemsize, dtype, t, h, hd, ts, hs), d, host, view


@pytest.mark.parametrize("cache", CACHES, ids=ref.NAME.get)
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("io,order,pad,shift", [(F32, "thd", 0, 0), (BF16, "thd", 192, 64), (F16, "htd", 8, 8), (F32, "htd", 1, 3), (BF16, "thd", 3, 1)],
                         ids=["f32", "bf16_slice", "f16_heads_outer", "f32_odd", "bf16_odd"])
def test_write_and_read(hip, cache, hd, io, order, pad, shift):
    """Every byte of both pools after a write: the rows' where they belong, the rest as it was; then the rows read back,
    each the value that the cache holds rounded once to the rows' type: exactly equal. Padding, rows and pages that do
    not exist are left out and read as zeros."""
    rng = np.random.default_rng(hd * 10 + cache)
    nkv, ps, layers = 3, 48, 2
    lens = [100, 1, 0, 47, 49]
    table, pages = tables(rng, lens, ps)
    table[4, 1] = pages + 5                        # a page that does not exist
    seqs, pos = zip(*[(s, p) for s, n in enumerate(lens) for p in rng.permutation(n)[:40]])
    seqs, pos = list(seqs) + [0, 0, 9, -1, 1], list(pos) + [-1, 100 * ps, 0, 0, ps]      # none of these exist
    t = len(seqs)
    x = {w: (rng.normal(size=(t, nkv, hd)) * 2).astype(np.float32) for w in "kv"}
    c = Cache(cache, layers, pages, ps, nkv, hd)
    rk, rv = device_rows(x["k"], io, order, pad, shift), device_rows(x["v"], io, order, pad, shift)
    from sapphire_amd.paged import PageTable
    dt, ds, dp = dev(table), dev(np.array(seqs, np.int32)), dev(np.array(pos, np.int32))
    pt = PageTable(dt, *table.shape)
    c.c.write(1, rk[0], rv[0], pt, dp, seqs=ds)
    sync()
    there, want = [], {w: np.zeros((t, nkv, hd), np.float32) for w in "kv"}
    for i, (s, p) in enumerate(zip(seqs, pos)):
        ok = 0 <= s < len(lens) and 0 <= p < table.shape[1] * ps and 0 <= table[s, p // ps] < pages
        there.append(ok)
        for w, r in (("k", rk), ("v", rv)):
            if ok:
                row = ref.from_type(io, r[3][i])
                c.pool[w].put(1, table[s, p // ps], p % ps, row)
                want[w][i] = ref.stored(cache, row)
    assert 0 < sum(there) < t
    for w in "kv":
        np.testing.assert_array_equal(c.on[w].numpy(), c.pool[w].a, err_msg=w)
    ok_, ov_ = device_rows(np.ones((t, nkv, hd), np.float32), io, order, pad, shift), device_rows(np.ones((t, nkv, hd), np.float32), io, order, pad, shift)
    c.c.read(1, ok_[0], ov_[0], pt, dp, seqs=ds)
    sync()
    for w, r in (("k", ok_), ("v", ov_)):
        r[3][...] = ref.to_type(io, want[w])       # the host copy with the rows in place: padding included
        np.testing.assert_array_equal(r[1].numpy(), r[2], err_msg=w)


@pytest.mark.parametrize("cache", CACHES, ids=ref.NAME.get)
def test_write_special_values(hip, cache):
    """Zeros of both signs, ties of the largest magnitude, subnormal blocks, halves between codes, NaN and infinities."""
    hd, ps, t = 64, 16, 12
    x = np.zeros((t, 1, hd), np.float32)
    x[0, 0, ::2] = -0.0
    x[1, 0, 5], x[1, 0, 9] = -3.0, 3.0
    x[2, 0, 5], x[2, 0, 9] = 3.0, -3.0
    x[3, 0] = np.float32(1e-41) * np.arange(hd)
    x[4, 0, :32] = np.arange(32) * 0.5 * 127 / 127
    x[4, 0, 0] = 127.0
    x[5, 0] = np.where(np.arange(hd) % 2, 1.5, -2.5)
    x[5, 0, 3] = 127.0
    x[6, 0, 7] = np.nan
    x[7, 0, 40] = np.inf
    x[8, 0, 1] = -np.inf
    x[9, 0] = 3e38
    x[9, 0, 2] = -3e38
    x[10, 0] = np.float32(1.4e-45)
    x[11, 0] = 65519.0
    c = Cache(cache, 1, 1, ps, 1, hd)
    from sapphire_amd.paged import PageTable
    dt, dp, ds = dev(np.zeros((1, 1), np.int32)), dev(np.arange(t, dtype=np.int32)), dev(np.zeros(t, np.int32))
    rk, rv = device_rows(x, F32), device_rows(-x, F32)
    c.c.write(0, rk[0], rv[0], PageTable(dt, 1, 1), dp, seqs=ds)
    ok_, ov_ = device_rows(np.ones_like(x), F32), device_rows(np.ones_like(x), F32)
    c.c.read(0, ok_[0], ov_[0], PageTable(dt, 1, 1), dp, seqs=ds)
    sync()
    for w, r, s in (("k", ok_, x), ("v", ov_, -x)):
        got = r[1].numpy()[:t * hd].reshape(t, hd)
        np.testing.assert_array_equal(got, ref.stored(cache, s)[:, 0], err_msg=w)
        if cache in (Q8_0, Q4_0):
            assert np.isnan(got[6, :32]).all() and np.isnan(got[7, 32:]).all() and np.isfinite(got[7, :32]).all() and np.isnan(got[8, :32]).all()


def attend_case(rng, cache, io, hd, nkv, heads, ps, lens, window=0, softcap=0.0, layers=1, layer=0, peak=2.0, max_length=None,
                broken=(), order="thd", pad=0, lse=True, stream=None, n_given=None):
    """Runs one call and compares it with 64 bits; returns (out, lse) as read."""
    from sapphire_amd.device import DeviceArray
    from sapphire_amd.paged import PageTable
    table, pages = tables(rng, lens, ps)
    c = Cache(cache, layers, pages, ps, nkv, hd)   # 0xff bytes: NaN wherever nothing is written, scales included
    ks, vs = [], []
    for s, n in enumerate(lens):
        k, v = (rng.normal(size=(n, nkv, hd)).astype(np.float32) for _ in range(2))
        ks.append(ref.stored(cache, k))
        vs.append(ref.stored(cache, v))
        c.fill(layer, table, s, k, v)
    c.upload()
    for s, i in broken:
        table[s, i] = pages + i if i % 2 else -7
    q = (rng.normal(size=(len(lens), heads, hd)) * peak).astype(np.float32)
    rq, ro = device_rows(q, io, order, pad), device_rows(q * 0 + 3, io, order, pad)
    qs = ref.from_type(io, rq[3])
    top = max_length or max(1, max(lens))
    dt, dl = dev(table), dev(np.array(lens if n_given is None else n_given, np.int32))
    dlse = dev(np.full((len(lens) + 1, heads), 5, np.float32))
    ws = DeviceArray(max(1, c.c.attention_workspace_bytes(len(lens), heads, top)))
    scale = 1.0 / np.sqrt(hd)
    c.c.attention(layer, rq[0], ro[0], PageTable(dt, *table.shape), dl, top, scale, window=window, softcap=softcap,
                  lse=dlse if lse else None, workspace=ws, stream=stream)
    sync()
    host = ro[2].copy()
    raw = ro[1].numpy()
    ro[2][...] = raw
    got, glse = ref.from_type(io, ro[3].copy()).astype(np.float64), dlse.numpy()
    ro[2][...] = host
    ro[3][...] = 0
    mask = np.ones(raw.shape, bool)
    host = np.ones_like(ro[2])
    np.lib.stride_tricks.as_strided(mask[:], q.shape, tuple(s // host.itemsize for s in ro[3].strides))[...] = False
    assert (raw[mask] == 7).all(), "elements between the rows were written"
    assert (glse[-1] == 5).all()
    rounded = io != F32
    for s, n in enumerate(lens):
        keep = np.ones(n, bool)
        lo = max(0, n - window) if window > 0 else 0
        keep[:lo] = False
        for bs, i in broken:
            if bs == s:
                keep[i * ps:(i + 1) * ps] = False
        out, l, size, mean = ref.attention64(qs[s], ks[s][keep], vs[s][keep], scale, 0, softcap)
        tol, ltol = ref.attention_bound(io, rounded, hd, n, out, l, size, mean, softcap)
        worst = np.max(np.abs(got[s] - out) / tol)
        assert worst <= 1, (s, n, worst)
        if lse:
            dead = np.isneginf(l)
            assert np.array_equal(np.isneginf(glse[s]), dead)
            assert (np.abs(glse[s][~dead] - l[~dead]) <= ltol[~dead]).all(), (s, n)
            assert (got[s][dead] == 0).all()
    if not lse:
        assert (glse == 5).all()
    return got, glse


IO = [(F32, F32), (BF16, F32), (F16, F32), (Q8_0, F32), (Q4_0, F32), (BF16, BF16), (F16, F16), (Q8_0, BF16), (Q8_0, F16), (Q4_0, BF16), (Q4_0, F16)]
IDS = [f"{ref.NAME[a]}-{ref.NAME[b]}" for a, b in IO]
LENS = [0, 1, 15, 16, 17, 63, 64, 65, 130, 511]


@pytest.mark.parametrize("cache,io", IO, ids=IDS)
@pytest.mark.parametrize("hd,nkv,heads,ps", [(64, 1, 4, 16), (128, 3, 3, 48), (256, 1, 4, 64), (128, 2, 16, 32), (64, 2, 34, 16), (256, 2, 10, 48)])
def test_attention(hip, cache, io, hd, nkv, heads, ps):
    """Lengths around the tiles and pages, NaN behind every sequence's last position, head groups of 1 to 17."""
    attend_case(np.random.default_rng(hd + heads), cache, io, hd, nkv, heads, ps, LENS)


@pytest.mark.parametrize("cache,io", IO, ids=IDS)
def test_attention_pieces(hip, cache, io):
    """Few sequences, cut into pieces and joined: short ones beside one of several thousand positions."""
    rng = np.random.default_rng(7)
    attend_case(rng, cache, io, 128, 1, 4, 64, [3001, 5, 0, 1024])
    attend_case(rng, cache, io, 256, 1, 4, 16, [1025], layers=2, layer=1)
    attend_case(rng, cache, io, 64, 2, 6, 1024, [2049, 2047], order="htd", pad=5)


@pytest.mark.parametrize("cache,io", [(F32, F32), (BF16, BF16), (Q8_0, F32), (Q4_0, F16)], ids=["f32", "bf16", "q8_0_f32", "q4_0_f16"])
def test_attention_of_very_many_pieces(hip, cache, io):
    """Two hundred pieces and more of one sequence, some of them without a page, beside short sequences; a window that
    starts inside a piece."""
    rng = np.random.default_rng(18)
    attend_case(rng, cache, io, 64, 1, 4, 256, [16500, 7, 0, 9000], broken=[(0, 0), (0, 1), (0, 40), (3, 35)])
    attend_case(rng, cache, io, 128, 1, 2, 128, [8300, 4097], window=6001)
    attend_case(rng, cache, io, 256, 1, 5, 64, [4200])


@pytest.mark.parametrize("cache,io", IO, ids=IDS)
@pytest.mark.parametrize("window,softcap", [(1, 0.0), (16, 0.0), (100, 0.0), (512, 30.0), (0, 5.0)])
def test_attention_window_and_cap(hip, cache, io, window, softcap):
    attend_case(np.random.default_rng(window), cache, io, 128, 2, 8, 48, [1, 16, 99, 100, 101, 700], window=window, softcap=softcap, peak=4.0)


@pytest.mark.parametrize("cache", CACHES, ids=ref.NAME.get)
def test_attention_pages_that_do_not_exist(hip, cache):
    attend_case(np.random.default_rng(3), cache, F32, 64, 1, 4, 16, [40, 16, 100, 700], broken=[(0, 1), (1, 0), (2, 0), (2, 6), (3, 5), (3, 43)])


@pytest.mark.parametrize("cache,io,batch,nkv", [(BF16, BF16, 257, 4), (Q4_0, F32, 1024, 1), (F32, F32, 1100, 1), (Q8_0, BF16, 64, 17), (F16, F32, 520, 2)],
                         ids=["257x4", "1024", "1100", "64x17", "520x2"])
def test_attention_of_many_sequences(hip, cache, io, batch, nkv):
    """Enough whole sequences to fill the chip, which the workgroups take by length: every one, empty ones and lengths out
    of range among them, gets its own output."""
    rng = np.random.default_rng(batch)
    lens = [int(n) for n in rng.integers(0, 80, batch)]
    lens[3], lens[7] = 0, 80
    given = np.array(lens)
    given[3], given[7] = -7, 10**9
    attend_case(rng, cache, io, 64, nkv, nkv * 2, 16, lens, n_given=given, max_length=80)


def test_attention_lengths_are_clamped(hip):
    rng = np.random.default_rng(4)
    attend_case(rng, F32, F32, 64, 1, 2, 16, [0, 50, 20], n_given=[-5, 1000, 20], max_length=50, lse=False)
    attend_case(rng, Q8_0, F32, 64, 1, 2, 16, [0, 50, 20], n_given=[-2**31, 2**31 - 1, 20], max_length=50)


@pytest.mark.parametrize("cache", [F32, Q8_0], ids=ref.NAME.get)
def test_attention_of_peaked_and_flat_scores(hip, cache):
    """Scores of hundreds (one weight carries all) and of zero (all are equal)."""
    rng = np.random.default_rng(5)
    attend_case(rng, cache, F32, 128, 1, 8, 32, [500, 33], peak=100.0)
    attend_case(rng, cache, F32, 128, 1, 8, 32, [500, 33], peak=0.0)


@pytest.mark.parametrize("io", [F32, BF16, F16], ids=ref.NAME.get)
def test_attention_infinite_and_nan_scores(hip, io):
    """-inf scores weigh nothing (a row of them only gives 0 and -inf, whatever V holds there); NaN and +inf reach the
    outputs of their heads and sequences only."""
    from sapphire_amd.device import DeviceArray
    from sapphire_amd.paged import PageTable
    rng = np.random.default_rng(6)
    hd, ps, heads = 64, 16, 2
    for n in (40, 700):
        table, pages = tables(rng, [n] * 5, ps)
        c = Cache(io, 1, pages, ps, 1, hd)
        k, v = (rng.normal(size=(5, n, 1, hd)).astype(np.float32) for _ in range(2))
        k[..., 0] = 1.0
        k[0, 3:20, 0, 0] = -np.inf             # some positions weigh nothing
        k[1, :, 0, 0] = -np.inf                # all of them
        v[1, :, 0, :] = np.nan
        k[2, 7, 0, 5] = np.nan
        k[3, n - 1, 0, 0] = np.inf
        for s in range(5):
            c.fill(0, table, s, k[s], v[s])
        c.upload()
        q = rng.normal(size=(5, heads, hd)).astype(np.float32)
        q[..., 0] = 1.0
        rq, ro = device_rows(q, io), device_rows(q * 0, io)
        dt, dl, dlse = dev(table), dev(np.full(5, n, np.int32)), DeviceArray.empty((5, heads))
        ws = DeviceArray(max(1, c.c.attention_workspace_bytes(5, heads, n)))
        c.c.attention(0, rq[0], ro[0], PageTable(dt, *table.shape), dl, n, 0.125, lse=dlse, workspace=ws)
        sync()
        got = ref.from_type(io, ro[1].numpy()[:5 * heads * hd]).reshape(5, heads, hd)
        lse = dlse.numpy()
        assert np.isnan(got[2]).all() and np.isnan(got[3]).all() and np.isnan(lse[2]).all() and np.isnan(lse[3]).all()
        assert (got[1] == 0).all() and np.isneginf(lse[1]).all()
        for s in (0, 4):
            out, l, size, mean = ref.attention64(ref.from_type(io, rq[3])[s], np.where(np.isneginf(k[s]), -1e30, ref.stored(io, k[s])), ref.stored(io, v[s]), 0.125)
            _, _, size, _ = ref.attention64(ref.from_type(io, rq[3])[s], np.where(np.isneginf(k[s]), 0, ref.stored(io, k[s])), ref.stored(io, v[s]), 0.125)
            tol, ltol = ref.attention_bound(io, io != F32, hd, n, out, l, size, mean)
            assert (np.abs(got[s] - out) <= tol).all() and (np.abs(lse[s] - l) <= ltol).all()


@pytest.mark.parametrize("io", [F32, BF16, F16], ids=ref.NAME.get)
def test_attention_of_many_small_weights(hip, io):
    """One position outweighs each of 2^17 - 1 others by 2^25: together they weigh 2^-8, which is the output (its value is
    0, theirs 1)."""
    from sapphire_amd.device import DeviceArray
    from sapphire_amd.paged import PagedCache, PageTable
    hd, ps, n = 64, 256, 1 << 17
    c = PagedCache(io, 1, n // ps, ps, 1, hd)
    k, v = np.zeros((n, 1, hd), np.float32), np.ones((n, 1, hd), np.float32)
    k[0, 0, 0], v[0] = 25 * np.log(2), 0
    rk, rv = device_rows(k, io), device_rows(v, io)
    q = np.zeros((1, 1, hd), np.float32)
    q[0, 0, 0] = 1
    rq, ro = device_rows(q, io), device_rows(q, io)
    dt, dp, ds = dev(np.arange(n // ps, dtype=np.int32)[None]), dev(np.arange(n, dtype=np.int32)), dev(np.zeros(n, np.int32))
    pt = PageTable(dt, 1, n // ps)
    c.write(0, rk[0], rv[0], pt, dp, seqs=ds)
    ws = DeviceArray(max(1, c.attention_workspace_bytes(1, 1, n)))
    c.attention(0, rq[0], ro[0], pt, dev(np.array([n], np.int32)), n, 1.0, workspace=ws)
    sync()
    got = ref.from_type(io, ro[1].numpy()[:hd]).astype(np.float64)
    out, l, size, mean = ref.attention64(q[0], ref.from_type(io, rk[3]), v, 1.0)
    tol, _ = ref.attention_bound(io, io != F32, hd, n, out, l, size, mean)
    assert (np.abs(got - out[0]) <= np.minimum(tol[0], out[0] / 50)).all()


@pytest.mark.parametrize("cache", CACHES, ids=ref.NAME.get)
@pytest.mark.parametrize("heads", [4, 7])
def test_attention_of_extreme_queries(hip, cache, heads):
    """Rows of zeros, of 1e-30 and of 1e30 (under scales that bring their scores back), one element a million times the
    others; a NaN makes its own head NaN and no other."""
    from sapphire_amd.device import DeviceArray
    from sapphire_amd.paged import PageTable
    rng = np.random.default_rng(13)
    hd, ps, n = 128, 16, 200
    table, pages = tables(rng, [n], ps)
    c = Cache(cache, 1, pages, ps, 1, hd)
    k, v = (rng.normal(size=(n, 1, hd)).astype(np.float32) for _ in range(2))
    c.fill(0, table, 0, k, v)
    c.upload()
    ks, vs = ref.stored(cache, k), ref.stored(cache, v)
    dt, dl, ws = dev(table), dev(np.array([n], np.int32)), DeviceArray(max(1, c.c.attention_workspace_bytes(1, heads, n)))
    for size in (0.0, 1e-30, 1.0, 1e30):
        q = (rng.normal(size=(1, heads, hd)) * size).astype(np.float32)
        if size == 1.0:
            q[0, 1, 77] = 1e6
            q[0, 2, 5] = np.nan
        scale = 0.1 / size if size else 0.1
        rq, ro = device_rows(q, F32), device_rows(np.ones_like(q), F32)
        c.c.attention(0, rq[0], ro[0], PageTable(dt, *table.shape), dl, n, scale, workspace=ws)
        sync()
        got = ro[1].numpy()[:heads * hd].reshape(heads, hd)
        if size == 1.0:
            assert np.isnan(got[2]).all()
            got, q = np.delete(got, 2, 0), np.delete(q, 2, 1)
        out, l, big, mean = ref.attention64(q[0], ks, vs, float(np.float32(scale)))
        tol, _ = ref.attention_bound(F32, False, hd, n, out, l, big, mean)
        assert (np.abs(got - out) <= tol).all(), size


def test_pages_past_four_gigabytes(hip):
    """Rows written, read and attended to in the last pages of pools of more than 2^32 bytes."""
    from sapphire_amd.device import DeviceArray
    from sapphire_amd.paged import PagedCache, PageTable
    hd, ps, pages = 256, 64, 70000
    c = PagedCache(F32, 1, pages, ps, 1, hd)
    assert c.nbytes > 2**32
    rng = np.random.default_rng(8)
    n = 100
    table = np.array([[pages - 1, pages - 3]], np.int32)
    k, v = (rng.normal(size=(n, 1, hd)).astype(np.float32) for _ in range(2))
    rk, rv = device_rows(k, F32), device_rows(v, F32)
    dt, dp, ds = dev(table), dev(np.arange(n, dtype=np.int32)), dev(np.zeros(n, np.int32))
    c.write(0, rk[0], rv[0], PageTable(dt, 1, 2), dp, seqs=ds)
    ok_, ov_ = device_rows(k * 0, F32), device_rows(v * 0, F32)
    c.read(0, ok_[0], ov_[0], PageTable(dt, 1, 2), dp, seqs=ds)
    q = rng.normal(size=(1, 2, hd)).astype(np.float32)
    rq, ro = device_rows(q, F32), device_rows(q * 0, F32)
    dl = dev(np.array([n], np.int32))
    ws = DeviceArray(max(1, c.attention_workspace_bytes(1, 2, n)))
    c.attention(0, rq[0], ro[0], PageTable(dt, 1, 2), dl, n, 1 / 16, workspace=ws)
    sync()
    np.testing.assert_array_equal(ok_[1].numpy(), rk[2])
    np.testing.assert_array_equal(ov_[1].numpy(), rv[2])
    out, l, size, mean = ref.attention64(q[0], k, v, 1 / 16)
    tol, _ = ref.attention_bound(F32, False, hd, n, out, l, size, mean)
    assert (np.abs(ro[1].numpy()[:2 * hd].reshape(2, hd) - out) <= tol).all()
    for d in (c.k, c.v):
        d.free()


@pytest.mark.parametrize("cache", CACHES, ids=ref.NAME.get)
@pytest.mark.parametrize("hd,nkv,ps", [(64, 2, 16), (128, 1, 48), (256, 1, 64)])
def test_reorder(hip, cache, hd, nkv, ps):
    """Tables, lengths and every byte of both pools; parents used several times and not at all, a parent and a spare page
    that do not exist, full and empty rows, lengths out of range."""
    from sapphire_amd.device import DeviceArray
    from sapphire_amd.paged import PageTable
    rng = np.random.default_rng(ps)
    ld, layers = 4, 3
    lens = np.array([0, 1, 17, ps, ps + 15, 2 * ps + 16, 4 * ps, 3 * ps + 1, -4, 100 * ps], np.int32)
    rows = len(lens)
    pages = rows * ld + rows + 2
    order = rng.permutation(pages).astype(np.int32)
    table, spare = order[:rows * ld].reshape(rows, ld).copy(), order[rows * ld:rows * ld + rows].copy()
    parents = np.array([4, 4, 2, 5, 7, 1, 9, 0, 12, 8], np.int32)
    spare[4] = pages                           # row 4 continues row 7, partly filled
    c = Cache(cache, layers, pages, ps, nkv, hd)
    for w in "kv":
        c.pool[w].a[...] = rng.integers(0, 256, c.pool[w].a.shape, np.uint8)
    c.upload()
    d = [dev(a) for a in (table, parents, lens, spare)]
    to, lo = DeviceArray.empty((rows, ld), np.int32), DeviceArray.empty(rows, np.int32)
    c.c.reorder(PageTable(d[0], rows, ld), d[1], d[2], d[3], PageTable(to, rows, ld), lo)
    sync()
    want_t, want_l = np.full((rows, ld), -1, np.int32), np.zeros(rows, np.int32)
    for b, p in enumerate(parents):
        if not 0 <= p < rows:
            continue
        n = int(np.clip(lens[p], 0, ld * ps))
        want_l[b] = n
        full, rem = divmod(n, ps)
        want_t[b, :full] = table[p, :full]
        if rem and 0 <= spare[b] < pages:
            want_t[b, full] = spare[b]
            held = -(-rem // 16) * 16
            for w in "kv":
                code = c.pool[w].code
                a = c.pool[w].a
                a[:, spare[b], :, :held * code] = a[:, table[p, full], :, :held * code]
                per = (c.pool[w].tile - ps * code) // ps
                a[:, spare[b], :, ps * code:ps * code + held * per] = a[:, table[p, full], :, ps * code:ps * code + held * per]
    np.testing.assert_array_equal(to.numpy(), want_t)
    np.testing.assert_array_equal(lo.numpy(), want_l)
    for w in "kv":
        np.testing.assert_array_equal(c.on[w].numpy(), c.pool[w].a)


class Graph:
    """What `work(stream)` enqueues, captured on a stream of its own through the HIP runtime that the library uses."""

    def __init__(self, work):
        path = next(line.split()[-1] for line in open("/proc/self/maps") if "libamdhip64" in line)
        self.rt, self.stream, self.graph, self.exec = C.CDLL(path), C.c_void_p(), C.c_void_p(), C.c_void_p()
        self.ok(self.rt.hipStreamCreateWithFlags(C.byref(self.stream), 1))
        self.ok(self.rt.hipStreamBeginCapture(self.stream, 2))
        work(self.stream)
        self.ok(self.rt.hipStreamEndCapture(self.stream, C.byref(self.graph)))
        self.ok(self.rt.hipGraphInstantiate(C.byref(self.exec), self.graph, None, None, C.c_size_t(0)))

    @staticmethod
    def ok(rc):
        assert rc == 0, rc

    def replay(self):
        self.ok(self.rt.hipGraphLaunch(self.exec, self.stream))

    def close(self):
        self.ok(self.rt.hipStreamSynchronize(self.stream))
        self.ok(self.rt.hipGraphExecDestroy(self.exec))
        self.ok(self.rt.hipGraphDestroy(self.graph))
        self.ok(self.rt.hipStreamDestroy(self.stream))


@pytest.mark.parametrize("cache,io", [(F32, F32), (Q8_0, F32), (BF16, BF16)], ids=["f32", "q8_0", "bf16"])
def test_captured_step(hip, cache, io):
    """A step (rotate, write, attend, select, reorder) captured into a graph and replayed as the lengths grow, against the
    same calls made eagerly on a second cache between the replays: the same bits."""
    from sapphire_amd import paged
    from sapphire_amd.device import DeviceArray
    from sapphire_amd.paged import PagedCache, PageTable, Rows
    rng = np.random.default_rng(9)
    b, heads, nkv, hd, ps, ld, n = 3, 4, 1, 64, 16, 20, 900
    order = rng.permutation(b * ld + b).astype(np.int32)
    table, spare = dev(order[:b * ld].reshape(b, ld)), dev(order[b * ld:])
    pos = np.array([0, 30, 7], np.int32)
    dpos, dlen = dev(pos), dev(pos + 1)
    freqs = dev(paged.rope_frequencies(hd, 1e4)[0])
    H, es = heads + 2 * nkv, 4 if io == F32 else 2
    qkv, logits, score = DeviceArray(b * H * hd * es), DeviceArray(b * n * 4), DeviceArray(4 * b)

    class Side:
        def __init__(self):
            self.c = PagedCache(cache, 1, b * ld + b, ps, nkv, hd)
            self.out, self.turned = DeviceArray.empty(b * heads * hd * es, np.uint8), DeviceArray(b * (heads + nkv) * hd * es)
            self.lse, self.table = DeviceArray.empty((b, heads)), DeviceArray.empty((b, ld), np.int32)
            self.ws, self.bws = (DeviceArray(max(1, x)) for x in (self.c.attention_workspace_bytes(b, heads, ld * ps),
                                                                    paged.beam_workspace_bytes(n, 1, b)))
            self.new = [DeviceArray.empty(b), *(DeviceArray.empty(b, np.int32) for _ in range(3))]
            for d in (self.c.k, self.c.v, self.out, self.lse, self.table, *self.new):
                d.zero()

        def step(self, stream):
            c, pt = self.c, PageTable(table, b, ld)
            def rows(d, first, count, width):
                return Rows(d.ptr + first * hd * es, io, b, count, hd, width * hd, hd)
            paged.rope(rows(qkv, 0, heads + nkv, H), rows(self.turned, 0, heads + nkv, heads + nkv), dpos, freqs, hd, stream=stream)
            c.write(0, rows(self.turned, heads, nkv, heads + nkv), rows(qkv, heads + nkv, nkv, H), pt, dpos, stream=stream)
            c.attention(0, rows(self.turned, 0, heads, heads + nkv), rows(self.out, 0, heads, heads), pt, dlen, ld * ps, 0.125,
                        lse=self.lse, workspace=self.ws, stream=stream)
            paged.beam_select(logits, n, n, 1, b, score, self.new[0], self.new[1], self.new[2], self.bws, stream=stream)
            c.reorder(pt, self.new[2], dlen, spare, PageTable(self.table, b, ld), self.new[3], stream=stream)

        def results(self):
            return [d.numpy() for d in (self.out, self.lse, self.table, *self.new, self.c.k, self.c.v)]

    def renew():
        qkv.upload(ref.to_type(io, rng.normal(size=(b, H, hd)).astype(np.float32)))
        logits.upload(rng.normal(size=(b, n)).astype(np.float32))
        score.upload(-np.abs(rng.normal(size=b)).astype(np.float32))
    replayed, eager = Side(), Side()
    renew()
    graph = Graph(replayed.step)
    for k in range(40):
        graph.replay()
        eager.step(None)
        sync()
        for i, (x, y) in enumerate(zip(replayed.results(), eager.results())):
            np.testing.assert_array_equal(x, y, err_msg=f"replay {k}, result {i}")
        assert np.isfinite(replayed.lse.numpy()).all()
        pos = pos + 5
        dpos.upload(pos)
        dlen.upload(pos + 1)
        renew()
    graph.close()


def test_streams(hip):
    """The same call on a stream of its own, beside another on the null stream with its own workspace."""
    from sapphire_amd import load
    L = load()
    s = L.sapphire_stream_create()
    rng = np.random.default_rng(10)
    attend_case(rng, F32, F32, 128, 1, 4, 32, [900, 40], stream=s)
    attend_case(rng, Q4_0, F32, 128, 1, 4, 32, [900, 40], stream=s)
    assert L.sapphire_stream_synchronize(s) == 0 and L.sapphire_stream_destroy(s) == 0


@pytest.mark.parametrize("cache,io,heads", [(F32, F32, 4), (F32, F32, 20), (F16, F16, 3), (Q8_0, BF16, 12)], ids=["few", "f32", "f16", "q8_0"])
@pytest.mark.parametrize("lens", [[40, 3], [3000, 200]], ids=["one", "pieces"])
def test_attention_in_place(hip, cache, io, heads, lens):
    """out is q itself: the bits of the call with an out of its own."""
    from sapphire_amd.device import DeviceArray
    from sapphire_amd.paged import PageTable
    rng = np.random.default_rng(16)
    hd, ps = 64, 16
    table, pages = tables(rng, lens, ps)
    c = Cache(cache, 1, pages, ps, 1, hd)
    for s, n in enumerate(lens):
        c.fill(0, table, s, rng.normal(size=(n, 1, hd)).astype(np.float32), rng.normal(size=(n, 1, hd)).astype(np.float32))
    c.upload()
    q = device_rows(rng.normal(size=(2, heads, hd)).astype(np.float32), io)
    out = device_rows(np.zeros((2, heads, hd), np.float32), io)
    dt, dl = dev(table), dev(np.array(lens, np.int32))
    ws = DeviceArray(max(16, c.c.attention_workspace_bytes(2, heads, max(lens))))
    for o in (out, q):
        c.c.attention(0, q[0], o[0], PageTable(dt, *table.shape), dl, max(lens), 0.2, workspace=ws)
    sync()
    np.testing.assert_array_equal(out[1].numpy(), q[1].numpy())


@pytest.mark.parametrize("cache,io,heads", [(F32, F32, 4), (BF16, BF16, 8), (F16, F32, 6), (Q8_0, F32, 4), (Q4_0, F16, 8)],
                         ids=["f32", "bf16", "f16_f32", "q8_0", "q4_0"])
def test_workspace_of_the_largest_call(hip, cache, io, heads):
    """One workspace, of the size for the largest batch and length, serves smaller calls: nothing behind it is written, and
    the outputs are the bits of a call with a workspace of its own."""
    from sapphire_amd.device import DeviceArray
    from sapphire_amd.paged import PageTable
    rng = np.random.default_rng(17)
    hd, ps, top = 64, 64, 9000
    lens = [top, 1, 4500, 700, 8999, 64, 0, 130]
    table, pages = tables(rng, [top], ps)                      # (all sequences read the same pages)
    table = np.repeat(table, 520, 0)
    c = Cache(cache, 1, pages, ps, 1, hd)
    c.fill(0, table, 0, rng.normal(size=(top, 1, hd)).astype(np.float32), rng.normal(size=(top, 1, hd)).astype(np.float32))
    c.upload()
    nbytes, guard = c.c.attention_workspace_bytes(520, heads, top), 8 << 20
    ws = DeviceArray.from_numpy(np.full(nbytes + guard, 0x5a, np.uint8))
    dt = dev(table)
    for batch, most in [(1, top), (2, top), (3, 5000), (8, top), (60, 2000), (129, top), (255, 300), (256, top), (511, top), (512, top), (520, top)]:
        n = np.minimum(np.resize(lens, batch), most).astype(np.int32)
        q = device_rows(rng.normal(size=(batch, heads, hd)).astype(np.float32), io)
        dl, outs = dev(n), []
        for w in (ws, DeviceArray(max(16, c.c.attention_workspace_bytes(batch, heads, most)))):
            outs.append(device_rows(np.zeros((batch, heads, hd), np.float32), io))
            c.c.attention(0, q[0], outs[-1][0], PageTable(dt, *table.shape), dl, most, 0.2, workspace=w)
            sync()
        np.testing.assert_array_equal(outs[0][1].numpy(), outs[1][1].numpy(), err_msg=f"{batch} {most}")
        assert (ws.numpy()[nbytes:] == 0x5a).all(), (batch, most)


def test_two_streams_at_once(hip):
    """Calls on two streams, each with its own workspace and outputs, over one cache: the bits of calls one after the other."""
    from sapphire_amd import load
    from sapphire_amd.device import DeviceArray
    from sapphire_amd.paged import PageTable
    L = load()
    rng = np.random.default_rng(14)
    hd, ps, heads, lens = 128, 32, 4, [1500, 700, 90]
    table, pages = tables(rng, lens, ps)
    c = Cache(Q8_0, 1, pages, ps, 1, hd)
    for s, n in enumerate(lens):
        c.fill(0, table, s, rng.normal(size=(n, 1, hd)).astype(np.float32), rng.normal(size=(n, 1, hd)).astype(np.float32))
    c.upload()
    dt, dl = dev(table), dev(np.array(lens, np.int32))
    streams = [L.sapphire_stream_create() for _ in range(2)]
    qs = [device_rows(rng.normal(size=(3, heads, hd)).astype(np.float32), F32) for _ in range(20)]
    ws = [DeviceArray(c.c.attention_workspace_bytes(3, heads, 1500)) for _ in range(2)]
    outs = [[device_rows(np.zeros((3, heads, hd), np.float32), F32) for _ in qs] for _ in range(2)]
    for side in range(2):
        for i, q in enumerate(qs):
            c.c.attention(0, q[0], outs[side][i][0], PageTable(dt, *table.shape), dl, 1500, 0.1, workspace=ws[i % 2 if side else 0],
                          stream=streams[i % 2] if side else None)
        sync()
    for a, b in zip(*outs):
        np.testing.assert_array_equal(a[1].numpy(), b[1].numpy())
    for s in streams:
        L.sapphire_stream_destroy(s)


@pytest.mark.parametrize("cache", CACHES, ids=ref.NAME.get)
def test_write_to_one_place_twice(hip, cache):
    """Which of two rows for one place is kept is open; every other byte is as it should be."""
    from sapphire_amd.paged import PageTable
    rng = np.random.default_rng(15)
    hd, ps, t = 128, 16, 40
    c = Cache(cache, 1, 3, ps, 2, hd)
    pos = np.arange(t, dtype=np.int32)
    pos[[7, 21]] = 30
    x = {w: rng.normal(size=(t, 2, hd)).astype(np.float32) for w in "kv"}
    rk, rv = device_rows(x["k"], F32), device_rows(x["v"], F32)
    dt, ds = dev(np.array([[2, 0, 1]], np.int32)), dev(np.zeros(t, np.int32))
    c.c.write(0, rk[0], rv[0], PageTable(dt, 1, 3), dev(pos), seqs=ds)
    sync()
    for w in "kv":
        got, spare = c.on[w].numpy(), ref.Pool(w, cache, 1, 3, ps, 2, hd)
        for p, page in ((q, [2, 0, 1][q // ps]) for q in range(3 * ps)):
            rows = np.flatnonzero(pos == p)
            if p == 30:                        # taken over as it is: what remains to be compared is the rest
                at, _ = spare._at(p % ps)
                for h in range(2):
                    a = np.unique(np.concatenate([np.ravel(at[:, None] + np.arange({F32: 4, BF16: 2, F16: 2}.get(cache, 1))),
                                                  np.ravel(spare._scale_at(p % ps)[:, None] + np.arange(4)) if cache in (Q8_0, Q4_0) else at[:0]]))
                    c.pool[w].a[0, page, h, a] = got[0, page, h, a]
            elif len(rows):
                c.pool[w].put(0, page, p % ps, x[w][rows[0]])
        np.testing.assert_array_equal(got, c.pool[w].a, err_msg=w)


def test_results_do_not_depend_on_the_batch(hip):
    """A sequence's bits beside others equal its bits in another place with other neighbours (same max_length and batch)."""
    from sapphire_amd.device import DeviceArray
    from sapphire_amd.paged import PageTable
    rng = np.random.default_rng(11)
    hd, ps, heads = 128, 32, 4
    lens = [700, 90, 33, 1]
    table, pages = tables(rng, lens, ps)
    c = Cache(Q8_0, 1, pages, ps, 1, hd)
    for s, n in enumerate(lens):
        c.fill(0, table, s, rng.normal(size=(n, 1, hd)).astype(np.float32), rng.normal(size=(n, 1, hd)).astype(np.float32))
    c.upload()
    q = rng.normal(size=(4, heads, hd)).astype(np.float32)
    got = []
    for order in ([0, 1, 2, 3], [3, 2, 1, 0], [1, 1, 0, 0]):
        rq, ro = device_rows(q[order], F32), device_rows(q * 0, F32)
        dt, dl = dev(table[order]), dev(np.array(lens, np.int32)[order])
        ws = DeviceArray(max(1, c.c.attention_workspace_bytes(4, heads, 700)))
        c.c.attention(0, rq[0], ro[0], PageTable(dt, *table.shape), dl, 700, 0.1, workspace=ws)
        sync()
        o = ro[1].numpy()[:q.size].reshape(q.shape)
        got.append({s: o[i] for i, s in enumerate(order)})
    for g in got[1:]:
        for s in g:
            np.testing.assert_array_equal(g[s], got[0][s])


@pytest.mark.parametrize("cache", [F32, Q8_0, Q4_0], ids=ref.NAME.get)
def test_beam_search_decode(hip, cache):
    """Fourteen steps of beam search (two requests of three beams, two layers) through rotary rows, cache writes,
    attention, selection and reordering, as a server runs them, against histories kept per beam in 64 bits."""
    from sapphire_amd import paged
    from sapphire_amd.device import DeviceArray
    from sapphire_amd.paged import PageTable, Rows
    rng = np.random.default_rng(12)
    R, W, L, heads, nkv, hd, ps, vocab, steps, end = 2, 3, 2, 4, 1, 64, 16, 50, 22, 1
    B, H = R * W, heads + 2 * nkv
    emb = rng.normal(size=(vocab, L, H, hd)).astype(np.float32)
    head = (rng.normal(size=(L * heads * hd, vocab)) * 0.3).astype(np.float32)
    freqs, _ = paged.rope_frequencies(hd, 1e4)
    ld = -(-steps // ps) + 1
    pages = 4 * B * ld
    c = Cache(cache, L, pages, ps, nkv, hd)
    free = list(rng.permutation(pages).astype(np.int32))
    table, spare = np.full((B, ld), -1, np.int32), np.array([free.pop() for _ in range(B)], np.int32)
    lens = np.zeros(B, np.int32)
    tok = rng.integers(2, vocab, R).repeat(W)
    score, done = np.tile([0, -np.inf, -np.inf], R).astype(np.float32), np.zeros(B, np.int32)
    hist = [[[] for _ in range(L)] for _ in range(B)]           # (k, v) as stored
    score64 = score.astype(np.float64)
    dfreqs = dev(freqs)
    ws = DeviceArray(max(1, c.c.attention_workspace_bytes(B, heads, ld * ps)))
    bws = DeviceArray(paged.beam_workspace_bytes(vocab, R, W))
    for step in range(steps):
        for b in range(B):                                     # a page for the new position where one begins
            if lens[b] % ps == 0:
                table[b, lens[b] // ps] = free.pop()
        dt, dpos, dlen = dev(table), dev(lens), dev(lens + 1)
        pt = PageTable(dt, B, ld)
        outs, outs64 = [], []
        for l in range(L):
            x = emb[tok, l]
            dx, dy = dev(x), DeviceArray.empty((B, heads + nkv, hd))
            do = DeviceArray.empty((B, heads, hd))
            rows = lambda d, first, n, width: Rows(d.ptr + 4 * first * hd, F32, B, n, hd, width * hd, hd)      # noqa: E731
            paged.rope(rows(dx, 0, heads + nkv, H), rows(dy, 0, heads + nkv, heads + nkv), dpos, dfreqs, hd)
            c.c.write(l, rows(dy, heads, nkv, heads + nkv), rows(dx, heads + nkv, nkv, H), pt, dpos)
            c.c.attention(l, rows(dy, 0, heads, heads + nkv), rows(do, 0, heads, heads), pt, dlen, ld * ps, 0.125, workspace=ws)
            sync()
            turned = dy.numpy()
            want = ref.rope64(x[:, :heads + nkv], lens, freqs, hd, False, 1.0)
            assert np.abs(turned - want).max() <= 2.0**-21 * np.abs(x).max()
            outs.append(do.numpy())
            o64 = np.zeros((B, heads, hd))
            for b in range(B):
                hist[b][l].append((ref.stored(cache, turned[b, heads:]), ref.stored(cache, x[b, heads + nkv:])))
                k, v = (np.stack([e[i] for e in hist[b][l]]) for i in (0, 1))
                o64[b], l64, size, mean = ref.attention64(turned[b, :heads], k, v, 0.125)
                tol, _ = ref.attention_bound(F32, False, hd, len(k), o64[b], l64, size, mean)
                assert (np.abs(outs[-1][b] - o64[b]) <= tol).all(), (step, l, b)
            outs64.append(o64)
        logits = (np.stack(outs, 1).reshape(B, -1) @ head).astype(np.float32)
        dl, ds, dd = dev(logits), dev(score), dev(done)
        so, to, po, eo = DeviceArray.empty(B), *(DeviceArray.empty(B, np.int32) for _ in range(3))
        paged.beam_select(dl, vocab, vocab, R, W, ds, so, to, po, bws, done=dd, done_out=eo, end_token=end)
        t2, l2, dsp = DeviceArray.empty((B, ld), np.int32), DeviceArray.empty(B, np.int32), dev(spare)
        dn = dev(lens + 1)
        c.c.reorder(pt, po, dn, dsp, PageTable(t2, B, ld), l2)
        sync()
        ws_, wt, wp, wd = ref.beams64(logits, score, done, R, W, end)
        np.testing.assert_array_equal(to.numpy(), wt)
        np.testing.assert_array_equal(po.numpy(), wp)
        np.testing.assert_array_equal(eo.numpy(), wd)
        assert np.abs(so.numpy() - ws_)[np.isfinite(ws_)].max() <= 1e-5 * np.abs(ws_[np.isfinite(ws_)]).max()
        parents = po.numpy()
        hist = [[list(hist[p][l]) for l in range(L)] for p in parents]
        old = table[:, lens[0] // ps].copy()
        lens = l2.numpy()
        assert (lens == step + 1).all()
        table = t2.numpy()
        if (step + 1) % ps:
            spare = old                                        # the pages copied from are the next spares
        tok, score, done = to.numpy(), so.numpy(), eo.numpy()
    assert len(set(parents)) < B or done.any()                 # beams were dropped along the way


def compare_special(got, lse, q, k, v, scale, io, n, weights=0.0):
    """Outputs against 64 bits where some are NaN or infinite: these have to be the same, the others within the bound of an fp32
    evaluation whose weights are off by `weights`, relative."""
    with np.errstate(all="ignore"):
        out, l, size, mean = ref.attention64(q, k, v, scale)
        assert np.array_equal(np.isnan(got), np.isnan(out)), np.argwhere(np.isnan(got) != np.isnan(out))[:4]
        inf = np.isinf(out)
        assert np.array_equal(got[inf], out[inf]) and np.array_equal(np.isinf(got), inf)
        tol, ltol = ref.attention_bound(io, False, q.shape[1], n, out, l, size, mean)
        tol = tol + 2 * weights * mean
        fin = np.isfinite(out)
        assert (np.abs(got - out)[fin] <= tol[fin]).all(), np.nanmax((np.abs(got - out) / tol)[fin])
        assert (np.abs(lse - l) <= ltol).all()


def attend(c, table, lens, q, io, scale, nkv):
    """(out, lse, q as it was rounded) of one call."""
    from sapphire_amd.device import DeviceArray
    from sapphire_amd.paged import PageTable
    rq, ro = device_rows(q, io), device_rows(q * 0, io)
    dt, dl, dlse = dev(table), dev(np.array(lens, np.int32)), DeviceArray.empty(q.shape[:2])
    ws = DeviceArray(max(16, c.c.attention_workspace_bytes(len(lens), q.shape[1], max(lens))))
    c.c.attention(0, rq[0], ro[0], PageTable(dt, *table.shape), dl, max(lens), scale, lse=dlse, workspace=ws)
    sync()
    return ref.from_type(io, ro[1].numpy()[:q.size]).reshape(q.shape).astype(np.float64), dlse.numpy(), ref.from_type(io, rq[3])


@pytest.mark.parametrize("cache", [Q8_0, Q4_0], ids=ref.NAME.get)
@pytest.mark.parametrize("io", [F32, BF16, F16], ids=ref.NAME.get)
@pytest.mark.parametrize("hd,heads", [(64, 4), (64, 7), (128, 4), (128, 8), (256, 1), (256, 4), (256, 5), (256, 8), (256, 20)])
def test_attention_nan_blocks_of_v(hip, cache, io, hd, heads):
    """A NaN or an infinity in a block of V makes that block's dims NaN, in every head that reads it, and no other."""
    rng = np.random.default_rng(hd + heads)
    lens, ps = [200, 200, 1500, 37, 40], 48
    table, pages = tables(rng, lens, ps)
    c = Cache(cache, 1, pages, ps, 1, hd)
    ks, vs = [], []
    for s, n in enumerate(lens):
        k, v = (rng.normal(size=(n, 1, hd)).astype(np.float32) for _ in range(2))
        if s == 0:
            v[5, 0, 3] = np.nan
        elif s == 1:
            v[77, 0, hd - 1], v[199, 0, hd - 1] = np.inf, np.nan
        elif s == 2:
            v[0, 0, 32], v[1499, 0, hd - 40] = -np.inf, np.nan
        elif s == 3:
            v[36, 0, ::32] = np.nan            # all of them
        ks.append(ref.stored(cache, k))
        vs.append(ref.stored(cache, v))
        c.fill(0, table, s, k, v)
    c.upload()
    got, lse, q = attend(c, table, lens, rng.normal(size=(len(lens), heads, hd)).astype(np.float32), io, 1 / np.sqrt(hd), 1)
    for s, n in enumerate(lens):
        assert np.isnan(got[s]).any() == (s < 4)
        # bf16 rows: the weights' first 16 bits
        compare_special(got[s], lse[s], q[s], ks[s], vs[s], 1 / np.sqrt(hd), io, n, 2.0**-15 if io == BF16 else 0.0)


@pytest.mark.parametrize("cache,io", [(BF16, BF16), (F16, F16), (F32, F32), (BF16, F32), (F16, F32)],
                         ids=["bf16", "f16", "f32", "bf16-f32", "f16-f32"])
@pytest.mark.parametrize("hd,heads", [(64, 1), (64, 20), (128, 4), (128, 7), (256, 4), (256, 16)])
def test_attention_infinite_v(hip, cache, io, hd, heads):
    """Infinities in V reach their own dim as infinities of their sign, NaN where both signs meet or one is there already."""
    rng = np.random.default_rng(hd + heads)
    lens, ps = [200, 33, 1500, 40, 700], 32
    table, pages = tables(rng, lens, ps)
    c = Cache(cache, 1, pages, ps, 1, hd)
    ks, vs = [], []
    for s, n in enumerate(lens):
        k, v = (rng.normal(size=(n, 1, hd)).astype(np.float32) for _ in range(2))
        if s == 0:
            v[5, 0, 3], v[199, 0, hd - 1] = np.inf, -np.inf
        elif s == 1:
            v[32, 0, 0], v[31, 0, 0], v[0, 0, 9], v[7, 0, 10] = -np.inf, -np.inf, np.nan, np.inf
        elif s == 2:
            v[0, 0, 32], v[1499, 0, 32] = np.inf, -np.inf      # both: NaN
            v[700:, 0, 33] = np.inf
        elif s == 3:
            k[:], v[:, 0, :20] = 0, np.inf                     # all weights alike
        ks.append(ref.stored(cache, k))
        vs.append(ref.stored(cache, v))
        c.fill(0, table, s, k, v)
    c.upload()
    got, lse, q = attend(c, table, lens, rng.normal(size=(len(lens), heads, hd)).astype(np.float32), io, 1 / np.sqrt(hd), 1)
    for s, n in enumerate(lens):
        assert np.isinf(got[s]).any() == (s < 4)
        compare_special(got[s], lse[s], q[s], ks[s], vs[s], 1 / np.sqrt(hd), io, n, 2.0**-16 if io != F32 else 0.0)


@pytest.mark.parametrize("cache,io", [(F32, F32), (BF16, BF16), (Q4_0, F16)], ids=["f32", "bf16", "q4_0"])
def test_slices_of_one_buffer(hip, cache, io):
    """q and out beside each other in every token's row, K and V read to interleaved heads and to the two halves of one row:
    the bits of calls with buffers of their own, and nothing between them written."""
    from sapphire_amd.device import DeviceArray
    from sapphire_amd.paged import PageTable, Rows
    rng = np.random.default_rng(19)
    hd, ps, heads, nkv, b = 64, 16, 4, 2, 3
    es, lens = 4 if io == F32 else 2, [40, 3, 900]
    table, pages = tables(rng, lens, ps)
    c = Cache(cache, 1, pages, ps, nkv, hd)
    for s, n in enumerate(lens):
        c.fill(0, table, s, rng.normal(size=(n, nkv, hd)).astype(np.float32), rng.normal(size=(n, nkv, hd)).astype(np.float32))
    c.upload()
    q = ref.to_type(io, rng.normal(size=(b, heads, hd)).astype(np.float32))
    dt, dl, pos = dev(table), dev(np.array(lens, np.int32)), dev(np.array(lens, np.int32) - 1)
    pt = PageTable(dt, *table.shape)
    ws = DeviceArray(max(16, c.c.attention_workspace_bytes(b, heads, max(lens))))
    dq, out, k, v = dev(q), dev(np.zeros_like(q)), dev(np.zeros_like(q[:, :nkv])), dev(np.zeros_like(q[:, :nkv]))
    plain = lambda d, h: Rows(d.ptr, io, b, h, hd)                      # noqa: E731
    c.c.attention(0, plain(dq, heads), plain(out, heads), pt, dl, max(lens), 0.2, workspace=ws)
    c.c.read(0, plain(k, nkv), plain(v, nkv), pt, pos)
    sync()
    want, wk, wv = out.numpy(), k.numpy(), v.numpy()
    for at in ([0, heads + 1], [heads + 2, 1]):        # q first, out first
        row = np.full((b, 2 * heads + 3, hd), 7, q.dtype)
        row[:, at[0]:at[0] + heads] = q
        d = dev(row)
        rows = [Rows(d.ptr + es * hd * i, io, b, heads, hd, token_stride=row.shape[1] * hd) for i in at]
        c.c.attention(0, *rows, pt, dl, max(lens), 0.2, workspace=ws)
        sync()
        row[:, at[1]:at[1] + heads] = want
        np.testing.assert_array_equal(d.numpy(), row)
    both = np.stack([wk, wv], 2)                       # [tokens][heads][2][hd]
    for shape, ts, hs, step, ans in ((both.shape, 2 * nkv * hd, 2 * hd, hd, both),
                                     ((b, 2, nkv, hd), 2 * nkv * hd, hd, nkv * hd, np.stack([wk, wv], 1)),
                                     ((nkv, b, 2, hd), 2 * hd, 2 * b * hd, hd, both.transpose(1, 0, 2, 3))):
        d = dev(np.zeros(shape, q.dtype))
        c.c.read(0, *(Rows(d.ptr + es * step * i, io, b, nkv, hd, ts, hs) for i in (0, 1)), pt, pos)
        sync()
        np.testing.assert_array_equal(d.numpy(), ans)
    hs = 2 * b * hd + hd                               # heads that start in the middle of a token's pair
    host = np.zeros(nkv * hs, q.dtype)
    d = dev(host)
    c.c.read(0, *(Rows(d.ptr + es * hd * i, io, b, nkv, hd, 2 * hd, hs) for i in (0, 1)), pt, pos)
    sync()
    host.reshape(nkv, hs)[:, :2 * b * hd] = both.transpose(1, 0, 2, 3).reshape(nkv, -1)
    np.testing.assert_array_equal(d.numpy(), host)


@pytest.mark.parametrize("cache,io", [(F32, F32), (BF16, F32), (BF16, BF16), (Q8_0, F32), (Q8_0, BF16), (Q4_0, F32), (Q4_0, BF16)],
                         ids=["f32", "bf16-f32", "bf16", "q8_0", "q8_0-bf16", "q4_0", "q4_0-bf16"])
@pytest.mark.parametrize("hd,heads", [(64, 4), (128, 8), (256, 4), (256, 8)])
def test_attention_of_the_largest_values(hip, cache, io, hd, heads):
    """V just below 2^119 (Q4_0: 2^115) over the number of positions, nearly all of them with weights of almost 2^8: the
    maximum stays that of the first tiles, which scores up to 8 log2 units above it do not move. Whole sequences, so that
    every wave's first tiles lie in the first 128 positions."""
    from sapphire_amd.device import DeviceArray
    from sapphire_amd.paged import PageTable
    rng = np.random.default_rng(hd)
    n, ps, batch = 2048, 256, 512
    table = np.repeat(rng.permutation(n // ps).astype(np.int32)[None], batch, 0)
    c = Cache(cache, 1, n // ps, ps, 1, hd)
    k, v = np.zeros((n, 1, hd), np.float32), np.empty((n, 1, hd), np.float32)
    k[128:, 0, 0] = 7.9 * np.log(2)
    v[...] = 2.0**(119 - 11 - (4 if cache == Q4_0 else 0)) * 0.99
    v[:, 0, ::3] *= -0.7
    c.fill(0, table, 0, k, v)
    c.upload()
    q = np.zeros((batch, heads, hd), np.float32)
    q[..., 0] = 1.0
    rq, ro = device_rows(q, io), device_rows(q, io)
    dt, dl, dlse = dev(table), dev(np.full(batch, n, np.int32)), DeviceArray.empty((batch, heads))
    ws = DeviceArray(max(16, c.c.attention_workspace_bytes(batch, heads, n)))
    c.c.attention(0, rq[0], ro[0], PageTable(dt, *table.shape), dl, n, 1.0, lse=dlse, workspace=ws)
    sync()
    got = ref.from_type(io, ro[1].numpy()[:q.size]).reshape(q.shape).astype(np.float64)
    assert (got == got[:1, :1]).all()
    compare_special(got[0], dlse.numpy()[0], q[0], ref.stored(cache, k), ref.stored(cache, v), 1.0, io, n,
                    0.0 if io == F32 else 2.0**-16 if cache == BF16 else 2.0**-15)


@pytest.mark.parametrize("cache", CACHES[:2] + CACHES[3:], ids=ref.NAME.get)
@pytest.mark.parametrize("hd,heads", [(64, 4), (128, 7), (256, 4), (256, 8)])
def test_attention_of_the_largest_keys(hip, cache, hd, heads):
    """K just below 2^85 in every dim, under queries of one sign that bring the scores back."""
    rng = np.random.default_rng(hd)
    n, ps = 150, 16
    table, pages = tables(rng, [n], ps)
    c = Cache(cache, 1, pages, ps, 1, hd)
    k = np.full((n, 1, hd), 2.0**85 * 0.99, np.float32)
    k[1::3] *= -1
    k[2::3, 0, ::2] *= -0.4
    v = rng.normal(size=(n, 1, hd)).astype(np.float32)
    c.fill(0, table, 0, k, v)
    c.upload()
    q = (rng.uniform(0.5, 1, (1, heads, hd)) * 2.0**-85).astype(np.float32)
    got, lse, q = attend(c, table, [n], q, F32, 1 / hd, 1)
    compare_special(got[0], lse[0], q[0], ref.stored(cache, k), ref.stored(cache, v), 1 / hd, F32, n)


# the weights' bits that meet V: two roundings to the rows' type over a cache of that type (fp16: of 2^-22, and of half the
# smallest subnormal, 2^-25, for a largest weight of 2^7 at least), over a quantized one the first 16 bits, truncated, for bf16 rows
# and all 24 otherwise
WEIGHTS = {(BF16, BF16): 2.0**-16, (F16, F16): 2.0**-21, (Q8_0, BF16): 2.0**-15, (Q4_0, BF16): 2.0**-15}


@pytest.mark.parametrize("cache,io", IO, ids=IDS)
@pytest.mark.parametrize("hd,heads", [(64, 8), (128, 4), (256, 5)])
def test_attention_weights_keep_their_bits(hip, cache, io, hd, heads):
    """Sums that nearly cancel show the weights' own rounding, which an output's would hide: half of the positions weigh 1 and
    have values about 1, the others weigh a third and have values of about -3. Beside them random rows. lse is fp32's."""
    rng = np.random.default_rng(hd)
    lens, ps, scale = [300, 300, 77, 1], 48, 1.0 if hd == 64 else 0.5
    table, pages = tables(rng, lens, ps)
    c = Cache(cache, 1, pages, ps, 1, hd)
    q = rng.normal(size=(len(lens), heads, hd)).astype(np.float32)
    q[0] = 0
    q[0, :, 0] = (1 + 0.01 * np.arange(heads)) / scale
    ks, vs = [], []
    for s, n in enumerate(lens):
        k, v = (rng.normal(size=(n, 1, hd)).astype(np.float32) for _ in range(2))
        if s == 0:
            k[:], v[:] = 0, 1
            k[1::2, 0, 0], v[1::2] = -np.log(3), -np.linspace(2.9, 3.1, hd)
        ks.append(ref.stored(cache, k))
        vs.append(ref.stored(cache, v))
        c.fill(0, table, s, k, v)
    c.upload()
    got, lse, q = attend(c, table, lens, q, io, scale, 1)
    for s, n in enumerate(lens):
        compare_special(got[s], lse[s], q[s], ks[s], vs[s], scale, io, n, WEIGHTS.get((cache, io), 0.0))


@pytest.mark.parametrize("cache,io", [(F32, F32), (BF16, F32), (BF16, BF16), (F16, F16)], ids=["f32", "bf16-f32", "bf16", "f16"])
@pytest.mark.parametrize("heads", [2, 9])
def test_attention_nan_v_where_scores_are_minus_infinity(hip, cache, io, heads):
    """A NaN of V makes its dim NaN whatever its weight, in a tile with others as in a wave's or a piece's share in which
    nothing else weighs; unless no score of the sequence is above -inf."""
    rng = np.random.default_rng(heads)
    hd, ps, lens = 64, 32, [40, 700, 3000, 50]
    table, pages = tables(rng, lens, ps)
    c = Cache(cache, 1, pages, ps, 1, hd)
    ks, vs = [], []
    for s, n in enumerate(lens):
        k, v = (rng.normal(size=(n, 1, hd)).astype(np.float32) for _ in range(2))
        k[:n // 2 if s < 3 else n, 0, 0] = -np.inf
        v[5, 0, 3], v[n // 2 - 1, 0, 60] = np.nan, np.nan
        ks.append(k)
        vs.append(ref.stored(cache, v))
        c.fill(0, table, s, k, v)
    c.upload()
    q = rng.normal(size=(len(lens), heads, hd)).astype(np.float32)
    q[..., 0] = 1.0
    got, lse, q = attend(c, table, lens, q, io, 0.125, 1)
    assert (got[3] == 0).all() and np.isneginf(lse[3]).all()
    for s, n in enumerate(lens[:3]):
        assert np.isnan(got[s][:, [3, 60]]).all(), s
        rest = np.arange(hd)[~np.isin(np.arange(hd), [3, 60])]
        k = ref.stored(cache, ks[s][n // 2:])
        out, l, size, mean = ref.attention64(q[s], k, vs[s][n // 2:], 0.125)
        tol, ltol = ref.attention_bound(io, False, hd, n, out, l, size, mean)
        tol = tol + 2 * WEIGHTS.get((cache, io), 0.0) * mean
        assert (np.abs(got[s] - out) <= tol)[:, rest].all() and (np.abs(lse[s] - l) <= ltol).all(), s
