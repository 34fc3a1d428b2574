"""Bounds of pages and the choice by them on the GPU against plain numpy. Bounds are 16-bit numbers and choices whole ones: both
have to be equal (scores of 64 bits on both sides; ties are made on purpose)."""
import numpy as np
import pytest

from tests import paged_ref as ref
from tests.paged_ref import BF16, F16, F32, Q4_0, Q8_0
from tests.test_paged_gpu import CACHES, Cache, Graph, dev, device_rows, sync, tables

pytestmark = pytest.mark.gpu


def outward(x, up, f16):
    """fp32 as the bits of the next 16-bit number up or down (NaN: NaN)."""
    if f16:
        return np.asarray(x, np.float16).view(np.uint16)
    b = ref.bf16_bits(x)
    r = ref.from_type(BF16, b)
    over = r < x if up else r > x
    away = (b & 0x8000 == 0) == up
    step = np.where(b & 0x7fff == 0, 1 if up else 0x8001, np.where(away, b + 1, b - 1)).astype(np.uint16)
    return np.where(over, step, b).astype(np.uint16)


def values(bits, f16):
    return (bits.view(np.float16) if f16 else ref.from_type(BF16, bits)).astype(np.float32)


def same_bounds(got, want, f16):
    g, w = values(got, f16), values(want, f16)
    np.testing.assert_array_equal(g, w)                # NaN equals NaN, -0 equals 0


def page_bounds(dtype, k):
    """(lo, hi) bits [heads][2][hd] of fp32 rows [positions][heads][hd] as a cache of that type holds them."""
    x = ref.stored(dtype, k)
    with np.errstate(invalid="ignore"):
        lo, hi = x.min(0), x.max(0)                    # NaN stays
    return np.stack([outward(lo, False, dtype == F16), outward(hi, True, dtype == F16)], 1)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("dtype", CACHES, ids=ref.NAME.get)
def test_bounds(hip, dtype, hd):
    """All pages of ragged rows, then the pages that a few more positions touch; pages of others, and pages that do not exist, stay."""
    rng = np.random.default_rng(dtype * 7 + hd)
    nkv, ps, layers = 3, 48, 2
    lens = [100, 1, 0, 48, 49, 17, 400]
    table, pages = tables(rng, lens, ps)
    table[0, 1] = pages + 4                            # does not exist
    table[6, 3] = -1
    k = [(rng.normal(size=(n, nkv, hd)) * 3).astype(np.float32) for n in lens]
    k[0][3, 1, 5], k[0][4, 1, 6], k[4][0, 0, 40], k[3][20, 2, 7] = np.nan, np.inf, -np.inf, -np.nan
    k[5][:, :, :32] = 0.0
    k[6][:, 0, 1] = np.float32(3.4e38)
    c = Cache(dtype, layers, pages, ps, nkv, hd)       # 0xff: NaN of the float types, behind the last positions
    for s in range(len(lens)):
        c.fill(1, np.where(table < pages, table, -1), s, k[s], k[s])
    c.upload()
    from sapphire_amd.paged import PageTable
    host = np.full((layers, pages, nkv, 2, hd), 0x1234, np.uint16)
    on = dev(host)
    assert c.c.bounds_bytes == host.nbytes
    dt, dn = dev(table), dev(np.array(lens, np.int32))
    pt = PageTable(dt, *table.shape)

    def make(start, ns):
        for s, n in enumerate(ns):
            for i in range(start[s] // ps, -(-n // ps)):
                if n > start[s] and 0 <= table[s, i] < pages:
                    host[1, table[s, i]] = page_bounds(dtype, k[s][i * ps:min(n, (i + 1) * ps)])

    c.c.bounds(1, on, pt, dn, 400)
    sync()
    make([0] * len(lens), lens)
    got = on.numpy()
    same_bounds(got[1], host[1], dtype == F16)
    assert (got[0] == 0x1234).all()
    # shorter, and from some position on; a length beyond the table, a start behind the length
    ns, start = [97, 1, -3, 40, 49, 16, 10**6], [96, 0, 0, 39, 48, 16, 384]
    top = table.shape[1] * ps
    k[6] = np.concatenate([k[6], np.full((top - 400, nkv, hd), np.nan, np.float32)])
    got[...] = 0x1234
    on.upload(got)
    host[...] = 0x1234
    c.c.bounds(1, on, pt, dev(np.array(ns, np.int32)), top - 384, start=dev(np.array(start, np.int32)))
    sync()
    ns = [min(max(n, 0), top) for n in ns]
    make(start, ns)                                    # (the 0xff bytes behind row 6 stand for NaN in all types)
    same_bounds(on.numpy()[1], host[1], dtype == F16)


def test_bounds_of_the_last_positions_only(hip):
    """More new positions than max_new says: the pages of the last ones, and no others."""
    rng = np.random.default_rng(1)
    ps, n = 16, 320
    table, pages = tables(rng, [n], ps)
    k = rng.normal(size=(n, 1, 64)).astype(np.float32)
    c = Cache(F32, 1, pages, ps, 1, 64)
    c.fill(0, table, 0, k, k)
    c.upload()
    from sapphire_amd.paged import PageTable
    for most in (1, 16, 17, 100):
        on = dev(np.full((pages, 1, 2, 64), 0x1234, np.uint16))
        c.c.bounds(0, on, PageTable(dev(table), *table.shape), dev(np.array([n], np.int32)), most)
        sync()
        got = on.numpy()
        made = [i for i in range(n // ps) if (got[table[0, i]] != 0x1234).any()]
        assert made == list(range(made[0], n // ps)) and made[0] * ps <= n - most and len(made) <= most // ps + 2
        for i in made:
            same_bounds(got[table[0, i]], page_bounds(F32, k[i * ps:(i + 1) * ps]), False)


def select64(q, bounds, table, lens, ps, k, first, last, pages, top):
    """q [batch][heads][hd] and bounds [pages][kv][2][hd] as fp32 -> the choice."""
    batch, heads, hd = q.shape
    kv = bounds.shape[1]
    out = np.full((batch, kv, k), -1)
    for b in range(batch):
        np_ = -(-min(max(lens[b], 0), top) // ps)
        there = [i for i in range(np_) if 0 <= table[b, i] < pages]
        for h in range(kv):
            key = []
            for i in there:
                lo, hi = bounds[table[b, i], h].astype(np.float64)
                with np.errstate(invalid="ignore"):
                    x = q[b, h * heads // kv:(h + 1) * heads // kv].astype(np.float64)
                    s = (np.maximum(x, 0) * hi).sum(-1) + (np.minimum(x, 0) * lo).sum(-1)
                    s = np.where(np.isnan(s), np.inf, s).max()
                key.append((0 if i < first or i >= np_ - last else 1, -s, i))
            chosen = sorted(i for _, _, i in sorted(key)[:k])
            out[b, h, :len(chosen)] = chosen
    return out


class Select:
    def __init__(self, rng, dtype, io, nkv, heads, hd, ps, lens, spread=1.0, extra=3):
        from sapphire_amd.device import DeviceArray
        from sapphire_amd.paged import PagedCache, PageTable, Rows
        self.dtype, self.ps, self.lens, self.f16 = dtype, ps, lens, dtype == F16
        self.table, self.pages = tables(rng, lens, ps, extra)
        mid = rng.normal(size=(self.pages, nkv, 1, hd)) * spread
        self.bits = ref.to_type(F16 if self.f16 else BF16, np.concatenate([mid - rng.random(mid.shape), mid + rng.random(mid.shape)], 2))
        self.bits = self.bits.view(np.uint16)
        self.q = ref.from_type(io, ref.to_type(io, rng.normal(size=(len(lens), heads, hd)) * 2))
        self.q_on = dev(ref.to_type(io, self.q))
        self.rows = Rows(self.q_on, io, len(lens), heads, hd)
        # K itself is not read
        self.c = PagedCache(dtype, 1, self.pages, ps, nkv, hd, k=1 << 20, v=1 << 20)
        self.top = max(1, max(lens))
        self.ws = DeviceArray(self.c.select_workspace_bytes(len(lens), self.top))
        self.on, self.dt, self.dn = dev(self.bits), dev(self.table), dev(np.array(lens, np.int32))
        self.pt = PageTable(self.dt, *self.table.shape)
        self.nkv = nkv

    def run(self, k, first, last, stream=None, out=None):
        out = dev(np.full((len(self.lens), self.nkv, k), 77, np.int32)) if out is None else out
        self.c.select(0, self.on, self.rows, self.pt, self.dn, self.top, out, k, first=first, last=last, workspace=self.ws, stream=stream)
        return out

    def want(self, k, first, last):
        return select64(self.q, values(self.bits, self.f16), self.table, self.lens, self.ps, k, first, last, self.pages, self.top)

    def check(self, k, first, last):
        out = self.run(k, first, last)
        sync()
        np.testing.assert_array_equal(out.numpy(), self.want(k, first, last), err_msg=str((k, first, last)))


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("dtype,io,nkv,heads", [(F32, F32, 1, 1), (BF16, BF16, 2, 8), (F16, F16, 3, 3), (Q8_0, F32, 2, 10), (Q4_0, BF16, 1, 17)])
def test_select(hip, hd, dtype, io, nkv, heads):
    rng = np.random.default_rng(hd + heads)
    s = Select(rng, dtype, io, nkv, heads, hd, 16, [16 * 700, 0, 1, 16 * 20 + 3, 16 * 21, 16 * 1000 + 1])
    s.table[3, 4], s.table[3, 7], s.table[5, 999] = -1, s.pages, s.pages + 100      # do not exist
    s.dt.upload(s.table)
    for k, first, last in ((1, 0, 0), (1, 1, 0), (1, 0, 1), (7, 2, 3), (21, 1, 2), (64, 0, 0), (64, 32, 32), (700, 5, 5), (2000, 1, 1)):
        s.check(k, first, last)


@pytest.mark.parametrize("n", [1023, 1024, 1025, 8191, 8192, 8193, 20000])
def test_many_pages(hip, n):
    """Around the numbers of pages at which threads and registers run out."""
    rng = np.random.default_rng(n)
    s = Select(rng, BF16, F32, 1, 2, 64, 16, [16 * n, 16 * n - 40], extra=0)
    for k in (1, 100, n // 2, n - 1, n, n + 5):
        s.check(k, 0, 1)


@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 255, 256, 257])
def test_few_pages(hip, n):
    """Around the number of pages that are ranked at once; some alike, some that do not exist."""
    rng = np.random.default_rng(n)
    s = Select(rng, BF16, F32, 2, 6, 128, 16, [16 * n, 16 * n - 15, 5], extra=0)
    for k in sorted({1, 2, 40, n // 3 + 1, n, n + 3}):
        s.check(k, 0, 0)
        s.check(k, 0, 1)
        if k > 3:
            s.check(k, 2, 2)
    s.bits[...] = s.bits[rng.integers(0, min(4, s.pages), s.pages)]
    s.on.upload(s.bits)
    s.table[0, rng.integers(0, n, n // 5)] = -1
    s.dt.upload(s.table)
    for k in sorted({1, 3, n // 2 + 1, n}):
        s.check(k, 0, 0)
        s.check(k, 1, 0)


def test_ties(hip):
    """Pages alike: the first ones. All alike, groups of alike ones, and many that differ in the last bits only."""
    rng = np.random.default_rng(3)
    s = Select(rng, BF16, F32, 2, 4, 64, 16, [16 * 3000])
    s.bits[...] = s.bits[:1]
    s.on.upload(s.bits)
    for k in (1, 5, 1500, 2999):
        s.check(k, 0, 0)
        s.check(k, 1, 0)
    kind = rng.integers(0, 5, s.pages)
    s.bits[...] = Select(rng, BF16, F32, 2, 4, 64, 16, [16 * 5], extra=0).bits[kind]
    s.on.upload(s.bits)
    for k in (4, 300, 600, 1200, 2400):
        s.check(k, 2, 2)
    # scores next to each other: one dim counts, and the others move it by 2^-40 of it
    q = np.zeros_like(s.q)
    q[:, :, 0], q[:, :, 1] = 1.0, 2.0**-40
    s.q = q
    s.q_on.upload(q)
    s.bits[...] = ref.bf16_bits(np.ones(s.bits.shape))
    s.bits[:, :, 1, 1] = ref.bf16_bits(rng.integers(0, 128, (s.pages, 2)).astype(np.float32))
    s.on.upload(s.bits)
    for k in (1, 40, 1500, 2980):
        s.check(k, 0, 0)


def test_not_finite(hip):
    """NaN and infinities in bounds and q; scores of both infinities."""
    rng = np.random.default_rng(4)
    s = Select(rng, F32, F32, 2, 2, 128, 16, [16 * 50, 16 * 40, 16 * 30])
    v = values(s.bits, False)
    v[s.table[0, 5], 0, 0, 3], v[s.table[0, 9], 0, 1, 4], v[s.table[0, 11], 1, 1, :] = np.nan, np.inf, np.nan
    v[s.table[1, 7], 0, :, 8] = np.inf, -np.inf
    s.bits[...] = ref.bf16_bits(v)
    s.on.upload(s.bits)
    s.q[1, 0, 9], s.q[2, 1] = np.nan, 0.0
    s.q[2, 0, 0] = -np.inf
    s.q_on.upload(s.q)
    for k in (1, 3, 10, 29):
        s.check(k, 0, 0)
        s.check(k, 0, 1)


def test_strides_streams_and_replays(hip):
    """q as a slice of a wider buffer at an odd place; the same choice on another stream, and replayed as lengths change."""
    from tests.test_paged_gpu import C
    rng = np.random.default_rng(5)
    s = Select(rng, BF16, BF16, 2, 6, 128, 32, [32 * 300, 32 * 100 + 5])
    for order, pad, shift in (("thd", 5, 3), ("htd", 2, 1)):
        r = device_rows(s.q, BF16, order, pad, shift)
        s.rows = r[0]
        s.check(20, 1, 1)
    st = hip.sapphire_stream_create()
    out = s.run(20, 1, 1, stream=st)
    sync()
    np.testing.assert_array_equal(out.numpy(), s.want(20, 1, 1))
    hip.sapphire_stream_destroy(st)
    g = Graph(lambda stream: s.run(20, 1, 1, stream=stream, out=out))
    for lens in ([32 * 300, 10], [5000, 0], [32 * 19, 32 * 21]):
        s.lens = lens
        s.dn.upload(np.array(lens, np.int32))
        g.replay()
        sync()
        np.testing.assert_array_equal(out.numpy(), s.want(20, 1, 1))
    g.close()
    assert C
