"""The paged cache's entry points on the CPU: sizes, refusals (before any device work) and the rotary frequencies."""
import ctypes as C
import math

import numpy as np
import pytest

import sapphire_amd
from sapphire_amd import paged
from sapphire_amd._lib import AttentionC, PagedCacheC, PageTableC, RopeC, RowsC
from tests import paged_ref as ref

F32, BF16, F16, Q4_0, Q8_0 = 0, 1, 2, 3, 4
P = 1 << 20                                    # stands for a device address: nothing here reaches the device


@pytest.fixture(scope="module")
def lib():
    return sapphire_amd.load()


def cache(dtype=F32, layers=2, pages=8, ps=32, nkv=2, hd=64, k=P, v=2 * P):
    return PagedCacheC(k, v, dtype, layers, pages, ps, nkv, hd)


def rows(tokens=3, heads=2, hd=64, dtype=F32, data=4 * P, ts=None, hs=None):
    return paged.Rows(data, dtype, tokens, heads, hd, ts, hs)


@pytest.mark.parametrize("dtype", [F32, BF16, F16, Q4_0, Q8_0])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_cache_bytes(lib, dtype, hd):
    c = cache(dtype, 3, 7, 48, 5, hd)
    assert lib.sapphire_paged_cache_bytes(C.byref(c)) == ref.Pool("k", dtype, 3, 7, 48, 5, hd).a.nbytes


@pytest.mark.parametrize("change", [dict(dtype=5), dict(dtype=-1), dict(layers=0), dict(pages=0), dict(ps=0), dict(ps=24),
                                    dict(ps=1040), dict(nkv=0), dict(hd=32), dict(hd=96), dict(hd=512),
                                    dict(pages=2**31 - 1, layers=2**31 - 1, nkv=60000, ps=1024, hd=256)])
def test_cache_refused(lib, change):
    c = cache(**change)
    assert lib.sapphire_paged_cache_bytes(C.byref(c)) == 0
    assert lib.sapphire_paged_attention_workspace_bytes(C.byref(c), 4, 8, 100) == 0
    t, r = PageTableC(P, 3, 4), rows()
    assert lib.sapphire_paged_write_dev(C.byref(c), 0, C.byref(r), C.byref(r), C.byref(t), None, P, None) == -1
    assert lib.sapphire_paged_cache_bytes(None) == 0


MOVES = [dict(c=dict(k=None)), dict(c=dict(v=None)), dict(c=dict(k=P + 8)), dict(layer=-1), dict(layer=2), dict(positions=None),
         dict(k=None), dict(k=dict(tokens=0)), dict(k=dict(tokens=-1)), dict(k=dict(heads=1)), dict(k=dict(hd=128)),
         dict(k=dict(dtype=BF16)), dict(k=dict(dtype=Q8_0), v=dict(dtype=Q8_0)), dict(k=dict(tokens=4)), dict(k=dict(data=4 * P + 2)),
         dict(k=dict(ts=-64)), dict(k=dict(hs=-64)), dict(t=dict(rows=0)), dict(t=dict(ld=0)), dict(t=dict(pages=None)),
         dict(t=dict(rows=2)), dict(k=dict(ts=2**62))]


@pytest.mark.parametrize("change", MOVES, ids=[str(m) for m in MOVES])
def test_moves_refused(lib, change):
    c = cache(**change.get("c", {}))
    r = [C.byref(rows(**change[n])) if change.get(n, 0) is not None and n in change else None if n in change else C.byref(rows())
         for n in ("k", "v")]
    t = PageTableC(**{"pages": P, "rows": 3, "ld": 4, **change.get("t", {})})
    for fn in (lib.sapphire_paged_write_dev, lib.sapphire_paged_read_dev):
        assert fn(C.byref(c), change.get("layer", 1), *r, C.byref(t), None, change.get("positions", P), None) == -1
        assert lib.sapphire_last_error()


def test_read_refuses_overlapping_rows(lib):
    c, t, good = cache(), PageTableC(P, 3, 4), rows()
    for bad in (rows(ts=0), rows(hs=0), rows(ts=64, hs=64), rows(ts=100), rows(hs=32, ts=1000)):
        for pair in ((bad, good), (good, bad)):
            assert lib.sapphire_paged_read_dev(C.byref(c), 0, C.byref(pair[0]), C.byref(pair[1]), C.byref(t), None, P, None) == -1


ATTEND = [dict(q=dict(heads=3)), dict(q=dict(hd=128)), dict(q=dict(dtype=BF16)), dict(c=dict(dtype=BF16), q=dict(dtype=F16), o=dict(dtype=F16)),
          dict(q=dict(dtype=BF16), o=dict(dtype=BF16)), dict(o=dict(tokens=2)), dict(o=dict(heads=2)), dict(o=dict(ts=0)),
          dict(lengths=None), dict(max_length=0), dict(max_length=129), dict(a=None), dict(a=dict(scale=math.nan)),
          dict(a=dict(scale=math.inf)), dict(a=dict(softcap=-1.0)), dict(a=dict(softcap=math.nan)), dict(a=dict(softcap=math.inf)),
          dict(t=dict(rows=2)), dict(layer=-1), dict(layer=2), dict(ws=None), dict(ws=P + 4), dict(c=dict(k=None)), dict(q=None), dict(o=None)]


@pytest.mark.parametrize("change", ATTEND, ids=[str(m) for m in ATTEND])
def test_attention_refused(lib, change):
    c = cache(**{**dict(ps=32), **change.get("c", {})})
    def one(n):
        return None if n in change and change[n] is None else C.byref(rows(**{**dict(heads=4), **change.get(n, {})}))
    t = PageTableC(**{"pages": P, "rows": 3, "ld": 4, **change.get("t", {})})
    a = change.get("a", {})
    a = None if a is None else C.byref(AttentionC(**{**dict(scale=1.0, window=0, softcap=0.0), **a}))
    top = change.get("max_length", 128)
    if "ws" in change:                          # one that is needed
        t, top = PageTableC(P, 3, 400), 12000
        assert lib.sapphire_paged_attention_workspace_bytes(C.byref(c), 3, 4, top) > 0
    assert lib.sapphire_paged_attention_dev(C.byref(c), change.get("layer", 0), one("q"), one("o"), C.byref(t), change.get("lengths", P),
                                            top, a, None, change.get("ws", P), None) == -1
    assert lib.sapphire_last_error()


# (data, token stride, head stride) of three tokens of two heads of 64 dims, in elements from a first one of [256][64]
OVERLAPS = [((0, 128, 64), (64, 128, 64)), ((0, 128, 64), (128, 128, 64)), ((128, 128, 64), (0, 128, 64)), ((0, 128, 64), (0, 256, 64)),
            ((0, 128, 64), (0, 256, 128)), ((0, 64, 192), (64, 64, 192)), ((0, 64, 192), (0, 128, 64)), ((0, 256, 64), (127, 256, 64)),
            ((0, 256, 64), (129, 256, 64)), ((0, 256, 128), (63, 256, 128)), ((0, 256, 128), (256, 256, 128)), ((0, 200, 64), (136, 200, 64)),
            ((0, 0, 64), (64, 128, 64))]


@pytest.mark.parametrize("dtype", [F32, BF16], ids=ref.NAME.get)
@pytest.mark.parametrize("a,b", OVERLAPS)
def test_overlapping_rows_refused(lib, dtype, a, b):
    """Rows that share elements in some other way than being each other: an attention's out with its q, a read's k with its v."""
    es = 4 if dtype == F32 else 2
    at = [{(off + t * ts + h * hs + d) for t in range(3) for h in range(2) for d in range(64)} for off, ts, hs in (a, b)]
    assert at[0] & at[1]
    c, t = cache(dtype), PageTableC(P, 3, 4)
    x, y = (rows(dtype=dtype, data=4 * P + es * off, ts=ts, hs=hs) for off, ts, hs in (a, b))
    assert lib.sapphire_paged_read_dev(C.byref(c), 0, C.byref(x), C.byref(y), C.byref(t), None, P, None) == -1
    assert lib.sapphire_paged_attention_dev(C.byref(c), 0, C.byref(x), C.byref(y), C.byref(t), P, 128, C.byref(AttentionC(1.0, 0, 0.0)),
                                            None, P, None) == -1
    assert b"overlap" in lib.sapphire_last_error()


def test_read_refuses_the_same_rows(lib):
    c, t, r = cache(), PageTableC(P, 3, 4), rows()
    assert lib.sapphire_paged_read_dev(C.byref(c), 0, C.byref(r), C.byref(r), C.byref(t), None, P, None) == -1
    assert b"overlap" in lib.sapphire_last_error()


@pytest.mark.parametrize("dtype", [F32, BF16, F16, Q8_0, Q4_0], ids=ref.NAME.get)
@pytest.mark.parametrize("nkv,heads", [(1, 1), (1, 40), (3, 12), (8, 64), (600, 600)])
def test_workspace_is_enough_for_smaller_calls(lib, dtype, nkv, heads):
    c = cache(dtype, nkv=nkv, hd=128)
    need = np.array([[lib.sapphire_paged_attention_workspace_bytes(C.byref(c), b, heads, n) for n in (1, 64, 65, 500, 2000, 9000, 131072, 2**30)]
                     for b in (1, 2, 3, 20, 63, 64, 65, 170, 171, 511, 512, 4000)], dtype=np.int64)
    assert (np.diff(need, axis=0) >= 0).all() and (np.diff(need, axis=1) >= 0).all()
    assert need[0, 0] == 0 and (need[:, -1] > 0).all() == (nkv < 512)


def test_reorder_refused(lib):
    c, t, o = cache(), PageTableC(P, 3, 4), PageTableC(2 * P, 3, 4)
    good = [C.byref(c), C.byref(t), 3 * P, 4 * P, 5 * P, C.byref(o), 6 * P, None]
    for i, bad in [(0, None), (1, None), (2, None), (3, None), (4, None), (5, None), (6, None), (5, C.byref(t)), (6, 4 * P), (6, 4 * P + 8),
                   (6, P + 44), (6, 2 * P), (5, C.byref(PageTableC(2 * P, 4, 4))), (5, C.byref(PageTableC(2 * P, 3, 5))),
                   (5, C.byref(PageTableC(P + 4, 3, 4))), (5, C.byref(PageTableC(3 * P, 3, 4))), (0, C.byref(cache(layers=20000)))]:
        args = list(good)
        args[i] = bad
        assert lib.sapphire_paged_reorder_dev(*args) == -1, (i, bad)


def test_rope_refused(lib):
    def call(x=None, y=None, pos=P, r=None, **kw):
        x, y = x or rows(), y or rows(data=8 * P)
        r = r or RopeC(P, kw.get("rot", 64), 0, kw.get("mag", 1.0))
        return lib.sapphire_rope_rows_dev(C.byref(x), C.byref(y), pos, C.byref(r), None)
    assert call(pos=None) == -1
    assert call(r=RopeC(None, 64, 0, 1.0)) == -1
    for rot in (0, -2, 1, 63, 66):
        assert call(rot=rot) == -1
    assert call(mag=math.nan) == -1 and call(mag=math.inf) == -1
    assert call(y=rows(data=8 * P, dtype=BF16)) == -1 and call(y=rows(data=8 * P, heads=1)) == -1
    assert call(y=rows(data=4 * P + 4)) == -1                  # overlaps x
    assert call(y=rows(ts=256)) == -1                          # x's place, other strides
    assert call(x=rows(dtype=Q8_0), y=rows(data=8 * P, dtype=Q8_0)) == -1
    assert call(y=rows(data=8 * P, ts=64)) == -1               # written rows overlap
    assert call(x=rows(hd=1026), y=rows(data=8 * P, hd=1026)) == -1
    assert lib.sapphire_rope_rows_dev(None, C.byref(rows()), P, C.byref(RopeC(P, 64, 0, 1.0)), None) == -1
    assert lib.sapphire_rope_rows_dev(C.byref(rows()), C.byref(rows()), P, None, None) == -1


def test_beam_refused(lib):
    good = dict(logits=P, ld=100, n=100, requests=2, beams=4, scores=P, done=P, end=1, so=P, tok=P, par=P, do=P, ws=P)
    for bad in (dict(logits=None), dict(ld=99), dict(n=3), dict(n=0), dict(requests=0), dict(beams=0), dict(beams=17), dict(scores=None),
                dict(done=None), dict(do=None), dict(so=None), dict(tok=None), dict(par=None), dict(ws=None), dict(ws=P + 8),
                dict(n=2**21 + 1, ld=2**21 + 1), dict(requests=20000)):
        assert lib.sapphire_beam_select_dev(*{**good, **bad}.values(), None) == -1, bad
    assert lib.sapphire_beam_workspace_bytes(3, 1, 4) == 0 and lib.sapphire_beam_workspace_bytes(100, 1, 17) == 0
    assert lib.sapphire_beam_workspace_bytes(262144, 8, 8) > 0


@pytest.mark.parametrize("n", [16, 2048, 2049, 5000, 262144, 2**21])
def test_beam_workspace_is_enough_for_smaller_calls(lib, n):
    """More of anything never needs less. What a call uses is a slot of `beams` keys (8 bytes) and a partial sum (16) for each
    row and chunk of it, min(2048 / rows, n / 2048) chunks, one at least."""
    need = np.array([[lib.sapphire_beam_workspace_bytes(n, r, w) for w in range(1, 17)] for r in range(1, 700)], dtype=np.int64)
    assert (np.diff(need, axis=0) >= 0).all() and (np.diff(need, axis=1) >= 0).all()
    assert lib.sapphire_beam_workspace_bytes(max(16, n - 1), 41, 7) <= lib.sapphire_beam_workspace_bytes(n, 41, 7)
    rows = np.arange(1, 700)[:, None] * np.arange(1, 17)
    chunks = np.minimum(np.maximum(1, 2048 // rows), -(-n // 2048))
    assert (need >= rows * chunks * (8 * np.arange(1, 17) + 16)).all()


@pytest.mark.parametrize("rot,base", [(2, 10000.0), (64, 10000.0), (256, 1e6), (18, 500.0)])
def test_frequencies(rot, base):
    """Each is one pow and at most a few more roundings in 64 bits."""
    i = np.arange(rot // 2)
    plain = np.exp(-2 * i / rot * np.log(base))
    close = dict(rtol=1e-13, atol=0)
    f, m = paged.rope_frequencies(rot, base)
    np.testing.assert_allclose(f, plain, **close)
    assert m == 1.0
    f, m = paged.rope_frequencies(rot, base, paged.ROPE_LINEAR, factor=8.0)
    np.testing.assert_allclose(f, plain / 8, **close)
    assert m == 1.0
    if rot > 2:
        f, m = paged.rope_frequencies(rot, base, paged.ROPE_BASE, factor=4.0)
        assert f[0] == 1.0 and m == 1.0
        np.testing.assert_allclose(f[-1], plain[-1] / 4, **close)
    f, m = paged.rope_frequencies(rot, base, paged.ROPE_PARTS, factor=16.0, trained=4096, low=1.0, high=32.0)
    turns = 4096 * plain / (2 * np.pi)
    g = np.clip((turns - 1) / 31, 0, 1)
    np.testing.assert_allclose(f, plain * ((1 - g) / 16 + g), **close)
    assert abs(m - (0.1 * math.log(16) + 1)) < 1e-7
    f, m = paged.rope_frequencies(rot, base, paged.ROPE_PARTS, factor=1.0, trained=4096, low=1.0, high=32.0)
    np.testing.assert_allclose(f, plain, **close)
    assert m == 1.0


def test_frequencies_refused():
    bad = [(0, 1e4), (3, 1e4), (64, 0.0), (64, -1.0), (64, math.nan), (64, math.inf)]
    for args in bad:
        with pytest.raises(RuntimeError):
            paged.rope_frequencies(*args)
    for kw in (dict(scaling=4), dict(scaling=-1), dict(scaling=1, factor=0.5), dict(scaling=1, factor=math.nan),
               dict(scaling=3, factor=2.0, trained=0.0, low=1.0, high=2.0), dict(scaling=3, factor=2.0, trained=10.0, low=2.0, high=2.0),
               dict(scaling=3, factor=2.0, trained=10.0, low=-1.0, high=2.0)):
        with pytest.raises(RuntimeError):
            paged.rope_frequencies(64, 1e4, **kw)
    with pytest.raises(RuntimeError):
        paged.rope_frequencies(2, 1e4, paged.ROPE_BASE, factor=2.0)


def test_reference_quantizer_reads_back():
    """The tests' own quantizer: values within half a step of the block's scale (Q4_0: one at the clipped end)."""
    x = np.random.default_rng(1).normal(size=(7, 256)).astype(np.float32)
    for dtype, steps in ((Q8_0, 0.5), (Q4_0, 1.0)):
        _, d = ref.quantize(dtype, x)
        err = np.abs(ref.stored(dtype, x) - x).reshape(7, 8, 32).max(-1)
        assert (err <= steps * np.abs(d) * 1.0001).all()
