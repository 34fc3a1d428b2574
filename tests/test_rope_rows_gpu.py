"""Rotary positions of many rows against 64-bit numpy."""
import numpy as np
import pytest

from tests import paged_ref as ref
from tests.paged_ref import BF16, F16, F32
from tests.test_paged_gpu import dev, device_rows, sync

pytestmark = pytest.mark.gpu


def check(io, x, xs, got, pos, freqs, rot, inter, mag):
    """The angle's 64-bit reduction leaves 2^-24 pi of rounding, sine and cosine a few 2^-24: at most 8 x 2^-24 of the
    pair's two magnitudes, and one rounding to the rows' type."""
    want = ref.rope64(xs.astype(np.float64), pos, freqs, rot, inter, mag)
    pair = np.abs(xs).max(-1, keepdims=True) * 2 * max(1.0, abs(mag))
    tol = 2.0**-24 * 8 * pair + ref.HALF_STEP[io] * np.abs(want) * 1.001 + (2.0**-25 if io == F16 else 0)
    tol[..., rot:] = 0                             # copied
    assert (np.abs(got - want) <= tol).all(), np.max(np.abs(got - want) / np.maximum(tol, 1e-30))


@pytest.mark.parametrize("io", [F32, BF16, F16], ids=ref.NAME.get)
@pytest.mark.parametrize("inter", [False, True], ids=["half", "pairs"])
@pytest.mark.parametrize("t,h,hd,rot", [(1, 5, 256, 256), (1, 64, 128, 128), (7, 3, 64, 64), (33, 2, 96, 32), (130, 6, 128, 66), (5, 1, 2, 2),
                                        (3, 2, 80, 18), (9, 4, 1024, 1024), (700, 9, 64, 16)])
def test_rope_rows(hip, io, inter, t, h, hd, rot):
    from sapphire_amd import paged
    rng = np.random.default_rng(t * hd + rot)
    x = rng.normal(size=(t, h, hd)).astype(np.float32)
    pos = rng.integers(-10, 1 << 20, t).astype(np.int32)
    pos[0] = 2**31 - 1 if t > 5 else 0
    freqs, _ = paged.rope_frequencies(rot, 1e4)
    dp, df = dev(pos), dev(freqs)
    for order, pad, shift, mag in (("thd", 0, 0, 1.0), ("thd", 2 * hd, 8, 1.25), ("htd", 1, 1, -0.5)):
        rx, ry = device_rows(x, io, order, pad, shift), device_rows(x * 0 + 9, io, order, pad + hd, shift)
        paged.rope(rx[0], ry[0], dp, df, rot, interleaved=inter, magnitude=mag)
        sync()
        xs = ref.from_type(io, rx[3])
        raw = ry[1].numpy()
        got = np.lib.stride_tricks.as_strided(raw[shift:], x.shape, ry[3].strides).copy()
        check(io, x, xs, ref.from_type(io, got), pos, freqs, rot, inter, mag)
        ry[3][...] = got
        np.testing.assert_array_equal(raw, ry[2], err_msg="elements between the rows")
        np.testing.assert_array_equal(rx[1].numpy(), rx[2], err_msg="x")
        paged.rope(rx[0], rx[0], dp, df, rot, interleaved=inter, magnitude=mag)          # in place: the same bits
        sync()
        raw = rx[1].numpy()
        np.testing.assert_array_equal(np.lib.stride_tricks.as_strided(raw[shift:], x.shape, rx[3].strides), got)
        rx[3][...] = got
        np.testing.assert_array_equal(raw, rx[2], err_msg="elements between the rows, in place")


@pytest.mark.parametrize("io", [F32, BF16], ids=ref.NAME.get)
@pytest.mark.parametrize("inter", [False, True], ids=["half", "pairs"])
@pytest.mark.parametrize("t,h,hd,rot", [(6001, 7, 128, 64), (5003, 5, 128, 66), (20000, 1, 64, 64), (257, 129, 64, 32)])
def test_rope_rows_of_long_prompts(hip, io, inter, t, h, hd, rot):
    """Rows enough that a thread takes many pieces, of several heads and tokens; to other rows and in place."""
    from sapphire_amd import paged
    rng = np.random.default_rng(t)
    x = rng.normal(size=(t, h, hd)).astype(np.float32)
    pos = rng.integers(0, 1 << 18, t).astype(np.int32)
    freqs, _ = paged.rope_frequencies(rot, 1e4)
    dp, df = dev(pos), dev(freqs)
    rx, ry = device_rows(x, io, "thd", 64, 0), device_rows(x * 0 + 9, io, "htd", 8, 8)
    for to in (ry, rx):
        paged.rope(rx[0], to[0], dp, df, rot, interleaved=inter)
        sync()
        raw = to[1].numpy()
        got = np.lib.stride_tricks.as_strided(raw[8 if to is ry else 0:], x.shape, to[3].strides).copy()
        if to is ry:
            check(io, x, ref.from_type(io, rx[3]), ref.from_type(io, got), pos, freqs, rot, inter, 1.0)
            first = got
        else:
            np.testing.assert_array_equal(got, first)
        to[3][...] = got
        np.testing.assert_array_equal(raw, to[2], err_msg="elements between the rows")


def test_rope_rows_agree_with_the_tables(hip, oracle):
    """The half layout over a whole head against the table form at the same position: the tables hold fp32 angles' sines
    (an angle of up to 2047 rounded to 2^-24 of itself and its fp32 frequency's error), so to 4e-4 of the values."""
    from sapphire_amd import paged
    from sapphire_amd.device import check as ok
    hd, heads, base = 256, 4, 1e4
    c, s = oracle.rope_tables(hd, 2048, base)
    dc, ds = dev(c), dev(s)
    x = np.random.default_rng(3).normal(size=(1, heads, hd)).astype(np.float32)
    df = dev(paged.rope_frequencies(hd, base)[0])
    for pos in (0, 1, 2047):
        a, b = dev(x), device_rows(x, F32)
        ok(hip.sapphire_rope_apply_dev(a.ptr, heads, hd, pos, dc.ptr, ds.ptr, None))
        paged.rope(b[0], b[0], dev(np.array([pos], np.int32)), df, hd)
        sync()
        assert np.abs(a.numpy().ravel() - b[1].numpy()[:x.size]).max() <= 2047 * 2.0**-23 * 3 * 2 * np.abs(x).max()


def test_rope_rows_undone_by_negative_positions(hip):
    from sapphire_amd import paged
    x = np.random.default_rng(4).normal(size=(50, 3, 64)).astype(np.float32)
    pos = np.arange(50, dtype=np.int32) * 1000
    df, r = dev(paged.rope_frequencies(64, 1e4)[0]), device_rows(x, F32)
    paged.rope(r[0], r[0], dev(pos), df, 64)
    paged.rope(r[0], r[0], dev(-pos), df, 64)
    sync()
    assert np.abs(r[1].numpy()[:x.size].reshape(x.shape) - x).max() <= 2.0**-24 * 32 * np.abs(x).max()


@pytest.mark.parametrize("io", [F32, BF16], ids=ref.NAME.get)
@pytest.mark.parametrize("inter", [False, True], ids=["half", "pairs"])
@pytest.mark.parametrize("rot", [64, 34])
def test_rope_rows_between_slices_of_one_buffer(hip, io, inter, rot):
    """From some heads of every token's row to others, behind them or ahead: the bits of a call with a y of its own, and
    nothing else written."""
    from sapphire_amd import paged
    from sapphire_amd.paged import Rows
    rng = np.random.default_rng(rot)
    t, h, hd, H = 37, 3, 64, 8
    es = 4 if io == F32 else 2
    x = ref.to_type(io, rng.normal(size=(t, H, hd)).astype(np.float32))
    dp, df = dev(rng.integers(0, 5000, t).astype(np.int32)), dev(paged.rope_frequencies(rot, 1e4)[0])
    for src, dst in ((0, 3), (0, 5), (5, 1)):
        dx, dy = dev(x), dev(x[:, :h] * 0)
        def rows(d, first, width):
            return Rows(d.ptr + es * hd * first, io, t, h, hd, token_stride=width * hd)
        paged.rope(rows(dx, src, H), rows(dy, 0, h), dp, df, rot, interleaved=inter)
        paged.rope(rows(dx, src, H), rows(dx, dst, H), dp, df, rot, interleaved=inter)
        sync()
        want = x.copy()
        want[:, dst:dst + h] = dy.numpy()
        np.testing.assert_array_equal(dx.numpy(), want)
