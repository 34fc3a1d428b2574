"""Beam search's selection against every candidate formed and sorted in 64 bits."""
import numpy as np
import pytest

from tests import paged_ref as ref
from tests.test_paged_gpu import dev, sync

pytestmark = pytest.mark.gpu


def select(logits, ld, score, done, R, W, end, in_place=False):
    from sapphire_amd import paged
    from sapphire_amd.device import DeviceArray
    n = logits.shape[1]
    wide = np.full((R * W, ld), 1e30, np.float32)  # what lies between the rows does not count
    wide[:, :n] = logits
    dl, ds, dd = dev(wide), dev(score), None if done is None else dev(done)
    so = ds if in_place else DeviceArray.empty(R * W)
    to, po, eo = (DeviceArray.empty(R * W, np.int32) for _ in range(3))
    eo = None if done is None else dd if in_place else eo
    ws = DeviceArray(paged.beam_workspace_bytes(n, R, W))
    paged.beam_select(dl, ld, n, R, W, ds, so, to, po, ws, done=dd, done_out=eo, end_token=end)
    sync()
    np.testing.assert_array_equal(dl.numpy(), wide)
    return so.numpy(), to.numpy(), po.numpy(), None if eo is None else eo.numpy()


def check(logits, score, done, R, W, end, ld=None, in_place=False):
    got = select(logits, ld or logits.shape[1], score, done, R, W, end, in_place)
    want = ref.beams64(logits, score, np.zeros(R * W, int) if done is None else done, R, W, end)
    for name, g, w in zip(("tokens", "parents", "done"), got[1:], want[1:]):
        if g is not None:
            np.testing.assert_array_equal(g, w, err_msg=name)
    fin = np.isfinite(want[0])
    np.testing.assert_array_equal(np.isfinite(got[0]), fin)
    # the normaliser is a sum of fp32 exponentials (2^-22 each, relative) in 64-bit and fp32 steps of at most 64
    size = np.abs(np.where(np.isfinite(logits), logits, 0)).max()
    tol = 2.0**-22 * 80 + 2.0**-23 * size * 4 + 2.0**-24 * np.abs(want[0][fin])
    assert (np.abs(got[0][fin] - want[0][fin]) <= tol).all()


@pytest.mark.parametrize("R,W,n,ld", [(1, 1, 1, 1), (1, 4, 4, 7), (1, 16, 16, 16), (3, 5, 63, 65), (2, 4, 2047, 2050), (2, 3, 2049, 2049), (8, 8, 5000, 5003),
                                      (1, 16, 100001, 100001), (1, 2, 262144, 262144), (70, 3, 300, 300)])
def test_beams(hip, R, W, n, ld):
    rng = np.random.default_rng(n)
    logits = (rng.normal(size=(R * W, n)) * 3).astype(np.float32)
    score = -np.abs(rng.normal(size=R * W) * 4).astype(np.float32)
    check(logits, score, None, R, W, -1, ld)
    done = (rng.random(R * W) < 0.3).astype(np.int32) * 5
    check(logits, score, done, R, W, min(1, n - 1), ld)
    check(logits, score, done, R, W, n - 1, ld, in_place=True)
    check(logits, score, np.ones(R * W, np.int32), R, W, 0, ld)


def test_first_step(hip):
    """All beams but the first at -inf: the first row's best tokens; and with fewer tokens above -inf than beams."""
    rng = np.random.default_rng(1)
    R, W, n = 2, 4, 3000
    logits = rng.normal(size=(R * W, n)).astype(np.float32)
    score = np.tile([0, -np.inf, -np.inf, -np.inf], R).astype(np.float32)
    check(logits, score, None, R, W, -1)
    logits[0, :] = -np.inf
    logits[0, [5, 2999]] = [1.0, 2.0]
    logits[4, 7:] = np.nan
    logits[4, :7] = -np.inf
    check(logits, score, None, R, W, -1)
    check(logits, score, np.array([1, 0, 0, 0, 0, 1, 0, 0], np.int32), R, W, 2)


def test_ties_masks_and_specials(hip):
    rng = np.random.default_rng(2)
    R, W, n = 3, 4, 5000
    logits = np.round(rng.normal(size=(R * W, n))).astype(np.float32)         # many equal ones
    logits[logits == 0] = np.where(rng.random((logits == 0).sum()) < 0.5, -0.0, 0.0)
    score = np.zeros(R * W, np.float32)
    logits[4:8] = logits[4]                                                     # beams that are alike
    check(logits, score, None, R, W, -1)
    logits[rng.random(logits.shape) < 0.5] = -np.inf
    logits[rng.random(logits.shape) < 0.1] = np.nan
    check(logits, score, None, R, W, -1)
    logits[0, 77] = np.inf
    logits[9] = -np.inf
    score[2], score[6], score[10] = np.nan, -np.inf, np.inf
    check(logits, score, None, R, W, -1)
    check(logits, score, (np.arange(12) % 3 == 0).astype(np.int32), R, W, 4999)
    check(logits, score, (np.arange(12) % 3 == 0).astype(np.int32), R, W, 5000)
    check(logits, score, np.ones(12, np.int32), R, W, -3)


@pytest.mark.parametrize("down", [False, True])
def test_sorted_logits(hip, down):
    """Rising logits, where every element enters the wave's list, and falling ones."""
    n = 40000
    x = np.linspace(-5, 5, n, dtype=np.float32)[::-1 if down else 1]
    check(np.stack([x, x - 1, x + 1, x]).astype(np.float32), np.array([-1, -1, -2, -1.5], np.float32), None, 1, 4, -1)


@pytest.mark.parametrize("R,W,n,ld", [(8, 8, 70001, 70003), (4, 16, 131072, 131072), (40, 8, 60000, 60001), (300, 1, 50000, 50000)])
def test_many_rows_of_a_large_vocabulary(hip, R, W, n, ld):
    """Rows enough that a workgroup takes thousands of logits, of the largest several batches: random ones, rising and
    falling ones, few above -inf, equal ones, and NaN of both kinds."""
    rng = np.random.default_rng(n + W)
    rows = R * W
    x = (rng.normal(size=(rows, n)) * 3).astype(np.float32)
    ramp = np.linspace(-9, 9, n, dtype=np.float32)
    x[1 % rows::7], x[2 % rows::7] = ramp, ramp[::-1]
    x[3 % rows::7] = np.round(x[3 % rows::7])
    few = x[4 % rows::7]
    few[rng.random(few.shape) < 0.9999] = -np.inf
    bad = x[5 % rows::7].view(np.uint32)
    bad[rng.random(bad.shape) < 0.01] = 0x7fc00000             # quiet, signalling, negative
    bad[rng.random(bad.shape) < 0.01] = 0x7f800001
    bad[rng.random(bad.shape) < 0.01] = 0xff923456
    score = -np.abs(rng.normal(size=rows) * 4).astype(np.float32)
    check(x, score, None, R, W, -1, ld)
    check(x, score, (rng.random(rows) < 0.2).astype(np.int32), R, W, 5, ld, in_place=True)


def test_far_logits(hip):
    """Magnitudes whose exponentials overflow or vanish."""
    x = np.array([[3e38, 2.9e38, -3e38, 0, 1], [-3e38, -3e38, -2e38, -2e38, -1e38], [88, 89, 90, 91, 1000], [0, 0, 0, 0, 0]], np.float32)
    check(x, np.array([0, 0, 0, 0], np.float32), None, 1, 4, -1)


FAR = [(4.3e9, 0.0), (1e10, 0.0), (1e10, -np.inf), (1e10, np.nan), (1e12, 9e11), (-1e10, -2e10), (-1e10, -np.inf), (-1e12, np.nan),
       (float(np.finfo(np.float32).min), -np.inf), (float(np.finfo(np.float32).max), -1e38)]


@pytest.mark.parametrize("top,rest", FAR)
@pytest.mark.parametrize("n", [5000, 100001])
def test_far_maxima(hip, n, top, rest):
    """Rows of one logit far from zero, the others far below it: their normaliser is that logit, so the row's best score is
    its beam's own, ahead of an ended beam at -5 and of an ordinary one at -3.

    A score is off by the normaliser's error, which does not grow with the logits: at most eight exponentials in a row of
    factors (2^-22 each, and their arguments, ln n in the mean, by 2^-23 of themselves) and sums in fp32 of 2^-22, together below
    2^-18; by the roundings of m + log s and of x - (m + log s) in 64 bits, here and in the oracle; and by that to fp32."""
    rng = np.random.default_rng(n)
    R, W = 3, 3
    logits = np.full((R * W, n), rest, np.float32)
    at = [0, n // 2 + 1, n - 1]
    for r in range(R):
        logits[r * W, at[r]] = top
        logits[r * W + 2] = rng.normal(size=n) * 3
    score = np.tile([0.0, -5.0, -3.0], R).astype(np.float32)
    done = np.tile([0, 1, 0], R).astype(np.int32)
    got = select(logits, n, score, done, R, W, 7)
    want = ref.beams64(logits, score, done, R, W, 7)
    for g, w in zip(got[1:], want[1:]):
        np.testing.assert_array_equal(g, w)
    for r in range(R):
        assert got[1][r * W] == at[r] and got[2][r * W] == r * W
    fin = np.isfinite(want[0])
    tol = 2.0**-18 + 4 * 2.0**-53 * abs(top) + 2.0**-24 * np.abs(want[0][fin])
    if abs(top) > 2e12:                        # there the oracle's own m + log s is coarse; the best score is 0 all the same
        np.testing.assert_array_equal(got[0][::W], 0.0)
    assert (np.abs(got[0][fin] - want[0][fin]) <= tol).all()


@pytest.mark.parametrize("shift", [0.0, 1000.0, -1e6])
@pytest.mark.parametrize("R,W,n", [(2, 4, 3000), (1, 16, 100001), (40, 8, 60000), (1, 1, 262144)])
def test_normaliser(hip, R, W, n, shift):
    """Scores within the normaliser's error (2^-18: see test_far_maxima; of rows whose maximum moves at a handful of
    batches), however far the logits are from zero. Those are multiples of 1/8, which a shift leaves as they are; the tokens
    and parents are compared where no other candidate is that near."""
    rng = np.random.default_rng(n)
    rows = R * W
    x = np.round(rng.normal(size=(rows, n)) * 24).astype(np.float32) / 8 + np.float32(shift)
    x[0] = np.round(np.linspace(-9, 9, n) * 8).astype(np.float32) / 8 + np.float32(shift)
    score = -np.abs(rng.normal(size=rows) * 4).astype(np.float32)
    got = select(x, n, score, None, R, W, -1)
    want = ref.beams64(x, score, np.zeros(rows, int), R, W, -1)
    tol = 2.0**-18 + 4 * 2.0**-53 * abs(shift) + 2.0**-24 * np.abs(want[0])
    assert (np.abs(got[0] - want[0]) <= tol).all()
    clear = np.array([np.sum(np.abs(want[0] - s) < 1e-5) == 1 for s in want[0]])
    clear[W - 1::W] = False                    # (the last one's rival may not be among them)
    np.testing.assert_array_equal(got[1][clear], want[1][clear])
    np.testing.assert_array_equal(got[2][clear], want[2][clear])
