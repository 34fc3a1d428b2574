"""The verification of drafted tokens on the GPU against plain numpy in 64 bits. Every output is a whole number and has to be
equal: the draws are not next to a border (1e-9 relative, where both sides are within 1e-11)."""
import numpy as np
import pytest

from tests.test_paged_gpu import Graph
from tests.verify_ref import probabilities, verify64

pytestmark = pytest.mark.gpu


def dev(a):
    from sapphire_amd.device import DeviceArray
    return DeviceArray.from_numpy(np.ascontiguousarray(a))


class Call:
    """One call's arrays on the device; `pad` elements behind each row of logits, `shift` ahead of the first."""

    def __init__(self, logits, draft, tokens, counts, draws, pad=0, shift=0):
        from sapphire_amd.device import DeviceArray
        from sapphire_amd.paged import verify_workspace_bytes
        self.requests, self.drafts = tokens.shape
        self.n, self.pad, self.shift = logits.shape[2], pad, shift
        self.logits, self.draft = self._rows(logits), None if draft is None else self._rows(draft)
        self.tokens, self.counts = dev(tokens.astype(np.int32)), None if counts is None else dev(np.array(counts, np.int32))
        self.draws = None if draws is None else dev(draws.astype(np.float32))
        self.out, self.kept = dev(np.full((self.requests, self.drafts + 1), 77, np.int32)), dev(np.full(self.requests, 77, np.int32))
        self.ws = DeviceArray(verify_workspace_bytes(self.n, self.requests, self.drafts))

    def _rows(self, x):
        flat = np.full((x.shape[0] * x.shape[1], self.n + self.pad), np.inf, np.float32)       # what is not a logit must not count
        flat[:, :self.n] = x.reshape(-1, self.n)
        return dev(np.concatenate([np.full(self.shift, np.inf, np.float32), flat.ravel()]))

    def run(self, temperature=1.0, stream=None):
        from sapphire_amd.paged import verify
        at = 4 * self.shift
        verify(self.logits.ptr + at, self.n + self.pad, self.n, self.requests, self.drafts, self.tokens, self.draws, self.out, self.kept, self.ws,
               draft_logits=None if self.draft is None else self.draft.ptr + at, draft_ld=0 if self.draft is None else self.n + self.pad,
               counts=self.counts, temperature=temperature, stream=stream)

    def result(self):
        from sapphire_amd import load
        assert load().sapphire_synchronize() == 0
        return self.out.numpy(), self.kept.numpy()


def inputs(rng, requests, drafts, n, near=0.7):
    """A draft near the target, its tokens drawn from it."""
    logits = (rng.normal(size=(requests, drafts + 1, n)) * 3).astype(np.float32)
    draft = (logits[:, :drafts] + rng.normal(size=(requests, drafts, n)) * near).astype(np.float32)
    tokens = np.array([[rng.choice(n, p=probabilities(draft[r, i], 1.0)) for i in range(drafts)] for r in range(requests)])
    return logits, draft, tokens, rng.random((requests, drafts + 1)).astype(np.float32)


@pytest.mark.parametrize("n", [1, 2, 5, 1000, 8189, 8192, 8193, 50257, 262144])
@pytest.mark.parametrize("requests,drafts", [(1, 1), (3, 4), (2, 64)])
def test_sizes(hip, n, requests, drafts):
    if n * drafts > 1 << 21:
        drafts = 6
    rng = np.random.default_rng(n + drafts)
    logits, draft, tokens, draws = inputs(rng, requests, drafts, n)
    counts = rng.integers(-1, drafts + 2, requests)
    for q, t, pad, shift in ((draft, 1.0, 0, 0), (None, 0.7, 1, 0), (draft, 1.6, 3, 1), (draft, 0.0, 2, 3)):
        for cnt in (None, counts):
            c = Call(logits, q, tokens, cnt, draws, pad, shift)
            c.run(t)
            got, want = c.result(), verify64(logits, q, tokens, cnt, draws, t)
            np.testing.assert_array_equal(got[1], want[1])
            np.testing.assert_array_equal(got[0], want[0])


def test_every_way_a_request_ends(hip):
    """Many requests over a small vocabulary: all numbers of kept drafts occur, with and without q."""
    rng = np.random.default_rng(8)
    logits, draft, tokens, draws = inputs(rng, 400, 3, 37, near=1.5)
    for q in (draft, None):
        c = Call(logits, q, tokens, None, draws)
        c.run()
        got, want = c.result(), verify64(logits, q, tokens, None, draws, 1.0)
        np.testing.assert_array_equal(got[0], want[0])
        np.testing.assert_array_equal(got[1], want[1])
        assert set(want[1]) == {0, 1, 2, 3}


def test_borders(hip):
    """Weights that are whole numbers of 1 / 2^14 over three chunks of a row (logits of 0 and -inf): draws on a border take the
    token behind it, as sums and products are exact."""
    n = 3 * 8192 - 5
    rng = np.random.default_rng(2)
    on = np.sort(rng.permutation(n)[:1 << 14])
    logits = np.full((1, 2, n), -np.inf, np.float32)
    logits[:, :, on] = 0.0
    for k in (0, 1, 8191, 8192, 12345, (1 << 14) - 1):
        # nothing kept: the drafted token has no weight in the target, and none is left over from it
        c = Call(logits, None, np.array([[(on[0] + 1) % n if (on[0] + 1) % n not in on[:2] else n - 1]]), [0], np.array([[0.5, k / 2.0**14]]))
        c.run()
        out, kept = c.result()
        assert kept[0] == 0 and out[0, 0] == on[k] and out[0, 1] == -1
    # the draft is kept exactly while draws * q < p: p = 2^-14, q = 1
    for u, kept in ((2.0**-14, 0), (np.nextafter(np.float32(2.0**-14), np.float32(0)), 1), (0.0, 1)):
        c = Call(logits, None, np.array([[on[5]]]), None, np.array([[u, 0.0]]))
        c.run()
        out = c.result()
        assert out[1][0] == kept
        assert out[0][0, 0] == (on[5] if kept else on[0])
    # max(p - q, 0) where q is half of p's tokens: what is left is the other half
    draft = np.full((1, 1, n), -np.inf, np.float32)
    draft[:, :, on[::2]] = 0.0
    for k in (0, 100, 8191):
        c = Call(logits, draft, np.array([[on[0]]]), None, np.array([[0.75, k / 2.0**13]]))
        c.run()
        out = c.result()
        assert out[1][0] == 0 and out[0][0, 0] == on[1::2][k]


def test_draws_at_the_ends(hip):
    """0, 1, beyond, NaN; a draft equal to the target, of which nothing is left over; one that holds all of it."""
    rng = np.random.default_rng(4)
    logits, draft, tokens, _ = inputs(rng, 1, 2, 9000)
    one = np.full((1, 3, 9000), -np.inf, np.float32)
    one[:, :, 8500] = 2.0
    with np.errstate(invalid="ignore"):
        for u in (0.0, 1.0, -3.0, 7.0, np.nan):
            for v in (0.0, 1.0, 0.5, -1.0, 2.0, np.nan):
                draws = np.array([[u, u, v]], np.float32)
                for lo, q, x in ((logits, draft, tokens), (logits, logits[:, :2], tokens), (logits, None, tokens), (one, None, np.full((1, 2), 8500)),
                                 (one, None, np.full((1, 2), 3))):
                    c = Call(lo, q, x, None, draws)
                    c.run()
                    got, want = c.result(), verify64(lo, q, x, None, draws, 1.0)
                    np.testing.assert_array_equal(got[0], want[0])
                    np.testing.assert_array_equal(got[1], want[1])


def test_odd_logits(hip):
    """NaN, infinities, rows without a finite logit, tokens that do not exist, temperatures at the ends of the range."""
    rng = np.random.default_rng(5)
    n = 8400
    logits, draft, tokens, draws = inputs(rng, 9, 2, n)
    logits[0, :, ::3] = np.nan
    logits[1, :, 17] = np.inf
    logits[2, 0, [5, 8300]] = np.inf
    logits[3] = -np.inf
    logits[4] = np.nan
    draft[5, 0, 99] = np.inf
    draft[6] = -np.inf
    logits[7] = np.float32(3e38) * np.sign(logits[7])
    tokens[8] = [n, -1]
    tokens[1, 0] = 17
    for t in (1.0, 1e-40, 3e38, 0.0, -1.0):
        for q in (draft, None):
            c = Call(logits, q, tokens, None, draws)
            c.run(t)
            got, want = c.result(), verify64(logits, q, tokens, None, draws, t)
            np.testing.assert_array_equal(got[1], want[1], err_msg=str(t))
            np.testing.assert_array_equal(got[0], want[0], err_msg=str(t))


def test_rows_behind_the_count_are_not_read_and_results_repeat(hip):
    """What stands behind a request's count does not matter; a call gives the same every time, on another stream, and after a
    call of other sizes in the same workspace."""
    rng = np.random.default_rng(6)
    logits, draft, tokens, draws = inputs(rng, 5, 4, 20000)
    counts = np.array([0, 1, 2, 3, 4])
    for r in range(5):
        logits[r, counts[r] + 1:], draft[r, counts[r]:] = np.nan, np.inf
    want = verify64(logits, draft, tokens, counts, draws, 1.0)
    c = Call(logits, draft, tokens, counts, draws)
    small = Call(logits[:1, :2, :100], None, tokens[:1, :1] % 100, None, draws[:1, :2])
    small.ws = c.ws
    s = hip.sapphire_stream_create()
    for stream in (None, s, None):
        c.run(stream=stream)
        got = c.result()
        small.run(stream=stream)
        np.testing.assert_array_equal(got[0], want[0])
        np.testing.assert_array_equal(got[1], want[1])
        small.result()
    hip.sapphire_stream_destroy(s)


def test_captured(hip):
    """A captured call, replayed with new draws."""
    rng = np.random.default_rng(7)
    logits, draft, tokens, draws = inputs(rng, 4, 3, 10000)
    c = Call(logits, draft, tokens, None, draws)
    g = Graph(lambda stream: c.run(stream=stream))
    for _ in range(4):
        draws = rng.random(draws.shape).astype(np.float32)
        c.draws.upload(draws)
        g.replay()
        got, want = c.result(), verify64(logits, draft, tokens, None, draws, 1.0)
        np.testing.assert_array_equal(got[0], want[0])
        np.testing.assert_array_equal(got[1], want[1])
    g.close()


def test_rows_past_four_gigabytes(hip):
    """Rows 2^30 elements apart, of both models: what rows next to each other give."""
    from sapphire_amd.device import DeviceArray
    from sapphire_amd.paged import verify, verify_workspace_bytes
    rng = np.random.default_rng(9)
    n, ld = 5000, 1 << 30
    logits, draft, tokens, draws = inputs(rng, 1, 3, n, near=0.1)
    draws[:, :3] *= 0.5
    on = [DeviceArray((len(x[0]) - 1) * ld * 4 + n * 4) for x in (logits, draft)]
    for d, x in zip(on, (logits, draft)):
        for i, row in enumerate(x[0]):
            assert hip.sapphire_memcpy_h2d(d.ptr + i * ld * 4, row.ctypes.data, row.nbytes) == 0
    ws, out, kept = DeviceArray(verify_workspace_bytes(n, 1, 3)), dev(np.zeros((1, 4), np.int32)), dev(np.zeros(1, np.int32))
    t, d = dev(tokens.astype(np.int32)), dev(draws)
    for temperature in (1.0, 0.0):
        verify(on[0], ld, n, 1, 3, t, d, out, kept, ws, draft_logits=on[1], draft_ld=ld, temperature=temperature)
        assert hip.sapphire_synchronize() == 0
        want = verify64(logits, draft, tokens, None, draws, temperature)
        np.testing.assert_array_equal(out.numpy(), want[0])
        np.testing.assert_array_equal(kept.numpy(), want[1])
    for x in on:
        x.free()


def test_calls_at_once(hip):
    """Two calls under way on two streams, each in a workspace of its own: the same as alone."""
    rng = np.random.default_rng(10)
    sets = [inputs(rng, 6, 4, 30000), inputs(rng, 2, 7, 5000)]
    calls = [Call(lo, q, x, None, u) for lo, q, x, u in sets]
    streams = [hip.sapphire_stream_create() for _ in calls]
    for _ in range(4):
        for _ in range(8):
            for c, s in zip(calls, streams):
                c.run(stream=s)
        for c, (lo, q, x, u) in zip(calls, sets):
            got, want = c.result(), verify64(lo, q, x, None, u, 1.0)
            np.testing.assert_array_equal(got[0], want[0])
            np.testing.assert_array_equal(got[1], want[1])
    for s in streams:
        hip.sapphire_stream_destroy(s)
