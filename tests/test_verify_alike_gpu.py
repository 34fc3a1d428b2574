"""Verification of drafted tokens where the draft model's probabilities are the target's: nothing is left over from them, so that the
next token is the target's own, wherever the rows of both lie in memory."""
import numpy as np
import pytest

from tests.test_verify_gpu import Call
from tests.verify_ref import probabilities, verify64

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,pad", [(37, 0), (37, 2), (5001, 0), (20000, 1), (20000, 2), (20000, 3), (262144, 1)])
@pytest.mark.parametrize("more", [0.0, 2.0], ids=["same", "shifted"])
def test_nothing_is_left(hip, n, pad, more):
    """Drafted tokens that do not exist are refused whatever their draw; the logits (multiples of 2^-10, so that the shifted ones are
    exact) of a draft's two rows lie 0 to 3 elements apart against 16 bytes."""
    rng = np.random.default_rng(n + pad)
    requests, drafts = (40, 3) if n < 10000 else (9, 2)
    logits = (np.rint(rng.normal(size=(requests, drafts + 1, n)) * 3 * 1024) / 1024).astype(np.float32)
    draft = logits[:, :drafts] + np.float32(more)
    tokens = np.argmax(logits[:, :drafts], -1)
    stop = rng.integers(0, drafts, requests)
    tokens[np.arange(requests), stop] = np.where(rng.random(requests) < 0.5, n, -1)
    draws = np.minimum(rng.random((requests, drafts + 1)), 0.99).astype(np.float32)
    c = Call(logits, draft, tokens, None, draws, pad)
    c.run(0.8)
    got, want = c.result(), verify64(logits, logits[:, :drafts], tokens, None, draws, 0.8)
    np.testing.assert_array_equal(got[1], stop)
    np.testing.assert_array_equal(got[1], want[1])
    np.testing.assert_array_equal(got[0], want[0])


def test_little_is_left(hip):
    """A draft whose probabilities are the target's but for one token that it holds for impossible, or 2^-20 less likely: that token
    is what is left."""
    rng = np.random.default_rng(3)
    requests, n = 12, 3001
    logits = (rng.normal(size=(requests, 2, n)) * 2).astype(np.float32)
    draft, x = logits[:, :1].copy(), rng.integers(0, n, requests)
    for r in range(requests):
        logits[r, 0, x[r]] = 3.0
        draft[r, 0, x[r]] = -np.inf if r % 2 else 3.0 - 2.0**-20
        assert probabilities(logits[r, 0], 1.0)[x[r]] > 2.0**-12
    draws = rng.random((requests, 2)).astype(np.float32)
    c = Call(logits, draft, np.full((requests, 1), n), None, draws, 1)
    c.run()
    got, want = c.result(), verify64(logits, draft, np.full((requests, 1), n), None, draws, 1.0)
    assert (want[0][:, 0] == x).all() and (want[1] == 0).all()
    np.testing.assert_array_equal(got[0], want[0])
    np.testing.assert_array_equal(got[1], want[1])


@pytest.mark.parametrize("n,pad", [((1 << 20) + 5, 3), (1 << 21, 0), ((1 << 21) - 3, 2)])
def test_the_largest_vocabularies(hip, n, pad):
    """More units of a row than a workgroup has threads; draws at both ends and between."""
    rng = np.random.default_rng(n)
    requests, drafts = 4, 1
    logits = (rng.normal(size=(requests, drafts + 1, n)) * 2).astype(np.float32)
    draft = (logits[:, :drafts] + rng.normal(size=(requests, drafts, n))).astype(np.float32)
    tokens = np.array([[5], [n], [-1], [n - 1]])
    logits[0, 0, 5] += 5.0
    draws = np.array([[0.25, 0.999], [0.5, 0.0], [0.1, 1.0], [0.9, 0.625]], np.float32)
    for q in (draft, None):
        for t in (1.0, 0.0):
            c = Call(logits, q, tokens, None, draws, pad)
            c.run(t)
            got, want = c.result(), verify64(logits, q, tokens, None, draws, t)
            np.testing.assert_array_equal(got[1], want[1])
            np.testing.assert_array_equal(got[0], want[0])
