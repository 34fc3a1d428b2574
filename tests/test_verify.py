"""The verification of drafted tokens on the CPU: refusals (before any device work), workspace sizes, and the plain form's own
property: its tokens are distributed as the target's."""
import math

import numpy as np
import pytest

import sapphire_amd
from tests.verify_ref import probabilities, verify64

P = 1 << 20                                    # stands for a device address: nothing here reaches the device


@pytest.fixture(scope="module")
def lib():
    return sapphire_amd.load()


GOOD = dict(logits=P, ld=100, draft=2 * P, draft_ld=100, n=100, requests=3, drafts=4, drafted=3 * P, counts=4 * P, temperature=1.0,
            draws=5 * P, tokens=6 * P, accepted=7 * P, ws=8 * P, stream=None)


@pytest.mark.parametrize("change", [
    dict(logits=None), dict(drafted=None), dict(tokens=None), dict(accepted=None), dict(ws=None), dict(ws=8 * P + 8), dict(ld=99),
    dict(draft_ld=99), dict(n=0), dict(n=-1), dict(n=(1 << 21) + 1, ld=1 << 22, draft_ld=1 << 22), dict(requests=0), dict(requests=-1),
    dict(drafts=0), dict(drafts=65), dict(requests=7282), dict(draws=None), dict(temperature=math.nan), dict(temperature=math.inf),
    dict(temperature=-math.inf), dict(tokens=3 * P), dict(tokens=3 * P + 44), dict(tokens=4 * P), dict(tokens=5 * P), dict(accepted=3 * P),
    dict(accepted=4 * P + 8), dict(accepted=5 * P + 56), dict(accepted=6 * P + 56)], ids=str)
def test_refused(lib, change):
    assert lib.sapphire_verify_dev(*{**GOOD, **change}.values()) == -1
    assert lib.sapphire_last_error()


def test_workspace_is_enough_for_smaller_calls(lib):
    need = np.array([[[lib.sapphire_verify_workspace_bytes(n, r, d) for n in (1, 8189, 8190, 262144, 1 << 21)] for r in (1, 2, 17, 508)]
                     for d in (1, 2, 5, 64)], dtype=np.int64)
    assert (need > 0).all() and all((np.diff(need, axis=i) >= 0).all() for i in range(3))
    for n, r, d in ((0, 1, 1), ((1 << 21) + 1, 1, 1), (5, 0, 1), (5, 1, 0), (5, 1, 65), (5, 509, 64)):
        assert lib.sapphire_verify_workspace_bytes(n, r, d) == 0


@pytest.mark.parametrize("with_q", [True, False])
def test_plain_form_keeps_the_targets_distribution(with_q):
    """One draft over five tokens: the first token's shares over a grid of draws, against p. The grid of 41 draws for the test
    and 41 for the draw behind it is exact up to its own step for each drafted token, whose own share is q."""
    rng = np.random.default_rng(3)
    logits, draft = rng.normal(size=(1, 2, 5)) * 1.5, rng.normal(size=(1, 1, 5))
    p, q = probabilities(logits[0, 0], 0.9), probabilities(draft[0, 0], 0.9)
    grid = (np.arange(41) + 0.5) / 41
    got = np.zeros(5)
    for x in range(5):
        share = q[x] if with_q else 0.2
        for u in grid:
            for v in grid:
                t, _ = verify64(logits, draft if with_q else None, np.array([[x]]), None, np.array([[u, v]]), 0.9)
                got[t[0, 0]] += share / 41**2
    assert np.abs(got - p).max() < 3 / 41
