"""Attention of rows that share positions on the CPU: refusals, before any device work, and workspace sizes."""
import ctypes as C
import math

import numpy as np
import pytest

import sapphire_amd
from sapphire_amd._lib import AttentionC, GroupsC, PageTableC
from tests import paged_ref as ref
from tests.test_paged import ATTEND, BF16, F16, F32, P, Q4_0, Q8_0, cache, rows


@pytest.fixture(scope="module")
def lib():
    return sapphire_amd.load()


CHANGES = [c for c in ATTEND if "ws" not in c] + [
    dict(g=None), dict(g=dict(shared=None)), dict(g=dict(rows=0)), dict(g=dict(rows=-1)), dict(g=dict(max_own=-1)), dict(a=dict(window=5)),
    dict(ws=None), dict(ws=P + 4)]


@pytest.mark.parametrize("change", CHANGES, ids=str)
def test_shared_attention_refused(lib, change):
    c = cache(**{**dict(ps=32), **change.get("c", {})})
    def one(n):
        return None if n in change and change[n] is None else C.byref(rows(**{**dict(heads=4), **change.get(n, {})}))
    t = PageTableC(**{"pages": P, "rows": 3, "ld": 4, **change.get("t", {})})
    a, g = change.get("a", {}), change.get("g", {})
    a = None if a is None else C.byref(AttentionC(**{**dict(scale=1.0, window=0, softcap=0.0), **a}))
    g = None if g is None else C.byref(GroupsC(**{**dict(shared=9 * P, rows=2, max_own=5), **g}))
    assert lib.sapphire_paged_shared_attention_dev(C.byref(c), change.get("layer", 0), one("q"), one("o"), C.byref(t), change.get("lengths", P),
                                                   change.get("max_length", 128), g, a, None, change.get("ws", P), None) == -1
    assert lib.sapphire_last_error()


PAGES = [c for c in ATTEND if "ws" not in c and "max_length" not in c] + [
    dict(selected=None), dict(pages=0), dict(pages=-1), dict(pages=2**30), dict(ws=None), dict(ws=P + 4), dict(a=dict(scale=-math.inf))]


@pytest.mark.parametrize("change", PAGES, ids=str)
def test_pages_attention_refused(lib, change):
    c = cache(**{**dict(ps=32), **change.get("c", {})})
    def one(n):
        return None if n in change and change[n] is None else C.byref(rows(**{**dict(heads=4), **change.get(n, {})}))
    t = PageTableC(**{"pages": P, "rows": 3, "ld": 4, **change.get("t", {})})
    a = change.get("a", {})
    a = None if a is None else C.byref(AttentionC(**{**dict(scale=1.0, window=0, softcap=0.0), **a}))
    pages = change.get("pages", 2)
    if "ws" in change:                          # one that is needed
        pages = 400
        assert lib.sapphire_paged_attention_workspace_bytes(C.byref(c), 3, 4, pages * 32) > 0
    assert lib.sapphire_paged_pages_attention_dev(C.byref(c), change.get("layer", 0), one("q"), one("o"), C.byref(t), change.get("lengths", P),
                                                  change.get("selected", 9 * P), pages, a, None, change.get("ws", P), None) == -1
    assert lib.sapphire_last_error()


@pytest.mark.parametrize("dtype", [F32, BF16, F16, Q8_0, Q4_0], ids=ref.NAME.get)
@pytest.mark.parametrize("nkv,heads", [(1, 1), (1, 40), (3, 12), (8, 64), (600, 600)])
def test_workspace_is_enough_for_smaller_calls(lib, dtype, nkv, heads):
    c = cache(dtype, nkv=nkv, hd=128)
    need = np.array([[lib.sapphire_paged_shared_attention_workspace_bytes(C.byref(c), b, heads, n) for n in (1, 64, 65, 500, 2000, 9000, 131072, 2**30)]
                     for b in (1, 2, 3, 20, 63, 64, 65, 170, 171, 511, 512, 4000)], dtype=np.int64)
    assert (np.diff(need, axis=0) >= 0).all() and (np.diff(need, axis=1) >= 0).all() and (need > 0).all()
    for b, h, n in ((0, heads, 5), (1, heads, 0), (1, nkv + 1 if nkv > 1 else 0, 5)):
        assert lib.sapphire_paged_shared_attention_workspace_bytes(C.byref(c), b, h, n) == 0
