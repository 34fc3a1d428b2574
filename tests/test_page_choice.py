"""Bounds of pages and the choice by them on the CPU: sizes and refusals, before any device work."""
import ctypes as C

import numpy as np
import pytest

import sapphire_amd
from sapphire_amd import paged
from sapphire_amd._lib import PageChoiceC, PageTableC
from tests.test_paged import BF16, F32, P, Q8_0, cache, rows


@pytest.fixture(scope="module")
def lib():
    return sapphire_amd.load()


def test_bounds_bytes(lib):
    assert lib.sapphire_paged_bounds_bytes(C.byref(cache(BF16, 3, 7, 48, 5, 128))) == 3 * 7 * 5 * 2 * 128 * 2
    assert lib.sapphire_paged_bounds_bytes(C.byref(cache(hd=96))) == 0
    assert lib.sapphire_paged_bounds_bytes(None) == 0


@pytest.mark.parametrize("change", [dict(c=dict(k=None)), dict(c=dict(ps=24)), dict(layer=-1), dict(layer=2), dict(bounds=None), dict(bounds=P + 8),
                                    dict(t=dict(rows=0)), dict(t=dict(pages=None)), dict(t=dict(rows=65536)), dict(lengths=None), dict(max_new=0)], ids=str)
def test_bounds_refused(lib, change):
    t = PageTableC(**{"pages": P, "rows": 3, "ld": 4, **change.get("t", {})})
    assert lib.sapphire_paged_bounds_dev(C.byref(cache(**change.get("c", {}))), change.get("layer", 1), change.get("bounds", 3 * P), C.byref(t), None,
                                         change.get("lengths", P), change.get("max_new", 5), None) == -1
    assert lib.sapphire_last_error()


SELECT = [dict(c=dict(v=None)), dict(layer=-1), dict(layer=2), dict(bounds=None), dict(bounds=P + 2), dict(q=None), dict(q=dict(heads=3)),
          dict(q=dict(hd=128)), dict(q=dict(dtype=Q8_0)), dict(q=dict(tokens=4)), dict(q=dict(ts=-1)), dict(t=dict(rows=2)), dict(t=dict(ld=0)),
          dict(lengths=None), dict(max_length=0), dict(max_length=129), dict(choice=None), dict(choice=(0, 0, 0)), dict(choice=(-1, 0, 0)),
          dict(choice=(3, 2, 2)), dict(choice=(3, -1, 2)), dict(choice=(3, 1, -1)), dict(choice=(3, 2**31 - 1, 2**31 - 1)), dict(choice=(2**30, 0, 0)), dict(choice=(2**31 - 1, 0, 0)), dict(selected=None),
          dict(ws=None), dict(ws=P + 8)]


@pytest.mark.parametrize("change", SELECT, ids=str)
def test_select_refused(lib, change):
    q = None if "q" in change and change["q"] is None else C.byref(rows(**{**dict(heads=4), **change.get("q", {})}))
    t = PageTableC(**{"pages": P, "rows": 3, "ld": 4, **change.get("t", {})})
    k = change.get("choice", (3, 1, 1))
    k = None if k is None else C.byref(PageChoiceC(*k))
    assert lib.sapphire_paged_select_dev(C.byref(cache(**change.get("c", {}))), change.get("layer", 0), change.get("bounds", 5 * P), q, C.byref(t),
                                         change.get("lengths", P), change.get("max_length", 128), k, change.get("selected", 6 * P),
                                         change.get("ws", 7 * P), None) == -1
    assert lib.sapphire_last_error()


def test_select_workspace(lib):
    c = cache(F32, nkv=3)
    need = np.array([[lib.sapphire_paged_select_workspace_bytes(C.byref(c), b, n) for n in (1, 32, 33, 5000, 1 << 20)] for b in (1, 2, 60)])
    assert (need > 0).all() and (np.diff(need, axis=0) >= 0).all() and (np.diff(need, axis=1) >= 0).all()
    for b, n in ((0, 5), (5, 0), (65536, 5), (5, 2**30 + 1)):
        assert lib.sapphire_paged_select_workspace_bytes(C.byref(c), b, n) == 0


def test_wrappers_raise(lib):
    c = paged.PagedCache(F32, 1, 2, 16, 1, 64, k=P, v=2 * P)
    assert c.bounds_bytes == 2 * 2 * 64 * 2
    with pytest.raises(RuntimeError, match="max_new"):
        c.bounds(0, 3 * P, paged.PageTable(P, 1, 2), P, 0)
    with pytest.raises(RuntimeError, match="paged select"):
        c.select(0, 3 * P, rows(1, 1), paged.PageTable(P, 1, 2), P, 16, P, 1, first=1, last=1, workspace=P)
