"""Attention of rows that share positions where a workgroup walks many of them: from one step to tens, in odd and even numbers,
with tiles of missing pages on the way, for every combination of sets, waves and types of the kernel that takes more than 32
columns. Groups of more rows than a wave has lanes, and pieces of many steps. Against plain numpy in 64 bits."""
import numpy as np
import pytest

from tests import paged_ref as ref
from tests.paged_ref import BF16, F16, F32, Q4_0, Q8_0
from tests.test_paged_gpu import IDS, IO, WEIGHTS, dev, device_rows, sync

pytestmark = pytest.mark.gpu

UNITS, WAVES = 256, 2048                               # compute units; waves of the shared positions at once


def step_of(cache, hd):
    """Positions of a step of a wide workgroup."""
    return 16 if cache == F32 or hd == 256 else 32


def wide_sets(cache, io, hd):
    """Sets of 16 columns that a wave of many columns takes at most."""
    if hd == 64:
        return 2
    return 2 if hd == 128 and (cache == F16 or (cache == BF16 and io == BF16)) else 1


def plan(cache, io, hd, nkv, groups, cols, top):
    """(sets, waves, pieces) of a call of more than 32 columns a group, as the library cuts it."""
    def of(sets):
        cs = 1 if cols <= 64 else sets
        nw = 4 if cols <= 64 * cs else 8
        wgs = groups * nkv * -(-cols // (16 * cs * nw))
        one = UNITS // wgs
        pieces = max(min(one // 2, -(-top // 32)), min(WAVES // (wgs * nw), top // (8 * step_of(cache, hd))))
        if pieces > one and 2 * pieces < 3 * one:
            pieces = one
        return cs, nw, min(max(1, pieces), 128)
    p = of(wide_sets(cache, io, hd))
    return of(1) if p[0] == 2 and top < 768 * p[2] else p


class Steps:
    """`groups` groups of `rows` rows over the same n positions of a cache; group g shares tiles[g] tiles, and its rows end up to 20
    positions behind them. broken: {group: pages of its rows that do not exist}; padded: rows of a group that have no
    position and no page. All K/V heads have the same q. k, v [n][nkv][hd], q [tokens][1][h][hd]: random ones if not given."""

    def __init__(self, rng, cache, io, hd, nkv, h, rows, tiles, n, ps=16, broken=None, padded=(), own=20,
                 k=None, v=None, q=None, scale=None):
        from sapphire_amd.device import DeviceArray
        from sapphire_amd.paged import PagedCache, PageTable
        self.cache, self.io, self.hd, self.nkv, self.h, self.rows, self.n, self.ps = cache, io, hd, nkv, h, rows, n, ps
        self.scale = scale or hd**-0.5
        groups = len(tiles)
        tokens, ld = groups * rows, -(-n // ps)
        order = rng.permutation(ld + 2)[:ld].astype(np.int32)
        table = np.repeat(order[None], tokens, 0)
        self.lens = np.array([[min(n, 16 * t + 1 + r * 7 % own) for r in range(rows)] for t in tiles])
        self.seen = np.arange(n)[None] < self.lens.reshape(-1, 1)      # [tokens][n]
        for g, pages in (broken or {}).items():
            for i in pages:
                table[g * rows:(g + 1) * rows, i] = ld + 2 + i if i % 2 else -1
                self.seen[g * rows:(g + 1) * rows, i * ps:(i + 1) * ps] = False
        for r in padded:
            self.lens[:, r] = 0
            table[r::rows] = -1
            self.seen[r::rows] = False
        self.tiles = [min(t, min(x for x in lens if x > 0) // 16) for t, lens in zip(tiles, self.lens)]
        self.shared = [16 * t + g * 5 % 16 for g, t in enumerate(tiles)]
        self.c = PagedCache(cache, 1, ld + 2, ps, nkv, hd)
        k, v = (rng.normal(size=(n, nkv, hd)).astype(np.float32) if x is None else x for x in (k, v))
        self.k, self.v = ref.stored(cache, k), ref.stored(cache, v)
        rk, rv, t = device_rows(k, F32), device_rows(v, F32), dev(order[None])
        self.c.write(0, rk[0], rv[0], PageTable(t, 1, ld), dev(np.arange(n, dtype=np.int32)), seqs=dev(np.zeros(n, np.int32)))
        sync()
        q = (rng.normal(size=(tokens, 1, h, hd)) * 2).astype(np.float32) if q is None else q
        q = np.broadcast_to(q, (tokens, nkv, h, hd)).reshape(tokens, nkv * h, hd)
        self.rq, self.ro = device_rows(q, io), device_rows(np.zeros((1, 1, hd), np.float32), io)
        self.q = ref.from_type(io, self.rq[3][:, :h].copy())
        self.out = DeviceArray.empty((tokens, nkv * h, hd), ref.np_type(io))
        self.dt, self.dn, self.ds = dev(table), dev(self.lens.astype(np.int32).ravel()), dev(np.array(self.shared, np.int32))
        self.pt = PageTable(self.dt, tokens, ld)
        self.lse = DeviceArray.empty((tokens, nkv * h))
        self.ws = DeviceArray(self.c.shared_attention_workspace_bytes(tokens, nkv * h, n))

    def steps(self):
        """(sets, waves, pieces), and the numbers of steps that workgroups take."""
        p = plan(self.cache, self.io, self.hd, self.nkv, len(self.tiles), self.rows * self.h, self.n)
        units = [-(-16 * t // step_of(self.cache, self.hd)) for t in self.tiles]
        return p, {u * (i + 1) // p[2] - u * i // p[2] for u in units for i in range(p[2])}

    def run(self, cap=0.0, own=20):
        from sapphire_amd.paged import Rows
        tokens, heads = self.lens.size, self.nkv * self.h
        self.c.shared_attention(0, self.rq[0], Rows(self.out, self.io, tokens, heads, self.hd), self.pt, self.dn, self.n, self.rows, self.ds,
                                self.scale, max_own=own, softcap=cap, lse=self.lse, workspace=self.ws)
        sync()
        return self.out.numpy(), self.lse.numpy()

    def check(self, heads, cap=0.0, own=20):
        """The columns of some K/V heads; of the others that they are finite."""
        raw, lse = self.run(cap, own)
        tokens, h, hd = self.lens.size, self.h, self.hd
        raw = raw.reshape(tokens, self.nkv, h, hd)
        assert np.isfinite(ref.from_type(self.io, raw)).all()
        lse = lse.reshape(tokens, self.nkv, h)
        q = self.q.reshape(tokens * h, hd).astype(np.float64)
        scale, seen = float(np.float32(self.scale)), np.repeat(self.seen, h, 0)
        for hk in heads:
            k, v = self.k[:, hk].astype(np.float64), self.v[:, hk].astype(np.float64)
            s = q @ k.T * scale
            size = np.where(seen, np.abs(q) @ np.abs(k).T * scale, 0).max(1)
            if cap:
                s = cap * np.tanh(s / cap)
            s[~seen] = -np.inf
            m = s.max(1, keepdims=True)
            dead = np.isneginf(m[:, 0])
            p = np.exp(s - np.where(np.isneginf(m), 0, m))
            total = np.where(dead, 1, p.sum(1))
            out, mean = p @ v / total[:, None], p @ np.abs(v) / total[:, None]
            l = np.where(dead, -np.inf, m[:, 0] + np.log(total))
            tol, ltol = ref.attention_bound(self.io, False, hd, self.n, out, l, size, mean, cap)
            tol = tol + 2 * WEIGHTS.get((self.cache, self.io), 0.0) * mean
            got = ref.from_type(self.io, raw[:, hk].reshape(-1, hd)).astype(np.float64)
            worst = np.abs(got - out) / tol
            at = np.unravel_index(worst.argmax(), worst.shape)
            row = at[0] // h
            assert worst.max() <= 1, (worst.max(), "group", row // self.rows, "tiles", self.tiles[row // self.rows], "row", row % self.rows, "dim", at[1])
            e = lse[:, hk].reshape(-1)
            assert np.array_equal(np.isneginf(e), dead) and (got[dead] == 0).all()
            assert (np.abs(e[~dead] - l[~dead]) <= ltol[~dead]).all()


def forms(cache, io, hd):
    """(sets, waves) -> (query heads of a K/V head, rows, groups, K/V heads, positions): one piece each."""
    two = wide_sets(cache, io, hd) == 2
    f = {(1, 4): (8, 5, 24, 22, 720), (1, 8): (4, 18, 24, 11, 720)}
    if two:
        f[2, 4] = (4, 25, 24, 22, 816)                 # 100 of 128 columns
        f[2, 8] = (3, 100, 12, 11, 816)                # 300 of 512
    return f


@pytest.mark.parametrize("cache,io", IO, ids=IDS)
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_steps(hip, cache, io, hd):
    """Every form in one piece: groups of all numbers of tiles around the first steps, and of tens; pages missing in the first,
    a middle and the last step, singly and two in a row."""
    rng = np.random.default_rng(hd + cache * 8 + io)
    for (cs, nw), (h, rows, groups, nkv, n) in forms(cache, io, hd).items():
        top = n // 16
        some = [1, 2, 3, 4, 5, 6, 7, 8] if groups == 12 else [*range(1, 17), 18, 19, 20, 21]       # steps
        tiles = some if step_of(cache, hd) == 16 else [2 * s - s % 2 for s in some]
        tiles = tiles + [top - 3, top - 2, top - 1, top]
        broken = {2: [0], 5: [4], 6: [6, 7], groups - 5: [2, 5], groups - 4: [8, 9, 21], groups - 3: [top - 3], groups - 2: [10, 13, 16, 19]}
        c = Steps(rng, cache, io, hd, nkv, h, rows, tiles, n, broken=broken)
        p, steps = c.steps()
        assert p == (cs, nw, 1) and {2, 3, 4, 5, 6, 7} <= steps and len({s % 2 for s in steps if s > 20}) == 2, (p, steps)
        c.check((0, nkv - 1))


@pytest.mark.parametrize("cache,io", IO, ids=IDS)
def test_pieces_of_many_steps(hip, cache, io):
    """Few groups over thousands of positions: pieces of eight steps and more each, with a cap and without."""
    rng = np.random.default_rng(cache * 8 + io)
    for hd, h, rows in ((64, 4, 40), (128, 8, 9), (256, 8, 9)):
        n = 16 * step_of(cache, hd) * 16 + 16
        c = Steps(rng, cache, io, hd, 2, h, rows, [n // 16 - 1, n // 48], n, ps=48, broken={0: [5, 40], 1: [0]})
        p, steps = c.steps()
        assert p[2] > 4 and max(steps) >= 8, (p, steps)
        c.check((0, 1))
        c.check((1,), cap=20.0)


@pytest.mark.parametrize("cache,io", [(F32, F32), (BF16, BF16), (F16, F32), (Q8_0, F32), (Q4_0, BF16)], ids=["f32", "bf16", "f16_f32", "q8_0", "q4_0_bf16"])
def test_groups_of_more_rows_than_lanes(hip, cache, io):
    """Groups whose first 64 rows and more are padding, of which the row that leads and the shortest one lie behind; the shortest
    one ends the shared positions for all."""
    rng = np.random.default_rng(cache + 50)
    for h, rows, padded in ((1, 130, tuple(range(67)) + (90, 129)), (2, 200, tuple(range(128)) + (131,)), (1, 70, tuple(range(64)))):
        c = Steps(rng, cache, io, 64, 2, h, rows, [30, 12], 500, padded=padded, own=20)
        short = rows - 3
        for g in range(2):
            c.lens[g, short] -= 75
            c.seen[g * rows + short, c.lens[g, short]:] = False
        c.dn.upload(c.lens.astype(np.int32).ravel())
        for own in (150, 30):
            c.check((0, 1), own=own)


@pytest.mark.parametrize("cache,io", [(F32, F32), (BF16, BF16), (Q4_0, F32)], ids=["f32", "bf16", "q4_0"])
def test_own_positions_of_unknown_number(hip, cache, io):
    """max_own = 0, where rows have thousands of positions of their own: cut as with the largest number, to the same bits."""
    c = Steps(np.random.default_rng(cache + 60), cache, io, 128, 1, 4, 3, [4], 4000)
    c.lens[0] = 4000, 3000, 64
    c.seen[...] = np.arange(c.n) < c.lens.reshape(-1, 1)
    c.dn.upload(c.lens.astype(np.int32).ravel())
    known = c.run(own=4000)
    for a, b in zip(known, c.run(own=0)):
        np.testing.assert_array_equal(a, b)
    c.check((0,), own=0)
