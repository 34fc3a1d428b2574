"""The paged cache, its attention, rotary rows and beam selection in plain numpy, for the tests: the cache's bytes
by index arithmetic over single elements, everything else in 64 bits."""
import numpy as np

F32, BF16, F16, Q4_0, Q8_0 = 0, 1, 2, 3, 4
NAME = {F32: "f32", BF16: "bf16", F16: "f16", Q4_0: "q4_0", Q8_0: "q8_0"}
HALF_STEP = {F32: 2.0**-24, BF16: 2.0**-8, F16: 2.0**-11}      # largest relative rounding error


def bf16_bits(x):
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    r = ((u + 0x7fff + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), ((u >> 16) | 0x40).astype(np.uint16), r)


def to_type(dtype, x):
    """fp32 values -> the array that holds them in `dtype` (uint16 for BF16)."""
    x = np.asarray(x, np.float32)
    with np.errstate(over="ignore"):
        return x if dtype == F32 else bf16_bits(x) if dtype == BF16 else x.astype(np.float16)


def from_type(dtype, a):
    if dtype == BF16:
        return (a.astype(np.uint32) << 16).view(np.float32)
    return a.astype(np.float32)


def np_type(dtype):
    return {F32: np.float32, BF16: np.uint16, F16: np.float16}[dtype]


def quantize(dtype, x):
    """(codes, scales) of fp32 [..., hd]: quantize.h's arithmetic, codes signed, scale NaN for a non-finite block."""
    b = np.ascontiguousarray(x, np.float32).reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    with np.errstate(all="ignore"):
        mag = np.abs(b).max(-1)
        if dtype == Q8_0:
            d = mag / np.float32(127)
        else:
            first = np.take_along_axis(b, np.abs(b).argmax(-1)[..., None], -1)[..., 0]
            d = first / np.float32(-8)
        inv = np.where(d == 0, np.float32(0), np.float32(1) / d).astype(np.float32)
        y = (b * inv[..., None]).astype(np.float32)
        if dtype == Q8_0:
            y = np.clip(np.where(np.isnan(y), np.float32(0), y), -127, 127).astype(np.float64)
            q = np.copysign(np.floor(np.abs(y) + 0.5), y)
        else:
            y = y + np.float32(8.5)
            q = np.trunc(np.clip(np.where(np.isnan(y), np.float32(8), y), 0, 15)) - 8
    bad = ~np.isfinite(b).all(-1)
    return np.where(bad[..., None], 0, q).astype(np.int8).reshape(x.shape), np.where(bad, np.float32(np.nan), d).astype(np.float32)


def stored(dtype, x):
    """The fp32 values that rows read back as."""
    if dtype in HALF_STEP:
        return from_type(dtype, to_type(dtype, x))
    q, d = quantize(dtype, x)
    with np.errstate(all="ignore"):
        return (q.reshape(*d.shape, 32).astype(np.float32) * d[..., None]).reshape(x.shape)


class Pool:
    """K or V of a cache as bytes, [layers][pages][heads][tile]."""

    def __init__(self, which, dtype, layers, pages, ps, nkv, hd, fill=0):
        self.which, self.dtype, self.ps, self.nkv, self.hd = which, dtype, ps, nkv, hd
        self.code = {F32: 4 * hd, BF16: 2 * hd, F16: 2 * hd, Q8_0: hd, Q4_0: hd // 2}[dtype]
        self.tile = ps * (self.code + (hd // 32 * 4 if dtype in (Q8_0, Q4_0) else 0))
        self.a = np.full((layers, pages, nkv, self.tile), fill, np.uint8)

    def _at(self, p):
        """(byte, shift) of every dim of position p."""
        hd, t = self.hd, self.dtype
        d = np.arange(hd)
        b, e, nb = d // 32, d % 32, hd // 32
        none = np.zeros(hd, int)
        es = {F32: 4, BF16: 2, F16: 2, Q8_0: 1, Q4_0: 0}[t]
        if self.which == "v":
            run, run_bytes = hd // 16, self.code // 16
            par = min(4, max(1, 16 // run_bytes))
            first = ((p // par * 16 + d // run) * par + p % par) * run_bytes
            if t == Q4_0:
                return first + d % run % (run // 2), d % run // (run // 2) * 4
            return first + d % run * es, none
        if t == Q8_0:
            return (((p // 16 * (nb // 2) + b // 2) * 4 + e // 8) * 16 + p % 16) * 16 + b % 2 * 8 + e % 8, none
        if t == Q4_0:
            g = min(4, nb)
            return (((p // 16 * (nb // g) + b // g) * 4 + e // 8) * 16 + p % 16) * (4 * g) + b % g * 4 + e % 4, e % 8 // 4 * 4
        per = 16 // es
        return ((p // 16 * (hd // per) + d // per) * 16 + p % 16) * 16 + d % per * es, none

    def _scale_at(self, p):
        b = np.arange(self.hd // 32)
        i = p * (self.hd // 32) + b if self.which == "k" else (p // 4 * (self.hd // 32) + b) * 4 + p % 4
        return self.ps * self.code + 4 * i

    def put(self, layer, page, p, x):
        """fp32 rows [heads][hd] at position p of a page."""
        at, shift = self._at(p)
        for h in range(self.nkv):
            t = self.a[layer, page, h]
            if self.dtype in HALF_STEP:
                raw = np.ascontiguousarray(to_type(self.dtype, x[h])).view(np.uint8).reshape(self.hd, -1)
                t[at[:, None] + np.arange(raw.shape[1])] = raw
                continue
            q, d = quantize(self.dtype, x[h])
            if self.dtype == Q8_0:
                t[at] = q.view(np.uint8)
            else:
                nib = (q & 15 if self.which == "k" else q + 8).astype(np.uint8)
                for s in (0, 4):
                    m = shift == s
                    t[at[m]] = (t[at[m]] & (0xf0 if s == 0 else 0x0f)) | (nib[m] << s)
            t[self._scale_at(p)[:, None] + np.arange(4)] = d.view(np.uint8).reshape(-1, 4)


def attention64(q, k, v, scale, window=0, softcap=0.0):
    """One sequence: q [heads][hd], k and v [positions][kv heads][hd] (what the cache stands for) -> out, lse and, for
    the error bounds, the largest scale * sum |q k| and sum p |v| / sum p."""
    q, k, v = (np.asarray(a, np.float64) for a in (q, k, v))
    heads, hd = q.shape
    n, nkv = k.shape[0], k.shape[1]
    g = heads // nkv
    out, lse = np.zeros((heads, hd)), np.full(heads, -np.inf)
    size, mean = np.zeros(heads), np.zeros((heads, hd))
    lo = max(0, n - window) if window > 0 else 0
    with np.errstate(all="ignore"):
        for h in range(heads):
            kk, vv = k[lo:, h // g], v[lo:, h // g]
            if n == lo:
                continue
            s = (kk @ q[h]) * scale
            size[h] = np.max((np.abs(kk) @ np.abs(q[h])) * abs(scale))
            if softcap > 0:
                s = softcap * np.tanh(s / softcap)
            m = np.max(s)
            if m == -np.inf:
                continue
            p = np.exp(s - m)
            out[h] = (p[:, None] * np.where(p[:, None] == 0, 0, vv)).sum(0) / p.sum()
            mean[h] = (p[:, None] * np.abs(np.where(p[:, None] == 0, 0, vv))).sum(0) / p.sum()
            lse[h] = m + np.log(p.sum())
    return out, lse, size, mean


def attention_bound(io, rounded_weights, hd, n, out, lse, size, mean, softcap=0.0):
    """How far an fp32 evaluation may be from 64 bits: a score is a sum of hd products, at most hd + 8 roundings of
    2^-24 of sum |q k|, then times scale and log2 e; exp2 of it is off by that, absolutely, and by 2^-22 (a softcap's quotient,
    tanh and product by a few 2^-24 of the cap). The sums over
    n positions run in at most n / 4 + 128 steps in any lane (four waves share a piece). Outputs are rounded once; 16-bit
    weights and values (rounded_weights) by half a step each."""
    u = 2.0**-24
    ds = u * (hd + 16) * size + 2.0**-22 + 16 * u * softcap
    steps = u * (n / 4 + 128)
    w = 3 * HALF_STEP[io] if rounded_weights else 0.0
    tol = (2 * ds[:, None] + 2 * steps + w) * mean + HALF_STEP[io] * np.abs(out) * (1 + 1e-3) + 1e-37
    if io == F16:
        tol = tol + 2.0**-25                   # half of the smallest subnormal
    return tol, ds + steps + 4 * u * np.abs(np.where(np.isfinite(lse), lse, 0)) + (w if rounded_weights else 0)


def rope64(x, pos, freqs, rot, interleaved, magnitude):
    """x [tokens][heads][hd] float64, turned."""
    y = np.array(x, np.float64)
    i = np.arange(rot // 2)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
    # the product in long double: its rounding does not matter at far positions
    ang = np.asarray(pos, np.longdouble)[:, None] * np.asarray(freqs, np.longdouble)
    c, s = ((f(ang) * magnitude).astype(np.float64)[:, None] for f in (np.cos, np.sin))
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    return y


def beams64(logits, scores, done, requests, beams, end):
    """(scores, tokens, parents, done) by the definition, every candidate formed and sorted."""
    n = logits.shape[1]
    x = np.where(np.isnan(logits), -np.inf, logits).astype(np.float64)
    out = ([], [], [], [])
    with np.errstate(all="ignore"):
        for r in range(requests):
            cand = []
            for b in range(beams):
                row = r * beams + b
                cum = float(scores[row])
                m = x[row].max()
                lse = m + np.log(np.exp(x[row] - m).sum())
                s = cum + (x[row] - lse)
                if done[row]:
                    s = np.full(n, -np.inf)
                    if 0 <= end < n:
                        s[end] = cum
                if not np.isfinite(cum) or np.isnan(s).all():
                    s = np.full(n, -np.inf)
                s = np.where(np.isnan(s) | (s == np.inf), -np.inf, s)
                if np.isposinf(m):
                    s = np.full(n, -np.inf) if not done[row] else s
                order = np.lexsort((np.arange(n), -np.where(np.isneginf(s), -np.inf, x[row] if not done[row] else s), -s))[:beams]
                cand += [(-s[v], b, k, int(v)) for k, v in enumerate(order)]
            for ns, b, _, v in sorted(cand)[:beams]:
                out[0].append(-ns)
                out[1].append(v)
                out[2].append(r * beams + b)
                out[3].append(int(bool(done[r * beams + b]) or v == end))
    return tuple(np.array(o) for o in out)
