"""The operators of a paged key-value cache and what serves it, as a program on the device-pointer API
uses them: rotary positions of many rows, the cache's writes and reads (fp32, 16-bit, Q8_0, Q4_0),
attention of one new token per sequence, beam search's selection and the reordering of its cache.

listed() names fixed cases, draw() gives others of the same ranges. prepare() makes what the program
holds before the call, run() is one pass: through the library where `own` is set, in elementary torch
operations where it is not. work() counts the bytes and operations that a pass cannot do without and
exact() gives the same outputs in 64-bit arithmetic, by its own indexing of the cache's bytes.

The cache holds its pages in the order of the matrix cores' operands. Of one page and K/V head
(page_size ps, head_dim hd, nb = hd / 32 blocks, position p, dim d):
  K  F32, BF16, F16   [ps/16][hd * es / 16][16 positions][16 bytes]
     Q8_0             [ps/16][nb/2][4][16 positions][2 blocks][8 codes]: dims 32 b + 8 m .. + 7
     Q4_0             [ps/16][nb/g][4][16 positions][g blocks][4 bytes], g = min(4, nb): dims 32 b + 8 m + i in the
                      low nibbles, + 4 + i in the high ones, as 4-bit two's complement
     scales           fp32 [ps][nb], behind the codes
  V  all              [ps/P][16][P positions][hd/16 dims], P = 16 / (bytes of hd/16 dims), within 1..4
     Q4_0             byte i of a run: dim i in the low nibble, dim hd/32 + i in the high one, value + 8
     scales           fp32 [ps/4][nb][4 positions], behind the codes
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda:0"
F32, BF16, F16, Q4_0, Q8_0 = 0, 1, 2, 3, 4
CODE = {"f32": F32, "bf16": BF16, "f16": F16, "q4_0": Q4_0, "q8_0": Q8_0}
TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ROW_BYTES = {"f32": 4.0, "bf16": 2.0, "f16": 2.0, "q8_0": 36 / 32, "q4_0": 20 / 32}     # per element, scales included
CODE_BYTES = {"f32": 4.0, "bf16": 2.0, "f16": 2.0, "q8_0": 1.0, "q4_0": 0.5}


def listed():
    return [
        # The q and k heads of one decode step of the 270M shape: the smallest call.
        {"name": "rope-token", "kind": "rope", "tokens": 1, "heads": 4, "kv": 1, "hd": 256, "rot": 256, "io": "f32",
         "interleaved": False, "top": 1024, "magnitude": 1.0},
        # A pass over long prompts, far positions, half of each head rotated in pairs.
        {"name": "rope-prompt", "kind": "rope", "tokens": 8192, "heads": 32, "kv": 8, "hd": 128, "rot": 64, "io": "bf16",
         "interleaved": True, "top": 131072, "magnitude": 1.2},
        # Sixteen sequences' new rows into an 8-bit cache, and back out.
        {"name": "rows-step", "kind": "rows", "seqs": 16, "tokens": 16, "len": 2048, "heads": 4, "kv": 1, "hd": 256,
         "page": 64, "layers": 2, "cache": "q8_0", "io": "f32", "padded": False},
        # Several prompts' rows into a 4-bit cache, and back out as a prompt pass over them reads them.
        {"name": "rows-prompt", "kind": "rows", "seqs": 5, "tokens": 8192, "len": 4000, "heads": 32, "kv": 8, "hd": 128,
         "page": 64, "layers": 1, "cache": "q4_0", "io": "bf16", "padded": True},
        # Chat: one sequence, a windowed layer of the 270M shape over an fp32 cache.
        {"name": "attend-chat", "kind": "attend", "batch": 1, "len": 1024, "window": 512, "heads": 4, "kv": 1, "hd": 256,
         "page": 64, "cache": "f32", "io": "f32", "cap": 0.0},
        # Sixteen sequences of the 1B shape in lock step, 8-bit cache, ragged lengths.
        {"name": "attend-batch", "kind": "attend", "batch": 16, "len": 2048, "window": 0, "heads": 4, "kv": 1, "hd": 256,
         "page": 64, "cache": "q8_0", "io": "f32", "cap": 0.0},
        # A full serving batch over a 16-bit cache with 16-bit rows: the most bytes.
        {"name": "attend-serve", "kind": "attend", "batch": 250, "len": 2000, "window": 0, "heads": 32, "kv": 8, "hd": 128,
         "page": 32, "cache": "bf16", "io": "bf16", "cap": 0.0},
        # A few long documents in a 4-bit cache.
        {"name": "attend-long", "kind": "attend", "batch": 3, "len": 131072, "window": 0, "heads": 32, "kv": 8, "hd": 128,
         "page": 64, "cache": "q4_0", "io": "f32", "cap": 0.0},
        # Four beams of one request over the small test vocabulary.
        {"name": "beams-small", "kind": "beams", "requests": 1, "beams": 4, "n": 4096, "done": False},
        # Eight requests of eight beams over the whole Gemma-3 vocabulary, some beams ended.
        {"name": "beams-vocab", "kind": "beams", "requests": 8, "beams": 8, "n": 262144, "done": True},
        # The cache of four beams of one request (18 layers) after a step.
        {"name": "reorder-small", "kind": "reorder", "requests": 1, "beams": 4, "len": 200, "layers": 18, "kv": 1, "hd": 256,
         "page": 16, "cache": "f32"},
        # Sixteen beams, 26 layers, larger pages.
        {"name": "reorder-large", "kind": "reorder", "requests": 4, "beams": 4, "len": 1000, "layers": 26, "kv": 1, "hd": 256,
         "page": 64, "cache": "bf16"},
    ]


def _log_int(rng, lo, hi, multiple=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return min(max(multiple, int(round(v / multiple)) * multiple), hi)


def _heads(rng):
    kv = rng.choice([1, 1, 2, 3, 8])
    return kv * rng.choice([1, 2, 4, 5, 8]), kv, rng.choice([64, 128, 256])


def draw(rng):
    kind = rng.choice(["rope", "rows", "attend", "attend", "attend", "beams", "reorder"])
    c = {"kind": kind}
    if kind == "rope":
        h, kv, hd = _heads(rng)
        most = 8192 * 48 * 128 // ((h + 2 * kv) * hd)
        c.update(tokens=_log_int(rng, 1, most), heads=h, kv=kv, hd=hd, rot=rng.choice([hd, hd, hd // 2, hd // 4 + 2]),
                 io=rng.choice(["f32", "bf16", "f16"]), interleaved=rng.random() < 0.5, top=_log_int(rng, 2, 1000000),
                 magnitude=rng.choice([1.0, 1.0, 1.3]))
    elif kind == "rows":
        h, kv, hd = _heads(rng)
        seqs, most = rng.randint(1, 40), 8192 * 8 * 128 // (kv * hd)
        c.update(seqs=seqs, tokens=_log_int(rng, 1, most), heads=h, kv=kv, hd=hd, page=16 * rng.randint(1, 8),
                 layers=rng.randint(1, 3), cache=rng.choice(sorted(CODE)), io=rng.choice(["f32", "bf16", "f16"]),
                 padded=rng.random() < 0.5)
        c["len"] = c["tokens"] // seqs + rng.randint(1, 2000)
    elif kind == "attend":
        h, kv, hd = _heads(rng)
        cache = rng.choice(sorted(CODE))
        batch = _log_int(rng, 1, 250)
        row = kv * hd * max(ROW_BYTES[cache], 1.0)      # the plain form's memory counts too
        most = int(250 * 1100 * 8 * 128 * 2 / row / (batch if batch < 3 else batch * 0.55))
        c.update(batch=batch, len=_log_int(rng, 1, min(131072, most)), window=rng.choice([0, 0, 0, 512, 1000]), heads=h, kv=kv,
                 hd=hd, page=16 * rng.randint(1, 8), cache=cache,
                 io=rng.choice(["f32", "f32"] + ([cache] if cache in ("bf16", "f16") else ["f32"] if cache == "f32" else ["bf16", "f16"])),
                 cap=rng.choice([0.0, 0.0, 30.0]))
    elif kind == "beams":
        b = rng.randint(1, 16)
        r = rng.randint(1, max(1, min(8, 64 // b)))
        c.update(requests=r, beams=b, n=_log_int(rng, 500, 262144), done=rng.random() < 0.5)
    else:
        b, hd = rng.randint(1, 8), rng.choice([64, 128, 256])
        c.update(requests=rng.randint(1, 4), beams=b, len=_log_int(rng, 1, 1000), layers=rng.randint(1, 26), kv=rng.choice([1, 2]),
                 hd=hd, page=16 * rng.randint(1, 4), cache=rng.choice(["f32", "bf16", "f16"]))
        while c["requests"] * b * c["layers"] * c["kv"] * hd * (c["len"] + 2 * c["page"]) > 1 << 28:
            c["layers"] = (c["layers"] + 1) // 2
            c["len"] = (c["len"] + 1) // 2
    return c


# ---- inputs ----

def _generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 1000003 + 29)
    return g


def _normal(g, *shape, std=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=g, device=DEV) * std).to(dtype)


def _ints(values):
    return torch.tensor(np.asarray(values, np.int32), device=DEV)


def _lengths(batch, top):
    """Ragged lengths: the first is `top`, every eighth sequence is a padded one of length 0."""
    f = np.arange(batch) * 0.6180339887498949 % 1.0
    n = np.maximum(1, np.rint(top * (1.0 - 0.9 * f))).astype(np.int64)
    n[7::8] = 0
    return n


def _page_bytes(c):
    """Bytes of one page of K (or V) of one K/V head."""
    quant = c["cache"] in ("q8_0", "q4_0")
    return int(c["page"] * c["hd"] * CODE_BYTES[c["cache"]]) + (c["page"] * c["hd"] // 32 * 4 if quant else 0)


def _pool(c, g, layers, pages):
    """K or V of a cache in use: [layers][pages][kv][bytes]. Values about N(0, 1) (4- and 8-bit codes: uniform)."""
    n = (layers, pages, c["kv"])
    if c["cache"] in TORCH:
        x = torch.empty(*n, c["page"] * c["hd"], dtype=TORCH[c["cache"]], device=DEV)
        for i in range(layers):
            x[i].normal_(generator=g)
        return x.view(torch.uint8)
    pool = torch.randint(-2**31, 2**31 - 1, (*n, _page_bytes(c) // 4), generator=g, device=DEV, dtype=torch.int32)
    codes = int(c["page"] * c["hd"] * CODE_BYTES[c["cache"]]) // 4
    if c["cache"] == "q8_0":
        b = pool.view(torch.int8)[..., :4 * codes]
        b.clamp_(min=-127)                              # what the quantizer emits
    scale = pool.view(torch.float32)[..., codes:]
    scale.uniform_(0.3, 1.5, generator=g)
    scale.mul_(0.0137 if c["cache"] == "q8_0" else 0.217)
    return pool.view(torch.uint8)


def _table(g, needed, ld, pages):
    """A page table [rows][ld]: `needed[r]` pages of the pool in no order, -1 behind them; and the pages left over."""
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32).cpu().numpy()
    t, at = np.full((len(needed), ld), -1, np.int32), 0
    for r, k in enumerate(needed):
        t[r, :k] = order[at:at + k]
        at += k
    return _ints(t), order[at:]


def _qkv(c, g, tokens):
    """The fused projection's rows, and its q, k and v heads as views."""
    h, kv, hd = c["heads"], c["kv"], c["hd"]
    x = _normal(g, tokens, h + 2 * kv, hd, dtype=TORCH[c["io"]])
    return x, x[:, :h], x[:, h:h + kv], x[:, h + kv:]


def _prepare_rope(c, seed):
    g = _generator(seed)
    x, _, _, _ = _qkv(c, g, c["tokens"])
    rot = c["rot"]
    inv = 10000.0 ** (-torch.arange(0, rot, 2, device=DEV, dtype=torch.float64) / rot)
    pos = torch.randint(0, c["top"], (c["tokens"],), generator=g, device=DEV, dtype=torch.int32)
    n = c["heads"] + c["kv"]
    return {"x": x, "n": n, "pos": pos, "inv": inv, "y": torch.empty(c["tokens"], n, c["hd"], dtype=x.dtype, device=DEV)}


def _row_places(c):
    """(sequence, position) of each token: an even share of consecutive positions per sequence, ending at a ragged length."""
    per = -(-c["tokens"] // c["seqs"])
    t = np.arange(c["tokens"])
    seq, ends = t // per, np.maximum(per, _lengths(c["seqs"], max(c["len"], per)))
    pos = ends[seq] - per + t % per
    if c["padded"]:
        pos = np.where(t % per >= per - per // 16, -1, pos)     # padding behind the prompt
    return seq, pos, int(ends.max())


def _prepare_rows(c, seed):
    g = _generator(seed)
    _, _, k, v = _qkv(c, g, c["tokens"])
    seq, pos, top = _row_places(c)
    ld = -(-top // c["page"])
    pages = c["seqs"] * ld + 3
    table, _ = _table(g, [ld] * c["seqs"], ld, pages)
    shape = (c["tokens"], c["kv"], c["hd"])
    return {"k": k, "v": v, "kp": _pool(c, g, c["layers"], pages), "vp": _pool(c, g, c["layers"], pages), "pages": pages,
            "table": table, "seq": _ints(seq), "pos": _ints(pos), "layer": c["layers"] - 1,
            "ko": torch.empty(shape, dtype=k.dtype, device=DEV), "vo": torch.empty(shape, dtype=k.dtype, device=DEV)}


def _prepare_attend(c, seed):
    g = _generator(seed)
    n = _lengths(c["batch"], c["len"])
    need = -(-n // c["page"])
    ld = max(1, int(need.max()))
    pages = int(need.sum()) + 5
    table, _ = _table(g, need, ld, pages)
    q = _normal(g, c["batch"], c["heads"], c["hd"], std=2.0, dtype=TORCH[c["io"]])
    return {"q": q, "kp": _pool(c, g, 1, pages), "vp": _pool(c, g, 1, pages), "pages": pages, "table": table, "len": _ints(n),
            "top": int(n.max()), "scale": 1.0 / math.sqrt(c["hd"]), "out": torch.empty_like(q),
            "lse": torch.empty(c["batch"], c["heads"], device=DEV)}


def _prepare_beams(c, seed):
    g = _generator(seed)
    rows, ld = c["requests"] * c["beams"], c["n"] + c["n"] % 3
    score = -_normal(g, rows, std=3.0).abs()
    done = torch.randint(0, 4, (rows,), generator=g, device=DEV, dtype=torch.int32) == 0
    done = done.to(torch.int32) * int(c["done"])
    out = {k: torch.empty(rows, dtype=torch.int32, device=DEV) for k in ("token", "parent", "done_out")}
    return {"logits": _normal(g, rows, ld, std=3.0), "ld": ld, "score": score, "done": done, "end": 1,
            "score_out": torch.empty(rows, device=DEV), **out}


def _prepare_reorder(c, seed):
    g = _generator(seed)
    rows = c["requests"] * c["beams"]
    n = np.repeat(np.maximum(1, _lengths(c["requests"], c["len"])), c["beams"])
    need = -(-n // c["page"])
    ld = int(need.max()) + 1
    pages = int(need.sum()) + rows + 2
    table, left = _table(g, need, ld, pages)
    first = torch.arange(rows, device=DEV) // c["beams"] * c["beams"]
    parent = first + torch.randint(0, c["beams"], (rows,), generator=g, device=DEV)
    return {"kp": _pool(c, g, c["layers"], pages), "vp": _pool(c, g, c["layers"], pages), "pages": pages, "table": table,
            "len": _ints(n), "parent": parent.to(torch.int32), "spare": _ints(left[:rows]),
            "table_out": torch.empty_like(table), "len_out": torch.empty(rows, dtype=torch.int32, device=DEV)}


# ---- the plain forms ----

def _views(c, pool, which):
    """(codes [pages.., page positions split.., ...], scales or None, to a head row): strided views of one layer's pool
    [pages][kv][bytes] whose leading dims, indexed by (page, position parts), give a position's codes of every head."""
    ps, hd, nb, t = c["page"], c["hd"], c["hd"] // 32, c["cache"]
    body = pool[..., :int(ps * hd * CODE_BYTES[t])]
    tail = pool[..., int(ps * hd * CODE_BYTES[t]):]
    if which == "k":
        if t in TORCH:
            e = 16 // int(CODE_BYTES[t])
            codes = body.view(TORCH[t]).unflatten(-1, (ps // 16, hd // e, 16, e)).permute(0, 2, 4, 1, 3, 5)
        elif t == "q8_0":      # pages kv tile pair m pos block 8 -> pages tile pos kv pair block m 8
            codes = body.view(torch.int8).unflatten(-1, (ps // 16, nb // 2, 4, 16, 2, 8)).permute(0, 2, 5, 1, 3, 6, 4, 7)
        else:                  # pages kv tile group m pos block 4 -> pages tile pos kv group block m 4
            gr = min(4, nb)
            codes = body.unflatten(-1, (ps // 16, nb // gr, 4, 16, gr, 4)).permute(0, 2, 5, 1, 3, 6, 4, 7)
        scales = None if t in TORCH else tail.view(torch.float32).unflatten(-1, (ps // 16, 16, nb)).permute(0, 2, 3, 1, 4)
        return codes, scales, 16, 16
    run = hd // 16
    p = min(4, max(1, int(16 // (run * CODE_BYTES[t]))))
    typed = body.view(TORCH[t]) if t in TORCH else body.view(torch.int8) if t == "q8_0" else body
    codes = typed.unflatten(-1, (ps // p, 16, p, run if t != "q4_0" else run // 2)).permute(0, 2, 4, 1, 3, 5)
    scales = None if t in TORCH else tail.view(torch.float32).unflatten(-1, (ps // 4, nb, 4)).permute(0, 2, 4, 1, 3)
    return codes, scales, p, 4


def _decode(c, codes, scales, which):
    """fp32 rows [..., kv, hd] of gathered codes [..., kv, parts] and scales [..., kv, nb]."""
    t, hd = c["cache"], c["hd"]
    if t in TORCH:
        return codes.flatten(-2).float()
    if t == "q8_0":
        x = codes.flatten(-4 if which == "k" else -2).float()
    else:
        low, high = (codes & 15).to(torch.int8), (codes >> 4).to(torch.int8)
        x = torch.stack([low, high], -2).flatten(-5 if which == "k" else -3)
        x = ((x ^ 8) - 8 if which == "k" else x - 8).float()
    return (x.unflatten(-1, (hd // 32, 32)) * scales[..., None]).flatten(-2)


def _gather(c, pool, which, page, pos):
    """fp32 rows [tokens, kv, hd] at (page, position in it)."""
    codes, scales, p, sp = _views(c, pool, which)
    return _decode(c, codes[page, pos // p, pos % p], None if scales is None else scales[page, pos // sp, pos % sp], which)


def _gather_pages(c, pool, which, pages):
    """fp32 rows [batch, positions, kv, hd] of whole pages [batch, n]."""
    codes, scales, _, _ = _views(c, pool, which)
    return _decode(c, codes[pages].flatten(1, 3), None if scales is None else scales[pages].flatten(1, 3), which)


def _encode(c, x, which):
    """(codes [tokens, kv, hd] as stored, nibbles unpacked; scales) of fp32 rows, each operation rounded on its own."""
    t, hd = c["cache"], c["hd"]
    if t in TORCH:
        return x.to(TORCH[t]), None
    b = x.unflatten(-1, (hd // 32, 32))
    mag = b.abs().amax(-1, keepdim=True)                        # NaN where the block has one
    if t == "q8_0":
        d = mag / torch.full_like(mag, 127.0)
    else:
        at = torch.arange(32, device=x.device)
        first = torch.where(b.abs() == mag, at, 31).amin(-1, keepdim=True)
        top = torch.where(torch.isnan(mag), mag, b.gather(-1, first))
        d = torch.where(mag == 0, 0.0, top) / torch.full_like(mag, -8.0)
    inv = torch.where(d == 0, 0.0, torch.ones_like(d) / d)
    y = b * inv
    if t == "q8_0":
        y = torch.nan_to_num(y, nan=0.0).clamp(-127.0, 127.0).double()
        q = torch.sign(y) * torch.floor(y.abs() + 0.5)          # halves away from zero, exactly
    else:
        q = torch.nan_to_num(y + 8.5, nan=8.0).clamp(0.0, 15.0).trunc() - 8.0
    return q.to(torch.int8).flatten(-2), d[..., 0]


def _store(c, pool, which, page, pos, x):
    codes, scales, p, sp = _views(c, pool, which)
    q, d = _encode(c, x, which)
    n, kv, hd, nb = q.shape[0], c["kv"], c["hd"], c["hd"] // 32
    if c["cache"] == "q4_0":
        if which == "k":        # elements 8 m + half * 4 + i of a block
            q = (q & 15).view(n, kv, nb, 4, 2, 4)
        else:                   # elements half * R + i of a run
            q = (q + 8).view(n, kv, 16, 2, hd // 32)
        q = (q.select(-2, 0) | (q.select(-2, 1) << 4)).to(torch.uint8)
    codes[page, pos // p, pos % p] = q.reshape(n, *codes.shape[3:])
    if scales is not None:
        scales[page, pos // sp, pos % sp] = d


def _plain_rope(c, s):
    x, rot = s["x"][:, :s["n"]].float(), c["rot"]
    ang = s["pos"].double()[:, None] * s["inv"]
    cos, sin = ((f(ang) * c["magnitude"]).float()[:, None] for f in (torch.cos, torch.sin))
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if c["interleaved"] else (x[..., :rot // 2], x[..., rot // 2:rot])
    ra, rb = a * cos - b * sin, b * cos + a * sin
    r = torch.stack([ra, rb], -1).flatten(-2) if c["interleaved"] else torch.cat([ra, rb], -1)
    return {"y": torch.cat([r, x[..., rot:]], -1).to(s["x"].dtype)}


def _plain_rows(c, s):
    pos, seq = s["pos"].long(), s["seq"].long()
    on = pos >= 0
    at = pos.clamp(min=0)
    page, off = s["table"].long()[seq, at // c["page"]], at % c["page"]
    keep = on.nonzero()[:, 0]
    out = {}
    for which in ("k", "v"):
        pool = s[which + "p"][s["layer"]]
        _store(c, pool, which, page[keep], off[keep], s[which][keep].float())
        rows = _gather(c, pool, which, page, off)
        out[which] = torch.where(on[:, None, None], rows, 0.0).to(s["k"].dtype)
    return out


def _plain_attend(c, s):
    b, g = c["batch"], c["heads"] // c["kv"]
    pages = s["table"].long()
    k, v = (_gather_pages(c, s[w + "p"][0], w, pages.clamp(min=0)) for w in ("k", "v"))     # [b, positions, kv, hd]
    at = torch.arange(k.shape[1], device=DEV)
    n = s["len"].long()[:, None]
    on = at < n
    if c["window"]:
        on = on & (at >= n - c["window"])
    on = on & (pages >= 0).repeat_interleave(c["page"], 1)
    q = s["q"].float().view(b, c["kv"], g, c["hd"])
    sc = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()) * s["scale"]                  # [b, kv, g, positions]
    if c["cap"]:
        sc = c["cap"] * torch.tanh(sc / c["cap"])
    on = on[:, None, None]
    sc = torch.where(on, sc, -math.inf)
    m = sc.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    p = torch.exp(sc - m)
    den = p.sum(-1, keepdim=True)
    v = torch.where(on[:, 0, 0, :, None, None], v, 0.0).permute(0, 2, 1, 3).contiguous()
    o = torch.matmul(p, v) / torch.where(den == 0, 1.0, den)
    return {"out": o.reshape(b, c["heads"], c["hd"]).to(s["q"].dtype), "lse": (m + torch.log(den)).reshape(b, c["heads"])}


def _plain_beams(c, s):
    r, w, n = c["requests"], c["beams"], c["n"]
    x = s["logits"][:, :n].double()
    x = torch.where(torch.isnan(x), -math.inf, x)
    m = x.amax(1, keepdim=True)
    lse = m + torch.log(torch.exp(x - m).sum(1, keepdim=True))
    sc = s["score"].double()[:, None] + (x - lse)
    sc = torch.where(torch.isnan(sc), -math.inf, sc)
    done = s["done"][:, None] != 0
    at = torch.arange(n, device=DEV)[None]
    sc = torch.where(done, torch.where(at == s["end"], s["score"].double()[:, None], -math.inf), sc)
    best, idx = torch.sort(sc.view(r, w * n), dim=1, descending=True, stable=True)
    best, idx = best[:, :w], idx[:, :w]
    parent = (idx // n + torch.arange(r, device=DEV)[:, None] * w).flatten()
    token = (idx % n).flatten()
    return {"score": best.flatten().float(), "token": token.to(torch.int32), "parent": parent.to(torch.int32),
            "done": ((s["done"][parent] != 0) | (token == s["end"])).to(torch.int32)}


def _plain_reorder(c, s):
    ps, table = c["page"], s["table"].long()
    parent, rows = s["parent"].long(), s["len"].shape[0]
    n = s["len"].long()[parent]
    full, rem = n // ps, n % ps
    at = torch.arange(table.shape[1], device=DEV)[None]
    out = torch.where(at < full[:, None], table[parent], -1)
    out = torch.where((at == full[:, None]) & (rem > 0)[:, None], s["spare"].long()[:, None], out)
    source = table[parent, full.clamp(max=table.shape[1] - 1)]
    tiles = ps // 16
    for w in ("k", "v"):
        pool = s[w + "p"].view(TORCH[c["cache"]])
        pool = pool.unflatten(-1, (tiles, -1)).permute(1, 3, 0, 2, 4)                       # pages, tiles, layers, kv, values
        row, tile = ((torch.arange(tiles, device=DEV)[None] * 16 < rem[:, None])).nonzero(as_tuple=True)
        pool[s["spare"].long()[row], tile] = pool[source[row], tile]
    return {"table": out.to(torch.int32), "len": n.to(torch.int32), "k": s["kp"].view(TORCH[c["cache"]]),
            "v": s["vp"].view(TORCH[c["cache"]])}


# ---- the library's calls ----

def _cache(c, s):
    """The program's handle of its cache, made once."""
    from sapphire_amd.paged import PagedCache
    if "cache" not in s:
        s["cache"] = PagedCache(CODE[c["cache"]], s["kp"].shape[0], s["pages"], c["page"], c["kv"], c["hd"],
                                k=s["kp"].data_ptr(), v=s["vp"].data_ptr())
    return s["cache"]


def _rows(x):
    from sapphire_amd.paged import Rows
    t, h, hd = x.shape
    return Rows(x.data_ptr(), {torch.float32: F32, torch.bfloat16: BF16, torch.float16: F16}[x.dtype], t, h, hd,
                token_stride=x.stride(0), head_stride=x.stride(1))


def _page_table(s, name="table"):
    from sapphire_amd.paged import PageTable
    return PageTable(s[name].data_ptr(), s[name].shape[0], s[name].shape[1])


def _own_rope(c, s):
    from sapphire_amd import paged
    paged.rope(_rows(s["x"][:, :s["n"]]), _rows(s["y"]), s["pos"].data_ptr(), s["inv"].data_ptr(), c["rot"],
               interleaved=c["interleaved"], magnitude=c["magnitude"])
    return {"y": s["y"]}


def _own_rows(c, s):
    cache, table = _cache(c, s), _page_table(s)
    cache.write(s["layer"], _rows(s["k"]), _rows(s["v"]), table, s["pos"].data_ptr(), seqs=s["seq"].data_ptr())
    cache.read(s["layer"], _rows(s["ko"]), _rows(s["vo"]), table, s["pos"].data_ptr(), seqs=s["seq"].data_ptr())
    return {"k": s["ko"], "v": s["vo"]}


def _own_attend(c, s):
    cache = _cache(c, s)
    if "ws" not in s:
        s["ws"] = torch.empty(max(1, cache.attention_workspace_bytes(c["batch"], c["heads"], s["top"])), dtype=torch.uint8, device=DEV)
    cache.attention(0, _rows(s["q"]), _rows(s["out"]), _page_table(s), s["len"].data_ptr(), s["top"], scale=s["scale"],
                    window=c["window"], softcap=c["cap"], lse=s["lse"].data_ptr(), workspace=s["ws"].data_ptr())
    return {"out": s["out"], "lse": s["lse"]}


def _own_beams(c, s):
    from sapphire_amd import paged
    if "ws" not in s:
        s["ws"] = torch.empty(max(1, paged.beam_workspace_bytes(c["n"], c["requests"], c["beams"])), dtype=torch.uint8, device=DEV)
    paged.beam_select(s["logits"].data_ptr(), s["ld"], c["n"], c["requests"], c["beams"], s["score"].data_ptr(),
                      s["score_out"].data_ptr(), s["token"].data_ptr(), s["parent"].data_ptr(), done=s["done"].data_ptr(),
                      done_out=s["done_out"].data_ptr(), end_token=s["end"], workspace=s["ws"].data_ptr())
    return {"score": s["score_out"], "token": s["token"], "parent": s["parent"], "done": s["done_out"]}


def _own_reorder(c, s):
    _cache(c, s).reorder(_page_table(s), s["parent"].data_ptr(), s["len"].data_ptr(), s["spare"].data_ptr(),
                         _page_table(s, "table_out"), s["len_out"].data_ptr())
    return {"table": s["table_out"], "len": s["len_out"], "k": s["kp"].view(TORCH[c["cache"]]), "v": s["vp"].view(TORCH[c["cache"]])}


# ---- the same in 64 bits ----

def _byte_of(c, which, p, d):
    """Byte offset of (position p, dim d) in a page's codes, and the nibble's shift (Q4_0)."""
    t, hd = c["cache"], c["hd"]
    b, e, nb = d // 32, d % 32, hd // 32
    none = torch.zeros_like(p + d)
    if which == "v":
        run = hd // 16
        bytes_ = run * CODE_BYTES[t]
        par = min(4, max(1, int(16 // bytes_)))
        first = ((p // par * 16 + d // run) * par + p % par) * int(bytes_)
        if t == "q4_0":
            return first + d % run % (run // 2), d % run // (run // 2) * 4 + none
        return first + d % run * int(CODE_BYTES[t]), none
    if t == "q8_0":
        return (((p // 16 * (nb // 2) + b // 2) * 4 + e // 8) * 16 + p % 16) * 16 + b % 2 * 8 + e % 8, none
    if t == "q4_0":
        g = min(4, nb)
        return (((p // 16 * (nb // g) + b // g) * 4 + e // 8) * 16 + p % 16) * (4 * g) + b % g * 4 + e % 4, e % 8 // 4 * 4 + none
    es = int(CODE_BYTES[t])
    per = 16 // es
    return ((p // 16 * (hd // per) + d // per) * 16 + p % 16) * 16 + d % per * es, none


def _rows64(c, pool, which, page, pos, head):
    """float64 [positions, hd] of one head at (page, position in it), read byte by byte."""
    t, hd, ps = c["cache"], c["hd"], c["page"]
    d = torch.arange(hd, device=DEV)[None]
    p = pos[:, None]
    start = ((page * c["kv"] + head) * pool.shape[-1])[:, None]
    at, shift = _byte_of(c, which, p, d)
    flat = pool.reshape(-1)
    if t in TORCH:
        return flat.view(TORCH[t])[(start + at) // int(CODE_BYTES[t])].double()
    tail = start + int(ps * hd * CODE_BYTES[t])
    sc = tail + ((p * (hd // 32) + d // 32) if which == "k" else ((p // 4 * (hd // 32) + d // 32) * 4 + p % 4)) * 4
    scale = flat.view(torch.float32)[sc // 4].double()
    if t == "q8_0":
        return flat.view(torch.int8)[start + at].double() * scale
    q = (flat[start + at].int() >> shift.int()) & 15
    q = torch.where(q > 7, q - 16, q) if which == "k" else q - 8
    return q.double() * scale


def _exact_rope(c, s):
    x = s["x"][:, :s["n"]].double()
    y, half = x.clone(), c["rot"] // 2
    z = torch.polar(torch.full_like(s["inv"], c["magnitude"])[None].expand(c["tokens"], -1).contiguous(), s["pos"].double()[:, None] * s["inv"])
    i = torch.arange(half, device=DEV)
    a, b = (2 * i, 2 * i + 1) if c["interleaved"] else (i, i + half)
    r = torch.complex(x[..., a], x[..., b]) * z[:, None]
    y[..., a], y[..., b] = r.real, r.imag
    return {"y": y}


def _quant64(t, x):
    """The values that fp32 rows [n, 32] are stored as, the quantizer's own fp32 operations in numpy."""
    with np.errstate(all="ignore"):
        mag = np.abs(x).max(1)
        if t == "q8_0":
            d = mag / np.float32(127)
        else:
            d = x[np.arange(len(x)), np.abs(x).argmax(1)] / np.float32(-8)
        y = x * np.where(d == 0, np.float32(0), np.float32(1) / d)[:, None]
        if t == "q8_0":
            q = np.copysign(np.floor(np.abs(y.astype(np.float64)) + 0.5), y)
        else:
            q = np.minimum(15, np.trunc(y + np.float32(8.5))) - 8.0
    return q * d.astype(np.float64)[:, None]


def _exact_rows(c, s):
    out = {}
    for w in ("k", "v"):
        x = s[w]
        if c["cache"] in TORCH:
            y = x.float().to(TORCH[c["cache"]]).double()
        else:
            y = _quant64(c["cache"], x.float().cpu().numpy().reshape(-1, 32))
            y = torch.from_numpy(y).reshape(x.shape).to(DEV)
        out[w] = y * (s["pos"] >= 0)[:, None, None]
    return out


def _exact_attend(c, s):
    out = torch.zeros(c["batch"], c["heads"], c["hd"], dtype=torch.float64, device=DEV)
    lse = torch.full((c["batch"], c["heads"]), -math.inf, dtype=torch.float64, device=DEV)
    g = c["heads"] // c["kv"]
    for b, n in enumerate(s["len"].tolist()):
        lo = max(0, n - c["window"]) if c["window"] else 0
        if n == lo:
            continue
        p = torch.arange(lo, n, device=DEV)
        page = s["table"][b].long()[p // c["page"]]
        for h in range(c["kv"]):
            k, v = (_rows64(c, s[w + "p"][0], w, page, p % c["page"], h) for w in ("k", "v"))
            sc = (s["q"][b, h * g:(h + 1) * g].double() @ k.T.contiguous()) * s["scale"]
            if c["cap"]:
                sc = c["cap"] * torch.tanh(sc / c["cap"])
            out[b, h * g:(h + 1) * g] = torch.softmax(sc, -1) @ v
            lse[b, h * g:(h + 1) * g] = torch.logsumexp(sc, -1)
    return {"out": out, "lse": lse}


def _exact_beams(c, s):
    w, n, score = c["beams"], c["n"], []
    lp = torch.log_softmax(s["logits"][:, :n].double(), 1) + s["score"].double()[:, None]
    for r in range(c["requests"]):
        rows = [s["score"][i].double()[None] if s["done"][i] else lp[i].topk(min(w, n)).values for i in range(r * w, r * w + w)]
        score.append(torch.cat(rows).sort(descending=True).values[:w])
    return {"score": torch.cat(score), "token": None, "parent": None, "done": None}


def _exact_reorder(c, s):
    return None         # copies only


# ---- what a pass cannot do without ----

def _work_rope(c):
    n = c["tokens"] * (c["heads"] + c["kv"])
    return {"bytes": 2 * n * c["hd"] * ROW_BYTES[c["io"]] + c["tokens"] * 4 + c["rot"] * 4, "flops": 3 * n * c["rot"]}


def _work_rows(c):
    row = c["kv"] * c["hd"]
    return {"bytes": c["tokens"] * (4 * row * (ROW_BYTES[c["io"]] + ROW_BYTES[c["cache"]]) + 16), "flops": 8 * c["tokens"] * row}


def _work_attend(c):
    n = _lengths(c["batch"], c["len"])
    n = int(np.minimum(n, c["window"]).sum() if c["window"] else n.sum())
    row = c["kv"] * c["hd"] * ROW_BYTES[c["cache"]]
    qo = c["batch"] * c["heads"] * (2 * c["hd"] * ROW_BYTES[c["io"]] + 4)
    return {"bytes": 2 * n * row + qo + n // c["page"] * 4 + c["batch"] * 4, "flops": 4 * n * c["heads"] * c["hd"]}


def _work_beams(c):
    rows = c["requests"] * c["beams"]
    return {"bytes": rows * (4 * c["n"] + 24), "flops": 4 * rows * c["n"]}


def _work_reorder(c):
    n = np.maximum(1, _lengths(c["requests"], c["len"]))
    tiles = int((-(-(n % c["page"]) // 16)).sum()) * c["beams"] * 16
    bytes_ = 4 * tiles * c["layers"] * c["kv"] * c["hd"] * ROW_BYTES[c["cache"]]
    return {"bytes": bytes_ + c["requests"] * c["beams"] * (8 * (int(n.max()) // c["page"] + 2) + 16), "flops": 0}


_KINDS = {"rope": (_prepare_rope, _plain_rope, _own_rope, _exact_rope, _work_rope),
          "rows": (_prepare_rows, _plain_rows, _own_rows, _exact_rows, _work_rows),
          "attend": (_prepare_attend, _plain_attend, _own_attend, _exact_attend, _work_attend),
          "beams": (_prepare_beams, _plain_beams, _own_beams, _exact_beams, _work_beams),
          "reorder": (_prepare_reorder, _plain_reorder, _own_reorder, _exact_reorder, _work_reorder)}


def prepare(case, seed):
    return case, _KINDS[case["kind"]][0](case, seed)


def run(state):
    case, held = state
    if own:
        return _KINDS[case["kind"]][2](case, held)
    return _KINDS[case["kind"]][1](case, held)


def work(case):
    return _KINDS[case["kind"]][4](case)


def exact(case, seed):
    return _KINDS[case["kind"]][3](case, _KINDS[case["kind"]][0](case, seed))
