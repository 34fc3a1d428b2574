"""Operators for prompts that many sequences share, for drafted tokens and for long contexts, as a program on the
device-pointer API uses them over its paged cache: attention of rows that share their first positions, the
verification of drafted tokens, bounds of K per page, the choice of pages by them, and attention over the chosen pages.

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
The bounds of K: [layers][pages][kv][2][hd], lowest and highest value of each dim, F16 over an F16 cache, else BF16.
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
        # Three drafted tokens of one sequence over the small test vocabulary: the smallest call.
        {"name": "verify-small", "kind": "verify", "requests": 1, "drafts": 3, "n": 4096, "draft": True, "temperature": 1.0},
        # A batch with five drafts each over the whole Gemma-3 vocabulary, by a draft model of the same one.
        {"name": "verify-vocab", "kind": "verify", "requests": 16, "drafts": 5, "n": 262144, "draft": True, "temperature": 0.75},
        # Drafts looked up in the prompt: no probabilities of their own.
        {"name": "verify-lookup", "kind": "verify", "requests": 8, "drafts": 4, "n": 262144, "draft": False, "temperature": 1.0},
        # The forward pass that verifies five drafts of one chat: six rows of the 270M shape over an fp32 cache.
        {"name": "shared-drafts", "kind": "shared", "groups": 1, "rows": 6, "shared": 1018, "own": 6, "drafts": True, "heads": 4, "kv": 1,
         "hd": 256, "page": 64, "cache": "f32", "io": "f32", "cap": 0.0},
        # A serving batch behind one long system prompt, 16-bit cache and rows, own turns of up to 1000 positions.
        {"name": "shared-serve", "kind": "shared", "groups": 1, "rows": 128, "shared": 32768, "own": 1000, "drafts": False, "heads": 32,
         "kv": 8, "hd": 128, "page": 32, "cache": "bf16", "io": "bf16", "cap": 0.0},
        # Two documents in a 4-bit cache, sixteen questions to each.
        {"name": "shared-long", "kind": "shared", "groups": 2, "rows": 16, "shared": 65536, "own": 300, "drafts": False, "heads": 32,
         "kv": 8, "hd": 128, "page": 64, "cache": "q4_0", "io": "f32", "cap": 0.0},
        # One decode step of sixteen sequences of the 1B shape, 8-bit cache: each one's last page.
        {"name": "bounds-step", "kind": "bounds", "batch": 16, "len": 2048, "new": 1, "kv": 1, "hd": 256, "page": 64, "cache": "q8_0"},
        # All pages of three long documents behind their prompt pass.
        {"name": "bounds-prompt", "kind": "bounds", "batch": 3, "len": 131072, "new": 131072, "kv": 8, "hd": 128, "page": 32, "cache": "bf16"},
        # The choice of 16 pages of one sequence.
        {"name": "select-small", "kind": "select", "batch": 1, "len": 4000, "heads": 4, "kv": 1, "hd": 256, "page": 16, "cache": "f32",
         "io": "f32", "pages": 16, "first": 1, "last": 2},
        # The choice of 128 pages of up to 4096 for four long documents.
        {"name": "select-long", "kind": "select", "batch": 4, "len": 131072, "heads": 32, "kv": 8, "hd": 128, "page": 32, "cache": "bf16",
         "io": "bf16", "pages": 128, "first": 1, "last": 4},
        # Attention over the 16 pages of that sequence.
        {"name": "pages-small", "kind": "pages", "batch": 1, "len": 4000, "heads": 4, "kv": 1, "hd": 256, "page": 16, "cache": "f32",
         "io": "f32", "pages": 16, "cap": 0.0},
        # A serving batch that attends to 64 pages of each long context.
        {"name": "pages-serve", "kind": "pages", "batch": 64, "len": 24000, "heads": 32, "kv": 8, "hd": 128, "page": 32, "cache": "bf16",
         "io": "bf16", "pages": 64, "cap": 0.0},
    ]


def _log_int(rng, lo, hi, multiple=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))
    return min(max(multiple, int(round(v / multiple)) * multiple), hi)


def _heads(rng):
    kv = rng.choice([1, 1, 2, 3, 8])
    return kv * rng.choice([1, 2, 4, 5, 8]), kv, rng.choice([64, 128, 256])


def _io(rng, cache):
    return rng.choice(["f32", "f32"] + ([cache] if cache in ("bf16", "f16") else ["f32"] if cache == "f32" else ["bf16", "f16"]))


def draw(rng):
    kind = rng.choice(["verify", "shared", "shared", "bounds", "select", "pages"])
    c = {"kind": kind}
    if kind == "verify":
        d = rng.randint(1, 8)
        c.update(drafts=d, n=_log_int(rng, 500, 262144), draft=rng.random() < 0.7, temperature=rng.choice([1.0, 0.75, 1.25, 0.0]))
        c["requests"] = _log_int(rng, 1, 176 // (2 * d + 1))
    elif kind == "shared":
        h, kv, hd = _heads(rng)
        cache = rng.choice(sorted(CODE))
        groups, drafts = rng.randint(1, 4), rng.random() < 0.3
        rows = rng.randint(1, 9) if drafts else _log_int(rng, 1, 128 // groups)
        most = int(min(1 << 17, (1 << 32) / (rows * groups * h * hd), (1 << 26) / (groups * kv * hd * ROW_BYTES[cache])))
        c.update(groups=groups, rows=rows, shared=_log_int(rng, 1, most), own=rows if drafts else _log_int(rng, 1, 1000), drafts=drafts,
                 heads=h, kv=kv, hd=hd, page=16 * rng.randint(1, 8), cache=cache, io=_io(rng, cache), cap=rng.choice([0.0, 0.0, 30.0]))
    elif kind == "bounds":
        _, kv, hd = _heads(rng)
        cache, batch = rng.choice(sorted(CODE)), rng.randint(1, 40)
        most = int(min(131072, (1 << 28) / (batch * kv * hd * max(ROW_BYTES[cache], 1.0))))
        c.update(batch=batch, len=_log_int(rng, 1, most), kv=kv, hd=hd, page=16 * rng.randint(1, 8), cache=cache)
        c["new"] = rng.choice([1, 1, _log_int(rng, 1, c["len"]), c["len"]])
    else:
        h, kv, hd = _heads(rng)
        cache, page = rng.choice(sorted(CODE)), 16 * rng.randint(1, 4)
        batch = _log_int(rng, 1, 64 if kind == "pages" else 24)
        most = int(min(131072, (1 << 30) / (batch * kv * hd * max(ROW_BYTES[cache], 1.0))))
        c.update(batch=batch, len=_log_int(rng, 1, most), heads=h, kv=kv, hd=hd, page=page, cache=cache, io=_io(rng, cache))
        c["pages"] = _log_int(rng, 1, 200) if kind == "select" else _log_int(rng, 1, max(1, (1 << 26) // (batch * kv * hd * page)))
        if kind == "select":
            c.update(first=rng.randint(0, 2), last=rng.randint(0, 4))
            c["pages"] = max(c["pages"], c["first"] + c["last"])
        else:
            c["cap"] = rng.choice([0.0, 0.0, 30.0])
    return c


# ---- inputs ----

def _generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 1000003 + 31)
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


def _pool(c, g, pages):
    """K or V of one layer in use: [pages][kv][bytes]. Values about N(0, 1) (4- and 8-bit codes: uniform)."""
    n = (pages, c["kv"])
    if c["cache"] in TORCH:
        x = torch.empty(*n, c["page"] * c["hd"], dtype=TORCH[c["cache"]], device=DEV)
        x.normal_(generator=g)
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


def _bound_type(c):
    return torch.float16 if c["cache"] == "f16" else torch.bfloat16


def _prepare_verify(c, seed):
    g = _generator(seed)
    r, d, n = c["requests"], c["drafts"], c["n"]
    ld = n + n % 3
    logits = _normal(g, r, d + 1, ld, std=3.0)
    # a draft model is near the target, and its tokens are its own draws
    draft = logits[:, :d] + _normal(g, r, d, ld, std=0.7)
    p = torch.softmax(draft[..., :n].float() / (c["temperature"] or 1.0), -1)
    tokens = torch.multinomial(p.view(r * d, n), 1, generator=g).view(r, d)
    if not c["draft"]:                                  # looked up: right more often than a draw would be
        best = logits[:, :d, :n].argmax(-1)
        tokens = torch.where(torch.rand(r, d, generator=g, device=DEV) < 0.5, best, tokens)
    counts = np.maximum(0, d - np.arange(r) % 4 // 3)   # every fourth request has one draft less
    return {"logits": logits, "draft": draft.contiguous(), "ld": ld, "token": tokens.to(torch.int32), "count": _ints(counts),
            "draws": torch.rand(r, d + 1, generator=g, device=DEV), "out": torch.empty(r, d + 1, dtype=torch.int32, device=DEV),
            "accepted": torch.empty(r, dtype=torch.int32, device=DEV)}


def _shared_sizes(c):
    """(shared positions of each group, lengths of all rows): drafted tokens follow one another, other rows have an own turn
    each, and every eighth row is a padded one."""
    f = np.arange(c["groups"]) * 0.6180339887498949 % 1.0
    shared = np.maximum(1, np.rint(c["shared"] * (1.0 - 0.5 * f))).astype(np.int64)
    if c["drafts"]:
        return shared, (shared[:, None] + 1 + np.arange(c["rows"])).reshape(-1)
    shared = -(-shared // c["page"]) * c["page"]        # whole pages are shared
    n = np.repeat(shared, c["rows"]) + np.maximum(1, _lengths(c["groups"] * c["rows"], c["own"]))
    row = np.arange(len(n)) % c["rows"]
    return shared, np.where((row % 8 == 7), 0, n)


def _prepare_shared(c, seed):
    g = _generator(seed)
    shared, n = _shared_sizes(c)
    ps, rows = c["page"], c["rows"]
    ld = -(-int(n.max()) // ps)
    group = np.arange(len(n)) // rows
    if c["drafts"]:                                     # all rows of a group are one sequence
        need = -(-n.reshape(-1, rows)[:, -1] // ps)
        first, behind = need, np.zeros(len(n), np.int64)
    else:
        first = shared // ps
        behind = np.maximum(0, -(-n // ps) - first[group])
    pages = int(first.sum() + behind.sum()) + 5
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32).cpu().numpy()
    table, at = np.full((len(n), ld), -1, np.int32), 0
    for i, k in enumerate(first):
        table[group == i, :k] = order[at:at + k]
        at += k
    for r, k in enumerate(behind):
        table[r, first[group[r]]:first[group[r]] + k] = order[at:at + k]
        at += k
    q = _normal(g, len(n), c["heads"], c["hd"], std=2.0, dtype=TORCH[c["io"]])
    return {"q": q, "kp": _pool(c, g, pages), "vp": _pool(c, g, pages), "pages": pages, "table": _ints(table), "len": _ints(n),
            "shared": _ints(shared), "top": int(n.max()), "most": int(shared.max()),
            "own": max(1, int((n - shared[group]).max())), "scale": 1.0 / math.sqrt(c["hd"]),
            "out": torch.empty_like(q), "lse": torch.empty(len(n), c["heads"], device=DEV)}


def _table(g, needed, ld, pages):
    """A page table [rows][ld]: `needed[r]` pages of the pool in no order, -1 behind them."""
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32).cpu().numpy()
    t, at = np.full((len(needed), ld), -1, np.int32), 0
    for r, k in enumerate(needed):
        t[r, :k] = order[at:at + k]
        at += k
    return _ints(t)


def _batch(c, g):
    n = _lengths(c["batch"], c["len"])
    need = -(-n // c["page"])
    ld, pages = max(1, int(need.max())), int(need.sum()) + 5
    return n, {"len": _ints(n), "top": int(n.max()), "pages": pages, "table": _table(g, need, ld, pages)}


def _prepare_bounds(c, seed):
    g = _generator(seed)
    n, s = _batch(c, g)
    s.update(kp=_pool(c, g, s["pages"]), vp=torch.empty(s["pages"], c["kv"], _page_bytes(c), dtype=torch.uint8, device=DEV),
             start=_ints(np.maximum(0, n - c["new"])),
             bounds=torch.zeros(s["pages"], c["kv"], 2, c["hd"], dtype=_bound_type(c), device=DEV))
    return s


def _prepare_select(c, seed):
    g = _generator(seed)
    _, s = _batch(c, g)
    mid = _normal(g, s["pages"], c["kv"], c["hd"], std=0.6)
    half = 1.0 + 0.5 * torch.rand(s["pages"], c["kv"], 2, c["hd"], generator=g, device=DEV)
    k = [torch.empty(s["pages"], c["kv"], _page_bytes(c), dtype=torch.uint8, device=DEV) for _ in range(2)]     # not read
    s.update(kp=k[0], vp=k[1], q=_normal(g, c["batch"], c["heads"], c["hd"], std=2.0, dtype=TORCH[c["io"]]),
             bounds=torch.stack([mid - half[:, :, 0], mid + half[:, :, 1]], 2).to(_bound_type(c)),
             selected=torch.empty(c["batch"], c["kv"], c["pages"], dtype=torch.int32, device=DEV))
    return s


def _chosen(c):
    """Pages of each row that its lists name."""
    return np.minimum(-(-_lengths(c["batch"], c["len"]) // c["page"]), c["pages"])


def _prepare_pages(c, seed):
    g = _generator(seed)
    n, s = _batch(c, g)
    need = -(-n // c["page"])
    k, top = c["pages"], int(need.max())
    # distinct pages in order, the last one of the sequence among them, -1 behind
    x = torch.rand(c["batch"], c["kv"], top, generator=g, device=DEV)
    at, last = torch.arange(top, device=DEV), torch.from_numpy(need).to(DEV)[:, None, None]
    x = torch.where(at < last, x + 2 * (at == last - 1), -1.0)
    sel = torch.full((c["batch"], c["kv"], k), 1 << 30, dtype=torch.int64, device=DEV)
    best = x.topk(min(k, top), -1)
    sel[..., :min(k, top)] = torch.where(best.values >= 0, best.indices, 1 << 30)
    sel = sel.sort(-1).values
    q = _normal(g, c["batch"], c["heads"], c["hd"], std=2.0, dtype=TORCH[c["io"]])
    s.update(q=q, kp=_pool(c, g, s["pages"]), vp=_pool(c, g, s["pages"]), selected=torch.where(sel == 1 << 30, -1, sel).to(torch.int32),
             scale=1.0 / math.sqrt(c["hd"]), out=torch.empty_like(q), lse=torch.empty(c["batch"], c["heads"], device=DEV))
    return s


# ---- the plain forms ----

def _views(c, pool, which):
    """Strided views of one layer's pool [pages][kv][bytes], codes and scales (or None), whose leading dims are (page, position
    split in two) and give a position's codes of every head, and the two splits."""
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


def _gather_pages(c, pool, which, pages):
    """fp32 rows [batch, positions, kv, hd] of whole pages [batch, n]."""
    codes, scales, _, _ = _views(c, pool, which)
    return _decode(c, codes[pages].flatten(1, 3), None if scales is None else scales[pages].flatten(1, 3), which)


def _gather_rows(c, pool, which, page, pos):
    """fp32 rows [..., kv, hd] at (page, position in it)."""
    codes, scales, p, sp = _views(c, pool, which)
    return _decode(c, codes[page, pos // p, pos % p], None if scales is None else scales[page, pos // sp, pos % sp], which)


def _plain_verify(c, s):
    r, d, n = c["requests"], c["drafts"], c["n"]
    x, token, count = s["logits"][..., :n].double(), s["token"].long(), s["count"].long()
    at = torch.arange(d + 1, device=DEV)
    row = torch.arange(r, device=DEV)
    if c["temperature"] == 0.0:
        best = x.argmax(-1)
        ok = (best[:, :d] == token) & (at[:d] < count[:, None])
        a = ok.long().cumprod(1).sum(1)
        last = best[row, a]
    else:
        p = torch.exp((x - x.amax(-1, keepdim=True)) / c["temperature"])
        p = p / p.sum(-1, keepdim=True)
        if c["draft"]:
            q = s["draft"][..., :n].double()
            q = torch.exp((q - q.amax(-1, keepdim=True)) / c["temperature"])
            q = q / q.sum(-1, keepdim=True)
        else:
            q = torch.zeros(r, d, n, dtype=torch.float64, device=DEV).scatter_(2, token[..., None], 1.0)
        px, qx = (y[:, :d].gather(2, token[..., None])[..., 0] for y in (p, q))
        ok = (s["draws"][:, :d].double() * qx < px) & (at[:d] < count[:, None])
        a = ok.long().cumprod(1).sum(1)
        w = p[row, a]
        refused = (a < count)[:, None]
        w = torch.where(refused, (w - q[row, a.clamp(max=d - 1)]).clamp(min=0.0), w)
        cum = w.cumsum(-1)
        past = cum > s["draws"][:, d:].double() * cum[:, -1:]
        last = past.to(torch.int8).argmax(-1)           # the first
    out = torch.where(at[:d + 1] < a[:, None], torch.cat([token, token[:, :1]], 1), -1)
    out[row, a] = last
    return {"token": out.to(torch.int32), "accepted": a.to(torch.int32)}


def _cap(c, sc):
    return c["cap"] * torch.tanh(sc / c["cap"]) if c["cap"] else sc


def _softmax(sc, on):
    """(weights, their sum, log of the sum of exp) over the last dim, rows without an `on` position: zeros, -inf."""
    sc = torch.where(on, sc, -math.inf)
    m = sc.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    p = torch.exp(sc - m)
    den = p.sum(-1, keepdim=True)
    return p, torch.where(den == 0, 1.0, den), (m + torch.log(den))[..., 0]


def _plain_shared(c, s):
    kv, hd, ps, rows = c["kv"], c["hd"], c["page"], c["rows"]
    g = c["heads"] // kv
    table, n, shared = s["table"].long(), s["len"].long(), s["shared"].long()
    most = -(-s["most"] // ps)
    out, lse = torch.empty_like(s["out"]), torch.empty_like(s["lse"])
    for i in range(c["groups"]):
        r = slice(i * rows, (i + 1) * rows)
        q = s["q"][r].float().view(rows, kv, g, hd)
        # the shared positions, once for all rows
        k, v = (_gather_pages(c, s[w + "p"], w, table[i * rows, :most].clamp(min=0)[None])[0] for w in ("k", "v"))   # [positions, kv, hd]
        qs = q.permute(1, 0, 2, 3).reshape(kv, rows * g, hd)
        sc = torch.bmm(qs, k.permute(1, 2, 0).contiguous()).view(kv, rows, g, -1).permute(1, 0, 2, 3)
        at = torch.arange(k.shape[0], device=DEV)
        on = (at < shared[i]) & (at < n[r, None])
        # each row's own
        pos = shared[i] + torch.arange(s["own"], device=DEV)
        page = table[r][:, (pos // ps).clamp(max=table.shape[1] - 1)].clamp(min=0)
        ko, vo = (_gather_rows(c, s[w + "p"], w, page, (pos % ps)[None].expand(rows, -1)) for w in ("k", "v"))       # [rows, own, kv, hd]
        so = torch.matmul(q, ko.permute(0, 2, 3, 1).contiguous())
        no = pos < n[r, None]
        p, den, e = _softmax(_cap(c, torch.cat([sc, so], -1) * s["scale"]), torch.cat([on, no], -1)[:, None, None])
        v = torch.where((at < shared[i])[:, None, None], v, 0.0)
        vo = torch.where(no[..., None, None], vo, 0.0)
        o = torch.bmm(p[..., :k.shape[0]].permute(1, 0, 2, 3).reshape(kv, rows * g, -1), v.permute(1, 0, 2).contiguous())
        o = o.view(kv, rows, g, hd).permute(1, 0, 2, 3) + torch.matmul(p[..., k.shape[0]:].contiguous(), vo.permute(0, 2, 1, 3).contiguous())
        out[r] = (o / den).reshape(rows, c["heads"], hd).to(out.dtype)
        lse[r] = e.reshape(rows, c["heads"])
    return {"out": out, "lse": lse}


def _outward(x, up, dtype):
    """fp32 rounded to 16 bits, up or down."""
    r = x.to(dtype)
    over = r.float() < x if up else r.float() > x
    bits = r.view(torch.int16).to(torch.int32) & 0xffff
    away = (bits & 0x8000 == 0) == up                   # the magnitude grows
    step = torch.where(bits & 0x7fff == 0, torch.full_like(bits, 1 if up else 0x8001), bits + torch.where(away, 1, -1))
    bits = torch.where(over, step, bits)
    return torch.where(bits > 0x7fff, bits - 0x10000, bits).to(torch.int16).view(dtype)


def _plain_bounds(c, s):
    ps = c["page"]
    row, i = ((torch.arange(s["table"].shape[1], device=DEV) * ps < s["len"][:, None])
              & ((torch.arange(s["table"].shape[1], device=DEV) + 1) * ps > s["start"][:, None])).nonzero(as_tuple=True)
    page = s["table"].long()[row, i]
    k = _gather_pages(c, s["kp"], "k", page[:, None])   # [pages, ps, kv, hd]
    on = (i[:, None] * ps + torch.arange(ps, device=DEV) < s["len"].long()[row, None])[..., None, None]
    lo, hi = torch.where(on, k, math.inf).amin(1), torch.where(on, k, -math.inf).amax(1)
    s["bounds"][page] = torch.stack([_outward(lo, False, s["bounds"].dtype), _outward(hi, True, s["bounds"].dtype)], 2)
    return {"bounds": s["bounds"]}


def _plain_select(c, s):
    b, kv, g, k = c["batch"], c["kv"], c["heads"] // c["kv"], c["pages"]
    need = (s["len"].long() + c["page"] - 1) // c["page"]
    q = s["q"].double().view(b, kv, g, c["hd"])
    out = torch.full((b, kv, k), 1 << 30, dtype=torch.int64, device=DEV)
    at = torch.arange(s["table"].shape[1], device=DEV)
    for r in range(b):
        x = s["bounds"][s["table"][r].long().clamp(min=0)].double()             # [pages, kv, 2, hd]
        up = torch.matmul(q[r].clamp(min=0.0), x[:, :, 1].permute(1, 2, 0).contiguous())
        sc = (up + torch.matmul(q[r].clamp(max=0.0), x[:, :, 0].permute(1, 2, 0).contiguous())).amax(1)     # [kv, pages]
        sc = torch.where((at < c["first"]) | (at >= need[r] - c["last"]), math.inf, sc)
        sc = torch.where(at < need[r], sc, -math.inf)
        best = sc.sort(dim=-1, descending=True, stable=True)
        m = min(k, sc.shape[-1])
        out[r, :, :m] = torch.where(best.values[:, :m] == -math.inf, 1 << 30, best.indices[:, :m])
    out = out.sort(-1).values
    return {"selected": torch.where(out == 1 << 30, -1, out).to(torch.int32)}


def _plain_pages(c, s):
    b, kv, g, hd, ps = c["batch"], c["kv"], c["heads"] // c["kv"], c["hd"], c["page"]
    sel = s["selected"].long()
    page = s["table"].long()[torch.arange(b, device=DEV)[:, None, None], sel.clamp(min=0)].clamp(min=0)
    out, lse = torch.empty_like(s["out"]).view(b, kv, g, hd), torch.empty_like(s["lse"]).view(b, kv, g)
    on = (sel[..., None] * ps + torch.arange(ps, device=DEV) < s["len"].long()[:, None, None, None]) & (sel >= 0)[..., None]
    on = on.flatten(-2)                                  # [b, kv, positions]
    q = s["q"].float().view(b, kv, g, hd)
    one = {**c, "kv": 1}
    for h in range(kv):
        k, v = (_gather_pages(one, s[w + "p"][:, h:h + 1], w, page[:, h])[:, :, 0] for w in ("k", "v"))      # [b, positions, hd]
        sc = _cap(c, torch.bmm(q[:, h], k.transpose(1, 2).contiguous()) * s["scale"])
        p, den, e = _softmax(sc, on[:, h, None])
        out[:, h] = (torch.bmm(p, torch.where(on[:, h, :, None], v, 0.0)) / den).to(out.dtype)
        lse[:, h] = e
    return {"out": out.view_as(s["out"]), "lse": lse.view_as(s["lse"])}


# ---- the library's calls ----

def _cache(c, s):
    """The program's handle of its cache, made once."""
    from sapphire_amd.paged import PagedCache
    if "cache" not in s:
        s["cache"] = PagedCache(CODE[c["cache"]], 1, s["pages"], c["page"], c["kv"], c["hd"], k=s["kp"].data_ptr(), v=s["vp"].data_ptr())
    return s["cache"]


def _rows(x):
    from sapphire_amd.paged import Rows
    t, h, hd = x.shape
    return Rows(x.data_ptr(), {torch.float32: F32, torch.bfloat16: BF16, torch.float16: F16}[x.dtype], t, h, hd,
                token_stride=x.stride(0), head_stride=x.stride(1))


def _page_table(s):
    from sapphire_amd.paged import PageTable
    return PageTable(s["table"].data_ptr(), s["table"].shape[0], s["table"].shape[1])


def _workspace(s, nbytes):
    if "ws" not in s:
        s["ws"] = torch.empty(max(1, nbytes()), dtype=torch.uint8, device=DEV)
    return s["ws"].data_ptr()


def _own_verify(c, s):
    from sapphire_amd import paged
    ws = _workspace(s, lambda: paged.verify_workspace_bytes(c["n"], c["requests"], c["drafts"]))
    paged.verify(s["logits"].data_ptr(), s["ld"], c["n"], c["requests"], c["drafts"], s["token"].data_ptr(), s["draws"].data_ptr(),
                 s["out"].data_ptr(), s["accepted"].data_ptr(), ws, draft_logits=s["draft"].data_ptr() if c["draft"] else None,
                 draft_ld=s["ld"] if c["draft"] else 0, counts=s["count"].data_ptr(), temperature=c["temperature"])
    return {"token": s["out"], "accepted": s["accepted"]}


def _own_shared(c, s):
    cache = _cache(c, s)
    ws = _workspace(s, lambda: cache.shared_attention_workspace_bytes(len(s["len"]), c["heads"], s["top"]))
    cache.shared_attention(0, _rows(s["q"]), _rows(s["out"]), _page_table(s), s["len"].data_ptr(), s["top"], rows=c["rows"],
                           shared=s["shared"].data_ptr(), max_own=c["own"], scale=s["scale"], softcap=c["cap"], lse=s["lse"].data_ptr(),
                           workspace=ws)
    return {"out": s["out"], "lse": s["lse"]}


def _own_bounds(c, s):
    _cache(c, s).bounds(0, s["bounds"].data_ptr(), _page_table(s), s["len"].data_ptr(), min(c["new"], s["top"]), start=s["start"].data_ptr())
    return {"bounds": s["bounds"]}


def _own_select(c, s):
    cache = _cache(c, s)
    ws = _workspace(s, lambda: cache.select_workspace_bytes(c["batch"], s["top"]))
    cache.select(0, s["bounds"].data_ptr(), _rows(s["q"]), _page_table(s), s["len"].data_ptr(), s["top"], s["selected"].data_ptr(), c["pages"],
                 first=c["first"], last=c["last"], workspace=ws)
    return {"selected": s["selected"]}


def _own_pages(c, s):
    cache = _cache(c, s)
    ws = _workspace(s, lambda: cache.attention_workspace_bytes(c["batch"], c["heads"], c["pages"] * c["page"]))
    cache.pages_attention(0, _rows(s["q"]), _rows(s["out"]), _page_table(s), s["len"].data_ptr(), s["selected"].data_ptr(), c["pages"],
                          scale=s["scale"], softcap=c["cap"], lse=s["lse"].data_ptr(), workspace=ws)
    return {"out": s["out"], "lse": s["lse"]}


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


def _attend64(c, s, q, k, v):
    """(out, lse) of q [heads, hd] over k and v [positions, hd]."""
    sc = (q.double() @ k.T.contiguous()) * s["scale"]
    if c["cap"]:
        sc = c["cap"] * torch.tanh(sc / c["cap"])
    return torch.softmax(sc, -1) @ v, torch.logsumexp(sc, -1)


def _exact_shared(c, s):
    shared, n = _shared_sizes(c)
    g, ps, rows = c["heads"] // c["kv"], c["page"], c["rows"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    lse = torch.full(s["lse"].shape, -math.inf, dtype=torch.float64, device=DEV)
    for i in range(c["groups"]):
        for h in range(c["kv"]):
            p = torch.arange(int(shared[i]), device=DEV)
            first = [_rows64(c, s[w + "p"], w, s["table"][i * rows].long()[p // ps], p % ps, h) for w in ("k", "v")]
            for r in range(i * rows, (i + 1) * rows):
                if n[r] == 0:
                    continue
                p = torch.arange(int(shared[i]), int(n[r]), device=DEV)
                k, v = (torch.cat([x, _rows64(c, s[w + "p"], w, s["table"][r].long()[p // ps], p % ps, h)]) for x, w in zip(first, ("k", "v")))
                out[r, h * g:(h + 1) * g], lse[r, h * g:(h + 1) * g] = _attend64(c, s, s["q"][r, h * g:(h + 1) * g], k, v)
    return {"out": out, "lse": lse}


def _exact_pages(c, s):
    n = _lengths(c["batch"], c["len"])
    g, ps = c["heads"] // c["kv"], c["page"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    lse = torch.full(s["lse"].shape, -math.inf, dtype=torch.float64, device=DEV)
    for b in range(c["batch"]):
        for h in range(c["kv"]):
            sel = s["selected"][b, h].long()
            p = (sel[sel >= 0][:, None] * ps + torch.arange(ps, device=DEV)).flatten()
            p = p[p < int(n[b])]
            if len(p) == 0:
                continue
            k, v = (_rows64(c, s[w + "p"], w, s["table"][b].long()[p // ps], p % ps, h) for w in ("k", "v"))
            out[b, h * g:(h + 1) * g], lse[b, h * g:(h + 1) * g] = _attend64(c, s, s["q"][b, h * g:(h + 1) * g], k, v)
    return {"out": out, "lse": lse}


def _exact_bounds(c, s):
    """The 16-bit numbers next to the extremes of the values in 64 bits."""
    n, ps, dtype = _lengths(c["batch"], c["len"]), c["page"], s["bounds"].dtype
    out = s["bounds"].double()
    every = torch.arange(-0x8000, 0x8000, device=DEV).to(torch.int16).view(dtype).double()
    every = torch.unique(every[torch.isfinite(every)])
    for b in range(c["batch"]):
        lo, end = max(0, int(n[b]) - c["new"]) // ps, -(-int(n[b]) // ps)
        p = torch.arange(lo * ps, end * ps, device=DEV)
        page = s["table"][b, lo:end].long()
        for h in range(c["kv"] if end > lo else 0):
            x = _rows64(c, s["kp"], "k", page.repeat_interleave(ps), p % ps, h)
            if c["cache"] in ("q4_0", "q8_0"):
                x = x.float().double()                  # values of a quantized cache are fp32 products
            here = (p < int(n[b]))[:, None]
            low, high = torch.where(here, x, math.inf).view(-1, ps, c["hd"]).amin(1), torch.where(here, x, -math.inf).view(-1, ps, c["hd"]).amax(1)
            out[page, h, 0] = every[torch.searchsorted(every, low, right=True) - 1]
            out[page, h, 1] = every[torch.searchsorted(every, high)]
    return {"bounds": out}


def _exact_none(c, s):
    return None         # whole numbers only


# ---- what a pass cannot do without ----

def _work_verify(c):
    rows = c["requests"] * (c["drafts"] * (2 if c["draft"] and c["temperature"] else 1) + 1)
    return {"bytes": 4 * rows * c["n"] + 4 * c["requests"] * (3 * c["drafts"] + 4), "flops": 4 * rows * c["n"]}


def _work_shared(c):
    shared, n = _shared_sizes(c)
    # drafted tokens read their predecessors' rows too, which are one sequence's
    behind = c["rows"] * c["groups"] if c["drafts"] else int(np.maximum(0, n - np.repeat(shared, c["rows"])).sum())
    read = int(shared.sum()) + behind
    qo = len(n) * c["heads"] * (2 * c["hd"] * ROW_BYTES[c["io"]] + 4)
    return {"bytes": 2 * read * c["kv"] * c["hd"] * ROW_BYTES[c["cache"]] + qo + read // c["page"] * 4 + len(n) * 4,
            "flops": 4 * int(n.sum()) * c["heads"] * c["hd"]}


def _work_bounds(c):
    n = _lengths(c["batch"], c["len"])
    start = np.maximum(0, n - c["new"]) // c["page"]
    positions = int((n - start * c["page"])[n > 0].sum())
    pages = int((-(-n // c["page"]) - start)[n > 0].sum())
    return {"bytes": c["kv"] * c["hd"] * (positions * ROW_BYTES[c["cache"]] + 4 * pages) + pages * 4, "flops": 2 * positions * c["kv"] * c["hd"]}


def _work_select(c):
    pages = int((-(-_lengths(c["batch"], c["len"]) // c["page"])).sum())
    qs = c["batch"] * (c["heads"] * c["hd"] * ROW_BYTES[c["io"]] + 4 * c["kv"] * c["pages"])
    return {"bytes": pages * (c["kv"] * c["hd"] * 4 + 4) + qs, "flops": 4 * pages * c["heads"] * c["hd"]}


def _work_pages(c):
    positions = int((_chosen(c) * c["page"]).sum())
    qo = c["batch"] * c["heads"] * (2 * c["hd"] * ROW_BYTES[c["io"]] + 4)
    return {"bytes": 2 * positions * c["kv"] * c["hd"] * ROW_BYTES[c["cache"]] + qo + 8 * c["batch"] * c["kv"] * c["pages"],
            "flops": 4 * positions * c["heads"] * c["hd"]}


_KINDS = {"verify": (_prepare_verify, _plain_verify, _own_verify, _exact_none, _work_verify),
          "shared": (_prepare_shared, _plain_shared, _own_shared, _exact_shared, _work_shared),
          "bounds": (_prepare_bounds, _plain_bounds, _own_bounds, _exact_bounds, _work_bounds),
          "select": (_prepare_select, _plain_select, _own_select, _exact_none, _work_select),
          "pages": (_prepare_pages, _plain_pages, _own_pages, _exact_pages, _work_pages)}


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
