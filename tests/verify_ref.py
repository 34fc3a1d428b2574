"""Verification of drafted tokens in plain numpy and 64 bits, for the tests."""
import numpy as np


def probabilities(logits, temperature):
    """softmax(logits / temperature) of one row: NaN as -inf, infinite maxima share it."""
    x = np.where(np.isnan(logits), -np.inf, logits).astype(np.float64)
    m = x.max()
    with np.errstate(over="ignore"):
        w = (x == m).astype(np.float64) if np.isinf(m) else np.exp((x - m) / temperature)
    return w / w.sum()


def first_best(logits):
    return int(np.where(np.isnan(logits), -np.inf, logits).argmax())


def verify64(logits, draft, tokens, counts, draws, temperature):
    """logits [requests][drafts + 1][n], draft [requests][drafts][n] or None -> (tokens, accepted)."""
    requests, drafts = tokens.shape
    temperature = float(np.float32(temperature))
    n = logits.shape[2]
    out, kept = np.full((requests, drafts + 1), -1), np.zeros(requests, int)
    for r in range(requests):
        count = drafts if counts is None else min(max(int(counts[r]), 0), drafts)
        a = 0
        if temperature <= 0:
            while a < count and tokens[r, a] == first_best(logits[r, a]):
                a += 1
            last = first_best(logits[r, a])
        else:
            u = np.where(np.isnan(draws[r]), 0.0, np.clip(draws[r], 0.0, 1.0)).astype(np.float64)
            w = None
            while w is None:
                p = probabilities(logits[r, a], temperature)
                if a == count:
                    w = p
                    break
                x = int(tokens[r, a])
                if draft is not None:
                    q = probabilities(draft[r, a], temperature)
                else:
                    q = (np.arange(n) == x).astype(np.float64)
                if 0 <= x < n and u[a] * q[x] < p[x]:
                    a += 1
                    continue
                w = np.maximum(p - q, 0.0)
                w = p if w.sum() == 0.0 else w
            cum = np.cumsum(w)
            past = np.flatnonzero((cum > u[drafts] * cum[-1]) & (w > 0))
            last = past[0] if len(past) else np.flatnonzero(w > 0)[-1]
        out[r, :a], out[r, a], kept[r] = tokens[r, :a], last, a
    return out, kept
