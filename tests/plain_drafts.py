"""Drafted tokens judged request by request in numpy's 64 bits: what `ops.verify_drafts` computes, stated plainly."""
import numpy as np


def softmax(row, t):
    """exp((l - max) / T) over its sum; NaN is no token, a row without one has no probabilities (all 0)."""
    l = np.where(np.isnan(row), -np.inf, row).astype(np.float64)
    top = l.max()
    if top == -np.inf:
        return np.zeros_like(l)
    with np.errstate(invalid="ignore", over="ignore"):
        below = l - top                                       # (infinitely far below, be it for l or for top: no weight, at an infinite temperature too)
        e = np.where(l == top, 1.0, np.where(below == -np.inf, 0.0, np.exp(below / np.float64(t))))
    return e / e.sum()


def draw(weights, u):
    running = np.cumsum(weights)
    if not running[-1] > 0:
        return None
    hit = np.flatnonzero(running > u * running[-1])
    return int(hit[0]) if hit.size else int(np.flatnonzero(weights)[-1])


def verify(logits, drafts, temperature, uniform, draft_logits=None, n_drafts=None, first_row=None):
    n, k = drafts.shape
    vocab = logits.shape[1]
    tokens, counts = np.full((n, k + 1), -1, dtype=np.int32), np.zeros(n, dtype=np.int32)
    for r in range(n):
        brought = k if n_drafts is None else min(max(int(n_drafts[r]), 0), k)
        first = r * (k + 1) if first_row is None else int(first_row[r])
        if first < 0 or first + brought >= logits.shape[0]:
            continue
        t, j = float(temperature[r]), 0
        while True:
            row = logits[first + j]
            x = int(drafts[r, j]) if j < brought else -1
            inside = 0 <= x < vocab
            if not t > 0:
                best = int(np.argmax(np.where(np.isnan(row), -np.inf, row)))
                token, stays = best, j < brought and inside and x == best
            else:
                p = softmax(row, t)
                rest = p
                stays = False
                if j < brought:
                    if draft_logits is not None:
                        q = softmax(draft_logits[r, j], t)
                        stays = inside and float(uniform[r, j]) * q[x] < p[x]
                        rest = np.maximum(p - q, 0.0)
                        rest = p if rest.sum() <= 1e-12 else rest
                    elif inside:
                        stays = float(uniform[r, j]) < p[x]
                        rest = p.copy()
                        rest[x] = 0.0
                token = x
                if not stays:
                    token = draw(rest, float(uniform[r, k]))
                    if token is None:
                        token = draw(p, float(uniform[r, k]))
                    token = 0 if token is None else token
            tokens[r, j] = token
            j += 1
            if not stays:
                break
        counts[r] = j
    return tokens, counts
