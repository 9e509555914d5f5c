"""Generation operators restated in float64 numpy -- TEST INFRASTRUCTURE ONLY.

Plain loops over sequences, heads and tokens: the paged key-value cache
(append, attention of one token, eviction) and sampling, as
include/tkm_b200.h defines them.  Arrays are numpy, caches float64.
"""
import math

import numpy as np


def rope_frequencies(D, theta, scale=1.0, low=1.0, high=4.0, octx=8192.0):
    """Angle per position of each pair of a head.  With scale > 1 the frequencies
    of wavelengths above octx/low are divided by it, and those of wavelengths
    from octx/high to octx/low by a ramp from the whole of it (at octx/high) to
    nothing (at octx/low): the engine's rule, which Llama 3's published one
    runs the other way round."""
    f = theta ** (-np.arange(D // 2) / D)
    if scale > 1.0:
        for i in range(D // 2):
            turns = octx * f[i] / (2 * math.pi)
            if turns < low:
                f[i] /= scale
            elif turns <= high:
                f[i] *= 1 - (turns - low) / (high - low) * (1 - 1 / scale)
    return f


def prepare_row(x, pos, Hq, Hkv, D, bias, gain, qknorm, freq):
    """One packed row after bias, QKNorm and RoPE at `pos` (freq None: no RoPE) -> [Hq + 2*Hkv, D]."""
    x = x + (0 if bias is None else bias)
    x = x.reshape(Hq + 2 * Hkv, D).copy()
    for h in range(Hq + Hkv):
        if qknorm:
            x[h] /= math.sqrt(np.mean(x[h] ** 2) + 1e-5)
            if gain is not None:
                x[h] *= gain[h * D:(h + 1) * D]
        if freq is not None:
            c, s = np.cos(pos * freq), np.sin(pos * freq)
            a, b = x[h, 0::2].copy(), x[h, 1::2].copy()
            x[h, 0::2], x[h, 1::2] = a * c - b * s, a * s + b * c
    return x


def attend(k, v, pages, n, q, scale):
    """(out [Hq, D], lse [Hq], p [Hq, n]) of one token's q [Hq, D] over the first n slots of `pages`."""
    Hkv, page, D = k.shape[1:]
    Hq = q.shape[0]
    out, lse, p = np.zeros((Hq, D)), np.full(Hq, -math.inf), np.zeros((Hq, n))
    if n == 0:
        return out, lse, p
    used = pages[:-(-n // page)]
    for h in range(Hq):
        g = h // (Hq // Hkv)
        kk = k[used, g].reshape(-1, D)[:n]
        vv = v[used, g].reshape(-1, D)[:n]
        s = kk @ q[h] * scale
        top = s.max()
        e = np.exp(s - top)
        p[h] = e / e.sum()
        lse[h] = top + math.log(e.sum())
        out[h] = p[h] @ vv
    return out, lse, p


def evict_moves(weight, pos, n, budget, seen, recent, sinks):
    """[(to, from)] of one (sequence, kv head) whose n slots have these weights and positions."""
    if n <= budget:
        return []

    def worth(j):
        if pos[j] >= seen - recent or pos[j] < sinks:
            return (0, 0.0)
        if math.isnan(weight[j]):
            return (2, 0.0)
        return (1, -float(weight[j]))

    kept = set(sorted(range(n), key=lambda j: (worth(j), j))[:budget])
    holes = [j for j in range(budget) if j not in kept]
    movers = sorted(j for j in kept if j >= budget)
    assert len(holes) == len(movers)
    return list(zip(holes, movers))


def sample_sets(x, temperature, top_k, top_p, min_p, slack=0.0):
    """The tokens kept of one row (their float64 weights, 0 where dropped), the
    bound of top-p moved by `slack` times the total: how far another rounding
    of the weights may move it."""
    x = np.where(np.isnan(x), -math.inf, x.astype(np.float64))
    top = x.max()
    if top == -math.inf:
        return np.zeros_like(x)
    with np.errstate(invalid="ignore", over="ignore"):
        z = np.where(x == top, 0.0, (top - x) / (temperature if temperature > 0 else 1.0))
    w = np.rint(np.exp(-z) * 2.0 ** 31)
    order = np.lexsort((np.arange(x.size), -x))
    if not temperature > 0:
        keep = order[:1]
    else:
        keep = order[:top_k] if top_k > 0 else order
        keep = keep[w[keep] > 0]
        if top_p < 1:
            before = np.cumsum(w[keep]) - w[keep]
            inside = before < (top_p + slack) * w[keep].sum()
            inside[0] = True
            keep = keep[inside]
        if min_p > 0:
            keep = keep[w[keep] >= min(min_p, 1.0) * 2.0 ** 31 * (1 - 4 * slack)]
    out = np.zeros_like(x)
    out[keep] = w[keep]
    return out
