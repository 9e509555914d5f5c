"""The operators that serve many requests at once restated in float64 --
TEST INFRASTRUCTURE ONLY.

Plain loops over sequences, rows and heads: attention of a chunk of new tokens
over the paged cache, block tables from lengths, low-rank adapters per row, as
include/tkm_b200.h defines them.  Arrays are numpy, caches float64.
"""
import math

import numpy as np


def softmax_rows(s):
    """(p, lse) of each row of s; a row of -inf alone gives p = 0 and -inf."""
    top = s.max(1, initial=-math.inf)
    with np.errstate(invalid="ignore", divide="ignore"):
        e = np.exp(s - np.where(np.isneginf(top), 0.0, top)[:, None])
        total = e.sum(1)
        return e / np.where(total == 0, 1.0, total)[:, None], np.where(np.isneginf(top), 0.0, top) + np.log(total)


def chunk(k, v, pages, held, q, scale):
    """(out [n, Hq, D], lse [n, Hq]) of the n newest of `held` tokens: q [n, Hq, D]; row i sees slots 0 .. held - n + i,
    those in a page below 0 or above the pool not among them.  What a row does not see does not enter its sums."""
    n, Hq, D = q.shape
    Hkv, page = k.shape[1:3]
    out, lse = np.zeros((n, Hq, D)), np.full((n, Hq), -math.inf)
    used = pages[:-(-max(held, 0) // page)]
    there = np.repeat((used >= 0) & (used < k.shape[0]), page)[:held]
    safe = np.where((used >= 0) & (used < k.shape[0]), used, 0)
    for h in range(Hkv):
        G = Hq // Hkv
        kk = k[safe, h].reshape(-1, D)[:held][there]
        vv = v[safe, h].reshape(-1, D)[:held][there]
        at = np.arange(held)[there]
        for i in range(n):
            m = int((at <= held - n + i).sum())
            if m == 0:
                continue
            s = q[i, h * G:(h + 1) * G] @ kk[:m].T * scale
            p, lse[i, h * G:(h + 1) * G] = softmax_rows(s)
            out[i, h * G:(h + 1) * G] = p @ vv[:m]
    return out, lse


def pages(table, held, lens, stack, page):
    """(table, held, stack, granted) after a call; `stack` is the list of free pages, its top last."""
    table, held, stack = table.copy(), held.copy(), list(stack)
    B, most = table.shape
    want = [min(most, -(-n // page)) for n in lens]
    for b in range(B):
        for e in range(want[b], held[b]):
            stack.append(int(table[b, e]))
            table[b, e] = -1
        held[b] = min(held[b], want[b])
    granted, asked, height = [], 0, len(stack)
    for b in range(B):
        need = want[b] - held[b]
        asked += need
        fits = need == 0 or asked <= height
        if fits:
            for e in range(held[b], want[b]):
                table[b, e] = stack.pop()
            held[b] = want[b]
        granted.append(int(fits and lens[b] <= most * page))
    return table, held, stack, granted


def slots(table, held, lens, page, row_start, rows):
    """The place of each row in the pool, -1 where it has none."""
    out = np.full(rows, -1, np.int64)
    for b in range(len(lens)):
        for r in range(row_start[b], row_start[b + 1]):
            j = lens[b] - (row_start[b + 1] - r)
            if 0 <= j < held[b] * page:
                out[r] = int(table[b, j // page]) * page + j % page
    return out


def lora(x, a, b, y, adapter, row_start, scale):
    """y + scale * (x A) B with the adapter of each row's sequence."""
    out = y.copy()
    for q, i in enumerate(adapter):
        if i >= 0:
            at = slice(row_start[q], row_start[q + 1])
            out[at] += (1.0 if scale is None else scale[i]) * ((x[at] @ a[i]) @ b[i])
    return out
