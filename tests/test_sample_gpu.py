"""tkb_sample_logits against the float64 oracle.

The weights are whole multiples of 2^-31 of the row's largest; the oracle's
exponential (64 bits) and the kernel's (32 bits, at most 2 ulp = 2^-22 off,
on a scaled distance of its own rounding, 2^-23 of up to 21.5) give weights
within 2^-18 of each other, so a running sum may differ by 2^-18 of the
total: the token must be one that u could select with the sums moved that
far, and the number of kept tokens must lie between the counts at top_p moved
by it.  log-probabilities: distances up to 21.5 rounded at 2^-23 twice: 1e-5.
"""
import math

import numpy as np
import pytest

from oracle import paged_oracle as ref

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

SLACK = 2.0 ** -18


def ops():
    from tokamak_b200 import ops as o
    return o


def dev(x, dtype=torch.float32):
    return torch.as_tensor(np.asarray(x)).to("cuda", dtype)


def check_rows(logits, u, t, k, p, m):
    rows = logits.shape[0]
    args = dict(temperature=None if t is None else dev(t), top_k=None if k is None else dev(k, torch.int32),
                top_p=None if p is None else dev(p), min_p=None if m is None else dev(m))
    token, logprob, kept = (x.cpu().numpy() for x in ops().sample_logits(logits, dev(u), **args))
    x = logits.float().cpu().numpy()
    u = np.asarray(u, np.float32).astype(np.float64)
    for r in range(rows):
        a = (float(np.float32(1 if t is None else t[r])), 0 if k is None else int(k[r]),
             float(np.float32(1 if p is None else p[r])), float(np.float32(0 if m is None else m[r])))
        less, more = (ref.sample_sets(x[r], *a, slack=s) for s in (-SLACK, SLACK))
        assert (less > 0).sum() <= kept[r] <= (more > 0).sum(), (r, kept[r])
        if not (more > 0).any():
            assert token[r] == -1 and logprob[r] == -math.inf
            continue
        i = token[r]
        assert 0 <= i < x.shape[1] and more[i] > 0, r
        if not a[0] > 0:
            assert i == np.nanargmax(np.where(np.isnan(x[r]), -np.inf, x[r])) and logprob[r] == 0
            continue
        # more and less differ by a few tokens of the last weight: both sums bracket the kernel's
        room = 4 * SLACK * more.sum() + (more.sum() - less.sum())
        at = u[r] * more.sum()
        upto = np.cumsum(more)
        assert upto[i] - more[i] - room <= at <= upto[i] + room, (r, i, upto[i], at)
        share = [math.log(more[i] / s.sum()) for s in (more, less)]
        # weights below 2^-20 of the top are whole numbers of few bits: their own logarithm is coarse
        tol = 1e-5 + 1.0 / more[i] + 8 * SLACK
        assert min(share) - tol <= logprob[r] <= max(share) + tol, (r, logprob[r], share)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,V", [(1, 32000), (5, 1), (7, 2), (33, 999), (9, 1024), (3, 49999), (2, 131072)])
@pytest.mark.parametrize("mode", ["plain", "top_k", "top_p", "min_p", "all"])
def test_sample(dtype, rows, V, mode):
    rng = np.random.default_rng(rows * 131 + V)
    logits = dev(2 * rng.standard_normal((rows, V)), dtype)
    u = rng.random(rows)
    u[0] = 0.0
    if rows > 1:
        u[-1] = 1 - 2.0 ** -24
    t = rng.uniform(0.3, 1.5, rows)
    t[rows // 2] = 0.0 if rows > 4 else t[rows // 2]
    k = rng.integers(1, 60, rows) if mode in ("top_k", "all") else None
    p = rng.uniform(0.1, 0.99, rows) if mode in ("top_p", "all") else None
    m = rng.uniform(0.001, 0.3, rows) if mode in ("min_p", "all") else None
    check_rows(logits, u, t, k, p, m)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V,ld", [(40000, 40000), (40001, 40003), (70000, 70016)])
def test_many_wide_rows(dtype, V, ld):
    """More rows than the GPU has SMs: one CTA per row, every truncation and odd value among them."""
    rng = np.random.default_rng(V)
    rows = 160
    x = 2 * rng.standard_normal((rows, ld)).astype(np.float32)
    x[3, :] = -np.inf
    x[4, 5:] = np.nan
    x[5, 100:30000] = -np.inf
    x[6, 30000:] = np.nan
    x[7, 39999] = np.inf
    x[8, :] = 1.0
    x[9] *= 10
    x[10] *= 0.01
    logits = dev(x, dtype)[:, :V]
    t = rng.uniform(0.3, 2.0, rows)
    t[11], t[12], t[13], t[14] = 0.0, 1e-30, 1e30, 50.0
    k = np.where(rng.random(rows) < 0.5, 0, rng.integers(1, 3000, rows))
    p = np.where(rng.random(rows) < 0.3, 1.0, rng.uniform(0.05, 0.999, rows))
    m = np.where(rng.random(rows) < 0.5, 0.0, rng.uniform(0.001, 0.3, rows))
    check_rows(logits, rng.random(rows), t, k, p, m)
    check_rows(logits, rng.random(rows), t, None, np.full(rows, 0.9), None)
    check_rows(logits, rng.random(rows), t, None, None, None)


def test_defaults_strides_and_whole_ranges():
    """No parameters at all; rows inside wider rows; parameters at their ends."""
    rng = np.random.default_rng(1)
    wide = dev(rng.standard_normal((6, 777)))
    check_rows(wide[:, 3:700], rng.random(6), None, None, None, None)
    logits = dev(rng.standard_normal((6, 777)))
    check_rows(logits, rng.random(6), np.ones(6), [0, -3, 777, 5000, 1, 776], [1.0, 2.0, 0.0, -1.0, 1e-9, 0.999999],
               [0.0, -1.0, 1.0, 5.0, 1e-12, 0.5])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [16, 5000, 70000])
def test_equal_logits_by_index(dtype, V):
    """Equal logits have equal weights: every count and token is known exactly."""
    rng = np.random.default_rng(V)
    on = rng.random((8, V)) < 0.4
    on[:, 3] = True
    logits = dev(np.where(on, 1.5, -np.inf), dtype)
    u = np.float32(rng.integers(0, 2 ** 24, 8) / 2 ** 24)
    k = [0, 1, 2, 5, 7, V // 2, V, 3]
    p = np.float32([1.0, 1.0, 0.5, 0.5, 0.25, 0.75, 0.125, 1.0])
    token, logprob, kept = (x.cpu().numpy() for x in ops().sample_logits(
        logits, dev(u), top_k=dev(k, torch.int32), top_p=dev(p)))
    for r in range(8):
        idx = np.flatnonzero(on[r])
        if k[r] > 0:
            idx = idx[:k[r]]
        if p[r] < 1:
            idx = idx[:math.ceil(float(p[r]) * len(idx))]
        assert kept[r] == len(idx)
        assert token[r] == idx[int(float(u[r]) * len(idx))]
        assert abs(logprob[r] + math.log(len(idx))) < 1e-5


def test_two_levels_across_the_cut():
    """Ties on both sides of top-k and top-p among two values."""
    V = 4096
    rng = np.random.default_rng(0)
    high = rng.permutation(V)[:100]
    x = np.zeros((4, V), np.float32)
    x[:, high] = 2.0
    high.sort()
    low = np.setdiff1d(np.arange(V), high)
    u = np.float32([0.0, 0.9999, 0.5, 0.25])
    token, _, kept = (a.cpu().numpy() for a in ops().sample_logits(
        dev(x), dev(u), temperature=dev([1.0, 1.0, 1.0, 2.0]), top_k=dev([150, 100, 30, 0], torch.int32),
        top_p=dev([1.0, 1.0, 0.5, 1.0])))
    for r, keep in enumerate((np.concatenate((high, low[:50])), high, high[:15], np.arange(V))):
        assert kept[r] == len(keep) and token[r] in keep
    assert token[0] == min(high[0], low[0]) and token[2] == high[7]


def test_masked_rows_and_odd_values():
    """-inf and NaN are never taken; +inf shares the whole weight; nothing left gives -1."""
    inf, nan = math.inf, math.nan
    x = np.full((8, 300), -inf, np.float32)
    x[0, 17] = -3e38                    # one finite logit
    x[2, [5, 9]] = inf                  # row 1: all masked
    x[2, 50:60] = 3.0
    x[3, :] = nan
    x[4, :] = nan
    x[4, 299] = 0.0
    x[5, 7], x[5, 8] = 3e38, -3e38      # a distance that overflows
    x[6, 100:200] = np.finfo(np.float32).min   # masks of the type's lowest value
    x[6, 150] = -1.0
    x[7, :] = np.finfo(np.float32).min
    u = np.float32([0.9, 0.5, 0.75, 0.1, 0.2, 0.99, 0.999, 0.5])
    for args in ({}, dict(top_k=dev([2] * 8, torch.int32)), dict(top_p=dev([0.9] * 8)), dict(min_p=dev([0.1] * 8)),
                 dict(temperature=dev([1e-30] * 8))):
        token, logprob, kept = (a.cpu().numpy() for a in ops().sample_logits(dev(x), dev(u), **args))
        assert token.tolist()[:7] == [17, -1, 9, -1, 299, 7, 150], args
        assert kept.tolist()[:7] == [1, 0, 2, 0, 1, 1, 1]
        assert np.isneginf(logprob[[1, 3]]).all() and abs(logprob[2] + math.log(2)) < 1e-6
    assert 0 <= token[7] < 300
    greedy, lp, kept = ops().sample_logits(dev(x), dev(u), temperature=dev([0.0] * 4 + [-1.0] * 4))
    assert greedy.tolist() == [17, -1, 5, -1, 299, 7, 150, 0] and kept.tolist() == [1, 0, 1, 0, 1, 1, 1, 1]
    assert lp.tolist() == [0.0, -inf, 0.0, -inf, 0.0, 0.0, 0.0, 0.0]


def test_small_negative_zero_and_uniform_ends():
    x = np.float32([[0.0, -0.0, 0.0, -0.0]])
    for u, want in ((0.0, 0), (0.25, 1), (0.4999, 1), (0.5, 2), (1.0, 3), (2.0, 3), (-1.0, 0), (math.nan, 0)):
        token, _, kept = ops().sample_logits(dev(x), dev([u]))
        assert token.item() == want and kept.item() == 4
    token, _, kept = ops().sample_logits(dev(x), dev([0.9]), top_k=dev([3], torch.int32))
    assert token.item() == 2 and kept.item() == 3


def test_frequencies():
    """The share of each token over a grid of u is its probability."""
    V, n = 50, 4096
    rng = np.random.default_rng(2)
    row = rng.standard_normal(V).astype(np.float32)
    logits = dev(np.tile(row, (n, 1)))
    u = (np.arange(n) + 0.5) / n
    token, _, _ = ops().sample_logits(logits, dev(u), temperature=dev([0.7] * n))
    want = np.exp(row.astype(np.float64) / np.float32(0.7))
    want /= want.sum()
    got = np.bincount(token.cpu().numpy(), minlength=V) / n
    assert np.abs(got - want).max() < 1.01 / n + 1e-6


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,V,ld", [(160, 262144, 262144), (149, 262143, 262151), (148, 260100, 260100),
                                       (3, 262144, 262144)])
def test_equal_weights_in_the_widest_rows(dtype, rows, V, ld):
    """Up to 2^18 tokens of the largest weight: equal logits, all +inf, a temperature that makes every exponential 1,
    and equal ones among masked ones.  Every count and token is known exactly."""
    rng = np.random.default_rng(V + rows)
    x = np.full((rows, ld), 1.5, np.float32)
    kind = np.arange(rows) % 4
    x[kind == 1] = np.inf
    spread = dev(2 * rng.standard_normal(ld).astype(np.float32), dtype)
    x[kind == 2] = spread.float().cpu().numpy()
    half = rng.random(ld) < 0.5
    half[0] = True
    x[kind == 3] = np.where(half, 1.5, -np.inf)
    logits = dev(x, dtype)[:, :V]
    t = np.where(kind == 2, 1e30, 1.0)
    p = np.float32(rng.integers(1, 2 ** 16, rows) / 2 ** 16)
    p[rows // 2] = 1.0
    p[:3] = np.float32([0.9, 0.5, 0.999])
    u = np.float32(rng.integers(0, 2 ** 24, rows) / 2 ** 24)
    token, logprob, kept = (a.cpu().numpy() for a in ops().sample_logits(logits, dev(u), temperature=dev(t),
                                                                         top_p=dev(p)))
    falling = np.lexsort((np.arange(V), -spread.float().cpu().numpy()[:V].astype(np.float64)))
    for r in range(rows):
        idx = falling if kind[r] == 2 else np.flatnonzero(half[:V]) if kind[r] == 3 else np.arange(V)
        if p[r] < 1:
            idx = np.sort(idx[:math.ceil(math.floor(float(p[r]) * 2 ** 32) * len(idx) / 2 ** 32)])
        assert kept[r] == len(idx), r
        at = math.floor(float(u[r]) * 2 ** 32) * len(idx) // 2 ** 32
        assert token[r] == np.sort(idx)[at], r
        assert abs(logprob[r] + math.log(len(idx))) < 1e-5


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_widest_rows_with_every_truncation(dtype):
    """The largest vocabulary, one CTA per row, on ordinary logits."""
    rng = np.random.default_rng(18)
    rows, V = 148, 262144
    logits = dev(2 * rng.standard_normal((rows, V)), dtype)
    t = rng.uniform(0.3, 2.0, rows)
    t[5], t[6] = 0.0, 50.0
    k = np.where(rng.random(rows) < 0.5, 0, rng.integers(1, 3000, rows))
    p = np.where(rng.random(rows) < 0.3, 1.0, rng.uniform(0.05, 0.999, rows))
    m = np.where(rng.random(rows) < 0.5, 0.0, rng.uniform(0.001, 0.3, rows))
    check_rows(logits, rng.random(rows), t, k, p, m)
