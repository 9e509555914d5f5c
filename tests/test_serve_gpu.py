"""Block tables and slot maps from request lengths (tkb_kv_pages) and low-rank
adapters of many requests (tkb_lora_plan, tkb_lora_add) against the oracle.

The tables are whole numbers: equal.  Adapters: out is rounded to its type
once, by up to half a step, eps / 2 of the value (bf16 2^-8, f16 2^-11).
Before that, sums of K and R products in fp32: the rounding of each of K
products and sums of mean size 1/sqrt(K) leaves 2^-24 sqrt(K) in the root mean
square, below 1e-5 of the whole for K up to 2^14; in 16-bit types the product
x A may be split into two 16-bit parts, off by 2^-17 of it (bf16), 2^-22 (f16).
"""
import numpy as np
import pytest

from oracle import serve_oracle as ref
from tests.conftest import rel_l2
from tests.test_paged_gpu import DTYPES, device_error, num, ops

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

LORA = {torch.float32: 1e-5, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def on_gpu(a, dtype=torch.int32):
    return torch.tensor(np.asarray(a), dtype=dtype, device="cuda")


class Pool:
    """Tables of B sequences over shuffled pages, its state on both sides."""

    def __init__(self, B, max_pages, page, lens, free, seed=0):
        rng = np.random.default_rng(seed)
        self.page = page
        self.held = np.array([-(-n // page) for n in lens])
        used = int(self.held.sum())
        self.n_pages = used + free + 2
        order = rng.permutation(self.n_pages)
        self.table = np.full((B, max_pages), -1)
        at = 0
        for b, n in enumerate(self.held):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.stack = order[used:used + free].tolist()
        self.t, self.h = on_gpu(self.table), on_gpu(self.held)
        self.f = torch.full((self.n_pages,), -5, dtype=torch.int32, device="cuda")
        self.f[:free] = on_gpu(self.stack) if free else 0
        self.n = on_gpu([free])

    def step(self, lens, row_start=None, rows=None):
        granted, slots = ops().kv_pages(self.t, self.h, on_gpu(lens), self.f, self.n, self.page,
                                        row_start=None if row_start is None else on_gpu(row_start), rows=rows)
        self.table, self.held, self.stack, want = ref.pages(self.table, self.held, lens, self.stack, self.page)
        assert np.array_equal(self.t.cpu().numpy(), self.table) and np.array_equal(self.h.cpu().numpy(), self.held)
        assert int(self.n) == len(self.stack) and self.f[:len(self.stack)].tolist() == self.stack
        assert granted.tolist() == want
        if rows is not None:
            start = np.arange(len(lens) + 1) if row_start is None else row_start
            assert slots.tolist() == ref.slots(self.table, self.held, lens, self.page, start, rows).tolist()
        return granted


@pytest.mark.parametrize("B", [1, 7, 64, 129, 1000, 4096])
@pytest.mark.parametrize("page", [16, 48, 1])
def test_pages(B, page):
    """A batch that grows, turns over, and meets an empty stack."""
    rng = np.random.default_rng(B + page)
    most = 40
    lens = rng.integers(0, most * page + 1, B)
    pool = Pool(B, most, page, lens, free=2 * B + 3)
    for step in range(6):
        new = np.minimum(most * page, lens + rng.integers(0, 2 * page + 2, B))
        if step % 2:
            new[rng.random(B) < 0.2] = 0
        rows = np.where(new > lens, new - lens, 0)
        start = np.concatenate(([0], np.cumsum(rows)))
        granted = pool.step(new, start, max(1, int(start[-1])))
        lens = np.where(granted.cpu().numpy() > 0, new, np.minimum(new, pool.held * page))
    assert device_error() == 0


def test_pages_of_single_tokens():
    pool = Pool(5, 4, 16, [16, 3, 0, 64, 31], free=2)
    pool.step([17, 4, 1, 64, 32], rows=5)
    pool.step([33, 5, 2, 64, 33], rows=5)    # the stack is empty: the first that needs a page goes without
    pool.step([0, 0, 0, 0, 0])
    pool.step([64, 64, 64, 1, 1])
    assert device_error() == 0


def test_pages_past_the_table():
    """A length past the table takes all of it and is not granted."""
    pool = Pool(2, 3, 16, [16, 16], free=8)
    granted = pool.step([49, 48])
    assert granted.tolist() == [0, 1]


def test_bad_counts_are_cut():
    """Counts outside their range: bit 2, and no access outside the arrays."""
    table = on_gpu([[3, 4], [5, 6]])
    guard = torch.full((12,), 77, dtype=torch.int32, device="cuda")
    free = guard[4:11]
    free.copy_(torch.arange(7))
    for held, lens, n_free in (([9, 1], [32, 16], [0]), ([-4, 1], [0, 16], [0]), ([1, 1], [-1, 16], [0]),
                               ([2, 2], [0, 0], [7]), ([2, 2], [0, 0], [99]), ([0, 0], [32, 32], [-3])):
        t = table.clone()
        ops().kv_pages(t, on_gpu(held), on_gpu(lens), free, on_gpu(n_free), 16)
        assert device_error() == 4, (held, lens, n_free)
        assert (guard[:4] == 77).all() and guard[11] == 77


@pytest.mark.parametrize("B", [1, 48, 49, 128, 129, 256, 257])
def test_pages_whatever_the_launch(B):
    """`tokens` chooses a launch; the tables are the same for every number, beside the oracle's."""
    rng, most, page = np.random.default_rng(B), 30, 16
    lens = rng.integers(0, most * page + 1, B)
    pool = Pool(B, most, page, lens, free=4 * B)
    for tokens in (0, 1024, 1025, 4096 * page + page, 1 << 40):
        new = np.where(rng.random(B) < 0.2, 0, np.minimum(most * page, lens + rng.integers(0, 3 * page, B)))
        granted, slots = ops().kv_pages(pool.t, pool.h, on_gpu(new), pool.f, pool.n, page, tokens=tokens)
        pool.table, pool.held, pool.stack, want = ref.pages(pool.table, pool.held, new, pool.stack, page)
        assert slots is None and granted.tolist() == want
        assert np.array_equal(pool.t.cpu().numpy(), pool.table) and np.array_equal(pool.h.cpu().numpy(), pool.held)
        assert int(pool.n) == len(pool.stack) and pool.f[:len(pool.stack)].tolist() == pool.stack
        lens = np.where(np.array(want) > 0, new, np.minimum(new, pool.held * page))
    assert device_error() == 0


@pytest.mark.parametrize("B", [3, 300])
@pytest.mark.parametrize("bad", [-1, 16, 1 << 30])
def test_numbers_that_name_no_page(B, bad):
    """A held entry that names no page: bit 2 when a row lies in it, when it is given back, and when another sequence gets
    it, which is then not granted; the other sequences are."""
    t = torch.full((B, 3), -1, dtype=torch.int32, device="cuda")
    t[0, :2], t[1, 0] = on_gpu([4, bad]), 7
    held, free, n_free = on_gpu([2, 1] + [0] * (B - 2)), torch.full((16,), -5, dtype=torch.int32, device="cuda"), on_gpu([0])

    def step(lens, rows=None):
        start = np.concatenate(([0], np.cumsum(rows))) if rows else None
        granted, slots = ops().kv_pages(t, held, on_gpu(lens + [0] * (B - len(lens))), free, n_free, 16,
                                        row_start=None if rows is None else on_gpu(list(start) + [start[-1]] * (B - len(rows))),
                                        rows=None if rows is None else int(start[-1]))
        return granted[:3].tolist(), None if slots is None else slots.tolist()

    assert step([32, 16]) == ([1, 1, 1], None) and device_error() == 0     # nothing moves
    assert step([18, 16], rows=[3, 1]) == ([1, 1, 1], [4 * 16 + 15, -1, -1, 7 * 16 + 15]) and device_error() == 4
    assert step([16, 16])[0] == [1, 1, 1] and device_error() == 4          # given back
    assert int(n_free) == 1 and int(free[0]) == bad
    assert step([16, 16, 5], rows=[0, 1, 5]) == ([1, 1, 0], [7 * 16 + 15] + [-1] * 5) and device_error() == 4
    assert held[:3].tolist() == [1, 1, 1] and int(n_free) == 0
    assert step([16, 16])[0] == [1, 1, 1] and device_error() == 4          # and back again
    free[0] = 9
    assert step([16, 16, 5])[0] == [1, 1, 1] and device_error() == 0


def test_pages_captured():
    """A captured call follows the lengths; the pages it takes are those of plain calls."""
    B, most, page = 9, 8, 16
    pool = Pool(B, most, page, [5] * B, free=40)
    lens = on_gpu([5] * B)
    granted = None
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        granted, _ = ops().kv_pages(pool.t, pool.h, lens, pool.f, pool.n, page)
    n = np.full(B, 5)
    for _ in range(5):
        n = np.minimum(n + np.arange(B) * 5, most * page)
        lens.copy_(on_gpu(n))
        graph.replay()
        pool.table, pool.held, pool.stack, want = ref.pages(pool.table, pool.held, n, pool.stack, page)
        assert np.array_equal(pool.t.cpu().numpy(), pool.table) and granted.tolist() == want
        assert int(pool.n) == len(pool.stack)


def lora_case(dtype, adapter, rows, n, K, N, R, seed=0, first=0, behind=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    T = first + sum(rows) + behind

    def randn(*shape, scale=1.0):
        return (scale * torch.randn(*shape, generator=g, device="cuda")).to(dtype)

    x, y = randn(T, K), randn(T, N)
    a, b = randn(n, K, R, scale=K ** -0.5), randn(n, R, N, scale=R ** -0.5)
    scale = 0.5 + torch.rand(n, generator=g, device="cuda")
    start = np.concatenate(([0], np.cumsum(rows))) + first
    return x, y, a, b, scale, start


def rows_close(got, want, dtype):
    assert rel_l2(got, want) < LORA[dtype]
    rms = np.sqrt((want ** 2).mean(1)) + 1e-30
    assert (np.sqrt(((got - want) ** 2).mean(1)) / rms < 3 * LORA[dtype]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("adapter,rows,n,K,N,R", [
    ([0], [1], 1, 64, 64, 8),
    ([2, -1, 0, 2, 1], [1, 1, 1, 1, 1], 3, 256, 688, 16),
    ([2, -1, 0, 2, 2, 1], [17, 5, 0, 64, 1, 130], 3, 688, 256, 8),     # no rows, edges of tiles
    ([1, 1, 1], [63, 65, 300], 2, 1040, 72, 64),                       # one adapter over several sequences
    ([5, 3], [33, 20], 6, 136, 1096, 128),
    ([-1, -1], [4, 4], 2, 64, 64, 24),                                 # nobody has one
    ([0], [1000], 1, 2048, 8, 16),
    ([0, 1], [40, 41], 2, 8, 2048, 40),
])
def test_lora(dtype, adapter, rows, n, K, N, R):
    x, y, a, b, scale, start = lora_case(dtype, adapter, rows, n, K, N, R)
    want = ref.lora(num(x), num(a), num(b), num(y), adapter, start, num(scale))
    plan = ops().lora_plan(on_gpu(adapter), n, x.shape[0], row_start=on_gpu(start))
    out = torch.full_like(y, 7.0)
    ops().lora_add(plan, x, a, b, y, scale=scale, out=out)
    rows_close(num(out), want, dtype)
    ops().lora_add(plan, x, a, b, y, scale=scale)  # in place
    assert torch.equal(y, out)
    assert device_error() == 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_lora_single_tokens(dtype):
    """One row a sequence, without row_start; adapters met once, often and never."""
    rng = np.random.default_rng(3)
    adapter = rng.integers(-1, 40, 300)
    adapter[adapter > 20] = 7
    x, y, a, b, scale, start = lora_case(dtype, adapter, [1] * 300, 40, 512, 264, 16)
    want = ref.lora(num(x), num(a), num(b), num(y), adapter, start, None)
    plan = ops().lora_plan(on_gpu(adapter), 40, 300)
    rows_close(num(ops().lora_add(plan, x, a, b, y)), want, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_lora_strides_and_rows_of_no_sequence(dtype):
    """Columns of wider rows (one projection of a fused one), rows before the first and behind the last sequence."""
    adapter, rows, K, N, R = [1, 0, -1], [20, 70, 9], 128, 192, 16
    x, y, a, b, scale, start = lora_case(dtype, adapter, rows, 2, K, N, R, first=3, behind=6)
    wide_x = torch.zeros(x.shape[0], K + 64, dtype=dtype, device="cuda")
    wide_x[:, 32:32 + K] = x
    wide_y = torch.full((y.shape[0], N + 128), 7.0, dtype=dtype, device="cuda")
    wide_y[:, 64:64 + N] = y
    plan = ops().lora_plan(on_gpu(adapter), 2, x.shape[0], row_start=on_gpu(start))
    out = torch.full((y.shape[0], N + 64), 5.0, dtype=dtype, device="cuda")
    ops().lora_add(plan, wide_x[:, 32:32 + K], a, b, wide_y[:, 64:64 + N], scale=scale, out=out[:, :N])
    want = ref.lora(num(x), num(a), num(b), num(y), adapter, start, num(scale))[3:-6]
    rows_close(num(out)[3:-6, :N], want, dtype)
    assert (out[:3] == 5).all() and (out[-6:] == 5).all() and (out[:, N:] == 5).all()
    assert torch.equal(out[93:-6, :N], y[93:-6])   # adapter -1
    ops().lora_add(plan, wide_x[:, 32:32 + K], a, b, wide_y[:, 64:64 + N], scale=scale)
    assert torch.equal(wide_y[3:-6, 64:64 + N], out[3:-6, :N])
    assert torch.equal(wide_y[:3, 64:64 + N], y[:3]) and torch.equal(wide_y[-6:, 64:64 + N], y[-6:])
    assert (wide_y[:, :64] == 7).all() and (wide_y[:, 64 + N:] == 7).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_lora_nan_stays_in_its_rows(dtype):
    adapter, rows = [0, 1, 0], [20, 1, 30]
    x, y, a, b, scale, start = lora_case(dtype, adapter, rows, 2, 256, 256, 16)
    plan = ops().lora_plan(on_gpu(adapter), 2, 51, row_start=on_gpu(start))
    clean = ops().lora_add(plan, x, a, b, y, out=torch.empty_like(y))
    x[7, 100], x[33, 5] = float("nan"), float("inf")
    out = ops().lora_add(plan, x, a, b, y, out=torch.empty_like(y))
    bad = torch.zeros(51, dtype=torch.bool, device="cuda")
    bad[7] = bad[33] = True
    assert torch.equal(out[~bad], clean[~bad]) and not out[bad].isfinite().any()
    a[1, 3, 2] = float("nan")
    out = ops().lora_add(plan, x, a, b, y, out=torch.empty_like(y))
    assert out[20].isnan().all() and out[:7].isfinite().all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R", [8, 16, 24, 64, 72])
@pytest.mark.parametrize("rows", [5, 200])
def test_lora_infinities_keep_their_sign(dtype, R, rows):
    """An infinite x beside adapters of one sign: rows of infinities, as in the formula; a scale below 0 turns them; a rank
    that is padded does not make them NaN, and neither does another large value of the row."""
    K, N = 128, 72
    x, y, a, b, _, start = lora_case(dtype, [0, 1], [rows, rows], 2, K, N, R)
    a, b, scale = a.abs() + 0.01, b.abs() + 0.01, on_gpu([1.0, -0.5], torch.float32)
    plan = ops().lora_plan(on_gpu([0, 1]), 2, 2 * rows, row_start=on_gpu(start))
    clean = ops().lora_add(plan, x, a, b, y, scale=scale, out=torch.empty_like(y))
    want = torch.full_like(y, float("inf"))
    x[1, 7], x[2, K - 1], x[rows + 3, 0] = float("inf"), -float("inf"), float("inf")
    x[2, 3] = 60000.0 if dtype == torch.float16 else 1e30
    want[2], want[rows + 3] = -float("inf"), -float("inf")
    out = ops().lora_add(plan, x, a, b, y, scale=scale, out=torch.empty_like(y))
    lost = torch.zeros(2 * rows, dtype=torch.bool, device="cuda")
    lost[[1, 2, rows + 3]] = True
    assert torch.equal(out[lost], want[lost]) and torch.equal(out[~lost], clean[~lost])


def test_lora_products_above_the_largest_bf16():
    """x A between the largest bf16 and the largest fp32, times a small B: finite."""
    K, N, R = 64, 64, 16
    x, y, a, b, _, start = lora_case(torch.bfloat16, [0], [3], 1, K, N, R)
    x.zero_()
    x[1, 0], x[1, 1] = torch.finfo(torch.bfloat16).max, 1e36
    a.fill_(1.0)
    b.fill_(2.0 ** -20)
    plan = ops().lora_plan(on_gpu([0]), 1, 3, row_start=on_gpu(start))
    out = ops().lora_add(plan, x, a, b, y, out=torch.empty_like(y))
    rows_close(num(out), ref.lora(num(x), num(a), num(b), num(y), [0], start, None), torch.bfloat16)


def test_lora_bad_adapters_and_row_starts():
    x, y, a, b, scale, _ = lora_case(torch.bfloat16, [0, 1], [4, 6], 2, 64, 64, 8)
    for adapter in ([2, 1], [-2, 1], [1 << 30, 1]):
        plan = ops().lora_plan(on_gpu(adapter), 2, 10, row_start=on_gpu([0, 4, 10]))
        out = ops().lora_add(plan, x, a, b, y, out=torch.empty_like(y))
        assert device_error() == 4 and torch.equal(out[:4], y[:4]) and not torch.equal(out[4:], y[4:])
    for start in ([0, 4, 99], [0, 8, 6], [-3, 4, 10], [0, 10, 0, 10], [0, 7, 2, 9]):
        ids = [0, 1, 1][:len(start) - 1]
        plan = ops().lora_plan(on_gpu(ids), 2, 10, row_start=on_gpu(start))
        ops().lora_add(plan, x, a, b, y, out=torch.empty_like(y))
        assert device_error() == 4, start


def test_lora_captured_and_again():
    """A captured plan and addition follow the adapters and row starts; equal inputs give equal bits."""
    x, y, a, b, scale, _ = lora_case(torch.bfloat16, [0] * 4, [30] * 4, 5, 512, 512, 16)
    adapter, start = on_gpu([0, 1, 2, 3]), on_gpu([0, 30, 60, 90, 120])
    out, ws = torch.empty_like(y), ops().lora_workspace(120, 16)
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=stream):
        plan = ops().lora_plan(adapter, 5, 120, row_start=start)
        ops().lora_add(plan, x, a, b, y, scale=scale, out=out, workspace=ws)
    for ids, begins in (([0, 1, 2, 3], [0, 30, 60, 90, 120]), ([4, -1, 4, 0], [0, 1, 2, 100, 120]),
                        ([3, 3, 3, 3], [0, 0, 0, 0, 120])):
        adapter.copy_(on_gpu(ids))
        start.copy_(on_gpu(begins))
        graph.replay()
        want = ref.lora(num(x), num(a), num(b), num(y), ids, begins, num(scale))
        rows_close(num(out), want, torch.bfloat16)
        first = out.clone()
        ws.fill_(255)
        graph.replay()
        assert torch.equal(first, out)


def test_lora_many_sequences():
    """4096 sequences of zero to three rows over 1000 adapters."""
    rng = np.random.default_rng(4)
    rows = rng.integers(0, 4, 4096)
    adapter = rng.integers(-1, 1000, 4096)
    x, y, a, b, scale, start = lora_case(torch.float16, adapter, rows, 1000, 128, 128, 8)
    plan = ops().lora_plan(on_gpu(adapter), 1000, x.shape[0], row_start=on_gpu(start))
    want = ref.lora(num(x), num(a), num(b), num(y), adapter, start, num(scale))
    rows_close(num(ops().lora_add(plan, x, a, b, y, scale=scale)), want, torch.float16)
