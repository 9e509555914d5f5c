"""Attention of a chunk of new tokens over the paged cache
(tkb_paged_attn_chunk) against the float64 oracle.

Tolerances, in relative L2, as for the attention of one token: storing a value
in a type of m mantissa bits is off by up to 2^-(m+1), and the probabilities
may be rounded to the same type before the product with V, another such error
in every term: 2^-7 for bf16, 2^-10 for f16.  fp32: products of up to 128 unit
values and sums of some thousand terms are off by some 1e-6, exponentials of
the scores by as much: 1e-5.  Log-sum-exps are fp32 in every type: 2e-5 of
their size.
"""
import numpy as np
import pytest

from oracle import serve_oracle as ref
from tests.conftest import rel_l2
from tests.test_paged_gpu import ATTN, DTYPES, Cache, device_error, num, ops

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def starts(rows, first=0):
    return np.concatenate(([0], np.cumsum(rows))).astype(np.int64) + first


def on_gpu(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


def want(c, q, Hq, lens, row_start, scale=None):
    """The oracle's out and lse for every row that belongs to a sequence, and which rows those are."""
    k, v, table, qn = num(c.k), num(c.v), c.table.cpu().numpy(), num(q)
    out, lse = np.zeros_like(qn), np.full((qn.shape[0], Hq), -np.inf)
    mine = np.zeros(qn.shape[0], bool)
    for b, n in enumerate(lens):
        at = slice(row_start[b], row_start[b + 1])
        m = row_start[b + 1] - row_start[b]
        o, l = ref.chunk(k, v, table[b], n, qn[at].reshape(m, Hq, c.D), c.D ** -0.5 if scale is None else scale)
        out[at], lse[at], mine[at] = o.reshape(m, Hq * c.D), l, True
    return out, lse, mine


def check(c, q, Hq, lens, row_start, out, lse, dtype, scale=None):
    want_o, want_l, mine = want(c, q, Hq, lens, row_start, scale)
    got_o, got_l = num(out)[mine], num(lse)[mine]
    want_o, want_l = want_o[mine], want_l[mine]
    assert np.isfinite(got_o).all()
    assert np.array_equal(np.isneginf(got_l), np.isneginf(want_l))
    fin = np.isfinite(want_l)
    assert np.abs(got_l[fin] - want_l[fin]).max(initial=0) < 2e-5 * max(1.0, np.abs(want_l[fin]).max(initial=0))
    assert rel_l2(got_o, want_o) < ATTN[dtype]
    # row by row, with room for the largest of many: a tile that went wrong in a long call does not hide
    scale_of = np.sqrt((want_o ** 2).mean(1)) + 1e-30
    assert (np.sqrt(((got_o - want_o) ** 2).mean(1)) / scale_of < 3 * ATTN[dtype]).all()
    empty = ~fin.any(1)
    assert (got_o[empty] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hkv,G,page,lens,rows", [
    (2, 1, 16, [5], [5]),                                       # a short prompt
    (1, 1, 16, [1], [1]),                                       # one token, nothing before it
    (2, 4, 16, [1, 0, 15, 16, 17, 128, 129, 300], [1, 0, 15, 1, 3, 128, 2, 40]),  # edges of pages and tiles
    (1, 8, 48, [700, 3, 0, 47, 49], [33, 3, 0, 1, 17]),         # pages that are no power of two
    (4, 7, 64, [65, 640], [65, 19]),                            # odd group: tiles of 18 tokens
    (2, 16, 32, [33, 257, 260], [9, 8, 17]),                    # eight tokens a tile, one more than that
    (1, 20, 128, [130, 1], [130, 1]),
    (1, 130, 16, [40, 9], [7, 9]),                              # more heads than a tile holds
    (3, 2, 1024, [1500, 31], [200, 31]),                        # large pages
    (1, 2, 16, [3000], [2]),                                    # few rows over many slots: split
    (1, 2, 16, [1000], [1000]),                                 # a whole prompt
    (2, 1, 64, [513, 900], [257, 129]),                         # one row more than a tile, than two tiles
    (1, 2, 16, [0], [0]),                                       # nothing at all
])
def test_chunk(dtype, D, Hkv, G, page, lens, rows):
    c = Cache(dtype, lens, Hkv, D, page).fill(lens)
    Hq, start = Hkv * G, starts(rows)
    q = c.randn(max(1, sum(rows)), Hq * D, dtype=dtype)
    out, lse = ops().paged_attn_chunk(c.handle, q, Hq, row_start=on_gpu(start))
    check(c, q, Hq, lens, start, out, lse, dtype)
    assert device_error() == 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_one_row_each_equals_the_attention_of_one_token(dtype):
    lens = [1, 0, 300, 17, 2000]
    c = Cache(dtype, lens, 2, 64, 16).fill(lens)
    q = c.randn(5, 8 * 64, dtype=dtype)
    out, lse = ops().paged_attn_chunk(c.handle, q, 8)
    # row 1: its token is not in the cache; bit 2 says so
    assert device_error() == 4
    check(c, q, 8, lens, starts([1] * 5), out, lse, dtype)
    single, single_lse = ops().paged_attn_decode(c.handle, q, 8)
    assert rel_l2(num(out), num(single)) < ATTN[dtype]
    ok = np.isfinite(num(single_lse))
    assert np.abs(num(lse)[ok] - num(single_lse)[ok]).max() < 2e-4


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_scale_shared_pages_and_rows_of_no_sequence(dtype):
    """A page stride above the page, rows inside wider rows, sequences that share their first pages, a scale of its own,
    rows before the first and behind the last sequence."""
    lens, rows, Hkv, G, D, page = [200, 100, 64], [20, 4, 30], 2, 3, 64, 32
    c = Cache(dtype, lens, Hkv, D, page, page_gap=64).fill(lens)
    c.table[1, :3] = c.table[0, :3]
    Hq, start = Hkv * G, starts(rows, 3)
    total = 3 + sum(rows) + 5
    wide = c.randn(total, Hq * D + 128, dtype=dtype)
    q = wide[:, 64:64 + Hq * D]
    room = torch.full((total, Hq * D + 64), 7.0, dtype=dtype, device="cuda")
    lse = torch.full((total, Hq), 7.0, device="cuda")
    ops().paged_attn_chunk(c.handle, q, Hq, row_start=on_gpu(start), scale=0.3, out=room[:, :Hq * D], lse=lse)
    check(c, q, Hq, lens, start, room[:, :Hq * D], lse, dtype, scale=0.3)
    assert (room[:, Hq * D:] == 7).all()
    for t in (room, lse):
        assert (t[:3] == 7).all() and (t[-5:] == 7).all()
    assert device_error() == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
def test_large_scores(dtype, D):
    """Scores in the hundreds, rising and falling along the slots: one key takes nearly all the weight, wherever it lies;
    the running maximum jumps in the middle of a tile, or never after the first."""
    lens, rows = [700, 700, 700], [40, 40, 40]
    c = Cache(dtype, lens, 2, D, 16).fill(lens)
    q = c.randn(120, 4 * D, dtype=dtype, scale=30.0 * (64 / D) ** 0.5)
    for b, j in enumerate((0, 350, 655)):  # a key along a query of each kv head
        for h in range(2):
            c.k[c.table[b, j // 16].long(), h, j % 16] = q[b * 40 + 7, h * 2 * D:h * 2 * D + D] * 0.2
    out, lse = ops().paged_attn_chunk(c.handle, q, 4, row_start=on_gpu(starts(rows)))
    want_o, want_l, _ = want(c, q, 4, lens, starts(rows))
    # scores up to 700 carry fp32 errors of 700 * 2^-22 and less: far below the storage bound
    assert rel_l2(num(out), want_o) < max(ATTN[dtype], 1e-3)
    assert np.abs(num(lse) - want_l).max() < 1e-3


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_small_weights_beside_a_large_one(dtype):
    """One key of weight 1 and 12000 of weight 2^-26, together 2^-12.4 of it: less than f16 can hold one by one, but not less
    than its step.  V is 1 for the small ones and 0 for the large one, so the output is their sum alone."""
    n, D = 12001, 64
    c = Cache(dtype, [n], 1, D, 64).fill([n])
    t, j = c.table[0].long(), torch.arange(n, device="cuda")
    c.k[t[j // 64], 0, j % 64] = 0.0
    c.v[t[j // 64], 0, j % 64] = 1.0
    c.k[t[5 // 64], 0, 5, 0] = 144.25   # scaled: 18.03, e^-18.03 = 2^-26.01
    c.v[t[5 // 64], 0, 5] = 0.0
    q = torch.zeros(3, D, dtype=dtype, device="cuda")
    q[:, 0] = 1.0
    out, _ = ops().paged_attn_chunk(c.handle, q, 1, row_start=on_gpu([0, 3]))
    big = float(c.k[t[0], 0, 5, 0].double()) / 8
    small = np.arange(n - 3, n) * np.exp(-big)
    assert rel_l2(num(out), np.repeat((small / (1 + small))[:, None], D, 1)) < 2 * ATTN[dtype]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_values_out_of_sight_do_not_matter(dtype, D, bad):
    """NaN and infinities in q, k and v: the rows that see them take them, the rows of the same tile before them do not."""
    lens, rows = [300, 140], [90, 140]
    Hq, start = 4, starts([90, 140])
    clean = Cache(dtype, lens, 2, D, 16).fill(lens)
    q = clean.randn(230, Hq * D, dtype=dtype)
    first, first_lse = ops().paged_attn_chunk(clean.handle, q, Hq, row_start=on_gpu(start))

    def spoil(pool, b, h, j, d):
        pool[clean.table[b, j // 16].long(), h, j % 16, d] = bad

    spoil(clean.v, 0, 0, 250, 3)          # token 250 = row 40 of 90: columns 3 of kv head 0
    spoil(clean.v, 1, 1, 130, D - 1)
    spoil(clean.k, 1, 0, 100, 5)
    q[200, 2 * D + 1] = bad               # row 110 of the second sequence, head 2
    out, lse = ops().paged_attn_chunk(clean.handle, q, Hq, row_start=on_gpu(start))
    got, was = num(out).reshape(230, Hq, D), num(first).reshape(230, Hq, D)
    lost = np.zeros_like(got, dtype=bool)
    lost[40:90, :2, 3] = True             # query heads 0 and 1 read kv head 0
    lost[90 + 130:, 2:, D - 1] = True
    assert not np.isfinite(got[lost]).any()
    if bad == bad:  # an infinite value keeps its sign, also beside probabilities far below 1
        assert (got[40:90, :2, 3] == bad).mean() > 0.9
    lost[90 + 100:, :2, :] = True         # these scores are NaN or infinite (of either sign)
    lost[200, 2, :] = True
    if bad != bad:
        assert np.isnan(got[90 + 100:, :2]).all() and np.isnan(got[200, 2]).all()
        assert np.isnan(num(lse)[90 + 100:, :2]).all() and np.isnan(num(lse)[200, 2])
    assert np.isfinite(got[~lost]).all()
    # rows that see none of it: as before, to the order of the sums
    assert rel_l2(got[~lost], was[~lost]) < ATTN[dtype]
    seen = np.ones((230, Hq), bool)
    seen[90 + 100:, :2] = False
    seen[200, 2] = False
    assert np.abs(num(lse)[seen] - num(first_lse)[seen]).max() < 2e-4


@pytest.mark.parametrize("dtype", DTYPES)
def test_keys_of_minus_infinity_score(dtype):
    """Keys whose scores are -inf take no weight, a row that sees only such keys is empty, and scores far below zero
    after them count in full."""
    lens, rows = [400], [200]
    c = Cache(dtype, lens, 1, 64, 16).fill(lens)
    q = torch.zeros(200, 64, dtype=dtype, device="cuda")
    q[:, 0] = 1.0
    q[:, 1] = 30.0
    t = c.table[0].long()
    flat = torch.arange(400, device="cuda")
    c.k[t[flat // 16], 0, flat % 16] = 0.0
    c.k[t[flat // 16], 0, flat % 16, 1] = -50.0               # scores of -187 in units of the exponent
    c.k[t[flat[:260] // 16], 0, flat[:260] % 16, 0] = -float("inf")
    out, lse = ops().paged_attn_chunk(c.handle, q, 1, row_start=on_gpu([0, 200]))
    got = num(out)
    v = num(c.v)
    seen = np.array([v[int(t[j // 16]), 0, j % 16] for j in range(400)])
    assert (got[:60] == 0).all() and np.isneginf(num(lse)[:60]).all()    # rows 200 .. 259 see none
    mean = np.array([seen[260:201 + i].mean(0) for i in range(60, 200)])
    assert rel_l2(got[60:], mean) < ATTN[dtype]
    wanted = -50 * 30 / 8 + np.log(np.arange(1, 141))
    assert np.abs(num(lse)[60:, 0] - wanted).max() < 2e-5 * np.abs(wanted).max()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
def test_bad_pages_lengths_and_row_starts(dtype, D):
    """Table entries that name no page do not count; lengths past the table and rows past a length see what there is;
    each sets bit 2, and nothing else changes."""
    lens, rows = [300, 290, 40], [50, 3, 40]
    c = Cache(dtype, lens, 2, D, 16, spare=1).fill(lens)
    c.table[0, 3], c.table[0, 17], c.table[1, 0] = -1, c.k.shape[0], 1 << 30
    q, start = c.randn(93, 6 * D, dtype=dtype), starts(rows)
    out, lse = ops().paged_attn_chunk(c.handle, q, 6, row_start=on_gpu(start))
    assert device_error() == 4
    check(c, q, 6, lens, start, out, lse, dtype)
    # a length past the table: its rows stand past the table's end and see all of it
    c = Cache(dtype, [64, 20], 2, D, 16).fill([64, 20])
    c.lens.copy_(on_gpu([70, 20]))
    q = c.randn(25, 6 * D, dtype=dtype)
    out, lse = ops().paged_attn_chunk(c.handle, q, 6, row_start=on_gpu([0, 3, 25]))
    assert device_error() == 4
    k, v, table = num(c.k), num(c.v), c.table.cpu().numpy()
    for r in range(3):
        o, l = ref.chunk(k, v, table[0], 64, num(q)[r].reshape(1, 6, D), D ** -0.5)
        assert rel_l2(num(out)[r], o.ravel()) < ATTN[dtype]
    # 22 rows of a sequence of 20 tokens: the first two see nothing
    assert (num(out)[3:5] == 0).all() and np.isneginf(num(lse)[3:5]).all()
    o, l = ref.chunk(k, v, table[1], 20, num(q)[5:25].reshape(20, 6, D), D ** -0.5)
    assert rel_l2(num(out)[5:25], o.reshape(20, -1)) < ATTN[dtype]
    # rows past the last, and a start that descends
    for bad in ([0, 3, 99], [0, 30, 25], [-5, 3, 25]):
        ops().paged_attn_chunk(c.handle, q, 6, row_start=on_gpu(bad))
        assert device_error() == 4
    c.lens.copy_(on_gpu([-3, 20]))
    out, lse = ops().paged_attn_chunk(c.handle, q, 6, row_start=on_gpu([0, 3, 23]))
    assert device_error() == 4 and (num(out)[:3] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_pieces_give_what_the_whole_gives(dtype):
    """A prompt of 500 tokens in pieces of 1, 128, 200 and 171: each row as in one call."""
    n, Hq, D = 500, 8, 128
    c = Cache(dtype, [n], 2, D, 32).fill([n])
    q = c.randn(n, Hq * D, dtype=dtype)
    whole, whole_lse = ops().paged_attn_chunk(c.handle, q, Hq, row_start=on_gpu([0, n]))
    done = 0
    for m in (1, 128, 200, 171):
        c.lens.fill_(done + m)
        out, lse = ops().paged_attn_chunk(c.handle, q[done:done + m], Hq, row_start=on_gpu([0, m]))
        assert rel_l2(num(out), num(whole)[done:done + m]) < ATTN[dtype]
        assert np.abs(num(lse) - num(whole_lse)[done:done + m]).max() < 2e-4
        done += m


def test_again_and_captured_gives_equal_bits():
    """Two calls, with others on the workspace between them, and a captured call replayed after the lengths, the rows'
    split over the sequences and the tables have changed."""
    lens, rows = [2000, 17, 900, 1], [60, 17, 1, 1]
    c = Cache(torch.bfloat16, lens, 2, 128, 16, spare=2).fill(lens)
    q = c.randn(sum(rows), 8 * 128, dtype=torch.bfloat16)
    ws = ops().paged_attn_chunk_workspace(c.handle, q.shape[0], 8)
    start = on_gpu(starts(rows))
    first = [t.clone() for t in ops().paged_attn_chunk(c.handle, q, 8, row_start=start, workspace=ws)]
    ws.fill_(255)
    again = ops().paged_attn_chunk(c.handle, q, 8, row_start=start, workspace=ws)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    out, lse = torch.empty_like(first[0]), torch.empty_like(first[1])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        ops().paged_attn_chunk(c.handle, q, 8, row_start=start, out=out, lse=lse, workspace=ws)
    new_lens, new_rows = [1024, 100, 900, 40], [1, 30, 20, 28]
    c.fill(new_lens)
    c.lens.copy_(on_gpu(new_lens))
    start.copy_(on_gpu(starts(new_rows)))
    for _ in range(2):
        out.fill_(7)
        graph.replay()
        check(c, q, 8, new_lens, starts(new_rows), out, lse, torch.bfloat16)


def test_offsets_past_32_bits():
    """Pages beyond the 2^31-th element of the pool."""
    page, Hkv, D = 64, 8, 128
    n_pages = (1 << 31) // (page * Hkv * D) + 40
    g = torch.Generator(device="cuda").manual_seed(0)
    k = torch.empty(n_pages, Hkv, page, D, dtype=torch.float16, device="cuda")
    v = torch.empty_like(k)
    used = torch.tensor([n_pages - 1, n_pages - 7, 3, n_pages - 20], device="cuda")
    for t in (k, v):
        t[used] = torch.randn(4, Hkv, page, D, generator=g, device="cuda").half()
    lens = torch.tensor([230], dtype=torch.int32, device="cuda")
    q = torch.randn(40, 16 * D, generator=g, device="cuda").half()
    far = ops().KVCache(k, v, used.int().view(1, 4), lens)
    near = ops().KVCache(k[used].contiguous(), v[used].contiguous(),
                         torch.arange(4, dtype=torch.int32, device="cuda").view(1, 4), lens)
    a = ops().paged_attn_chunk(far, q, 16, row_start=on_gpu([0, 40]))
    b = ops().paged_attn_chunk(near, q, 16, row_start=on_gpu([0, 40]))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_many_sequences():
    """4096 sequences, most of them with a row or none."""
    rng = np.random.default_rng(2)
    lens = rng.integers(0, 40, 4096)
    rows = np.minimum(lens, rng.integers(0, 3, 4096))
    c = Cache(torch.bfloat16, [48] * 4096, 1, 64, 16)
    c.k.normal_(generator=c.g)
    c.v.normal_(generator=c.g)
    c.lens.copy_(on_gpu(lens))
    q, start = c.randn(int(rows.sum()), 2 * 64, dtype=torch.bfloat16), starts(rows)
    out, lse = ops().paged_attn_chunk(c.handle, q, 2, row_start=on_gpu(start))
    check(c, q, 2, lens.tolist(), start, out, lse, torch.bfloat16)
    assert device_error() == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
def test_nan_scores_reach_rows_that_span_ctas(dtype, D):
    """Rows whose slots are dealt out to several CTAs, every score of some of the parts NaN: a query of NaN, and sequences
    that end in a block of one slot whose key is NaN.  None of them may look like a part that sees nothing."""
    lens = [3000, 20000]
    c = Cache(dtype, lens, 1, D, 16).fill(lens)
    q = c.randn(5, 2 * D, dtype=dtype)
    q[0, :D] = float("nan")
    q[4, D + 3] = float("nan")
    out, lse = ops().paged_attn_chunk(c.handle, q, 2, row_start=on_gpu([0, 2, 5]))
    lost = np.zeros((5, 2), bool)
    lost[0, 0] = lost[4, 1] = True
    assert np.array_equal(np.isnan(num(out).reshape(5, 2, D)), np.repeat(lost[:, :, None], D, 2))
    assert np.array_equal(np.isnan(num(lse)), lost)
    lens = [128 * k + 1 for k in range(2, 42)]
    c = Cache(dtype, lens, 1, D, 16).fill(lens)
    for b, n in enumerate(lens):
        c.k[c.table[b, (n - 1) // 16].long(), 0, (n - 1) % 16] = float("nan")
    q = c.randn(len(lens), D, dtype=dtype)
    out, lse = ops().paged_attn_chunk(c.handle, q, 1)
    assert num(out).shape == (40, D) and np.isnan(num(out)).all() and np.isnan(num(lse)).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,G,n,rows", [(64, 1, 100000, 20), (128, 1, 100000, 20), (128, 4, 60000, 50), (64, 8, 130000, 9)])
def test_a_value_out_of_sight_in_a_long_context(dtype, D, G, n, rows):
    """A value of V that is not finite near the end of long contexts, in a call that gives every CTA several of them and short
    sequences behind: rows before it as ever, the others lose its column alone, the other sequences nothing, and no
    wait runs out.  (The sequences share their pages.)"""
    B, page, few = 320 // G, 64, 64
    pages = -(-n // page)
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.randn(pages + few, 1, page, D, generator=g, device="cuda").to(dtype) for _ in "kv")
    table = torch.full((B + few, pages), -1, dtype=torch.int32, device="cuda")
    table[:B] = torch.arange(pages, device="cuda")
    table[B:, 0] = torch.arange(pages, pages + few, device="cuda")
    c = ops().KVCache(k, v, table, on_gpu([n] * B + [40] * few))
    start = on_gpu(starts([rows] * B + [3] * few))
    q = torch.randn(B * rows + 3 * few, G * D, generator=g, device="cuda").to(dtype)
    clean, clean_lse = ops().paged_attn_chunk(c, q, G, row_start=start)
    spoilt = []
    for slot, d, bad in ((n - rows // 2, 5, float("nan")), (n - 2, D - 1, float("inf"))):
        v[slot // page, 0, slot % page, d] = bad
        spoilt.append((slot - (n - rows), d))
    out, lse = ops().paged_attn_chunk(c, q, G, row_start=start)
    again, _ = ops().paged_attn_chunk(c, q, G, row_start=start)
    assert device_error() == 0
    assert torch.equal(out[B * rows:], clean[B * rows:]) and torch.equal(lse, clean_lse)
    lost = torch.zeros(B, rows, G, D, dtype=torch.bool, device="cuda")
    for row, d in spoilt:
        lost[:, row:, :, d] = True
    out, again, clean = (t[:B * rows].view(B, rows, G, D) for t in (out, again, clean))
    assert torch.equal(out.isfinite(), ~lost)
    assert torch.equal(out[~lost], again[~lost])
    want = clean[~lost].double()
    assert float((out[~lost].double() - want).norm() / want.norm()) < ATTN[dtype]
