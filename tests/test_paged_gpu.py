"""The paged key-value cache on the GPU (tkb_kv_append, tkb_paged_attn_decode,
tkb_kv_evict, tkb_kv_lens) against the float64 oracle.

Tolerances, in relative L2.  Storing a value in a type of m mantissa bits is
off by up to 2^-(m+1), 0.58 of that in the root mean square: 2^-m for stores
(2^-8 for bf16, 2^-11 for f16).  The attention may round its probabilities to
the same type before the product with V, another such error in every term:
twice that bound, 2^-7 and 2^-10.  fp32: sums of D (128) products of unit values are off by some
1e-6, exponentials of the scores by as much, so 1e-5; log-sum-exps and
accumulated weights are fp32 in every type: 2e-5.
"""
import numpy as np
import pytest

from oracle import paged_oracle as ref
from tests.conftest import rel_l2

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
STORE = {torch.float32: 1e-5, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
ATTN = {torch.float32: 1e-5, torch.bfloat16: 2.0 ** -7, torch.float16: 2.0 ** -10}


def ops():
    from tokamak_b200 import ops as o
    return o


def device_error():
    import ctypes
    from tokamak_b200 import check, lib
    code = ctypes.c_uint(0)
    check(lib().tkb_device_error(ctypes.byref(code), None))
    return code.value


def num(t):
    return t.double().cpu().numpy()


class Cache:
    """A cache with shuffled pages, every slot NaN where nothing was put."""

    def __init__(self, dtype, lens, Hkv, D, page, seed=0, extra=2, spare=0, page_gap=0):
        self.g = torch.Generator(device="cuda").manual_seed(seed)
        B = len(lens)
        per = max(1, max(-(-n // page) for n in lens) + spare)
        n_pages = B * per + extra
        size = Hkv * page * D
        shape, stride = (n_pages, Hkv, page, D), (size + page_gap, page * D, D, 1)

        def pool():
            t = torch.full((n_pages * (size + page_gap),), float("nan"), dtype=dtype, device="cuda")
            return t.as_strided(shape, stride)

        self.k, self.v = pool(), pool()
        self.pos = torch.full((n_pages, Hkv, page), -7, dtype=torch.int32, device="cuda")
        self.weight = torch.full((n_pages, Hkv, page), float("nan"), device="cuda")
        order = torch.randperm(n_pages, generator=self.g, device="cuda")[:B * per]
        self.table = order.view(B, per).int().contiguous()
        self.lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
        self.handle = ops().KVCache(self.k, self.v, self.table, self.lens, pos=self.pos, weight=self.weight)
        self.page, self.Hkv, self.D = page, Hkv, D

    def fill(self, lens, weights=None):
        """Random tokens in the first lens[b] slots of each sequence."""
        for b, n in enumerate(lens):
            for i in range(-(-n // self.page)):
                p, m = int(self.table[b, i]), min(self.page, n - i * self.page)
                for t in (self.k, self.v):
                    t[p, :, :m] = torch.randn(self.Hkv, m, self.D, generator=self.g, device="cuda").to(t.dtype)
                self.pos[p, :, :m] = torch.arange(i * self.page, i * self.page + m, device="cuda")
                w = torch.rand(self.Hkv, m, generator=self.g, device="cuda")
                self.weight[p, :, :m] = w if weights is None else weights(w)
        return self

    def randn(self, *shape, dtype=torch.float32, scale=1.0):
        return (scale * torch.randn(*shape, generator=self.g, device="cuda")).to(dtype)


def check_attention(c, q, Hq, lens, out, lse, dtype, before=None, scale=None):
    k, v, table, qn = num(c.k), num(c.v), c.table.cpu().numpy(), num(q)
    want_o, want_l, want_w = [], [], None if before is None else before.copy()
    scale = c.D ** -0.5 if scale is None else scale
    for b, n in enumerate(lens):
        o, l, p = ref.attend(k, v, table[b], n, qn[b].reshape(Hq, c.D), scale)
        want_o.append(o.ravel())
        want_l.append(l)
        if before is not None:
            G = Hq // c.Hkv
            for h in range(c.Hkv):
                for j in range(n):
                    want_w[table[b, j // c.page], h, j % c.page] += p[h * G:(h + 1) * G, j].sum()
    want_l = np.array(want_l)
    got_l = num(lse)
    assert np.array_equal(np.isneginf(got_l), np.isneginf(want_l))
    fin = np.isfinite(want_l)
    assert np.abs(got_l[fin] - want_l[fin]).max(initial=0) < 2e-5 * max(1.0, np.abs(want_l[fin]).max(initial=0))
    assert np.isfinite(num(out)).all()
    assert rel_l2(num(out), np.array(want_o)) < ATTN[dtype]
    empty = np.array(lens) == 0
    assert (num(out)[empty] == 0).all()
    if before is not None:
        got = num(c.weight)
        assert np.array_equal(np.isnan(got), np.isnan(want_w))
        ok = ~np.isnan(want_w)
        assert rel_l2(got[ok], want_w[ok]) < 2e-5


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hkv,G,page,lens", [
    (4, 1, 16, [77]),                                  # one short sequence
    (2, 4, 16, [1, 0, 15, 16, 17, 128, 129, 300]),     # empty, one token, page and tile edges
    (1, 8, 48, [1000, 3, 0, 47, 49]),                  # pages that are no power of two
    (8, 7, 64, [65, 640]),                             # odd group
    (2, 16, 32, [33, 257]),                            # a full tile of query heads
    (1, 20, 128, [130, 1]),                            # more query heads per kv head than a tile holds
    (3, 2, 1024, [1500, 31]),                          # large pages
    (1, 1, 16, [0]),                                   # nothing at all
    (1, 2, 16, [5000]),                                # long enough for many splits of one head
])
def test_decode(dtype, D, Hkv, G, page, lens):
    c = Cache(dtype, lens, Hkv, D, page).fill(lens)
    Hq = Hkv * G
    q = c.randn(len(lens), Hq * D, dtype=dtype)
    out, lse = ops().paged_attn_decode(c.handle, q, Hq)
    check_attention(c, q, Hq, lens, out, lse, dtype)
    before = num(c.weight)
    out2, lse2 = ops().paged_attn_decode(c.handle, q, Hq, accumulate=True)
    check_attention(c, q, Hq, lens, out2, lse2, dtype, before=before)
    assert device_error() == 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_decode_strides_scale_and_shared_pages(dtype):
    """A page stride above the page, query and output rows inside wider rows,
    two sequences that share their first pages, a scale of its own."""
    lens, Hkv, G, D, page = [200, 100, 64], 2, 3, 64, 32
    c = Cache(dtype, lens, Hkv, D, page, page_gap=64).fill(lens)
    c.table[1, :3] = c.table[0, :3]
    Hq = Hkv * G
    wide = c.randn(3, Hq * D + 128, dtype=dtype)
    q = wide[:, 64:64 + Hq * D]
    room = torch.full((3, Hq * D + 64), 7.0, dtype=dtype, device="cuda")
    out, lse = ops().paged_attn_decode(c.handle, q, Hq, scale=0.3, out=room[:, :Hq * D])
    check_attention(c, q, Hq, lens, out, lse, dtype, scale=0.3)
    assert (room[:, Hq * D:] == 7).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_decode_large_scores(dtype):
    """Scores in the hundreds: one key takes nearly all the weight, wherever it lies."""
    lens = [700, 700, 700]
    c = Cache(dtype, lens, 2, 64, 16).fill(lens)
    q = c.randn(3, 4 * 64, dtype=dtype, scale=30.0)
    for b, j in enumerate((0, 350, 699)):  # a key along the first query of each kv head
        for h in range(2):
            c.k[c.table[b, j // 16].long(), h, j % 16] = q[b, h * 128:h * 128 + 64] * 0.2
    out, lse = ops().paged_attn_decode(c.handle, q, 4)
    # scores up to 700 carry fp32 errors of 700 * 2^-22 and less: far below the storage bound
    k, v, t = num(c.k), num(c.v), c.table.cpu().numpy()
    for b in range(3):
        o, l, _ = ref.attend(k, v, t[b], lens[b], num(q)[b].reshape(4, 64), 0.125)
        assert rel_l2(num(out)[b].reshape(4, 64), o) < max(ATTN[dtype], 1e-3)
        assert np.abs(num(lse)[b] - l).max() < 1e-3


def test_decode_again_gives_equal_bits():
    """Two calls on one workspace, with other work between them on it."""
    lens = [3000, 17, 900, 1]
    c = Cache(torch.bfloat16, lens, 2, 128, 16).fill(lens)
    q = c.randn(4, 8 * 128, dtype=torch.bfloat16)
    ws = ops().paged_attn_workspace(c.handle, 8)
    first = [t.clone() for t in ops().paged_attn_decode(c.handle, q, 8, workspace=ws)]
    keep = c.lens.clone()
    for other in ([1, 1, 1, 1], [0, 0, 0, 0], [3000, 2000, 900, 600]):
        c.lens.copy_(torch.tensor(other))
        c.fill(other) if max(other) <= 1 else None
        ops().paged_attn_decode(c.handle, q, 8, workspace=ws)
    c.lens.copy_(keep)
    again = ops().paged_attn_decode(c.handle, q, 8, workspace=ws)
    fresh = ops().paged_attn_decode(c.handle, q, 8)
    for a, f in zip(again, fresh):
        assert torch.equal(a.isnan(), f.isnan()) and torch.equal(a.nan_to_num(), f.nan_to_num())
    assert first[0].shape == again[0].shape


def test_decode_follows_lengths_in_a_graph_and_on_a_stream():
    lens = [40, 100]
    c = Cache(torch.bfloat16, [500, 500], 2, 64, 16).fill([500, 500])
    q = c.randn(2, 4 * 64, dtype=torch.bfloat16)
    c.lens.copy_(torch.tensor(lens))
    ws = ops().paged_attn_workspace(c.handle, 4)
    out, lse = torch.empty_like(q), torch.empty(2, 4, device="cuda")
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        ops().paged_attn_decode(c.handle, q, 4, out=out, lse=lse, workspace=ws)
    st.synchronize()
    check_attention(c, q, 4, lens, out, lse, torch.bfloat16)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops().paged_attn_decode(c.handle, q, 4, out=out, lse=lse, workspace=ws)
    for lens in ([500, 1], [0, 333], [499, 500]):
        c.lens.copy_(torch.tensor(lens))
        graph.replay()
        torch.cuda.synchronize()
        check_attention(c, q, 4, lens, out, lse, torch.bfloat16)


def test_decode_beyond_32_bit_offsets():
    """Pages far into a pool of more than 2^32 bytes and 2^31 elements."""
    Hkv, page, D, stride = 1, 16, 128, 1 << 27
    n_pages = 20  # 20 * 2^27 elements: 5.4 GB each for k and v
    pools = [torch.empty(n_pages * stride, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    k, v = (p.as_strided((n_pages, Hkv, page, D), (stride, page * D, D, 1)) for p in pools)
    g = torch.Generator(device="cuda").manual_seed(3)
    for t in (k, v):
        for p in (19, 17, 3):
            t[p] = torch.randn(Hkv, page, D, generator=g, device="cuda").bfloat16()
    table = torch.tensor([[19, 17, 3]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([45], dtype=torch.int32, device="cuda")
    cache = ops().KVCache(k, v, table, lens)
    q = torch.randn(1, D, generator=g, device="cuda").bfloat16()
    out, lse = ops().paged_attn_decode(cache, q, 1)
    used = [19, 17, 3]
    kk, vv = num(k[used]), num(v[used])
    o, l, _ = ref.attend(kk, vv, np.arange(3), 45, num(q).reshape(1, D), D ** -0.5)
    assert rel_l2(num(out), o) < ATTN[torch.bfloat16]
    assert abs(num(lse)[0, 0] - l[0]) < 1e-4


@pytest.mark.parametrize("dtype", DTYPES)
def test_bad_pages_and_lengths_are_left_out(dtype):
    """A page the pool does not have counts as not held and sets bit 2."""
    c = Cache(dtype, [64, 40], 2, 64, 16).fill([64, 40])
    q = c.randn(2, 4 * 64, dtype=dtype)
    good = c.table.clone()
    c.table[0, 1] = 10 ** 6
    c.table[0, 3] = -1
    out, lse = ops().paged_attn_decode(c.handle, q, 4)
    assert device_error() == 4 and device_error() == 0
    k, v, t = num(c.k), num(c.v), good.cpu().numpy()
    o, l, _ = ref.attend(k, v, t[0][[0, 2]], 32, num(q)[0].reshape(4, 64), 0.125)
    assert rel_l2(num(out)[0].reshape(4, 64), o) < ATTN[dtype]
    assert np.abs(num(lse)[0] - l).max() < 2e-5 * max(1.0, np.abs(l).max())
    o, _, _ = ref.attend(k, v, t[1], 40, num(q)[1].reshape(4, 64), 0.125)
    assert rel_l2(num(out)[1].reshape(4, 64), o) < ATTN[dtype]
    c.table.copy_(good)
    c.lens[1] = -5  # nothing held
    out, lse = ops().paged_attn_decode(c.handle, q, 4)
    assert device_error() == 4
    assert (num(out)[1] == 0).all() and np.isneginf(num(lse)[1]).all()


# ------------------------------------------------------------------ append
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("qknorm,rope,scale", [(False, True, 1.0), (True, True, 8.0), (False, False, 1.0),
                                               (True, False, 1.0)])
def test_append_step(dtype, D, qknorm, rope, scale):
    """One token per sequence, at positions that are not the slots; strided rows."""
    Hq, Hkv, page, lens = 5, 1, 16, [1, 16, 17, 40]
    C = (Hq + 2 * Hkv) * D
    c = Cache(dtype, lens, Hkv, D, page)
    k0, v0 = num(c.k), num(c.v)
    seen = torch.tensor([1, 16, 100000, 41], dtype=torch.int32, device="cuda")
    rows = c.randn(4, C + 64, dtype=dtype)[:, :C]
    bias = c.randn(C, scale=0.1)
    gain = 1 + c.randn((Hq + Hkv) * D, scale=0.1) if qknorm else None
    out = ops().kv_append(c.handle, rows, Hq, seen=seen, bias=bias, qk_gain=gain, qknorm=qknorm, rope=rope,
                          theta=500000.0, rope_scale=scale)
    freq = ref.rope_frequencies(D, 500000.0, scale) if rope else None
    table = c.table.cpu().numpy()
    want_out = []
    for b, n in enumerate(lens):
        pos = int(seen[b]) - 1
        x = ref.prepare_row(num(rows)[b], pos, Hq, Hkv, D, num(bias), None if gain is None else num(gain), qknorm, freq)
        want_out.append(x[:Hq].ravel())
        j = n - 1
        k0[table[b, j // page], :, j % page] = x[Hq:Hq + Hkv]
        v0[table[b, j // page], :, j % page] = x[Hq + Hkv:]
        assert (c.pos[table[b, j // page], :, j % page] == pos).all()
        assert (c.weight[table[b, j // page], :, j % page] == 0).all()
    assert rel_l2(num(out), np.array(want_out)) < STORE[dtype]
    for got, want in ((num(c.k), k0), (num(c.v), v0)):
        assert np.array_equal(np.isnan(got), np.isnan(want))  # nothing else was written
        ok = ~np.isnan(want)
        assert rel_l2(got[ok], want[ok]) < STORE[dtype]
    assert int((c.pos != -7).sum()) == 4 and device_error() == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("full", [False, True])
def test_append_prompts(dtype, full):
    """Ragged prompts, one empty, one into a sequence that holds tokens already;
    with the packed rows wanted, they are tkb_qkv_prep_fwd's bit for bit."""
    Hq, Hkv, D, page = 4, 2, 64, 32
    fresh, held = [70, 0, 1, 33], [70, 5, 1, 50]
    C = (Hq + 2 * Hkv) * D
    c = Cache(dtype, held, Hkv, D, page)
    start = torch.tensor([0, 70, 70, 71, 104], dtype=torch.int32, device="cuda")
    rows = c.randn(104, C, dtype=dtype)
    out = ops().kv_append(c.handle, rows, Hq, row_start=start, theta=10000.0, full=full)
    freq = ref.rope_frequencies(D, 10000.0)
    table, x = c.table.cpu().numpy(), num(rows)
    r, want = 0, []
    for b in range(4):
        for i in range(fresh[b]):
            j = held[b] - fresh[b] + i
            y = ref.prepare_row(x[r], j, Hq, Hkv, D, None, None, False, freq)
            at = table[b, j // page], slice(None), j % page
            assert rel_l2(num(c.k[at]), y[Hq:Hq + Hkv]) < STORE[dtype]
            assert rel_l2(num(c.v[at]), y[Hq + Hkv:]) < STORE[dtype]
            assert (c.pos[at] == j).all()
            want.append(y.ravel() if full else y[:Hq].ravel())
            r += 1
    assert rel_l2(num(out), np.array(want)) < STORE[dtype]
    assert int((c.pos != -7).sum()) == 104 * Hkv and device_error() == 0
    if full:
        whole, _ = ops().qkv_prep_fwd(rows[:70].contiguous(), None, None, 70, Hq, Hkv, D)
        assert torch.equal(whole, out[:70])


def test_append_without_a_slot():
    """Rows that find no slot or page write nothing and set bit 2."""
    c = Cache(torch.bfloat16, [16, 16, 16], 1, 64, 16)
    c.lens.copy_(torch.tensor([0, 17, 16]))
    c.table[2, 0] = 99999
    rows = c.randn(3, 3 * 64, dtype=torch.bfloat16)
    out = ops().kv_append(c.handle, rows, 1)
    assert device_error() == 4
    assert c.k.isnan().all() and c.v.isnan().all() and (c.pos == -7).all()
    assert not out.isnan().any()


def test_lens():
    o = ops()
    lens = torch.tensor([0, 5, 99, 100], dtype=torch.int32, device="cuda")
    seen = torch.tensor([0, 50, 990, 1000], dtype=torch.int32, device="cuda")
    o.kv_lens(lens, 101, seen=seen, add=1)
    assert lens.tolist() == [1, 6, 100, 101] and seen.tolist() == [1, 51, 991, 1001] and device_error() == 0
    o.kv_lens(lens, 101, add=1)
    assert lens.tolist() == [2, 7, 101, 101] and device_error() == 4
    o.kv_lens(lens, 50)
    assert lens.tolist() == [2, 7, 50, 50] and device_error() == 0
    start = torch.tensor([0, 3, 3, 10, 11], dtype=torch.int32, device="cuda")
    o.kv_lens(lens, 1000, seen=seen, row_start=start)
    assert lens.tolist() == [5, 7, 57, 51] and seen.tolist() == [4, 51, 998, 1002] and device_error() == 0


# ------------------------------------------------------------------ eviction
def evict_case(dtype, lens, Hkv, D, page, budget, recent, sinks, weights=None, seed=0, shuffle=True):
    c = Cache(dtype, lens, Hkv, D, page, seed=seed).fill(lens, weights)
    seen = [3 * n + 1 for n in lens]
    if shuffle:  # positions in any order, other ones in every head; the newest is seen - 1
        rng = np.random.default_rng(seed)
        for b, n in enumerate(lens):
            for h in range(Hkv):
                pos = np.sort(rng.choice(np.arange(0, 3 * n + 1), size=n, replace=False)) if n else np.zeros(0, int)
                if n:
                    pos[-1] = 3 * n
                rng.shuffle(pos)
                for j in range(n):
                    c.pos[c.table[b, j // page].long(), h, j % page] = int(pos[j])
    k, v, w, pos = num(c.k), num(c.v), num(c.weight), c.pos.cpu().numpy().copy()
    table = c.table.cpu().numpy()
    ops().kv_evict(c.handle, budget, torch.tensor(seen, dtype=torch.int32, device="cuda"), recent=recent, sinks=sinks)
    total = 0
    for b, n in enumerate(lens):
        for h in range(Hkv):
            at = [(table[b, j // page], h, j % page) for j in range(n)]
            moves = ref.evict_moves([w[a] for a in at], [pos[a] for a in at], n, budget, seen[b], recent, sinks)
            total += len(moves)
            for to, frm in moves:
                for t in (k, v, w, pos):
                    t[at[to]] = t[at[frm]]
    for got, want in ((num(c.k), k), (num(c.v), v), (num(c.weight), w), (c.pos.cpu().numpy(), pos)):
        assert np.array_equal(got, want, equal_nan=got.dtype.kind == "f")
    assert device_error() == 0
    return total


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens,Hkv,D,page,budget,recent,sinks", [
    ([100, 64, 65, 0, 1, 63], 2, 64, 16, 64, 16, 4),    # over by one, at, below the budget; nothing held
    ([3000], 1, 128, 48, 100, 30, 1),                   # far over it
    ([2100, 1500], 3, 64, 64, 1024, 0, 0),              # no protected tokens
    ([50], 2, 64, 16, 49, 40, 9),                       # every kept place protected, or nearly
    ([40, 30], 1, 64, 32, 1, 1, 0),                     # a budget of one token
])
def test_evict(dtype, lens, Hkv, D, page, budget, recent, sinks):
    assert evict_case(dtype, lens, Hkv, D, page, budget, recent, sinks) > 0


@pytest.mark.parametrize("name", ["equal", "few", "nan", "signed"])
def test_evict_ties_and_odd_weights(name):
    """Equal weights go by the lower slot; NaN is the lowest, below -inf; -0 equals 0."""
    def weights(w):
        if name == "equal":
            return torch.full_like(w, 0.25)
        if name == "few":
            return (w * 4).floor()
        if name == "nan":
            return torch.where(w < 0.3, float("nan"), torch.where(w < 0.4, -float("inf"), w))
        return torch.where(w < 0.5, -0.0, 0.0)
    evict_case(torch.bfloat16, [300, 77], 2, 64, 16, 70, 8, 2, weights=weights, seed=5)


def test_evict_then_attend():
    """After an eviction the attention sees the kept tokens, whatever their order."""
    lens = [400, 90]
    c = Cache(torch.bfloat16, lens, 2, 64, 16).fill(lens)
    seen = c.lens.clone()
    ops().kv_evict(c.handle, 64, seen, recent=16, sinks=2)
    ops().kv_lens(c.lens, 64)
    assert c.lens.tolist() == [64, 64]
    q = c.randn(2, 4 * 64, dtype=torch.bfloat16)
    out, lse = ops().paged_attn_decode(c.handle, q, 4)
    check_attention(c, q, 4, [64, 64], out, lse, torch.bfloat16)
    for b in range(2):  # the newest 16 and the first 2 are still there
        for h in range(2):
            kept = set(c.pos[c.table[b, :4].long(), h].flatten().tolist())
            assert set(range(lens[b] - 16, lens[b])) | {0, 1} <= kept and len(kept) == 64


# ------------------------------------------------------------------ many sequences, long caches
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_decode_more_sequences_than_threads(dtype):
    """Each thread counts several sequences' tiles, empty ones among them."""
    rng = np.random.default_rng(3)
    lens = rng.integers(0, 40, 1100).tolist()
    lens[700] = 900
    c = Cache(dtype, lens, 1, 64, 16)
    g = c.g
    c.k.copy_(torch.randn(c.k.shape, generator=g, device="cuda"))
    c.v.copy_(torch.randn(c.v.shape, generator=g, device="cuda"))
    q = c.randn(len(lens), 2 * 64, dtype=dtype)
    out, lse = ops().paged_attn_decode(c.handle, q, 2)
    check_attention(c, q, 2, lens, out, lse, dtype)
    assert device_error() == 0


def test_append_many_prompts():
    rng = np.random.default_rng(4)
    fresh = rng.integers(0, 12, 700).tolist()
    total = sum(fresh)
    c = Cache(torch.float32, fresh, 1, 64, 16)
    start = torch.from_numpy(np.concatenate(([0], np.cumsum(fresh))).astype(np.int32)).cuda()
    rows = c.randn(total, 3 * 64)
    out = ops().kv_append(c.handle, rows, 1, row_start=start, rope=False)
    assert torch.equal(out, rows[:, :64])
    seq = np.repeat(np.arange(700), fresh)
    slot = np.concatenate([np.arange(n) for n in fresh]).astype(np.int64)
    pages = c.table[torch.from_numpy(seq).cuda(), 0].long()
    at = torch.from_numpy(slot).cuda()
    assert torch.equal(c.k[pages, 0, at], rows[:, 64:128]) and torch.equal(c.v[pages, 0, at], rows[:, 128:])
    assert int((c.pos != -7).sum()) == total and device_error() == 0


def test_evict_from_caches_too_long_for_shared_memory():
    """Above 49152 slots a sequence's keys are kept in the workspace."""
    assert evict_case(torch.bfloat16, [60000, 100], 1, 64, 1024, 500, 50, 4, shuffle=False) > 400


@pytest.mark.parametrize("dtype", DTYPES)
def test_decode_workspace_serves_every_shape(dtype):
    """One workspace, zeroed once, for caches of other batches, head counts and head widths in turn, and with
    accumulated weights between them: the bits of a workspace of each cache's own, and the oracle's values."""
    rng = np.random.default_rng(11)
    shapes = [([3000], 8, 4, 128, False), (rng.integers(0, 2000, 32).tolist(), 8, 2, 64, False),
              (rng.integers(500, 900, 20).tolist(), 2, 20, 64, True), ([1500, 0, 700], 1, 1, 128, True)]
    caches = []
    for lens, Hkv, G, D, acc in shapes:
        c = Cache(dtype, lens, Hkv, D, 16)
        for t in (c.k, c.v):
            t.copy_(torch.randn(t.shape, generator=c.g, device="cuda"))
        caches.append((c, c.randn(len(lens), Hkv * G * D, dtype=dtype)))
    need = [ops().paged_attn_workspace(c.handle, Hkv * G, acc).numel()
            for (c, _), (_, Hkv, G, _, acc) in zip(caches, shapes)]
    ws = torch.zeros(max(need), dtype=torch.uint8, device="cuda")
    fresh = {}
    for i in (0, 1, 0, 1, 2, 1, 3, 0, 2, 3, 1):
        (c, q), (lens, Hkv, G, D, acc) = caches[i], shapes[i]

        def call(workspace):
            c.weight.zero_()
            out, lse = torch.full_like(q, 7.0), torch.full((len(lens), Hkv * G), 7.0, device="cuda")
            ops().paged_attn_decode(c.handle, q, Hkv * G, accumulate=acc, out=out, lse=lse, workspace=workspace)
            return out, lse, c.weight.clone()

        if i not in fresh:
            fresh[i] = call(None)
            check_attention(c, q, Hkv * G, lens, fresh[i][0], fresh[i][1], dtype)
        for got, want in zip(call(ws), fresh[i]):
            assert torch.equal(got, want), i


@pytest.mark.parametrize("dtype", DTYPES)
def test_decode_nan_is_not_an_empty_cache(dtype):
    """NaN in a query, in every key of a kv head and in one key reaches the heads that use it, and no others; a
    sequence that holds nothing still gives 0 and -inf."""
    lens, Hkv, G, D, page = [40, 0, 600, 40, 3], 2, 4, 64, 16
    c = Cache(dtype, lens, Hkv, D, page).fill(lens)
    Hq = Hkv * G
    q = c.randn(5, Hq * D, dtype=dtype)
    good = [t.clone() for t in ops().paged_attn_decode(c.handle, q, Hq)]
    q.view(5, Hq, D)[0, 3, 5] = float("nan")
    c.k[c.table[2].long(), 1, :, 7] = float("nan")
    c.k[c.table[3, 1].long(), 0, 2, 0] = float("nan")
    bad = torch.zeros(5, Hq, dtype=torch.bool, device="cuda")
    bad[0, 3] = bad[2, G:] = bad[3, :G] = True
    for acc in (False, True):
        c.weight.zero_()
        out, lse = ops().paged_attn_decode(c.handle, q, Hq, accumulate=acc)
        assert torch.equal(out.view(5, Hq, D).isnan(), bad.unsqueeze(-1).expand(5, Hq, D))
        assert torch.equal(lse.isnan(), bad)
        for got, want in zip((out.view(5, Hq, D), lse), (good[0].view(5, Hq, D), good[1])):
            assert torch.equal(got[~bad], want[~bad])
        assert (out[1] == 0).all() and torch.isneginf(lse[1]).all()


@pytest.mark.parametrize("D,dtype", [(64, torch.bfloat16), (128, torch.float32)])
def test_rows_past_the_capacity_are_left_out(D, dtype):
    """Sequences that grow past their last page: what is held stays, the rows that fit are written, the others set
    bit 2; the attention then sees the full cache."""
    Hq, Hkv, page = 4, 2, 16
    held, fresh = [30, 32, 31, 5, 30, 32], [5, 1, 1, 2, 50, 40]
    c = Cache(dtype, held, Hkv, D, page).fill(held)
    cap = c.handle.capacity
    assert cap == 32
    k0, v0, pos0, w0 = num(c.k), num(c.v), c.pos.cpu().numpy().copy(), num(c.weight)
    seen = torch.tensor([h + 1000 for h in held], dtype=torch.int32, device="cuda")
    start = torch.tensor(np.concatenate(([0], np.cumsum(fresh))), dtype=torch.int32, device="cuda")
    C = (Hq + 2 * Hkv) * D
    rows = c.randn(sum(fresh), C, dtype=dtype)
    ops().kv_lens(c.lens, seen=seen, row_start=start)
    out = ops().kv_append(c.handle, rows, Hq, seen=seen, row_start=start, rope=False)
    assert device_error() == 4
    assert torch.equal(out, rows[:, :Hq * D])
    table, x = c.table.cpu().numpy(), num(rows).reshape(-1, Hq + 2 * Hkv, D)
    for b in range(len(held)):
        for i in range(fresh[b]):
            j = held[b] + i
            if j < cap:
                at = table[b, j // page], slice(None), j % page
                k0[at], v0[at] = x[int(start[b]) + i, Hq:Hq + Hkv], x[int(start[b]) + i, Hq + Hkv:]
                pos0[at], w0[at] = j + 1000, 0
    for got, want in ((num(c.k), k0), (num(c.v), v0), (num(c.weight), w0)):
        assert np.array_equal(got, want, equal_nan=True)
    assert np.array_equal(c.pos.cpu().numpy(), pos0)
    # and one token more for every sequence, of which one still has room
    before = [t.clone() for t in (c.k, c.v, c.pos)]
    ops().kv_lens(c.lens, seen=seen, add=1)
    one = c.randn(len(held), C, dtype=dtype)
    ops().kv_append(c.handle, one, Hq, seen=seen, rope=False)
    assert device_error() == 4
    at = int(c.table[3, 0]), slice(None), 7
    for t, was, part in ((c.k, before[0], one[3, Hq * D:(Hq + Hkv) * D]), (c.v, before[1], one[3, (Hq + Hkv) * D:])):
        was[at] = part.view(Hkv, D)
        assert torch.equal(t.isnan(), was.isnan()) and torch.equal(t.nan_to_num(), was.nan_to_num())
    before[2][at] = 1007
    assert torch.equal(c.pos, before[2])
    q = c.randn(len(held), Hq * D, dtype=dtype)
    out, lse = ops().paged_attn_decode(c.handle, q, Hq)
    assert device_error() == 4
    check_attention(c, q, Hq, [cap, cap, cap, 8, cap, cap], out, lse, dtype)
    # an eviction brings the lengths back below the budget
    ops().kv_evict(c.handle, 16, seen, recent=4)
    ops().kv_lens(c.lens, 16)
    assert device_error() == 4 and c.lens.tolist() == [16, 16, 16, 8, 16, 16]


def test_a_host_tensor_among_device_tensors_is_refused():
    from tokamak_b200 import TkbError
    c = Cache(torch.bfloat16, [5, 9], 2, 64, 16).fill([5, 9])
    q, rows = c.randn(2, 4 * 64, dtype=torch.bfloat16), c.randn(2, 8 * 64, dtype=torch.bfloat16)
    seen = c.lens.clone()
    o = ops()
    ws, ews = o.paged_attn_workspace(c.handle, 4), o.kv_evict_workspace(c.handle)
    for call in (lambda: o.kv_lens(c.lens, seen=seen.cpu(), add=1), lambda: o.kv_append(c.handle, rows.cpu(), 4),
                 lambda: o.kv_append(c.handle, rows, 4, seen=seen.cpu()),
                 lambda: o.kv_append(c.handle, rows, 4, bias=torch.zeros(8 * 64)),
                 lambda: o.kv_append(c.handle, rows, 4, row_start=torch.tensor([0, 1, 2], dtype=torch.int32)),
                 lambda: o.kv_append(c.handle, rows, 4, out=q.cpu()),
                 lambda: o.paged_attn_decode(c.handle, q.cpu(), 4, out=q.clone()),
                 lambda: o.paged_attn_decode(c.handle, q, 4, lse=torch.zeros(2, 4)),
                 lambda: o.paged_attn_decode(c.handle, q, 4, workspace=ws.cpu()),
                 lambda: o.kv_evict(c.handle, 4, seen.cpu()), lambda: o.kv_evict(c.handle, 4, seen, workspace=ews.cpu()),
                 lambda: o.sample_logits(q, torch.zeros(2)),
                 lambda: o.sample_logits(q, torch.zeros(2, device="cuda"), top_p=torch.ones(2)),
                 lambda: o.KVCache(c.k, c.v, c.table, c.lens.cpu())):
        with pytest.raises(TkbError, match="expected"):
            call()
    out, lse = o.paged_attn_decode(c.handle, q, 4, workspace=ws)
    check_attention(c, q, 4, [5, 9], out, lse, torch.bfloat16)


def test_strides_of_single_rows_heads_and_pages_mean_nothing():
    """torch gives a dimension of size one any stride: one sequence's rows, one kv head, one page, one token's logits."""
    lens, D, page = [11], 64, 16
    c = Cache(torch.bfloat16, lens, 1, D, page, extra=0).fill(lens)
    odd = [torch.empty(page * D + 8, dtype=torch.bfloat16, device="cuda").as_strided((1, 1, page, D), s)
           for s in ((24, 3, D, 1), (7, 5, D, 1))]
    for t, src in zip(odd, (c.k, c.v)):
        t.copy_(src)
    cache = ops().KVCache(*odd, c.table, c.lens, pos=c.pos, weight=c.weight)
    rows = c.randn(1, 4 * D, dtype=torch.bfloat16)
    same = rows.as_strided(rows.shape, (1, 1))
    want = ops().kv_append(c.handle, rows, 2)
    room = torch.empty_like(want)
    got = ops().kv_append(cache, same, 2, out=room.as_strided(room.shape, (3, 1)))
    assert torch.equal(want, room) and torch.equal(got, room)
    for t, src in zip(odd, (c.k, c.v)):  # the slots past the length are NaN in both
        assert np.array_equal(num(t), num(src), equal_nan=True)
    want, lse = ops().paged_attn_decode(c.handle, room, 2)
    out = torch.empty_like(want)
    _, lse2 = ops().paged_attn_decode(cache, got, 2, out=out.as_strided(out.shape, (1, 1)))
    assert torch.equal(out, want) and torch.equal(lse, lse2)
    token, _, kept = ops().sample_logits(torch.zeros(6, 2, device="cuda")[:, ::2].as_strided((3, 1), (2, 9)),
                                         torch.zeros(3, device="cuda"))
    assert token.tolist() == [0, 0, 0] and kept.tolist() == [1, 1, 1] and device_error() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,G", [(64, 8), (128, 8), (64, 16), (128, 4)])
def test_decode_rounds_only_the_output(dtype, D, G):
    """The probabilities are not rounded to the type: the error is the output's own rounding r.  P goes in with 16
    significant bits or more, so it adds at most 2^-16 of the result's size, and the fp32 sums 1e-5: against r (1.7e-3
    for bf16, 2.1e-4 for f16) that is sqrt(1 + (2.5e-5 / r)^2) < 1.01.  One rounding of P would add an error of the
    size of r itself (a factor of about 1.2 to 1.4)."""
    lens = [1500, 700, 64, 333]
    c = Cache(dtype, lens, 2, D, 16).fill(lens)
    q = c.randn(4, 2 * G * D, dtype=dtype)
    out, _ = ops().paged_attn_decode(c.handle, q, 2 * G)
    k, v, table = num(c.k), num(c.v), c.table.cpu().numpy()
    want = np.array([ref.attend(k, v, table[b], n, num(q)[b].reshape(2 * G, D), D ** -0.5)[0].ravel()
                     for b, n in enumerate(lens)])
    r = rel_l2(num(torch.from_numpy(want).to(dtype)), want)
    assert rel_l2(num(out), want) < 1.01 * r


@pytest.mark.parametrize("dtype", DTYPES)
def test_decode_of_the_same_inputs_gives_the_same_bits(dtype):
    """Twice on one workspace and on a fresh one, with calls of other lengths between; nothing is filled again."""
    lens = [3000, 17, 900, 1]
    c = Cache(dtype, lens, 2, 128, 16)
    for t in (c.k, c.v):
        t.copy_(torch.randn(t.shape, generator=c.g, device="cuda"))
    q = c.randn(4, 8 * 128, dtype=dtype)
    ws = ops().paged_attn_workspace(c.handle, 8)
    first = ops().paged_attn_decode(c.handle, q, 8, workspace=ws)
    for other in ([1, 1, 1, 1], [0, 0, 0, 0], [3000, 2000, 900, 600]):
        c.lens.copy_(torch.tensor(other))
        ops().paged_attn_decode(c.handle, q, 8, workspace=ws)
    c.lens.copy_(torch.tensor(lens))
    check_attention(c, q, 8, lens, *first, dtype)
    for again in (ops().paged_attn_decode(c.handle, q, 8, workspace=ws), ops().paged_attn_decode(c.handle, q, 8)):
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Hkv,G,D,lens", [(2, 4, 64, [700, 33, 5]), (1, 12, 128, [2000, 16, 1])])
def test_decode_infinite_values_stay_infinite(dtype, Hkv, G, D, lens):
    """An infinity in v is the sum's, in its column and for the heads that use it; two of both signs make NaN; slots
    past the length do not count."""
    c = Cache(dtype, lens, Hkv, D, 16).fill(lens)
    B, Hq = len(lens), Hkv * G
    q = c.randn(B, Hq * D, dtype=dtype)
    good = ops().paged_attn_decode(c.handle, q, Hq)[0].clone().view(B, Hkv, G, D)
    inf = float("inf")
    want = good.clone()
    for b, n in enumerate(lens):
        for j, col, x in ((0, 3, inf), (n // 2, 10, -inf), (n - 1, 40, inf)):
            c.v[c.table[b, j // 16].long(), 0, j % 16, col] = x
            want[b, 0, :, col] = x
    c.v[c.table[0, 20].long(), 0, 4, 3] = -inf   # the other sign in the same column of another key
    want[0, 0, :, 3] = float("nan")
    out, lse = ops().paged_attn_decode(c.handle, q, Hq)
    out = out.view(B, Hkv, G, D)
    assert torch.equal(out.isnan(), want.isnan()) and torch.equal(out.nan_to_num(), want.nan_to_num())
    assert torch.isfinite(lse).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("held", [0, 20])
def test_append_leaves_out_sequences_that_take_no_part(dtype, held):
    """seen below 0: nothing stored and no bit set, whatever the sequence holds; the other rows as ever."""
    c = Cache(dtype, [9, held, 33], 2, 64, 16).fill([9, held, 33])
    c.table[1] = -1
    seen = torch.tensor([9, -1, 33], dtype=torch.int32, device="cuda")
    before = [t.clone() for t in (c.k, c.v, c.pos, c.weight)]
    rows = c.randn(3, 8 * 64, dtype=dtype)
    out = ops().kv_append(c.handle, rows, 4, seen=seen, rope=False)
    assert device_error() == 0 and torch.equal(out, rows[:, :256])
    for t, part in ((before[0], rows[:, 256:384]), (before[1], rows[:, 384:])):
        for b, slot in ((0, 8), (2, 32)):
            t[c.table[b, slot // 16].long(), :, slot % 16] = part[b].view(2, 64)
    for b, slot in ((0, 8), (2, 32)):
        before[2][c.table[b, slot // 16].long(), :, slot % 16] = slot
        before[3][c.table[b, slot // 16].long(), :, slot % 16] = 0
    for got, want in zip((c.k, c.v, c.pos, c.weight), before):
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())
