"""Refusals of the entry points that serve many requests at once: bad arguments
are turned down with a message before any CUDA call."""
import ctypes

import numpy as np
import pytest

import tokamak_b200
from oracle import serve_oracle as ref
from tests.test_generate_cpu import cache, message

vp = ctypes.c_void_p


def chunk(c, rows=2, Hq=4, q=256, out=512, stride=256, out_stride=256, start=256, scale=0.1, ws=256, n=1 << 40):
    L = tokamak_b200.lib()
    return L.tkb_paged_attn_chunk(ctypes.byref(c) if c else None, vp(q), stride, vp(out), out_stride, None, vp(start),
                                  rows, Hq, scale, vp(ws), n, None)


@pytest.mark.parametrize("over,code", [
    (dict(k=0), -1), (dict(seq_lens=0), -1), (dict(block_table=0), -1), (dict(k=264), -1), (dict(dtype=7), -1),
    (dict(B=0), -1), (dict(B=5000), -3), (dict(D=96), -3), (dict(page_size=24), -1), (dict(page_size=2048), -1),
    (dict(page_stride=2 * 16 * 64 - 8), -1), (dict(max_pages=1 << 28), -1), (dict(n_pages=0), -1), (dict(Hkv=0), -1)])
def test_chunk_bad_caches(over, code):
    c = cache(**over)
    assert chunk(c) == code and message()
    assert tokamak_b200.lib().tkb_paged_attn_chunk_workspace(ctypes.byref(c), 2, 4) == 0


def test_chunk_refusals():
    c = cache()
    assert chunk(None) == -1
    assert chunk(c, Hq=3) == -1 and "multiple" in message()
    assert chunk(c, Hq=0) == -1 and chunk(c, rows=0) == -1 and chunk(c, rows=(1 << 26) + 1) == -3
    assert chunk(c, rows=3, start=0) == -1 and "row_start" in message()
    assert chunk(c, q=0) == -1 and chunk(c, out=0) == -1
    assert chunk(c, q=264) == -1 and chunk(c, stride=128) == -1 and chunk(c, out_stride=260) == -1
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        assert chunk(c, scale=scale) == -1 and "scale" in message()
    assert chunk(c, ws=0) == -4 and chunk(c, n=8) == -4 and chunk(c, ws=272) == -4
    L = tokamak_b200.lib()
    assert L.tkb_paged_attn_chunk_workspace(ctypes.byref(c), 0, 4) == 0
    assert L.tkb_paged_attn_chunk_workspace(ctypes.byref(c), 2, 3) == 0
    small, large = (L.tkb_paged_attn_chunk_workspace(ctypes.byref(c), n, 4) for n in (2, 4096))
    assert 0 < small <= large


def test_pages_refusals():
    def call(table=256, held=256, lens=256, free=256, n_free=256, slots=0, start=0, rows=0, B=2, most=4, page=16, n=8):
        return tokamak_b200.lib().tkb_kv_pages(vp(table), vp(held), vp(lens), vp(free), vp(n_free), None, vp(slots),
                                               vp(start), rows, B, most, page, n, None)
    for name in ("table", "held", "lens", "free", "n_free"):
        assert call(**{name: 0}) == -1 and "null" in message()
    assert call(B=0) == -1 and call(B=5000) == -3 and call(most=0) == -1 and call(n=0) == -1
    assert call(page=0) == -1 and call(page=1025) == -1 and call(most=1 << 29, B=2) == -3
    assert call(slots=256, rows=0) == -1 and call(slots=256, rows=3) == -1 and "row_start" in message()
    assert call(slots=260, rows=2) == -1 and "aligned" in message()


def test_lora_refusals():
    L = tokamak_b200.lib()

    def plan(adapter=256, start=256, B=2, rows=9, n=3, at=256, size=1 << 30):
        return L.tkb_lora_plan(vp(adapter), vp(start), B, rows, n, vp(at), size, None)
    assert plan(adapter=0) == -1 and plan(B=0) == -1 and plan(rows=0) == -1 and plan(n=0) == -1 and plan(B=5000) == -3
    assert plan(start=0) == -1 and "row_start" in message()
    assert plan(at=0) == -4 and plan(size=8) == -4 and plan(at=264) == -4
    assert L.tkb_lora_plan_bytes(0, 1, 1) == 0 and L.tkb_lora_plan_bytes(1, 1, 0) == 0
    assert L.tkb_lora_workspace(0, 8) == 0 and L.tkb_lora_workspace(8, 0) == 0

    def add(p=256, x=256, xs=64, a=256, b=256, y=256, ys=64, out=512, os=64, B=2, rows=9, n=3, K=64, N=64, R=8, dt=1,
            ws=256, size=1 << 30):
        return L.tkb_lora_add(vp(p), vp(x), xs, vp(a), vp(b), None, vp(y), ys, vp(out), os, B, rows, n, K, N, R, dt,
                              vp(ws), size, None)
    for name in ("p", "x", "a", "b", "y", "out"):
        assert add(**{name: 0}) == -1, name
    assert add(R=0) == -3 and add(R=12) == -3 and add(R=136) == -3
    assert add(K=60) == -1 and add(N=4) == -1 and add(K=0) == -1 and add(n=0) == -1 and add(dt=5) == -1
    assert add(xs=56) == -1 and add(ys=68) == -1 and add(os=0) == -1 and add(x=264) == -1 and add(a=264) == -1
    assert add(out=256, y=256, os=128) == -1 and "stride" in message()
    assert add(ws=0) == -4 and add(size=16) == -4 and add(ws=264) == -4


def test_python_checks():
    torch = pytest.importorskip("torch")
    from tokamak_b200 import TkbError, ops
    k = torch.zeros(4, 2, 16, 64)
    table, lens = torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    c = ops.KVCache(k, k.clone(), table, lens)
    q, start = torch.zeros(7, 4 * 64), torch.tensor([0, 3, 7], dtype=torch.int32)
    for args, more in (((q[:, :64], 4), {}), ((q.bfloat16(), 4), {}), ((q.view(-1), 4), {}), ((q, 4), dict(row_start=lens)),
                       ((q, 4), dict(row_start=start.long())), ((q, 4), dict(row_start=start, out=q[:3])),
                       ((q, 4), dict(row_start=start, lse=torch.zeros(7, 3))), ((q, 3), dict(row_start=start)),
                       ((q.t().contiguous().t(), 4), dict(row_start=start))):
        with pytest.raises(TkbError):
            ops.paged_attn_chunk(c, *args, **more)
    one = torch.zeros(1, dtype=torch.int32)
    free = torch.zeros(9, dtype=torch.int32)
    for bad in (dict(held=one), dict(lens=lens.long()), dict(n_free=lens), dict(block_table=table.t()),
                dict(row_start=lens, rows=4), dict(free_pages=free[::2])):
        with pytest.raises(TkbError):
            ops.kv_pages(**{**dict(block_table=table, held=lens, lens=lens, free_pages=free, n_free=one, page_size=16),
                            **bad})
    with pytest.raises(TkbError):
        ops.lora_plan(lens.long(), 2, 7, row_start=start)
    with pytest.raises(TkbError):
        ops.lora_plan(lens, 2, 7, row_start=lens)
    plan = ops.LoraPlan(torch.zeros(256, dtype=torch.uint8), 2, 7, 3)
    good = dict(x=torch.zeros(7, 64), A=torch.zeros(3, 64, 8), B=torch.zeros(3, 8, 32), y=torch.zeros(7, 32))
    for bad in (dict(x=torch.zeros(6, 64)), dict(x=torch.zeros(7, 64).half()), dict(A=torch.zeros(2, 64, 8)),
                dict(B=torch.zeros(3, 16, 32)), dict(y=torch.zeros(7, 40)), dict(out=torch.zeros(7, 31)),
                dict(scale=torch.zeros(2)), dict(x=torch.zeros(64, 7).t()), dict(A=torch.zeros(3, 8, 64).transpose(1, 2))):
        with pytest.raises(TkbError):
            ops.lora_add(plan, **{**good, **bad})


def test_tensors_of_the_host_are_refused():
    torch = pytest.importorskip("torch")
    from tokamak_b200 import TkbError, ops
    k = torch.zeros(4, 2, 16, 64)
    table, lens = torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    c = ops.KVCache(k, k.clone(), table, lens)
    start = torch.tensor([0, 3, 7], dtype=torch.int32)
    plan = ops.LoraPlan(torch.zeros(256, dtype=torch.uint8), 2, 7, 3)
    calls = [lambda: ops.paged_attn_chunk(c, torch.zeros(7, 4 * 64), 4, row_start=start),
             lambda: ops.kv_pages(table, lens, lens.clone(), torch.zeros(9, dtype=torch.int32), lens[:1], 16),
             lambda: ops.lora_plan(lens, 3, 7, row_start=start),
             lambda: ops.lora_add(plan, torch.zeros(7, 64), torch.zeros(3, 64, 8), torch.zeros(3, 8, 32),
                                  torch.zeros(7, 32))]
    for call in calls:
        with pytest.raises(TkbError, match="CUDA device"):
            call()


def test_oracle_of_the_chunk_against_differences_and_single_tokens():
    """The oracle itself: rows of a chunk are single tokens over ever more slots, and d lse / d score is the weight of
    its key, by differences."""
    from oracle import paged_oracle
    rng = np.random.default_rng(0)
    k, v = rng.standard_normal((2, 3, 2, 16, 8))
    pages, q = np.array([2, 0]), rng.standard_normal((5, 4, 8))
    out, lse = ref.chunk(k, v, pages, 20, q, 0.3)
    for i in range(5):
        o, l, p = paged_oracle.attend(k, v, pages, 16 + i, q[i], 0.3)
        assert np.allclose(out[i], o) and np.allclose(lse[i], l)
    # moving key 3 along the query by eps moves its score by eps |q|^2 scale
    eps, h = 1e-6, 0
    _, _, p = paged_oracle.attend(k, v, pages, 20, q[4], 0.3)
    moved = k.copy()
    moved[2, h, 3] += eps * q[4, 0]
    _, more = ref.chunk(moved, v, pages, 20, q, 0.3)
    assert abs((more[4, 0] - lse[4, 0]) / (eps * (q[4, 0] ** 2).sum() * 0.3) - p[0, 3]) < 1e-5


def test_oracle_of_the_pages_keeps_every_page_once():
    rng = np.random.default_rng(1)
    table, held, stack = np.full((6, 5), -1), np.zeros(6, int), list(range(17))
    for _ in range(50):
        lens = rng.integers(0, 81, 6)
        table, held, stack, granted = ref.pages(table, held, lens, stack, 16)
        used = [int(p) for b in range(6) for p in table[b, :held[b]]]
        assert sorted(used + stack) == list(range(17)) and (table[np.arange(5) >= held[:, None]] == -1).all()
        assert all(bool(g) == (h * 16 >= n) for g, h, n in zip(granted, held, lens))


def small(**more):
    from tests.test_generate_cpu import small_generator
    return small_generator(**more)


def test_generator_refusals():
    from tokamak_b200 import TkbError
    for bad in (dict(chunk=-1), dict(pool=-1)):
        with pytest.raises(TkbError):
            small(**bad)
    cfg, gen = small()
    for pieces in ([[1]], [[], []], [[1], [2], [3]]):
        with pytest.raises(TkbError, match="extend"):
            gen.extend(pieces)
    with pytest.raises(TkbError, match="max_tokens"):
        gen.extend([[1] * 65, []])
    with pytest.raises(TkbError, match="token ids"):
        gen.extend([[], [cfg["vocab"]]])
    for bad in ([2], [-1]):
        with pytest.raises(TkbError, match="release"):
            gen.release(bad)
    _, gen = small(pool=1, page_size=16)
    for call in (lambda: gen.prefill([[1] * 9, [2]]), lambda: gen.extend([[1], [2]]), lambda: gen.generate([[1], [2]], 4)):
        with pytest.raises(TkbError, match="2 pages are needed, the pool has 1"):
            call()


def test_released_sequences_take_no_part_in_steps(monkeypatch):
    """Lengths, positions and pages of a batch whose sequences end, wait and start again, the calls restated on the host: a
    sequence that holds nothing after a release, or after an extend that brought it nothing, gets no token from a step."""
    torch = pytest.importorskip("torch")
    from tokamak_b200 import TkbError, generate

    def kv_lens(lens, limit=None, seen=None, add=0, row_start=None):
        n = torch.full_like(lens, add) if row_start is None else row_start.diff()
        lens += n
        seen += n

    def kv_pages(table, held, lens, free, n_free, page, tokens=0):
        stack = free[:int(n_free)].tolist()
        t, h, stack, _ = ref.pages(table.numpy(), held.numpy(), lens.tolist(), stack, page)
        table.copy_(torch.from_numpy(t))
        held.copy_(torch.from_numpy(h))
        free[:len(stack)] = torch.tensor(stack, dtype=torch.int32)
        n_free.fill_(len(stack))

    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(generate.ops, "kv_lens", kv_lens)
    monkeypatch.setattr(generate.ops, "kv_pages", kv_pages)
    monkeypatch.setattr(generate.ops, "paged_attn_chunk_workspace", lambda *a: None)
    monkeypatch.setattr(generate.ops, "gemm", lambda x, w, **more: torch.zeros(x.shape[0], w.shape[1]))
    for pool in (0, 2):
        cfg, gen = small(pool=pool, page_size=16)
        gen._forward = lambda x, attend, row_start=None: torch.zeros(x.shape[0], cfg["d_model"])
        gen.extend([[1] * 5, [2] * 7])
        assert gen.lens.tolist() == gen.held == [5, 7]
        gen.release([1])
        for n in (6, 7, 8):
            gen.decode()
            assert gen.lens.tolist() == gen.held == [n, 0] and int(gen.seen[0]) == n
            assert int(gen.seen[1]) < 0  # the append leaves such a sequence out
            if pool:
                assert gen.pages_held.tolist() == [1, 0]
        gen.release([1])  # once more
        gen.extend([[], [3, 4]])
        assert gen.lens.tolist() == gen.seen.tolist() == gen.held == [8, 2]
        gen.decode()
        assert gen.lens.tolist() == gen.seen.tolist() == gen.held == [9, 3]
        # a full pool refuses only steps that need a page
        gen.release([0])
        gen.extend([[], [5] * 14])
        assert gen.held == [0, 17]
        gen.decode()
        assert gen.lens.tolist() == gen.held == [0, 18]
        if pool:
            with pytest.raises(TkbError, match="3 pages are needed"):
                gen.extend([[1], []])
            assert gen.lens.tolist() == gen.held == [0, 18] and int(gen.seen[0]) < 0
        gen.prefill([[1], [2]])
        gen.decode()
        assert gen.lens.tolist() == gen.seen.tolist() == gen.held == [2, 2]
        # slots that no request has taken yet wait too; without any request, steps start from self.token
        _, gen = small(pool=pool, page_size=16)
        gen._forward = lambda x, attend, row_start=None: torch.zeros(x.shape[0], cfg["d_model"])
        gen.decode()
        assert gen.lens.tolist() == gen.seen.tolist() == gen.held == [1, 1]
        _, gen = small(pool=pool, page_size=16)
        gen._forward = lambda x, attend, row_start=None: torch.zeros(x.shape[0], cfg["d_model"])
        gen.extend([[], [3] * 4])
        gen.decode()
        assert gen.lens.tolist() == gen.held == [0, 5]


def test_adapter_refusals(tmp_path):
    from tokamak_b200 import TkbError, configs, generate
    cfg = dict(configs.C1, layers=1)
    z = lambda *s: np.zeros(s, np.float32)  # noqa: E731
    good = (z(3, 256, 8), z(3, 8, 256))
    assert generate.Adapters(cfg, [dict(wo=good)], scale=z(3)).rank == 8
    for layers in ([], [{}], [dict(wo=good)] * 2, [dict(wq=good)], [dict(wo=(good[0], z(3, 16, 256)))],
                   [dict(wo=(z(3, 128, 8), good[1]))], [dict(wo=good, wd=(z(2, 688, 8), z(2, 8, 256)))],
                   [dict(wo=(z(256, 8), good[1]))]):
        with pytest.raises(TkbError):
            generate.Adapters(cfg, layers)
    with pytest.raises(TkbError):
        generate.Adapters(cfg, [dict(wo=good)], scale=z(2))
    path = tmp_path / "a.npz"
    np.savez(path, **{"0.wo.A": good[0], "0.wo.B": good[1]})
    assert generate.Adapters.load(cfg, path).n == 3
    for arrays in ({"0.wo.A": good[0]}, {"1.wo.A": good[0], "1.wo.B": good[1]}, {"wo.A": good[0]}, {}):
        np.savez(path, **arrays)
        with pytest.raises(TkbError):
            generate.Adapters.load(cfg, path)


def test_adapters_of_ranks_that_no_kernel_has_are_refused_at_once():
    """Before a forward pass has counted tokens that it cannot take."""
    from tokamak_b200 import TkbError, configs, generate
    cfg = dict(configs.C1, layers=1)

    def build(R):
        return generate.Adapters(cfg, [dict(wo=(np.zeros((3, 256, R), np.float32), np.zeros((3, R, 256), np.float32)))])
    for R in (8, 24, 128):
        assert build(R).rank == R
    for R in (0, 4, 12, 136, 256):
        with pytest.raises(TkbError, match="rank"):
            build(R)
    with pytest.raises(TkbError):
        generate.Adapters(cfg, [dict(wo=(np.zeros((0, 256, 8), np.float32), np.zeros((0, 8, 256), np.float32)))])


def test_arrays_beside_an_adapters_are_not_passed_over(tmp_path):
    """A misnamed array beside a good pair would be left out without a word."""
    from tokamak_b200 import TkbError, configs, generate
    cfg, path = dict(configs.C1, layers=1), tmp_path / "a.npz"
    a, b = np.zeros((3, 256, 8), np.float32), np.zeros((3, 8, 256), np.float32)
    for name in ("0.wo.", "0.wo.AB", "0.wo.C", "00.wo.A", "².wo.A"):
        np.savez(path, **{"0.wo.A": a, "0.wo.B": b, name: a})
        with pytest.raises(TkbError, match="unexpected array"):
            generate.Adapters.load(cfg, path)
