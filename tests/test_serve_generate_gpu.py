"""The Generator on the operators that serve many requests at once: prompts in
pieces, conversations that go on, a pool of pages, adapters."""
import numpy as np
import pytest

from tests.conftest import rel_l2
from tests.test_generate_gpu import make, weights
from tests.test_paged_gpu import device_error

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

# both sides run in bf16 with other roundings in between: the bound of the engine's own bf16 tests
LOGITS = 2e-2


def table(cfg, seed=0):
    return np.random.default_rng(seed).standard_normal((cfg["vocab"], cfg["d_model"])).astype(np.float32)


def num(t):
    return t.double().cpu().numpy()


@pytest.mark.parametrize("gqa", [False, True])
@pytest.mark.parametrize("chunk", [1, 16, 23, 64])
def test_prompts_in_pieces(gqa, chunk):
    from tokamak_b200 import generate
    cfg = make(gqa=gqa)
    ckpt, embed, rng = weights(cfg), table(cfg), np.random.default_rng(1)
    prompts = [rng.integers(0, cfg["vocab"], n).tolist() for n in (40, 3, 70, 16)]
    whole = generate.Generator(cfg, ckpt, embed, 4, 96, page_size=16)
    pieces = generate.Generator(cfg, ckpt, embed, 4, 96, page_size=16, chunk=chunk)
    want, got = whole.prefill(prompts), pieces.prefill(prompts)
    assert rel_l2(num(got), num(want)) < LOGITS
    assert pieces.held == whole.held == [40, 3, 70, 16] and pieces.lens.tolist() == pieces.held
    for _ in range(3):
        for gen in (whole, pieces):
            gen.token.copy_(torch.tensor([5, 6, 7, 8]))
        assert rel_l2(num(pieces.decode()), num(whole.decode())) < LOGITS
    assert device_error() == 0


def test_a_conversation_goes_on():
    """Turns of any length, some sequences without one, after decode steps: the logits of the whole conversation."""
    from tokamak_b200 import generate
    cfg = make(gqa=True)
    ckpt, embed, rng = weights(cfg), table(cfg), np.random.default_rng(2)
    turn = lambda *n: [rng.integers(0, cfg["vocab"], m).tolist() for m in n]  # noqa: E731
    gen = generate.Generator(cfg, ckpt, embed, 3, 128, page_size=16, chunk=20)
    said = turn(9, 30, 4)
    gen.prefill(said)
    gen.token.copy_(torch.tensor([1, 2, 3]))
    gen.decode()
    said = [s + [t] for s, t in zip(said, (1, 2, 3))]
    more = turn(33, 0, 1)
    got = num(gen.extend(more))
    said = [s + m for s, m in zip(said, more)]
    assert (got[1] == 0).all() and gen.held == [len(s) for s in said] == gen.lens.tolist()
    want = num(generate.Generator(cfg, ckpt, embed, 3, 128, page_size=16).prefill(said))
    assert rel_l2(got[[0, 2]], want[[0, 2]]) < LOGITS
    gen.token.copy_(torch.tensor([9, 9, 9]))
    got = num(gen.decode())
    want = num(generate.Generator(cfg, ckpt, embed, 3, 128, page_size=16).prefill([s + [9] for s in said]))
    assert rel_l2(got, want) < LOGITS


def test_a_shared_pool_gives_the_same_tokens():
    """The tables' pages come from a pool, in the captured step too; sequences leave and others take their pages."""
    from tokamak_b200 import TkbError, generate
    cfg = make()
    ckpt, embed = weights(cfg), table(cfg)
    prompts = [[1, 2, 3], list(range(50)), [7]]
    options = dict(temperature=0.0)
    want = generate.Generator(cfg, ckpt, embed, 3, 128, page_size=16).generate(prompts, 40, **options)
    gen = generate.Generator(cfg, ckpt, embed, 3, 128, page_size=16, pool=12)
    for _ in range(2):  # the second time over pages in another order
        assert torch.equal(gen.generate(prompts, 40, **options), want)
        used = [int(n) for n in gen.pages_held]
        assert used == [-(-n // 16) for n in gen.held] and int(gen.n_free) == 12 - sum(used)
        mine = [int(p) for b in range(3) for p in gen.table[b, :used[b]]]
        assert sorted(mine + gen.free_pages[:int(gen.n_free)].tolist()) == list(range(12))
    with pytest.raises(TkbError, match="pages"):
        gen.extend([[1] * 80, [], []])
    gen.release([1])
    assert int(gen.pages_held[1]) == 0 and (gen.table[1] == -1).all()
    # a new request in the place of the one that left
    got = num(gen.extend([[], list(range(20, 45)), []]))
    alone = generate.Generator(cfg, ckpt, embed, 1, 128, page_size=16)
    assert rel_l2(got[1], num(alone.prefill([list(range(20, 45))]))[0]) < LOGITS
    assert gen.held == [42, 25, 40] and device_error() == 0


@pytest.mark.parametrize("pool", [0, 12])
@pytest.mark.parametrize("captured", [False, True])
def test_a_released_sequence_stays_empty(pool, captured):
    """A request ends while the others decode; the next one in its place gets the logits of its tokens alone, and the others
    those of a batch where nobody left."""
    from tokamak_b200 import generate
    cfg = make(gqa=True)
    ckpt, embed, rng = weights(cfg), table(cfg), np.random.default_rng(3)
    said = [rng.integers(0, cfg["vocab"], n).tolist() for n in (30, 16, 5)]
    gen = generate.Generator(cfg, ckpt, embed, 3, 128, page_size=16, pool=pool)
    gen.prefill(said)
    said[1] = []
    graph, logits = torch.cuda.CUDAGraph(), None
    if captured:  # while all three are there
        gen.token.zero_()
        gen.decode()
        said = [s + [0] if s else s for s in said]
        with torch.cuda.graph(graph):
            logits = gen.decode()
    gen.release([1])

    def step(tokens):
        gen.token.copy_(torch.tensor(tokens))
        if not captured:
            return num(gen.decode())
        graph.replay()
        gen.held = [n + a for n, a in zip(gen.held, gen.live)]
        return num(logits)

    def alone(b):
        return num(generate.Generator(cfg, ckpt, embed, 1, 128, page_size=16).prefill([said[b]]))[0]

    for s in range(20):
        got = step([s, 100 + s, 50 + s])
        said = [t + [n] if t else t for t, n in zip(said, (s, 0, 50 + s))]
        assert gen.lens.tolist() == gen.held == [len(t) for t in said]
        if pool:
            assert gen.pages_held.tolist() == [-(-n // 16) for n in gen.held]
    assert rel_l2(got[0], alone(0)) < LOGITS and rel_l2(got[2], alone(2)) < LOGITS
    said[1] = rng.integers(0, cfg["vocab"], 21).tolist()
    got = num(gen.extend([[], said[1], []]))
    assert rel_l2(got[1], alone(1)) < LOGITS and gen.held == [len(t) for t in said]
    got = step([7, 8, 9])
    said = [t + [n] for t, n in zip(said, (7, 8, 9))]
    for b in range(3):
        assert rel_l2(got[b], alone(b)) < LOGITS
    assert gen.lens.tolist() == gen.seen.tolist() == gen.held and device_error() == 0


def test_pool_and_budget():
    """Evictions give pages back."""
    from tokamak_b200 import generate
    cfg = make()
    ckpt, embed = weights(cfg), table(cfg)
    prompts = [list(range(90)), [5, 6]]
    args = dict(page_size=16, budget=48, slack=16, recent=8, sinks=2)
    want = generate.Generator(cfg, ckpt, embed, 2, 96, **args).generate(prompts, 100, temperature=0.0)
    gen = generate.Generator(cfg, ckpt, embed, 2, 96, pool=10, **args)
    assert torch.equal(gen.generate(prompts, 100, temperature=0.0), want)
    assert [int(n) for n in gen.pages_held] == [-(-n // 16) for n in gen.held] and device_error() == 0


def test_pieces_with_a_budget():
    """A piece adds its last tokens' attention to the weights, and the cut cache goes on."""
    from tokamak_b200 import generate
    cfg = make(gqa=True)
    gen = generate.Generator(cfg, weights(cfg), table(cfg), 2, 96, page_size=16, budget=48, slack=16, recent=8, sinks=2,
                             window=4, chunk=24)
    gen.prefill([list(range(90)), [5, 6]])
    D, Hkv = cfg["head_dim"], cfg["kv_heads"]
    for c in gen.caches:  # four queries of each of four pieces (24, 24, 24, 18 tokens), summed over the heads' slots
        w = c.weight[c.block_table[0].long()]
        assert torch.allclose(w.sum((0, 2)), torch.full((Hkv,), 16.0 * cfg["q_heads"] / Hkv, device="cuda"), rtol=1e-4)
        w = c.weight[c.block_table[1].long()]
        assert torch.allclose(w.sum((0, 2)), torch.full((Hkv,), 2.0 * cfg["q_heads"] / Hkv, device="cuda"), rtol=1e-4)
    gen.evict()
    assert gen.held == [48, 2]
    gen.extend([[1, 2, 3], []])
    assert gen.held == [51, 2] and gen.lens.tolist() == gen.held and device_error() == 0


def adapters(cfg, n, R, names, seed=5, size=0.1):
    from tokamak_b200 import generate
    rng = np.random.default_rng(seed)
    d, F = cfg["d_model"], cfg["ffn"]
    q, kv = cfg["q_heads"] * cfg["head_dim"], cfg["kv_heads"] * cfg["head_dim"]
    sizes = dict(wqkv=(d, q + 2 * kv), wo=(q, d), wgu=(d, 2 * F), wd=(F, d))

    def low(K, N):
        a = rng.standard_normal((n, K, R)) * K ** -0.5
        return a.astype(np.float32), (size * rng.standard_normal((n, R, N)) * R ** -0.5).astype(np.float32)

    layers = [{k: low(*sizes[k]) for k in names} for _ in range(cfg["layers"])]
    return generate.Adapters(cfg, layers, scale=np.linspace(0.5, 1.5, n).astype(np.float32))


def merged(cfg, ckpt, low, i):
    """The checkpoint with adapter i in its matrices."""
    from tokamak_b200 import generate
    out = [t.copy() for t in ckpt]
    layers, _ = generate.split_checkpoint(cfg, out)
    for w, ab in zip(layers, low.layers):
        for name, (a, b) in ab.items():
            w[name] += (low.scale[i] * (a[i].astype(np.float64) @ b[i].astype(np.float64))).astype(np.float32).ravel()
    return out


@pytest.mark.parametrize("names", [("wqkv", "wo", "wgu", "wd"), ("wqkv",)])
def test_adapters_equal_merged_weights(names):
    """Every sequence with its own adapter or none, prompts and steps: the logits of a decoder whose matrices hold it."""
    from tokamak_b200 import generate
    cfg = make(gqa=True)
    ckpt, embed, rng = weights(cfg), table(cfg), np.random.default_rng(4)
    low, ids = adapters(cfg, 3, 16, names), [2, -1, 0, 2]
    prompts = [rng.integers(0, cfg["vocab"], n).tolist() for n in (40, 3, 70, 16)]
    gen = generate.Generator(cfg, ckpt, embed, 4, 96, page_size=16, chunk=32, adapters=low)
    gen.adapter.copy_(torch.tensor(ids, dtype=torch.int32))
    got = [num(gen.prefill(prompts))]
    gen.token.copy_(torch.tensor([5, 6, 7, 8]))
    got.append(num(gen.decode()))
    plain = generate.Generator(cfg, ckpt, embed, 4, 96, page_size=16)
    base, effect = num(plain.prefill(prompts)), []
    for b, i in enumerate(ids):
        one = generate.Generator(cfg, merged(cfg, ckpt, low, i) if i >= 0 else ckpt, embed, 1, 96, page_size=16)
        want = [num(one.prefill([prompts[b]]))[0]]
        one.token.fill_(5 + b)
        want.append(num(one.decode())[0])
        for s in range(2):
            assert rel_l2(got[s][b], want[s]) < LOGITS
        effect.append(rel_l2(base[b], want[0]))
    # and, all of them, they matter: logits without them, within LOGITS of base, would be further than LOGITS from some of
    # those wanted (those of wqkv alone move the logits less: the next test looks at its rows)
    assert effect[1] < LOGITS and (len(names) < 4 or max(effect) > 2 * LOGITS)
    assert device_error() == 0


def test_adapted_rows_of_the_first_projection():
    """What enters the cache of the first layer: the plain rows plus the adapters' products, each rounded to bf16 (half a
    step, 2^-9 at most, of the plain row and of the sum)."""
    from tokamak_b200 import generate, ops
    cfg = make(gqa=True)
    ckpt, embed, rng = weights(cfg), table(cfg), np.random.default_rng(6)
    low, ids = adapters(cfg, 3, 16, ("wqkv",)), [1, -1, 2]
    prompts = [rng.integers(0, cfg["vocab"], n).tolist() for n in (20, 9, 1)]
    rows = []
    for more in (dict(), dict(adapters=low)):
        gen = generate.Generator(cfg, ckpt, embed, 3, 96, page_size=16, **more)
        gen.adapter.copy_(torch.tensor(ids, dtype=torch.int32))
        seen, append = [], gen._append
        gen._append = lambda i, qkv, **kw: (seen.append(qkv.clone()), append(i, qkv, **kw))[1]
        gen.prefill(prompts)
        rows.append(num(seen[0]))
    x = gen.embed[torch.tensor(sum(prompts, []), device="cuda")]
    y = num(ops.add_rmsnorm_fwd(x, None, gen.layers[0]["norm1"])[1])
    a, b = (num(m) for m in gen.low[0]["wqkv"])
    want = rows[0].copy()
    for i, at in zip(ids, (slice(0, 20), slice(20, 29), slice(29, 30))):
        if i >= 0:
            want[at] += low.scale[i] * (y[at] @ a[i] @ b[i])
    assert rel_l2(rows[1], want) < 2 * 2.0 ** -9 and rel_l2(rows[0], want) > 0.05
    assert np.array_equal(rows[1][20:29], rows[0][20:29])


def test_command_with_everything(tmp_path, capsys):
    from tokamak_b200 import configs, generate
    low = adapters(configs.C1, 2, 8, ("wo", "wd"))
    arrays = {f"{i}.{k}.{x}": m for i, w in enumerate(low.layers) for k, ab in w.items() for x, m in zip("AB", ab)}
    np.savez(tmp_path / "low.npz", scale=low.scale, **arrays)
    generate.main(["--steps", "40", "--batch", "3", "--prompt", "150", "--chunk", "64", "--pool", "9", "--adapters",
                   str(tmp_path / "low.npz"), "--adapter-ids", "1,-1,0"])
    assert "3 x 40 tokens" in capsys.readouterr().out
