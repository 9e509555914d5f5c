"""The generation path as a whole: prompts and single tokens through the paged
cache give the logits that the engine's forward gives for the whole sequence."""
import numpy as np
import pytest

from tests.conftest import rel_l2

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def make(layers=2, gqa=False):
    from tokamak_b200 import configs
    cfg = dict(configs.C1, layers=layers)
    if gqa:
        cfg.update(kv_heads=2)
    return cfg


def weights(cfg, seed=3):
    from tokamak_b200 import generate
    rng = np.random.default_rng(seed)
    out = generate.random_checkpoint(cfg, seed)
    for t in out:  # biases and gains that matter
        if t.size < 4096:
            t += 0.1 * rng.standard_normal(t.size).astype(np.float32)
    return out


@pytest.mark.parametrize("gqa", [False, True])
@pytest.mark.parametrize("prompt", [1, 40, 63])
def test_logits_equal_the_engines(gqa, prompt):
    from tokamak_b200 import configs, generate, runtime
    cfg, S, B = make(gqa=gqa), 64, 2
    ckpt = weights(cfg)
    rng = np.random.default_rng(1)
    embed = rng.standard_normal((cfg["vocab"], cfg["d_model"])).astype(np.float32)
    tokens = rng.integers(0, cfg["vocab"], (B, S))
    rt = runtime.Runtime.from_dsl(configs.dsl_for(dict(cfg, seq=S)), B)
    rt.load_weights(runtime.tkm1_pack(ckpt))
    rt.step(embed[tokens], np.zeros(B * S, np.int32), 0.0)
    want = rt.logits(B * S * cfg["vocab"]).reshape(B, S, -1)
    rt.close()
    gen = generate.Generator(cfg, ckpt, embed, B, S, page_size=16)
    got = [gen.prefill([t[:prompt].tolist() for t in tokens])]
    for s in range(prompt, S):
        gen.token.copy_(torch.from_numpy(tokens[:, s].astype(np.int32)))
        got.append(gen.decode())
    got = torch.stack(got, 1).float().cpu().numpy()
    # both run in bf16 with other roundings in between: the bound of the engine's own bf16 tests
    assert rel_l2(got, want[:, prompt - 1:]) < 2e-2


def test_generation_is_reproducible_and_greedy_follows_the_logits():
    from tokamak_b200 import generate
    cfg = make()
    embed = np.random.default_rng(0).standard_normal((cfg["vocab"], cfg["d_model"])).astype(np.float32)
    prompts = [[1, 2, 3], list(range(50)), [7]]
    gen = generate.Generator(cfg, weights(cfg), embed, 3, 128, page_size=16)
    runs = [gen.generate(prompts, 20, temperature=0.9, top_k=20, top_p=0.9,
                         generator=torch.Generator(device="cuda").manual_seed(5)).cpu() for _ in range(2)]
    assert torch.equal(runs[0], runs[1]) and runs[0].shape == (3, 20)
    assert ((runs[0] >= 0) & (runs[0] < cfg["vocab"])).all()
    greedy = gen.generate(prompts, 12, temperature=0.0).cpu()
    logits = gen.prefill(prompts)
    for s in range(12):
        assert torch.equal(logits.argmax(1).cpu().int(), greedy[:, s])
        gen.token.copy_(greedy[:, s])
        logits = gen.decode()


def test_generation_with_a_budget():
    """The cache is cut during generation and never holds more than budget + slack tokens."""
    from tokamak_b200 import generate
    cfg = make()
    embed = np.random.default_rng(0).standard_normal((cfg["vocab"], cfg["d_model"])).astype(np.float32)
    gen = generate.Generator(cfg, weights(cfg), embed, 2, 96, page_size=16, budget=48, slack=16, recent=8, sinks=2)
    out = gen.generate([list(range(90)), [5, 6]], 120, temperature=0.7, top_p=0.9).cpu()
    assert out.shape == (2, 120) and (out >= 0).all()
    assert gen.seen.tolist() == [90 + 119, 2 + 119] and gen.lens.tolist() == gen.held and max(gen.held) <= 64
    for c in gen.caches:  # distinct tokens, the newest and the first among them
        for b in range(2):
            n = gen.held[b]
            for h in range(cfg["kv_heads"]):
                pos = c.pos[c.block_table[b].long(), h].flatten()[:n].tolist()
                assert len(set(pos)) == n and {0, 1} <= set(pos) and max(pos) == int(gen.seen[b]) - 1


def test_command():
    from tokamak_b200 import generate
    generate.main(["--steps", "8", "--batch", "2", "--prompt", "20", "--budget", "16"])


def test_refusals():
    from tokamak_b200 import TkbError, generate
    cfg = make()
    embed = np.zeros((cfg["vocab"], cfg["d_model"]), np.float32)
    with pytest.raises(TkbError):
        generate.Generator(dict(cfg, layers=1), weights(cfg), embed, 1, 64)
    gen = generate.Generator(cfg, weights(cfg), embed, 1, 64)
    with pytest.raises(TkbError):
        gen.prefill([[]])
    with pytest.raises(TkbError):
        gen.generate([[1] * 60], 10)


@pytest.mark.parametrize("prompts", [(90, 40), (64, 90), (90, 3)])
def test_a_long_prompt_is_cut_by_its_own_attention(prompts):
    """A prompt longer than the budget is weighed by the attention of its last `window` tokens, each over the tokens up
    to itself, and the first cut keeps the heaviest wherever they lie."""
    from oracle import paged_oracle as ref
    from tokamak_b200 import generate
    cfg = make(gqa=True)
    rng = np.random.default_rng(6)
    embed = rng.standard_normal((cfg["vocab"], cfg["d_model"])).astype(np.float32)
    budget, recent, sinks, window, page = 48, 10, 2, 7, 16
    gen = generate.Generator(cfg, weights(cfg), embed, 2, 96, page_size=page, budget=budget, slack=16, recent=recent,
                             sinks=sinks, window=window)
    seen_rows = []
    append = gen._append

    def record(i, qkv, **more):
        out = append(i, qkv, **more)
        seen_rows.append(out.double().cpu().numpy())
        return out

    gen._append = record
    tokens = [rng.integers(0, cfg["vocab"], n).tolist() for n in prompts]
    gen.prefill(tokens)
    Hq, Hkv, D = cfg["q_heads"], cfg["kv_heads"], cfg["head_dim"]
    G, start = Hq // Hkv, np.concatenate(([0], np.cumsum(prompts)))
    want = {}
    for layer, rows in enumerate(seen_rows):
        table = gen.table.cpu().numpy()
        got = gen.caches[layer].weight.double().cpu().numpy()
        pos = gen.caches[layer].pos.cpu().numpy()
        for b, n in enumerate(prompts):
            x = rows[start[b]:start[b + 1]].reshape(n, Hq + 2 * Hkv, D)
            for h in range(Hkv):
                w = np.zeros(n)
                for i in range(max(0, n - window), n):
                    for g in range(G):
                        s = x[:i + 1, Hq + h] @ x[i, h * G + g] * D ** -0.5
                        e = np.exp(s - s.max())
                        w[:i + 1] += e / e.sum()
                have = np.array([got[table[b, j // page], h, j % page] for j in range(n)])
                # fp32 softmax of bf16 rows that both sides share: the bound of the decode attention's weights
                assert rel_l2(have, w) < 2e-5
                at = [pos[table[b, j // page], h, j % page] for j in range(n)]
                moves = ref.evict_moves(have, at, n, budget, n, recent, sinks)
                kept = set(range(min(n, budget))) - {m[0] for m in moves} | {m[1] for m in moves}
                want[layer, b, h] = {at[j] for j in kept}
    gen.evict()
    for (layer, b, h), kept in want.items():
        c = gen.caches[layer]
        n = min(prompts[b], budget)
        pos = c.pos[c.block_table[b].long(), h].flatten()[:n].tolist()
        assert set(pos) == kept
        if prompts[b] > budget:  # not merely the first ones and the newest
            assert kept != set(range(budget - recent)) | set(range(prompts[b] - recent, prompts[b]))


@pytest.mark.parametrize("budget", [1, 16, 40])
def test_command_with_a_small_budget(budget):
    """The command goes past its first cut whatever the budget."""
    from tokamak_b200 import generate
    generate.main(["--steps", "90", "--batch", "2", "--prompt", "20", "--budget", str(budget)])


def test_command_runs_a_given_model(tmp_path, capsys):
    """Checkpoint, embedding and prompts from files: the tokens of a Generator on the same."""
    from tokamak_b200 import configs, generate, runtime
    cfg = configs.C1
    ckpt = weights(cfg)
    embed = np.random.default_rng(8).standard_normal((cfg["vocab"], cfg["d_model"])).astype(np.float32)
    prompts = [[5, 6, 7, 8], [9], list(range(40))]
    (tmp_path / "model.tkmw").write_bytes(runtime.tkm1_pack(ckpt))
    np.save(tmp_path / "table.npy", embed)
    (tmp_path / "prompts.txt").write_text("\n".join(" ".join(map(str, p)) for p in prompts))
    generate.main(["--checkpoint", str(tmp_path / "model.tkmw"), "--embedding", str(tmp_path / "table.npy"), "--tokens",
                   str(tmp_path / "prompts.txt"), "--steps", "10", "--temperature", "0"])
    lines = [[int(t) for t in row.split()] for row in capsys.readouterr().out.splitlines()[-3:]]
    want = generate.Generator(cfg, ckpt, embed, 3, 64).generate(prompts, 10, temperature=0.0)
    assert lines == want.tolist()
