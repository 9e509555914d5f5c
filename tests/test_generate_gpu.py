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
