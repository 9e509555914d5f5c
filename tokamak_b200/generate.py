"""Text generation with the Llama-style decoders of ``configs`` on the paged
key-value cache: prompts in one pass, then one token per sequence and step,
the step captured as a CUDA graph.

    python -m tokamak_b200.generate [--config C1|C4] [--checkpoint model.tkmw] [--embedding table.npy]
        [--tokens prompts.txt | --batch 8 --prompt 100] [--steps 64] [--budget 0] [--top-k 50] [--top-p 0.95]
        [--temperature 0.8]

Weights come from a TKM1 checkpoint that the engine trained on the same
configuration; the embedding table [vocab, d_model], which the engine takes as
its input rows, from the caller; prompts as token ids, one prompt a line.
Each is random where it is not given.  Kernels: tkb_add_rmsnorm_fwd,
tkb_gemm, tkb_gemm_swiglu, tkb_gqa_attn_fwd (prompts), tkb_kv_append,
tkb_paged_attn_decode, tkb_kv_evict, tkb_sample_logits.  torch only holds the
tensors and looks embeddings up.
"""
import numpy as np
import torch

from . import TkbError, ops


def split_checkpoint(cfg, tensors):
    """The TKM1 tensors of a configuration's graph (configs.dsl_for) by name:
    a list of layers and the head.  Registration order per layer: norm gain,
    fused QKV matrix, its bias and (unused) QKNorm gain, the K and V matrices
    and biases that the fusion removed, output matrix and bias, norm gain,
    fused [gate | up] matrix, gate bias, removed up matrix, up bias, down
    matrix and bias; then norm gain, matrix and bias of the head."""
    d, F, V = cfg["d_model"], cfg["ffn"], cfg["vocab"]
    q, kv = cfg["q_heads"] * cfg["head_dim"], cfg["kv_heads"] * cfg["head_dim"]
    sizes = [("norm1", d), ("wqkv", d * (q + 2 * kv)), ("bqkv", q + 2 * kv), (None, q + 2 * kv), (None, d * kv),
             (None, kv), (None, d * kv), (None, kv), ("wo", q * d), ("bo", d), ("norm2", d), ("wgu", d * 2 * F),
             ("bg", F), (None, d * F), ("bu", F), ("wd", F * d), ("bd", d)]
    tail = [("norm", d), ("w", d * V), ("b", V)]
    want = [n for _, n in sizes] * cfg["layers"] + [n for _, n in tail]
    if [t.size for t in tensors] != want:
        raise TkbError("the checkpoint does not fit the configuration")
    it = iter(tensors)
    layers = [{k: t for (k, _), t in zip(sizes, it) if k} for _ in range(cfg["layers"])]
    return layers, {k: t for (k, _), t in zip(tail, it)}


def random_checkpoint(cfg, seed=0):
    """TKM1 tensors N(0, 0.02) with unit gains, as the engine's own initial weights are distributed."""
    rng = np.random.default_rng(seed)
    d, F, V = cfg["d_model"], cfg["ffn"], cfg["vocab"]
    q, kv = cfg["q_heads"] * cfg["head_dim"], cfg["kv_heads"] * cfg["head_dim"]
    w = lambda *s: (0.02 * rng.standard_normal(int(np.prod(s)), dtype=np.float32))  # noqa: E731
    one, zero = lambda n: np.ones(n, np.float32), lambda n: np.zeros(n, np.float32)  # noqa: E731
    out = []
    for _ in range(cfg["layers"]):
        out += [one(d), w(d, q + 2 * kv), zero(q + 2 * kv), one(q + 2 * kv), w(d, kv), zero(kv), w(d, kv), zero(kv),
                w(q, d), zero(d), one(d), w(d, 2 * F), zero(F), w(d, F), zero(F), w(F, d), zero(d)]
    return out + [one(d), w(d, V), zero(V)]


class Generator:
    """Generation state of `batch` sequences of at most max_tokens tokens.

    budget: tokens a (sequence, kv head) keeps in the cache (0: all).  Once
    the sequences hold `slack` more, the cache is cut to the budget by
    accumulated attention weight; the newest `recent` tokens and the first
    `sinks` stay.  A decode step adds its token's attention to the weights; a
    prompt longer than the budget starts with that of its last `window` tokens,
    since it may be cut before any step (8 prompts of 2048 tokens on C4: 29 ms,
    and 0.5 ms for each of them)."""

    def __init__(self, cfg, checkpoint, embed, batch, max_tokens, page_size=64, budget=0, slack=64, recent=32, sinks=4,
                 device="cuda", window=8):
        if window < 1:
            raise TkbError("Generator: window must be positive")
        self.cfg, self.batch, self.max_tokens = cfg, batch, max_tokens
        self.budget, self.slack, self.recent, self.sinks, self.window = budget, slack, recent, sinks, window
        layers, head = split_checkpoint(cfg, checkpoint)
        Hq, Hkv, D = cfg["q_heads"], cfg["kv_heads"], cfg["head_dim"]
        self.Hq, self.Hkv, self.D = Hq, Hkv, D

        def put(t, cols=None):
            t = torch.from_numpy(np.ascontiguousarray(t)).to(device)
            return t if cols is None else t.view(-1, cols).bfloat16()

        d, F, V = cfg["d_model"], cfg["ffn"], cfg["vocab"]
        self.layers = [dict(norm1=put(w["norm1"]), wqkv=put(w["wqkv"], (Hq + 2 * Hkv) * D), bqkv=put(w["bqkv"]),
                            wo=put(w["wo"], d), bo=put(w["bo"]), norm2=put(w["norm2"]), wgu=put(w["wgu"], 2 * F),
                            bg=put(w["bg"]), bu=put(w["bu"]), wd=put(w["wd"], d), bd=put(w["bd"])) for w in layers]
        self.head = dict(norm=put(head["norm"]), w=put(head["w"], V), b=put(head["b"]))
        self.embed = torch.as_tensor(embed, dtype=torch.bfloat16, device=device)
        # a look-up past its end would be a device assert; rows past the vocabulary may hold prompt-only tokens
        if self.embed.dim() != 2 or self.embed.shape[0] < V or self.embed.shape[1] != d:
            raise TkbError(f"Generator: embed is {tuple(self.embed.shape)}, not {(V, d)}")
        pages = -(-max_tokens // page_size)
        self.table = torch.arange(batch * pages, dtype=torch.int32, device=device).view(batch, pages)
        self.lens = torch.zeros(batch, dtype=torch.int32, device=device)   # tokens held in the cache
        self.seen = torch.zeros(batch, dtype=torch.int32, device=device)   # tokens so far
        self.caches = []
        for _ in self.layers:
            k, v = (torch.zeros(batch * pages, Hkv, page_size, D, dtype=torch.bfloat16, device=device) for _ in "kv")
            meta = torch.zeros(2, batch * pages, Hkv, page_size, device=device)
            self.caches.append(ops.KVCache(k, v, self.table, self.lens, pos=meta[0].view(torch.int32), weight=meta[1]))
        self.workspace = ops.paged_attn_workspace(self.caches[0], Hq, budget > 0)
        self.evict_workspace = ops.kv_evict_workspace(self.caches[0]) if budget else None
        # the same caches up to a token of the prompt, for its attention weights
        self.upto = torch.zeros_like(self.lens)
        self.prefixes = [ops.KVCache(c.k, c.v, self.table, self.upto, pos=c.pos, weight=c.weight)
                         for c in self.caches if budget]
        self.token = torch.zeros(batch, dtype=torch.int32, device=device)
        self.u = torch.zeros(batch, device=device)
        self.held = [0] * batch  # the lengths, known on the host too: nothing is read back
        self.graph = None
        self.sampling = {}

    def _forward(self, x, attend):
        """Logits' input rows: the decoder on rows x [rows, d_model]; attend(layer, qkv) gives the heads' outputs."""
        skip, y = x, None
        for i, w in enumerate(self.layers):
            if i == 0:
                _, y, _ = ops.add_rmsnorm_fwd(x, None, w["norm1"])
            a = ops.gemm(attend(i, ops.gemm(y, w["wqkv"])), w["wo"], bias=w["bo"])
            skip, y, _ = ops.add_rmsnorm_fwd(a, skip, w["norm2"])
            _, h = ops.gemm_swiglu(y, w["wgu"], self.cfg["ffn"], w["bg"], w["bu"])
            f = ops.gemm(h, w["wd"], bias=w["bd"])
            gain = self.layers[i + 1]["norm1"] if i + 1 < len(self.layers) else self.head["norm"]
            skip, y, _ = ops.add_rmsnorm_fwd(f, skip, gain)
        return y

    def _append(self, i, qkv, **more):
        return ops.kv_append(self.caches[i], qkv, self.Hq, seen=self.seen, bias=self.layers[i]["bqkv"],
                             theta=float(self.cfg["theta"]), **more)

    def _weigh(self, i, rows, ends, lens):
        """Adds the attention of the prompts' last tokens to layer i's weights: step j takes the rows ends[j] as
        queries over the first lens[j] tokens of each sequence (none where the prompt is shorter)."""
        for j in range(ends.shape[0]):
            self.upto.copy_(lens[j])
            ops.paged_attn_decode(self.prefixes[i], rows[ends[j], :self.Hq * self.D], self.Hq, accumulate=True,
                                  workspace=self.workspace)

    def prefill(self, prompts):
        """Prompts (lists of token ids, none empty) enter the empty caches; returns the logits [batch, vocab]
        after each prompt's last token."""
        n = [len(p) for p in prompts]
        if len(n) != self.batch or min(n) < 1 or max(n) > self.max_tokens:
            raise TkbError("prefill: one prompt of 1 to max_tokens tokens per sequence")
        if min(map(min, prompts)) < 0 or max(map(max, prompts)) >= self.embed.shape[0]:
            raise TkbError(f"prefill: token ids are 0 to {self.embed.shape[0] - 1}")
        dev = self.token.device
        start = np.concatenate(([0], np.cumsum(n))).astype(np.int32)
        row_start = torch.from_numpy(start).to(dev)
        tokens = torch.tensor([t for p in prompts for t in p], dtype=torch.int64, device=dev)
        self.lens.zero_()
        self.seen.zero_()
        ops.kv_lens(self.lens, seen=self.seen, row_start=row_start)
        self.held = list(n)
        if self.budget and max(n) > self.budget:
            back = np.arange(self.window)[:, None]
            ends = torch.from_numpy(np.maximum(start[1:] - 1 - back, start[:-1]).astype(np.int64)).to(dev)
            upto = torch.from_numpy(np.maximum(np.diff(start) - back, 0).astype(np.int32)).to(dev)

        def attend(i, qkv):
            rows = self._append(i, qkv, row_start=row_start, full=True)
            if self.budget and max(n) > self.budget:
                self._weigh(i, rows, ends, upto)
            out = torch.empty(rows.shape[0], self.Hq * self.D, dtype=rows.dtype, device=dev)
            for b in range(self.batch):
                part = rows[start[b]:start[b + 1]]
                out[start[b]:start[b + 1]] = ops.gqa_attn_fwd(part, 1, n[b], self.Hq, self.Hkv, self.D)[0][0]
            return out

        y = self._forward(self.embed[tokens], attend)
        last = y[torch.from_numpy(start[1:].astype(np.int64) - 1).to(dev)]
        return ops.gemm(last, self.head["w"], bias=self.head["b"], out_dtype=torch.float32)

    def decode(self):
        """One step: the tokens in self.token (rows of embed) enter the caches; returns the next logits [batch, vocab]."""
        ops.kv_lens(self.lens, seen=self.seen, add=1)

        def attend(i, qkv):
            q = self._append(i, qkv)
            return ops.paged_attn_decode(self.caches[i], q, self.Hq, accumulate=self.budget > 0,
                                         workspace=self.workspace)[0]

        y = self._forward(self.embed[self.token.long()], attend)
        return ops.gemm(y, self.head["w"], bias=self.head["b"], out_dtype=torch.float32)

    def _step(self):
        token, _, _ = ops.sample_logits(self.decode(), self.u, **self.sampling)
        self.token.copy_(token)

    def evict(self):
        """Cut every layer's cache to the budget."""
        for c in self.caches:
            ops.kv_evict(c, self.budget, self.seen, recent=self.recent, sinks=self.sinks,
                         workspace=self.evict_workspace)
        ops.kv_lens(self.lens, self.budget)
        self.held = [min(n, self.budget) for n in self.held]

    def generate(self, prompts, steps, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, generator=None):
        """[batch, steps] sampled token ids (int32, on the device) after the prompts.  The decode step is captured
        as a CUDA graph on its second run and replayed; evictions run between replays."""
        dev, B = self.token.device, self.batch
        if not self.budget and max(len(p) for p in prompts) + steps - 1 > self.max_tokens:
            raise TkbError("generate: more tokens than max_tokens and no budget")
        if self.budget and self.budget + self.slack > self.max_tokens:
            raise TkbError("generate: max_tokens must hold budget + slack tokens")
        if self.budget and self.recent + self.sinks > self.budget and \
                max(len(p) for p in prompts) + steps - 2 >= self.budget + self.slack:
            raise TkbError("generate: the budget must hold recent + sinks tokens")
        full = lambda v, dt: torch.full((B,), v, dtype=dt, device=dev)  # noqa: E731
        sampling = dict(temperature=full(temperature, torch.float32), top_k=full(top_k, torch.int32) if top_k else None,
                        top_p=full(top_p, torch.float32) if top_p < 1 else None,
                        min_p=full(min_p, torch.float32) if min_p > 0 else None)
        self.sampling, self.graph = sampling, None
        u = torch.rand(steps, B, device=dev, generator=generator)
        out = torch.empty(steps, B, dtype=torch.int32, device=dev)
        logits = self.prefill(prompts)
        self.u.copy_(u[0])
        token, _, _ = ops.sample_logits(logits, self.u, **sampling)
        self.token.copy_(token)
        out[0] = token
        for s in range(1, steps):
            if self.budget and max(self.held) >= self.budget + self.slack:
                self.evict()
            self.u.copy_(u[s])
            if s == 1:
                self._step()
            else:
                if self.graph is None:
                    self.graph = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(self.graph):
                        self._step()
                self.graph.replay()
            self.held = [n + 1 for n in self.held]
            out[s] = self.token
        return out.t()


def read_prompts(path):
    """Lists of token ids from a text file, one prompt a line, empty lines left out."""
    with open(path) as f:
        try:
            prompts = [[int(t) for t in line.split()] for line in f if line.strip()]
        except ValueError as e:
            raise TkbError(f"{path}: {e}")
    if not prompts:
        raise TkbError(f"{path}: no prompts")
    return prompts


def main(argv=None):
    import argparse
    import time

    from . import configs, runtime
    ap = argparse.ArgumentParser(description="Generate tokens with a decoder of tokamak_b200.configs.")
    ap.add_argument("--config", default="C1", choices=("C1", "C4"))
    ap.add_argument("--checkpoint", help="TKM1 file of that configuration (default: random weights)")
    ap.add_argument("--embedding", help=".npy file of the embedding table [vocab, d_model] (default: a random one)")
    ap.add_argument("--tokens", help="text file of prompts, token ids, one prompt a line (default: random ones)")
    ap.add_argument("--batch", type=int, default=8)
    ap.add_argument("--prompt", type=int, default=100, help="tokens per (random) prompt")
    ap.add_argument("--steps", type=int, default=64)
    ap.add_argument("--budget", type=int, default=0, help="cached tokens per sequence and kv head (0: all)")
    ap.add_argument("--temperature", type=float, default=0.8)
    ap.add_argument("--top-k", type=int, default=50)
    ap.add_argument("--top-p", type=float, default=0.95)
    ap.add_argument("--min-p", type=float, default=0.0)
    ap.add_argument("--seed", type=int, default=0)
    a = ap.parse_args(argv)
    cfg = getattr(configs, a.config)
    if a.checkpoint:
        with open(a.checkpoint, "rb") as f:
            weights = runtime.tkm1_unpack(f.read())
    else:
        weights = random_checkpoint(cfg, a.seed)
    rng = np.random.default_rng(a.seed)
    if a.embedding:
        embed = np.load(a.embedding)
    else:
        embed = rng.standard_normal((cfg["vocab"], cfg["d_model"]), dtype=np.float32)
    if a.tokens:
        prompts = read_prompts(a.tokens)
    else:
        prompts = [rng.integers(0, cfg["vocab"], a.prompt).tolist() for _ in range(a.batch)]
    batch, longest = len(prompts), max(map(len, prompts))
    most = max(longest, a.budget + 64) if a.budget else longest + a.steps
    # protected tokens that a small budget has room for
    recent = 32 if a.budget >= 36 else a.budget // 2
    gen = Generator(cfg, weights, embed, batch, most, budget=a.budget, recent=recent, sinks=min(4, a.budget - recent))
    options = dict(temperature=a.temperature, top_k=a.top_k, top_p=a.top_p, min_p=a.min_p)
    gen.generate(prompts, min(4, a.steps), **options)  # warm-up
    g = torch.Generator(device="cuda").manual_seed(a.seed)
    torch.cuda.synchronize()
    t = time.perf_counter()
    tokens = gen.generate(prompts, a.steps, generator=g, **options).cpu()
    t = time.perf_counter() - t
    print(f"{a.config}: {batch} x {a.steps} tokens in {t * 1e3:.1f} ms ({batch * a.steps / t:.0f} tokens/s, prompts included)")
    if a.tokens:  # one line for each prompt's
        for row in tokens.tolist():
            print(*row)
    else:
        print("first sequence:", tokens[0].tolist())


if __name__ == "__main__":
    main()
