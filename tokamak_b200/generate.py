"""Text generation with the Llama-style decoders of ``configs`` on the paged
key-value cache: prompts in one pass, then one token per sequence and step,
the step captured as a CUDA graph.

    python -m tokamak_b200.generate [--config C1|C4] [--checkpoint model.tkmw] [--embedding table.npy]
        [--tokens prompts.txt | --batch 8 --prompt 100] [--steps 64] [--budget 0] [--top-k 50] [--top-p 0.95]
        [--temperature 0.8] [--chunk 512] [--pool 100] [--adapters adapters.npz --adapter-ids 0,-1,1]

Weights come from a TKM1 checkpoint that the engine trained on the same
configuration; the embedding table [vocab, d_model], which the engine takes as
its input rows, from the caller; prompts as token ids, one prompt a line.
Each is random where it is not given.  Prompts may enter in pieces (--chunk),
conversations go on with further ones (Generator.extend), sequences share one
pool of pages (--pool), and each may have a low-rank adapter of its own
(--adapters).  Kernels: tkb_add_rmsnorm_fwd, tkb_gemm, tkb_gemm_swiglu,
tkb_gqa_attn_fwd (whole prompts), tkb_paged_attn_chunk (pieces), tkb_kv_append,
tkb_kv_pages, tkb_paged_attn_decode, tkb_kv_evict, tkb_lora_plan, tkb_lora_add,
tkb_sample_logits.  torch only holds the tensors and looks embeddings up.
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


ADAPTED = ("wqkv", "wo", "wgu", "wd")  # the projections of a layer that may have adapters


class Adapters:
    """Low-rank adapters of a configuration's layers: layers[i][name] = (A [n, in, R], B [n, R, out]) for the projections
    of layer i that have them (names of ADAPTED; wgu is the fused [gate | up] matrix), all of n adapters and one rank, a
    multiple of 8 up to 128; scale [n] is usually alpha / R.  Where a layer has adapters of wgu, its gate and up values are
    rounded to bf16 once more for every sequence, also for those without one: the adapters' sum comes between the matrix
    and the activation."""

    def __init__(self, cfg, layers, scale=None):
        d, F = cfg["d_model"], cfg["ffn"]
        q, kv = cfg["q_heads"] * cfg["head_dim"], cfg["kv_heads"] * cfg["head_dim"]
        sizes = dict(wqkv=(d, q + 2 * kv), wo=(q, d), wgu=(d, 2 * F), wd=(F, d))
        first = next((ab[0] for w in layers for ab in w.values()), None)
        if len(layers) != cfg["layers"] or first is None or np.ndim(first) != 3:
            raise TkbError("Adapters: one dictionary of (A, B) for every layer, one of them at least")
        self.n, _, self.rank = first.shape
        if self.n < 1 or self.rank % 8 or not 8 <= self.rank <= 128:
            raise TkbError(f"Adapters: {self.n} of rank {self.rank}; one at least, and ranks are multiples of 8 up to 128")
        for w in layers:
            for name, (a, b) in w.items():
                if name not in sizes:
                    raise TkbError(f"Adapters: {name} is none of {', '.join(ADAPTED)}")
                K, N = sizes[name]
                if tuple(a.shape) != (self.n, K, self.rank) or tuple(b.shape) != (self.n, self.rank, N):
                    raise TkbError(f"Adapters: {name} is {tuple(a.shape)}, {tuple(b.shape)}, not "
                                   f"{(self.n, K, self.rank)}, {(self.n, self.rank, N)}")
        if scale is not None and np.shape(scale) != (self.n,):
            raise TkbError(f"Adapters: scale is {np.shape(scale)}, not {(self.n,)}")
        self.layers, self.scale = layers, scale

    @classmethod
    def load(cls, cfg, path):
        """From an .npz file of arrays "<layer>.<name>.A", "<layer>.<name>.B" and, if there is one, "scale"."""
        with np.load(path) as f:
            layers = [{} for _ in range(cfg["layers"])]
            for key in f.files:
                part = key.split(".")
                if key == "scale":
                    continue
                if len(part) != 3 or part[2] not in ("A", "B") or part[0] not in map(str, range(len(layers))) or \
                        f"{part[0]}.{part[1]}.{'B' if part[2] == 'A' else 'A'}" not in f.files:
                    raise TkbError(f"{path}: unexpected array {key}")
                if part[2] == "A":
                    layers[int(part[0])][part[1]] = (f[key], f[key[:-1] + "B"])
            return cls(cfg, layers, f["scale"] if "scale" in f.files else None)


class Generator:
    """Generation state of `batch` sequences of at most max_tokens tokens.

    budget: tokens a (sequence, kv head) keeps in the cache (0: all).  Once
    the sequences hold `slack` more, the cache is cut to the budget by
    accumulated attention weight; the newest `recent` tokens and the first
    `sinks` stay.  A decode step adds its token's attention to the weights; a
    prompt longer than the budget starts with that of its last `window` tokens,
    since it may be cut before any step (8 prompts of 2048 tokens on C4: 29 ms,
    and 0.5 ms for each of them).

    chunk: prompts enter in pieces of at most so many tokens a sequence, each
    over what is cached (0: whole).  pool: pages that all sequences share, taken
    as they grow and given back by release (0: each has room for max_tokens).
    adapters: Adapters; self.adapter [batch] is each sequence's, -1 for none."""

    def __init__(self, cfg, checkpoint, embed, batch, max_tokens, page_size=64, budget=0, slack=64, recent=32, sinks=4,
                 device="cuda", window=8, chunk=0, pool=0, adapters=None):
        if window < 1:
            raise TkbError("Generator: window must be positive")
        if chunk < 0 or pool < 0:
            raise TkbError("Generator: chunk and pool must not be negative")
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
        n_pages = pool or batch * pages
        self.chunk, self.pool, self.page_size = chunk, pool, page_size
        if pool:  # the table, the pages that each sequence holds, and the stack of free ones
            self.table = torch.full((batch, pages), -1, dtype=torch.int32, device=device)
            self.pages_held = torch.zeros(batch, dtype=torch.int32, device=device)
            self.free_pages = torch.arange(pool - 1, -1, -1, dtype=torch.int32, device=device)
            self.n_free = torch.full((1,), pool, dtype=torch.int32, device=device)
        else:
            self.table = torch.arange(n_pages, dtype=torch.int32, device=device).view(batch, pages)
        self.adapters = adapters
        self.adapter = torch.full((batch,), -1, dtype=torch.int32, device=device)
        if adapters is not None:
            self.scale = None if adapters.scale is None else \
                torch.as_tensor(adapters.scale, dtype=torch.float32, device=device).contiguous()
            self.low = [{k: tuple(torch.as_tensor(m, dtype=torch.bfloat16, device=device).contiguous() for m in ab)
                         for k, ab in w.items()} for w in adapters.layers]
        self.lens = torch.zeros(batch, dtype=torch.int32, device=device)   # tokens held in the cache
        self.seen = torch.zeros(batch, dtype=torch.int32, device=device)   # tokens so far; -1: takes no part in steps
        self.live = [True] * batch                                         # takes part in steps
        self.step_rows = torch.arange(batch + 1, dtype=torch.int32, device=device)  # row starts of a step's new tokens
        self.caches = []
        for _ in self.layers:
            k, v = (torch.zeros(n_pages, Hkv, page_size, D, dtype=torch.bfloat16, device=device) for _ in "kv")
            meta = torch.zeros(2, n_pages, Hkv, page_size, device=device)
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

    def _forward(self, x, attend, row_start=None):
        """Logits' input rows: the decoder on rows x [rows, d_model] of the sequences (row_start; None: one each);
        attend(layer, qkv) gives the heads' outputs."""
        plan = None
        if self.adapters is not None:
            plan = ops.lora_plan(self.adapter, self.adapters.n, x.shape[0], row_start=row_start)
            low_ws = ops.lora_workspace(x.shape[0], self.adapters.rank, x.device)

        def adapt(i, name, rows, y):
            if plan is not None and name in self.low[i]:
                ops.lora_add(plan, rows, *self.low[i][name], y, scale=self.scale, workspace=low_ws)
            return y

        skip, y = x, None
        for i, w in enumerate(self.layers):
            if i == 0:
                _, y, _ = ops.add_rmsnorm_fwd(x, None, w["norm1"])
            heads = attend(i, adapt(i, "wqkv", y, ops.gemm(y, w["wqkv"])))
            a = adapt(i, "wo", heads, ops.gemm(heads, w["wo"], bias=w["bo"]))
            skip, y, _ = ops.add_rmsnorm_fwd(a, skip, w["norm2"])
            if plan is not None and "wgu" in self.low[i]:  # before the activation
                h = ops.swiglu_fwd(adapt(i, "wgu", y, ops.gemm(y, w["wgu"])), w["bg"], w["bu"])
            else:
                _, h = ops.gemm_swiglu(y, w["wgu"], self.cfg["ffn"], w["bg"], w["bu"])
            f = adapt(i, "wd", h, ops.gemm(h, w["wd"], bias=w["bd"]))
            gain = self.layers[i + 1]["norm1"] if i + 1 < len(self.layers) else self.head["norm"]
            skip, y, _ = ops.add_rmsnorm_fwd(f, skip, gain)
        return y

    def _room(self, held):
        """Refuses lengths that the pool has no pages for.  (The lengths are known here: nothing is read back.)"""
        need = sum(-(-n // self.page_size) for n in held)
        if self.pool and need > self.pool:
            raise TkbError(f"Generator: {need} pages are needed, the pool has {self.pool}")

    def _pages(self, tokens=0):
        """The pages of the sequences as their lengths want them now, about so many tokens after the last time."""
        if self.pool:
            ops.kv_pages(self.table, self.pages_held, self.lens, self.free_pages, self.n_free, self.page_size, tokens=tokens)

    def _take_part(self, live):
        """Which sequences take part in decode steps.  Captured steps follow: they read step_rows and seen.  Those that
        change hold nothing."""
        if live == self.live:
            return
        for b, (was, now) in enumerate(zip(self.live, live)):
            if was != now:
                self.seen[b:b + 1].fill_(0 if now else -1)
        self.live = live
        self.step_rows.copy_(torch.from_numpy(np.concatenate(([0], np.cumsum(live))).astype(np.int32)))

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

    def _check_tokens(self, who, pieces):
        pieces = [p for p in pieces if p]
        if min(map(min, pieces)) < 0 or max(map(max, pieces)) >= self.embed.shape[0]:
            raise TkbError(f"{who}: token ids are 0 to {self.embed.shape[0] - 1}")

    def prefill(self, prompts):
        """Prompts (lists of token ids, none empty) enter the empty caches; returns the logits [batch, vocab]
        after each prompt's last token."""
        n = [len(p) for p in prompts]
        if len(n) != self.batch or min(n) < 1 or max(n) > self.max_tokens:
            raise TkbError("prefill: one prompt of 1 to max_tokens tokens per sequence")
        self._check_tokens("prefill", prompts)
        self._room(n)
        self._take_part([True] * self.batch)
        self.lens.zero_()
        self.seen.zero_()
        left, self.held = sum(self.held), [0] * self.batch
        if self.chunk and max(n) > self.chunk:
            logits = torch.empty(self.batch, self.cfg["vocab"], dtype=torch.float32, device=self.token.device)
            self._pages(left)  # what the sequences held goes back before the first piece
            for at in range(0, max(n), self.chunk):
                pieces = [p[at:at + self.chunk] for p in prompts]
                got, last = self._enter(pieces), [b for b, p in enumerate(pieces) if p and at + self.chunk >= n[b]]
                if last:
                    logits[last] = got[last]
            return logits
        dev = self.token.device
        start = np.concatenate(([0], np.cumsum(n))).astype(np.int32)
        row_start = torch.from_numpy(start).to(dev)
        tokens = torch.tensor([t for p in prompts for t in p], dtype=torch.int64, device=dev)
        ops.kv_lens(self.lens, seen=self.seen, row_start=row_start)
        self._pages(left + sum(n))
        self.held = list(n)
        if self.budget and max(n) > self.budget:
            ends, upto = self._last(start, n)

        def attend(i, qkv):
            rows = self._append(i, qkv, row_start=row_start, full=True)
            if self.budget and max(n) > self.budget:
                self._weigh(i, rows, ends, upto)
            out = torch.empty(rows.shape[0], self.Hq * self.D, dtype=rows.dtype, device=dev)
            for b in range(self.batch):
                part = rows[start[b]:start[b + 1]]
                out[start[b]:start[b + 1]] = ops.gqa_attn_fwd(part, 1, n[b], self.Hq, self.Hkv, self.D)[0][0]
            return out

        y = self._forward(self.embed[tokens], attend, row_start)
        last = y[torch.from_numpy(start[1:].astype(np.int64) - 1).to(dev)]
        return ops.gemm(last, self.head["w"], bias=self.head["b"], out_dtype=torch.float32)

    def _last(self, start, held):
        """For _weigh: the rows of each sequence's last `window` new tokens, the last first, and how many slots each
        sees (0 where there is no such token)."""
        dev, back = self.token.device, np.arange(self.window)[:, None]
        new = np.diff(start)
        ends = np.minimum(np.maximum(start[1:] - 1 - back, start[:-1]), start[-1] - 1)
        upto = np.where(back < new, np.asarray(held) - back, 0)
        return torch.from_numpy(ends.astype(np.int64)).to(dev), torch.from_numpy(upto.astype(np.int32)).to(dev)

    def _enter(self, pieces):
        """New tokens of each sequence (lists, some empty) enter behind what it holds; logits [batch, vocab] after each
        one's last, 0 where there is none."""
        dev, n = self.token.device, [len(p) for p in pieces]
        start = np.concatenate(([0], np.cumsum(n))).astype(np.int32)
        row_start = torch.from_numpy(start).to(dev)
        tokens = torch.tensor([t for p in pieces for t in p], dtype=torch.int64, device=dev)
        ops.kv_lens(self.lens, seen=self.seen, row_start=row_start)
        self._pages(sum(n))
        self.held = [h + m for h, m in zip(self.held, n)]
        workspace = ops.paged_attn_chunk_workspace(self.caches[0], len(tokens), self.Hq)
        if self.budget:
            ends, upto = self._last(start, self.held)

        def attend(i, qkv):
            rows = self._append(i, qkv, row_start=row_start, full=self.budget > 0)
            if self.budget:
                self._weigh(i, rows, ends, upto)
            return ops.paged_attn_chunk(self.caches[i], rows[:, :self.Hq * self.D], self.Hq, row_start=row_start,
                                        workspace=workspace)[0]

        y = self._forward(self.embed[tokens], attend, row_start)
        new = [b for b in range(self.batch) if n[b]]
        last = ops.gemm(y[torch.from_numpy(start[1:].astype(np.int64)[new] - 1).to(dev)], self.head["w"],
                        bias=self.head["b"], out_dtype=torch.float32)
        if len(new) == self.batch:
            return last
        logits = torch.zeros(self.batch, last.shape[1], dtype=last.dtype, device=dev)
        logits[new] = last
        return logits

    def extend(self, pieces):
        """Conversations go on: new tokens of each sequence (lists of token ids, empty for those that bring none) enter
        behind what it holds, in pieces of at most `chunk` tokens; returns the logits [batch, vocab] after each one's last
        (0 for sequences without new tokens).  A sequence that holds nothing starts with them; those that still hold
        nothing take no part in decode steps until they get some.  With a budget, a piece adds the attention of its last
        `window` tokens to the weights."""
        n = [len(p) for p in pieces]
        if len(n) != self.batch or max(n) < 1:
            raise TkbError("extend: a list of tokens per sequence, one of them not empty")
        held = [h + m for h, m in zip(self.held, n)]
        if max(held) > self.max_tokens:
            raise TkbError("extend: more tokens than max_tokens")
        self._check_tokens("extend", pieces)
        self._room(held)
        self._take_part([h > 0 for h in held])
        step = self.chunk or max(n)
        if step >= max(n):
            return self._enter(pieces)
        logits = torch.zeros(self.batch, self.cfg["vocab"], dtype=torch.float32, device=self.token.device)
        for at in range(0, max(n), step):
            part = [p[at:at + step] for p in pieces]
            got, last = self._enter(part), [b for b, p in enumerate(part) if p and at + step >= n[b]]
            if last:
                logits[last] = got[last]
        return logits

    def release(self, sequences):
        """These sequences (indices) end: they hold nothing, their pages go back to the pool, and decode steps leave them out
        until they start again with extend."""
        which = sorted(set(int(b) for b in sequences))
        if which and (which[0] < 0 or which[-1] >= self.batch):
            raise TkbError(f"release: sequences are 0 to {self.batch - 1}")
        left = sum(self.held[b] for b in which)
        for b in which:
            self.lens[b:b + 1].zero_()
            self.held[b] = 0
        self._take_part([a and b not in which for b, a in enumerate(self.live)])
        self._pages(left)

    def decode(self):
        """One step: the tokens in self.token (rows of embed) enter the caches; returns the next logits [batch, vocab].  The
        rows of sequences that have been released, or have had nothing from extend yet, mean nothing: their tokens enter
        nowhere."""
        if not torch.cuda.is_current_stream_capturing():  # a captured step's lengths are its replays'
            held = [n + a for n, a in zip(self.held, self.live)]
            self._room(held)
            self.held = held
        ops.kv_lens(self.lens, seen=self.seen, row_start=self.step_rows)
        self._pages()

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
        self._pages(sum(max(0, n - self.budget) for n in self.held))
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
        grown = [len(p) + steps - 1 for p in prompts]
        self._room([min(n, max(len(p), self.budget + self.slack)) if self.budget else n for n, p in zip(grown, prompts)])
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
    ap.add_argument("--chunk", type=int, default=0, help="prompts enter in pieces of so many tokens (0: whole)")
    ap.add_argument("--pool", type=int, default=0, help="pages of 64 tokens that all sequences share (0: room for all)")
    ap.add_argument("--adapters", help=".npz file of low-rank adapters (Adapters.load)")
    ap.add_argument("--adapter-ids", help="the prompts' adapters, separated by commas, -1 for none (default: in turn)")
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
    adapters = Adapters.load(cfg, a.adapters) if a.adapters else None
    gen = Generator(cfg, weights, embed, batch, most, budget=a.budget, recent=recent, sinks=min(4, a.budget - recent),
                    chunk=a.chunk, pool=a.pool, adapters=adapters)
    if adapters is not None:
        ids = [b % adapters.n for b in range(batch)]
        if a.adapter_ids:
            ids = [int(i) for i in a.adapter_ids.split(",")]
        if len(ids) != batch or min(ids) < -1 or max(ids) >= adapters.n:
            raise TkbError(f"--adapter-ids: one of -1 to {adapters.n - 1} for each of {batch} prompts")
        gen.adapter.copy_(torch.tensor(ids, dtype=torch.int32))
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
