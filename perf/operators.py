"""The cases of the generation operators: a paged key-value cache, the
attention that reads it, its eviction, and sampling.

Each case names one operator ("op") and its sizes.  ``run`` makes one pass:
with ``own`` false in plain torch operations, with ``own`` true through
``tokamak_b200.ops``.  Sizes are those of the decoders in
``tokamak_b200/configs.py`` (4 heads of 64; 32 query and 8 key-value heads of
64; 64 and 8 heads of 128 for long contexts; vocabulary 32000) or generic.
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # the first tokens of one conversation on the smallest decoder: latency
        dict(name="decode-one", op="decode", dtype="bf16", B=1, Hq=4, Hkv=4, D=64, page=16, lo=77, hi=77, weights=False),
        # a serving batch of the 1B decoder, every sequence of another length
        dict(name="decode-batch", op="decode", dtype="bf16", B=32, Hq=32, Hkv=8, D=64, page=16, lo=1, hi=2048,
             weights=False),
        # long contexts, with the attention weights kept for the eviction
        dict(name="decode-long", op="decode", dtype="bf16", B=16, Hq=64, Hkv=8, D=128, page=64, lo=15001, hi=16384,
             weights=True),
        # the fp32 mode, one key-value head per query head, pages that are no power of two
        dict(name="decode-f32", op="decode", dtype="f32", B=3, Hq=16, Hkv=16, D=128, page=48, lo=511, hi=4097,
             weights=True),
        # one token of each of 64 sequences enters the cache
        dict(name="append-step", op="append", dtype="bf16", B=64, Hq=32, Hkv=8, D=64, page=16, lo=1, hi=2048, rows=1,
             qknorm=False, bias=True, rope_scale=1.0, full=False),
        # eight prompts enter the cache at once; the packed rows go on to the prompt's own attention
        dict(name="append-prompt", op="append", dtype="f16", B=8, Hq=64, Hkv=8, D=128, page=64, lo=1000, hi=2048,
             rows=2048, qknorm=True, bias=True, rope_scale=8.0, full=True),
        # a batch that has grown some tokens over its budget
        dict(name="evict-step", op="evict", dtype="bf16", B=32, Hkv=8, D=64, page=16, lo=1000, hi=1088, budget=1024,
             recent=128, sinks=4),
        # long prompts cut to an eighth
        dict(name="evict-prompt", op="evict", dtype="f16", B=4, Hkv=8, D=128, page=64, lo=12001, hi=16384, budget=2048,
             recent=256, sinks=4),
        # the next token of one conversation: latency
        dict(name="sample-one", op="sample", dtype="bf16", B=1, V=32000, top_k=50, top_p=0.95, min_p=0.0),
        # a serving batch; every request has its own temperature and top-k
        dict(name="sample-batch", op="sample", dtype="f32", B=64, V=32000, top_k=40, top_p=0.9, min_p=0.02),
        # a large vocabulary and a large batch, nucleus only
        dict(name="sample-wide", op="sample", dtype="bf16", B=512, V=131072, top_k=0, top_p=0.9, min_p=0.0),
        # a small odd vocabulary, no truncation but min-p
        dict(name="sample-odd", op="sample", dtype="f16", B=200, V=999, top_k=0, top_p=1.0, min_p=0.05),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["decode", "decode", "append", "evict", "sample", "sample"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "sample":
        V = log(500, 131072)
        B = max(1, min(log(1, 512), (512 * 131072 * 2) // (V * BYTES[dtype])))
        return dict(op=op, dtype=dtype, B=B, V=V, top_k=rng.choice([0, 1, log(2, 500)]),
                    top_p=rng.choice([1.0, round(rng.uniform(0.3, 0.99), 3)]),
                    min_p=rng.choice([0.0, round(rng.uniform(0.005, 0.2), 3)]))
    D = rng.choice([64, 128])
    Hkv = rng.choice([1, 2, 4, 8])
    page = rng.choice([16, 32, 48, 64, 128])
    B = log(1, 64)
    # cached values in all sequences: at most a third of the longest listed case's
    most = 16 * 16384 * 8 * 128 // 3
    top = max(2, min(16384, most // (B * Hkv * D * (BYTES[dtype] // 2))))
    hi = log(2, top)
    lo = rng.choice([1, hi, max(1, hi // 2)])
    base = dict(op=op, dtype=dtype, B=B, Hkv=Hkv, D=D, page=page, lo=lo, hi=hi)
    if op == "decode":
        if rng.random() < 0.2:
            base["lo"] = 0  # sequences that hold nothing yet among the others
        return dict(base, Hq=Hkv * rng.choice([1, 2, 4, 7, 8, 16]), weights=rng.random() < 0.4)
    if op == "append":
        rows = rng.choice([1, 1, hi])
        Hq = Hkv * rng.choice([1, 4, 8])
        if rows > 1 and B * hi * (Hq + 2 * Hkv) * D > 8 * 2048 * 80 * 128:
            rows = 1
        return dict(base, Hq=Hq, rows=rows, qknorm=rng.random() < 0.5, bias=rng.random() < 0.5,
                    rope_scale=rng.choice([1.0, 8.0]), full=rows > 1)
    budget = max(1, min(hi, log(1, hi)))
    recent = rng.randint(0, budget // 2)
    return dict(base, budget=budget, recent=recent, sinks=rng.randint(0, min(4, budget - recent)))


def lengths(case):
    """Sequence lengths between lo and hi, spread evenly; a function of the case alone."""
    lo, hi = case["lo"], case["hi"]
    return [lo + int(((b + 1) * 0.6180339887498949) % 1.0 * (hi - lo + 1)) for b in range(case["B"])]


def fresh_rows(case):
    """Rows that each sequence of an append case brings: one, or its whole prompt."""
    return [min(n, case["rows"]) for n in lengths(case)]


# ------------------------------------------------------------------ inputs
ROPE = dict(theta=500000.0, low=1.0, high=4.0, octx=8192.0)


def rope_frequencies(D, scale):
    """Angle per position of each pair i of a head: theta^(-i/D), with the long
    wavelengths stretched by `scale` (smoothly between octx/high and octx/low)."""
    freq = []
    for i in range(D // 2):
        f = ROPE["theta"] ** (-i / D)
        if scale > 1.0:
            turns = ROPE["octx"] * f / (2 * math.pi)
            if turns < ROPE["low"]:
                f /= scale
            elif turns <= ROPE["high"]:
                f *= 1 - (turns - ROPE["low"]) / (ROPE["high"] - ROPE["low"]) * (1 - 1 / scale)
        freq.append(f)
    return torch.tensor(freq, dtype=torch.float64, device=DEV)


class State:
    pass


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = State()
    s.case = case
    dt = DTYPES[case["dtype"]]

    def normal(*shape, dtype=torch.float32, scale=1.0):
        x = torch.empty(*shape, dtype=dtype, device=DEV)
        return x.normal_(0, scale, generator=g)

    def uniform(*shape):
        return torch.rand(*shape, generator=g, device=DEV)

    if case["op"] == "sample":
        B, V = case["B"], case["V"]
        s.logits = normal(B, V, dtype=dt, scale=2.0)
        s.u = uniform(B)
        s.temperature = 0.5 + uniform(B)
        if B > 8:
            s.temperature[::8] = 0.0  # greedy requests among the others
        s.top_k = s.top_p = s.min_p = None
        if case["top_k"]:
            s.top_k = torch.randint(1, 2 * case["top_k"], (B,), generator=g, device=DEV, dtype=torch.int32)
        if case["top_p"] < 1:
            s.top_p = torch.full((B,), case["top_p"], device=DEV)
        if case["min_p"] > 0:
            s.min_p = torch.full((B,), case["min_p"], device=DEV)
        if own:
            from tokamak_b200 import ops
            s.ops = ops
        return s

    B, Hkv, D, page = case["B"], case["Hkv"], case["D"], case["page"]
    lens = lengths(case)
    per = -(-case["hi"] // page)
    n_pages = B * per + 3
    s.k = normal(n_pages, Hkv, page, D, dtype=dt)
    s.v = normal(n_pages, Hkv, page, D, dtype=dt)
    s.table = torch.randperm(n_pages, generator=g, device=DEV)[:B * per].view(B, per).int()
    s.lens = torch.tensor(lens, dtype=torch.int32, device=DEV)
    # positions and accumulated weights of the slots, in one allocation
    s.meta = torch.zeros(2, n_pages, Hkv, page, dtype=torch.int32, device=DEV)
    s.pos, s.weight = s.meta[0], s.meta[1].view(torch.float32)
    if case["op"] == "decode":
        s.q = normal(B, case["Hq"] * D, dtype=dt)
        if case["weights"]:
            s.weight.copy_(uniform(n_pages, Hkv, page))
    elif case["op"] == "append":
        rows = fresh_rows(case)
        s.C = (case["Hq"] + 2 * Hkv) * D
        s.qkv = normal(sum(rows), s.C, dtype=dt)
        s.row_start = None
        if case["rows"] > 1:
            s.row_start = torch.tensor([sum(rows[:b]) for b in range(B + 1)], dtype=torch.int32, device=DEV)
        # sequences whose cache has evicted tokens before have seen more than they hold
        s.seen = s.lens + (torch.randint(0, 4096, (B,), generator=g, device=DEV, dtype=torch.int32)
                           if case["rows"] == 1 else 0)
        s.bias = normal(s.C, scale=0.1) if case["bias"] else None
        s.gain = 1 + normal((case["Hq"] + Hkv) * D, scale=0.02) if case["qknorm"] else None
        s.freq = rope_frequencies(D, case["rope_scale"])
    else:
        # heavy-tailed weights; older tokens lie in any order below the newest `budget` / 16
        L = per * page
        s.seen = s.lens * 2
        fresh = case["budget"] // 16
        slot = torch.arange(L, device=DEV)
        old = slot < (s.lens.view(B, 1, 1) - fresh)
        order = torch.where(old, uniform(B, Hkv, L), 1.0 + slot).argsort(-1)
        pos = order + (s.seen - s.lens).view(B, 1, 1)
        w = normal(B, Hkv, L).mul_(2.0).exp_()
        t = s.table.long()
        s.pos[t] = pos.view(B, Hkv, per, page).transpose(1, 2).int()
        s.weight[t] = w.view(B, Hkv, per, page).transpose(1, 2)
        s.meta0 = s.meta.clone()
    if own:
        from tokamak_b200 import ops
        s.ops = ops
        s.cache = ops.KVCache(s.k, s.v, s.table, s.lens, pos=s.pos, weight=s.weight)
        if case["op"] == "decode":
            s.workspace = ops.paged_attn_workspace(s.cache, case["Hq"], case["weights"])
        elif case["op"] == "evict":
            s.workspace = ops.kv_evict_workspace(s.cache)
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    return {"decode": run_decode, "append": run_append, "evict": run_evict, "sample": run_sample}[s.case["op"]](s)


def by_sequence(pages, table):
    """[pages][heads][page]... and [B][per] -> [B][heads][per * page]..."""
    return pages[table.long()].movedim(2, 1).flatten(2, 3)


def run_decode(s):
    c = s.case
    B, Hq, Hkv, D = c["B"], c["Hq"], c["Hkv"], c["D"]
    if own:
        out, lse = s.ops.paged_attn_decode(s.cache, s.q, Hq, accumulate=c["weights"], workspace=s.workspace)
        return [out, lse, s.weight] if c["weights"] else [out, lse]
    k, v = by_sequence(s.k, s.table).float(), by_sequence(s.v, s.table).float()
    L = k.shape[2]
    held = torch.arange(L, device=DEV) < s.lens.view(B, 1, 1)
    q = s.q.float().view(B, Hkv, Hq // Hkv, D)
    x = (q @ k.transpose(-1, -2)) * D ** -0.5
    x = x.masked_fill(~held.unsqueeze(2), -math.inf)
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total > 0, total, 1.0)
    v = torch.where(held.unsqueeze(-1), v, 0.0)
    out = (p @ v).to(s.q.dtype).view(B, Hq * D)
    lse = (top + torch.log(total)).view(B, Hq)
    if not c["weights"]:
        return [out, lse]
    per, page = s.table.shape[1], c["page"]
    s.weight.index_put_((s.table.long(),), p.sum(2).view(B, Hkv, per, page).transpose(1, 2), accumulate=True)
    return [out, lse, s.weight]


def run_append(s):
    c = s.case
    Hq, Hkv, D, page = c["Hq"], c["Hkv"], c["D"], c["page"]
    if own:
        out = s.ops.kv_append(s.cache, s.qkv, Hq, seen=s.seen, row_start=s.row_start, bias=s.bias, qk_gain=s.gain,
                              qknorm=c["qknorm"], rope_scale=c["rope_scale"], full=c["full"], **ROPE)
        return [out, s.k, s.v, s.pos]
    T = s.qkv.shape[0]
    row = torch.arange(T, device=DEV)
    if s.row_start is None:
        seq, back = row, torch.ones_like(row)
    else:
        start = s.row_start.long()
        seq = torch.searchsorted(start, row, right=True) - 1
        back = start[seq + 1] - row
    slot, pos = s.lens[seq] - back, s.seen[seq] - back
    x = s.qkv.float()
    if s.bias is not None:
        x = x + s.bias
    x = x.view(T, Hq + 2 * Hkv, D)
    qk = x[:, :Hq + Hkv]
    if c["qknorm"]:
        qk = qk * torch.rsqrt((qk * qk).mean(-1, keepdim=True) + 1e-5) * s.gain.view(Hq + Hkv, D)
    angle = pos.double()[:, None] * s.freq  # large angles: reduced in 64 bits before the 32-bit sine
    angle = (angle - 2 * math.pi * torch.floor(angle / (2 * math.pi))).float().unsqueeze(1)
    cs, sn = torch.cos(angle), torch.sin(angle)
    a, b = qk[..., 0::2], qk[..., 1::2]
    qk = torch.stack((a * cs - b * sn, a * sn + b * cs), -1).flatten(-2)
    x = torch.cat((qk, x[:, Hq + Hkv:]), 1).to(s.qkv.dtype)
    at = s.table.long()[seq, slot // page]
    inside = slot % page
    s.k[at, :, inside] = x[:, Hq:Hq + Hkv]
    s.v[at, :, inside] = x[:, Hq + Hkv:]
    s.pos[at, :, inside] = pos.int()[:, None].expand(T, Hkv)
    s.weight[at, :, inside] = 0.0
    out = x.view(T, -1) if c["full"] else x[:, :Hq].reshape(T, -1)
    return [out, s.k, s.v, s.pos]


def run_evict(s):
    c = s.case
    B, Hkv, page, budget = c["B"], c["Hkv"], c["page"], c["budget"]
    # the positions and weights as the decode steps since the last eviction left them
    s.meta.copy_(s.meta0)
    if own:
        s.ops.kv_evict(s.cache, budget, s.seen, recent=c["recent"], sinks=c["sinks"], workspace=s.workspace)
        return [s.k, s.v, s.pos, s.weight]
    w, pos = by_sequence(s.weight, s.table), by_sequence(s.pos, s.table)
    L = w.shape[2]
    slot = torch.arange(L, device=DEV).expand(B, Hkv, L)
    held = slot < s.lens.view(B, 1, 1)
    safe = (pos >= (s.seen - c["recent"]).view(B, 1, 1)) | (pos < c["sinks"])
    worth = torch.where(safe, math.inf, w).masked_fill(~held, -math.inf)
    order = worth.sort(dim=-1, descending=True, stable=True).indices
    kept = torch.zeros_like(held).scatter_(2, order[..., :budget], True) & held
    over = (s.lens > budget).view(B, 1, 1)
    hole = over & ~kept & (slot < budget)
    mover = over & kept & (slot >= budget)
    b, h, to = hole.nonzero(as_tuple=True)
    _, _, frm = mover.nonzero(as_tuple=True)
    table = s.table.long()
    dst, src = (table[b, to // page], h, to % page), (table[b, frm // page], h, frm % page)
    for pages in (s.k, s.v, s.pos, s.weight):
        pages[dst] = pages[src]
    return [s.k, s.v, s.pos, s.weight]


def scaled(total, part):
    """(floor, whether exact) of total * part / 2^32 for whole numbers total < 2^56, part < 2^32."""
    low = total & 0xFFFFFF
    q = ((total >> 24) * part + ((low * part) >> 24)) >> 8
    return q, (total * part - (q << 32)) == 0


def run_sample(s):
    if own:
        return list(s.ops.sample_logits(s.logits, s.u, temperature=s.temperature, top_k=s.top_k, top_p=s.top_p,
                                        min_p=s.min_p))
    B, V = s.logits.shape
    x = s.logits.float()
    x = torch.where(torch.isnan(x), -math.inf, x)
    greedy = ~(s.temperature > 0)
    inv = torch.where(greedy, 1.0, 1.0 / s.temperature).unsqueeze(1)
    top = x.amax(1, keepdim=True)
    z = torch.where(x == top, 0.0, (top - x) * inv)
    # whole weights: their sums do not depend on the order of the terms
    w = torch.round(torch.exp(-z).double() * 2.0 ** 31).long().masked_fill(top == -math.inf, 0)
    order = x.sort(dim=1, descending=True, stable=True).indices
    sw = w.gather(1, order)
    rank = torch.arange(V, device=DEV).expand(B, V)
    keep = sw > 0
    if s.top_k is not None:
        keep &= (rank < s.top_k.unsqueeze(1)) | (s.top_k.unsqueeze(1) <= 0)
    if s.top_p is not None:
        sw_k = torch.where(keep, sw, 0)
        before = sw_k.cumsum(1) - sw_k
        part = (s.top_p.double() * 2.0 ** 32).long().clamp(0, 2 ** 32 - 1)
        bound, whole = scaled(sw_k.sum(1), part)
        bound = torch.where(whole, bound, bound + 1).unsqueeze(1)
        keep &= (before < bound) | (rank == 0) | (s.top_p >= 1).unsqueeze(1)
    if s.min_p is not None:
        keep &= sw >= torch.ceil(s.min_p.double() * 2.0 ** 31).long().clamp(0, 2 ** 31).unsqueeze(1)
    keep &= (rank == 0) | ~greedy.unsqueeze(1)
    w = torch.where(torch.zeros_like(keep).scatter_(1, order, keep), w, 0)
    upto = w.cumsum(1)
    total = upto[:, -1]
    target, _ = scaled(total, (s.u.double() * 2.0 ** 32).long().clamp(0, 2 ** 32 - 1))
    token = (upto <= target.unsqueeze(1)).sum(1)
    none = total == 0
    at = token.clamp(max=V - 1).unsqueeze(1)
    logprob = -z.gather(1, at).squeeze(1) - torch.log(total.float() * 2.0 ** -31)
    logprob = torch.where(greedy, 0.0, logprob)
    return [torch.where(none, -1, token).int(), torch.where(none, -math.inf, logprob), keep.sum(1).int()]


# ------------------------------------------------------------------ work
def work(case):
    e = BYTES[case["dtype"]]
    if case["op"] == "sample":
        return {"bytes": case["B"] * (case["V"] * e + 32), "flops": case["B"] * case["V"] * 8}
    lens, Hkv, D = lengths(case), case["Hkv"], case["D"]
    n = sum(lens)
    if case["op"] == "decode":
        io = case["B"] * case["Hq"] * (2 * D * e + 4) + 4 * -(-n // case["page"])
        return {"bytes": 2 * n * Hkv * D * e + io + (8 * n * Hkv if case["weights"] else 0),
                "flops": 4 * n * case["Hq"] * D}
    if case["op"] == "append":
        rows, C = sum(fresh_rows(case)), (case["Hq"] + 2 * Hkv) * D
        out = C if case["full"] else case["Hq"] * D
        return {"bytes": rows * (C * e + out * e + Hkv * (2 * D * e + 8)), "flops": rows * C * 8}
    total = 0.0
    for m in lens:
        if m <= case["budget"]:
            continue
        # tokens kept at `budget` or above: the protected newest, and their share of the heavy ones
        fresh = min(case["budget"] // 16, case["recent"])
        above = m - case["budget"]
        moved = min(fresh, above) + (case["budget"] - fresh) * max(0, above - fresh) / (m - fresh)
        total += Hkv * (8 * m + moved * 2 * (2 * D * e + 8))
    return {"bytes": total + 4 * case["B"], "flops": n * Hkv}


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "decode":
        B, Hq, Hkv, D, page = case["B"], case["Hq"], case["Hkv"], case["D"], case["page"]
        out = torch.zeros(B, Hq, D, dtype=torch.float64, device=DEV)
        lse = torch.full((B, Hq), -math.inf, dtype=torch.float64, device=DEV)
        weight = s.weight.double()
        for b, n in enumerate(lengths(case)):
            for h in range(Hkv):
                pages = s.table[b, :-(-n // page)].long()
                k = s.k[pages, h].reshape(-1, D)[:n].double()
                v = s.v[pages, h].reshape(-1, D)[:n].double()
                G = Hq // Hkv
                q = s.q[b].view(Hq, D)[h * G:(h + 1) * G].double()
                x = q @ k.T / math.sqrt(D)
                lse[b, h * G:(h + 1) * G] = torch.logsumexp(x, 1)
                p = torch.softmax(x, 1)
                out[b, h * G:(h + 1) * G] = p @ v
                slots = torch.arange(n, device=DEV)
                weight[pages[slots // page], h, slots % page] += p.sum(0)
        got = [out.view(B, Hq * D), lse]
        return got + [weight] if case["weights"] else got
    if case["op"] == "append":
        Hq, Hkv, D, page = case["Hq"], case["Hkv"], case["D"], case["page"]
        k, v, outs, r = s.k.double(), s.v.double(), [], 0
        half = D // 2
        for b, (n, m) in enumerate(zip(lengths(case), fresh_rows(case))):
            x = s.qkv[r:r + m].double()
            r += m
            if s.bias is not None:
                x = x + s.bias.double()
            x = x.view(m, Hq + 2 * Hkv, D)
            if s.gain is not None:
                y = x[:, :Hq + Hkv]
                y = y / torch.sqrt(y.pow(2).mean(2, keepdim=True) + 1e-5) * s.gain.double().view(1, Hq + Hkv, D)
                x = torch.cat((y, x[:, Hq + Hkv:]), 1)
            at = torch.arange(m, device=DEV, dtype=torch.float64) + int(s.seen[b]) - m
            turn = torch.polar(torch.ones(m, half, dtype=torch.float64, device=DEV), at[:, None] * s.freq[None])
            z = torch.view_as_complex(x[:, :Hq + Hkv].reshape(m, Hq + Hkv, half, 2).contiguous()) * turn[:, None]
            x = torch.cat((torch.view_as_real(z).reshape(m, Hq + Hkv, D), x[:, Hq + Hkv:]), 1)
            slots = torch.arange(n - m, n, device=DEV)
            pages = s.table[b].long()[slots // page]
            k[pages, :, slots % page] = x[:, Hq:Hq + Hkv]
            v[pages, :, slots % page] = x[:, Hq + Hkv:]
            outs.append(x.reshape(m, -1) if case["full"] else x[:, :Hq].reshape(m, -1))
        return [torch.cat(outs), k, v, None]
    if case["op"] == "evict":
        k, v, weight = s.k.double(), s.v.double(), s.weight.double()
        page, budget = case["page"], case["budget"]
        for b, n in enumerate(lengths(case)):
            if n <= budget:
                continue
            pages, slots = s.table[b].long(), torch.arange(n, device=DEV)
            for h in range(case["Hkv"]):
                at, inside = pages[slots // page], slots % page
                pos, w = s.pos[at, h, inside], s.weight[at, h, inside].double()
                w[(pos >= int(s.seen[b]) - case["recent"]) | (pos < case["sinks"])] = math.inf
                best = torch.argsort(-w, stable=True)[:budget].sort().values
                src = best[best >= budget]
                dst = slots[:budget][~torch.isin(slots[:budget], best)]
                for t in (k, v, weight):
                    t[pages[dst // page], h, dst % page] = t[pages[src // page], h, src % page]
        return [k, v, None, weight]
    # the token itself is a whole number; its probability comes from the definition in 64 bits
    B, V = s.logits.shape
    token, logprob, kept = [], [], []
    for b in range(B):
        x = s.logits[b].double()
        if not s.temperature[b] > 0:
            logprob.append(0.0)
            continue
        z = (x.max() - x) / float(s.temperature[b])
        w = torch.round(torch.exp(-z) * 2.0 ** 31)
        order = torch.argsort(-x, stable=True)
        sw = w[order]
        n = int((sw > 0).sum())
        if s.top_k is not None:
            n = min(n, int(s.top_k[b]))
        cum = sw[:n].cumsum(0)
        m = n
        if s.top_p is not None:
            m = int((cum - sw[:n] < float(s.top_p[b]) * cum[-1]).sum())
        if s.min_p is not None:
            m = min(m, int((sw[:n] >= float(s.min_p[b]) * 2.0 ** 31).sum()))
        chosen = order[:max(m, 1)].sort().values
        upto = w[chosen].cumsum(0)
        at = chosen[int((upto <= torch.floor(upto[-1] * float(s.u[b]))).sum())]
        logprob.append(float(-z[at] - torch.log(upto[-1] * 2.0 ** -31)))
    return [None, torch.tensor(logprob, dtype=torch.float64, device=DEV), None]
