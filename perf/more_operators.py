"""The cases of the operators that serve many requests at once: attention of a
chunk of new tokens over the paged cache, block tables and slot maps built on
the GPU from request lengths, and the requests' own low-rank adapters beside a
shared projection.

Each case names one operator ("op") and its sizes.  ``run`` makes one pass:
with ``own`` false in plain torch operations, with ``own`` true through
``tokamak_b200.ops``.  Sizes are those of the decoders in
``tokamak_b200/configs.py`` (4 heads of 64; 32 query and 8 key-value heads of
64; 64 and 8 heads of 128 for long contexts; rows of 2048, 5632 and 2 x 5632)
or generic.
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
        # four drafted tokens and the one before them, of one conversation on the smallest decoder: latency
        dict(name="chunk-draft", op="chunk", dtype="bf16", B=1, Hq=4, Hkv=4, D=64, page=16, lo=333, hi=333, new=5),
        # a serving batch of the 1B decoder: some sequences bring one token, some a piece of a prompt
        dict(name="chunk-mixed", op="chunk", dtype="bf16", B=32, Hq=32, Hkv=8, D=64, page=16, lo=1, hi=2048, new=100),
        # few drafted tokens on long contexts: the cache is read once, whatever the number of queries
        dict(name="chunk-verify", op="chunk", dtype="bf16", B=8, Hq=64, Hkv=8, D=128, page=64, lo=12001, hi=16384,
             new=6),
        # eight whole prompts of the 1B decoder, from empty caches
        dict(name="chunk-prompt", op="chunk", dtype="f16", B=8, Hq=32, Hkv=8, D=64, page=64, lo=1000, hi=2048,
             new=2048),
        # a piece of 2048 tokens of two long prompts
        dict(name="chunk-long", op="chunk", dtype="bf16", B=2, Hq=64, Hkv=8, D=128, page=64, lo=14001, hi=16384,
             new=2048),
        # the fp32 mode, one key-value head per query head, pages that are no power of two
        dict(name="chunk-f32", op="chunk", dtype="f32", B=3, Hq=16, Hkv=16, D=128, page=48, lo=300, hi=1025, new=129),
        # one token more for each of 64 sequences, some of which need a page for it
        dict(name="pages-step", op="pages", B=64, page=16, hi=2048, new=1, full=0.0),
        # a large batch turns over: sequences leave, prompts come, the pool runs short for the last ones
        dict(name="pages-turn", op="pages", B=1000, page=16, hi=4096, new=128, full=0.2),
        # one token of each of 64 requests over 16 adapters, the adapted projections of a layer of the 1B decoder
        dict(name="lora-step", op="lora", dtype="bf16", B=64, lo=1, hi=1, adapters=16, R=16,
             proj="2048x2048 2048x11264 5632x2048"),
        # prompts of the 1B decoder
        dict(name="lora-prompt", op="lora", dtype="bf16", B=8, lo=1000, hi=2048, adapters=8, R=16,
             proj="2048x2048 2048x11264 5632x2048"),
        # pieces of prompts and single tokens, larger ranks, odd numbers of rows
        dict(name="lora-mixed", op="lora", dtype="f16", B=33, lo=1, hi=100, adapters=64, R=64,
             proj="4096x4096"),
        # the fp32 mode on the smallest decoder
        dict(name="lora-f32", op="lora", dtype="f32", B=8, lo=1, hi=77, adapters=3, R=8, proj="256x256 688x256"),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))

    op = rng.choice(["chunk", "chunk", "chunk", "pages", "lora", "lora"])
    if op == "pages":
        B = log(1, 1000)
        return dict(op=op, B=B, page=rng.choice([16, 32, 48, 64, 128]), hi=log(2, 4096), new=log(1, 128),
                    full=rng.choice([0.0, 0.0, 0.1, 0.5]))
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "lora":
        small = dtype == "f32"
        B = log(1, 64)
        hi = log(1, 512 if small else 2048)
        count = rng.choice([1, 1, 3])
        proj = " ".join(f"{8 * log(16, 704)}x{8 * log(16, 1408)}" for _ in range(count))
        rows = max(B, 8 * 2048 // (2 if small else 1) // count)
        hi = max(1, min(hi, rows // B))
        return dict(op=op, dtype=dtype, B=B, lo=rng.choice([1, hi, max(1, hi // 2)]), hi=hi, adapters=log(1, 64),
                    R=8 * rng.choice([1, 2, 2, 3, 4, 8]), proj=proj)
    D = rng.choice([64, 128])
    Hkv = rng.choice([1, 2, 4, 8])
    Hq = Hkv * rng.choice([1, 2, 4, 7, 8, 16])
    B = log(1, 32)
    new = rng.choice([1, log(2, 16), log(16, 2048)])
    # cached values in all sequences, and products of all queries, within the long listed case's
    hi = log(1, max(1, min(16384, 2 * 16384 * 8 * 128 // (B * Hkv * D))))
    most = 1.5e12 if dtype != "f32" else 5e10
    while 4.0 * B * Hq * D * min(new, hi) * hi > most:
        if new > 1:
            new = max(1, new // 2)
        else:
            hi = max(1, hi // 2)
    lo = rng.choice([1, hi, max(1, hi // 2), 0])
    return dict(op=op, dtype=dtype, B=B, Hq=Hq, Hkv=Hkv, D=D, page=rng.choice([16, 32, 48, 64, 128]), lo=lo, hi=hi,
                new=new)


def spread(case, lo, hi, turn):
    """B whole numbers between lo and hi, spread evenly; a function of the case alone."""
    return [lo + int(((b + 1) * turn) % 1.0 * (hi - lo + 1)) for b in range(case["B"])]


def lengths(case):
    return spread(case, case["lo"], case["hi"], 0.6180339887498949)


def fresh_rows(case):
    """Rows that each sequence of a chunk case brings: up to `new`, one of four sequences a single token."""
    most = spread(case, max(1, case["new"] // 2), case["new"], 0.7548776662466927)
    return [min(n, 1 if b % 4 == 3 else m) for b, (n, m) in enumerate(zip(lengths(case), most))]


def turnover(case):
    """Tokens of each sequence of a page case before and after: each grows by `new` tokens or fewer; where prompts come,
    one of eight sequences is a new one and another one leaves."""
    hi, new = case["hi"], case["new"]
    before = spread(case, 1, hi, 0.6180339887498949)
    after = [min(hi, m + n) for m, n in zip(before, spread(case, 1, new, 0.7548776662466927))]
    if new > 1:
        for b in range(2, case["B"], 8):
            before[b], after[b] = 0, before[b]
        for b in range(5, case["B"], 8):
            after[b] = 0
    return before, after


def projections(case):
    """(columns in, columns out) of each adapted projection."""
    return [tuple(int(n) for n in p.split("x")) for p in case["proj"].split()]


# ------------------------------------------------------------------ inputs
class State:
    pass


def starts(rows):
    return torch.tensor([sum(rows[:b]) for b in range(len(rows) + 1)], dtype=torch.int32, device=DEV)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = State()
    s.case = case

    def normal(*shape, dtype=torch.float32, scale=1.0):
        return torch.empty(*shape, dtype=dtype, device=DEV).normal_(0, scale, generator=g)

    def randint(lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=g, device=DEV, dtype=torch.int32)

    if own:
        from tokamak_b200 import ops
        s.ops = ops
    if case["op"] == "chunk":
        dt = DTYPES[case["dtype"]]
        B, Hq, Hkv, D, page = case["B"], case["Hq"], case["Hkv"], case["D"], case["page"]
        rows = fresh_rows(case)
        per = max(1, -(-case["hi"] // page))
        n_pages = B * per + 3
        s.k = normal(n_pages, Hkv, page, D, dtype=dt)
        s.v = normal(n_pages, Hkv, page, D, dtype=dt)
        s.table = torch.randperm(n_pages, generator=g, device=DEV)[:B * per].view(B, per).int()
        s.lens = torch.tensor(lengths(case), dtype=torch.int32, device=DEV)
        s.q = normal(max(1, sum(rows)), Hq * D, dtype=dt)
        s.row_start = starts(rows)
        # rows of no sequence keep what they hold: the outputs of an earlier layer or batch
        s.out, s.lse = torch.zeros_like(s.q), torch.zeros(s.q.shape[0], Hq, device=DEV)
        if own:
            s.cache = ops.KVCache(s.k, s.v, s.table, s.lens)
            s.workspace = ops.paged_attn_chunk_workspace(s.cache, s.q.shape[0], Hq)
    elif case["op"] == "pages":
        B, page, hi = case["B"], case["page"], case["hi"]
        s.max_pages = -(-hi // page)
        before, after = turnover(case)
        held, want = [-(-n // page) for n in before], [-(-n // page) for n in after]
        grow = sum(max(0, w - h) for h, w in zip(held, want))
        back = sum(max(0, h - w) for h, w in zip(held, want))
        # free pages: enough for all, or for all but a part of the growth
        free = max(0, grow - back) + 5 if case["full"] == 0 else max(0, int(grow * (1 - case["full"])) - back)
        used = sum(held)
        s.n_pages = used + free + 1
        s.lens = torch.tensor(after, dtype=torch.int32, device=DEV)
        held = torch.tensor(held, dtype=torch.int32, device=DEV)
        order = torch.randperm(s.n_pages, generator=g, device=DEV).int()
        # table, pages held, the stack of free pages and its height, in one allocation
        n = B * s.max_pages
        s.meta = torch.full((n + B + s.n_pages + 1,), -1, dtype=torch.int32, device=DEV)
        s.table = s.meta[:n].view(B, s.max_pages)
        s.held, s.free, s.n_free = s.meta[n:n + B], s.meta[n + B:n + B + s.n_pages], s.meta[n + B + s.n_pages:]
        mine = torch.arange(s.max_pages, device=DEV) < held.unsqueeze(1)
        s.table[mine] = order[:used]
        s.held.copy_(held)
        s.free[:free] = order[used:used + free]
        s.n_free.fill_(free)
        s.meta0 = s.meta.clone()
        rows = [max(0, n - m) for m, n in zip(before, after)]
        s.row_start, s.rows = starts(rows), max(1, sum(rows))
    else:
        dt = DTYPES[case["dtype"]]
        rows = lengths(case)
        R, n, T = case["R"], case["adapters"], sum(rows)
        s.row_start = starts(rows) if case["hi"] > 1 else None
        s.adapter = randint(-1, n, case["B"])  # -1: a request without one
        s.scale = 0.5 + torch.rand(n, generator=g, device=DEV)
        s.x = [normal(T, K, dtype=dt) for K, _ in projections(case)]
        s.y = [normal(T, N, dtype=dt) for _, N in projections(case)]
        s.a = [normal(n, K, R, dtype=dt, scale=K ** -0.5) for K, _ in projections(case)]
        s.b = [normal(n, R, N, dtype=dt, scale=R ** -0.5) for _, N in projections(case)]
        s.out = [torch.empty_like(y) for y in s.y]
        if own:
            s.workspace = ops.lora_workspace(T, R)
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    return {"chunk": run_chunk, "pages": run_pages, "lora": run_lora}[s.case["op"]](s)


def run_chunk(s):
    c = s.case
    Hq, Hkv, D = c["Hq"], c["Hkv"], c["D"]
    if own:
        return list(s.ops.paged_attn_chunk(s.cache, s.q, Hq, row_start=s.row_start, out=s.out, lse=s.lse,
                                           workspace=s.workspace))
    G, first = Hq // Hkv, 0
    for b, (n, m) in enumerate(zip(lengths(c), fresh_rows(c))):
        if m == 0:
            continue
        pages = s.table[b, :-(-n // c["page"])].long()
        # row i of the m new ones sees the slots up to its own
        upto = torch.arange(n - m, n, device=DEV).view(m, 1, 1)
        hidden = torch.arange(n, device=DEV) > upto
        for h in range(Hkv):
            k = s.k[pages, h].flatten(0, 1)[:n].float()
            v = s.v[pages, h].flatten(0, 1)[:n].float()
            q = s.q[first:first + m].view(m, Hkv, G, D)[:, h].float()
            x = (q.reshape(m * G, D) @ k.T * D ** -0.5).view(m, G, n).masked_fill_(hidden, -math.inf)
            top = x.amax(-1, keepdim=True)
            x.sub_(top).exp_()
            total = x.sum(-1, keepdim=True)
            o = (x.view(m * G, n) @ v).view(m, G, D) / total
            s.out[first:first + m].view(m, Hkv, G, D)[:, h] = o.to(s.q.dtype)
            s.lse[first:first + m].view(m, Hkv, G)[:, h] = (top + torch.log(total)).squeeze(-1)
        first += m
    return [s.out, s.lse]


def run_pages(s):
    c = s.case
    B, page, most = c["B"], c["page"], s.max_pages
    # the state as the step before left it
    s.meta.copy_(s.meta0)
    if own:
        granted, slots = s.ops.kv_pages(s.table, s.held, s.lens, s.free, s.n_free, page, row_start=s.row_start,
                                        rows=s.rows)
        return [s.table, s.held, s.free, s.n_free, granted, slots]
    want = torch.clamp(-(-s.lens // page), max=most)
    entry = torch.arange(most, device=DEV)
    # surplus pages onto the stack, in the order of the sequences and of their entries
    surplus = (entry >= want.unsqueeze(1)) & (entry < s.held.unsqueeze(1))
    back = s.table[surplus]
    top = s.n_free + torch.arange(back.numel(), device=DEV)
    s.free[top] = back
    s.table[surplus] = -1
    height = s.n_free + back.numel()
    s.held.copy_(torch.minimum(s.held, want))
    # missing ones from its top, for the sequences whose sum of needs it covers
    need = want - s.held
    upto = need.cumsum(0)
    fits = (upto <= height) | (need == 0)
    need = torch.where(fits, need, 0)
    fresh = (entry >= s.held.unsqueeze(1)) & (entry < (s.held + need).unsqueeze(1))
    taken = int(fresh.sum())
    s.table[fresh] = s.free[height - 1 - torch.arange(taken, device=DEV)]
    s.held.add_(need)
    s.n_free.copy_(height - taken)
    # where the new rows go
    row = torch.arange(s.rows, device=DEV)
    start = s.row_start.long()
    seq = (torch.searchsorted(start, row, right=True) - 1).clamp(max=B - 1)
    slot = s.lens[seq] - (start[seq + 1] - row)
    has = (row < start[-1]) & (slot >= 0) & (slot < s.held[seq] * page)
    slot = torch.where(has, slot, 0)
    slots = torch.where(has, s.table[seq, slot // page].long() * page + slot % page, -1)
    return [s.table, s.held, s.free, s.n_free, fits.int(), slots]


def row_adapters(s):
    """The adapter of every row."""
    if s.row_start is None:
        return s.adapter
    return torch.repeat_interleave(s.adapter, (s.row_start[1:] - s.row_start[:-1]).long())


def run_lora(s):
    c = s.case
    if own:
        plan = s.ops.lora_plan(s.adapter, c["adapters"], s.x[0].shape[0], row_start=s.row_start)
        for x, y, a, b, out in zip(s.x, s.y, s.a, s.b, s.out):
            s.ops.lora_add(plan, x, a, b, y, scale=s.scale, out=out, workspace=s.workspace)
        return s.out
    of_row = row_adapters(s)
    groups = [(of_row == i).nonzero().squeeze(1) for i in range(c["adapters"])]
    for x, y, a, b, out in zip(s.x, s.y, s.a, s.b, s.out):
        out.copy_(y)
        for i, rows in enumerate(groups):
            if rows.numel():
                more = x[rows].float() @ a[i].float() @ b[i].float() * s.scale[i]
                out[rows] = (y[rows].float() + more).to(out.dtype)
    return s.out


# ------------------------------------------------------------------ work
def work(case):
    if case["op"] == "pages":
        # lengths, pages held, row starts and answers; an entry of the table and of the stack for each page; the slots
        before, after = turnover(case)
        moved = sum(abs(-(-n // case["page"]) + -m // case["page"]) for m, n in zip(before, after))
        return {"bytes": 20 * case["B"] + 8 * moved + 8 * sum(max(0, n - m) for m, n in zip(before, after)),
                "flops": case["B"]}
    e = BYTES[case["dtype"]]
    if case["op"] == "lora":
        T, R = sum(lengths(case)), case["R"]
        used = min(case["adapters"], case["B"])
        total = {"bytes": 4.0 * case["B"], "flops": 0.0}
        for K, N in projections(case):
            total["bytes"] += T * (K + 2 * N) * e + used * R * (K + N) * e
            total["flops"] += 2.0 * T * R * (K + N)
        return total
    lens, new, Hq, Hkv, D = lengths(case), fresh_rows(case), case["Hq"], case["Hkv"], case["D"]
    pairs = sum(m * (n - m) + m * (m + 1) / 2 for n, m in zip(lens, new))
    read = sum(n for n, m in zip(lens, new) if m)
    return {"bytes": 2 * read * Hkv * D * e + sum(new) * Hq * (2 * D * e + 4) + 4 * -(-read // case["page"]),
            "flops": 4 * pairs * Hq * D}


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "pages":
        return None  # whole numbers
    if case["op"] == "lora":
        outs = []
        row_start = list(range(case["B"] + 1)) if s.row_start is None else s.row_start.tolist()
        for x, y, a, b in zip(s.x, s.y, s.a, s.b):
            out = y.double()
            for q, i in enumerate(s.adapter.tolist()):
                if i >= 0:
                    at = slice(row_start[q], row_start[q + 1])
                    out[at] += float(s.scale[i]) * torch.einsum("tr,rn->tn", torch.einsum("tk,kr->tr", x[at].double(),
                                                                a[i].double()), b[i].double())
            outs.append(out)
        return outs
    Hq, Hkv, D, page = case["Hq"], case["Hkv"], case["D"], case["page"]
    out, lse, r = s.out.double(), s.lse.double(), 0
    for b, (n, m) in enumerate(zip(lengths(case), fresh_rows(case))):
        slots = torch.arange(n, device=DEV)
        at, inside = s.table[b].long()[slots // page], slots % page
        for hq in range(Hq):
            h = hq // (Hq // Hkv)
            k, v = s.k[at, h, inside].double(), s.v[at, h, inside].double()
            q = s.q[r:r + m, hq * D:(hq + 1) * D].double()
            x = torch.einsum("id,jd->ij", q, k) / math.sqrt(D)
            x = torch.where(torch.ones(m, n, dtype=torch.bool, device=DEV).tril(n - m), x, -math.inf)
            lse[r:r + m, hq] = torch.logsumexp(x, 1)
            out[r:r + m, hq * D:(hq + 1) * D] = torch.softmax(x, 1) @ v
        r += m
    return [out, lse]
