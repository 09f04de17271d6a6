"""Operators over device buffers for serving many continuations of one prompt, as cases whose time is measured.

Four of them: attention of a batch whose lanes share their first pages (the shared keys read once for all lanes), verification of
drafted tokens against the target's distribution from given random numbers, copies of whole or partly filled pages (forks, moves), and
the gathering of kept tokens into the first rows of a lane's pages.  Head layouts, vocabularies, pages and lengths are those of the
benchmark's model shapes and workloads.

`run` computes them in elementary torch operations, or, where `own` is true, through the framework's entry points.  `exact` states them
again in 64 bits, lane by lane.
"""
import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}

_device_ops = None


def framework():
    """The framework's operators over device buffers, imported with the first call."""
    global _device_ops
    if _device_ops is None:
        import importlib

        import __graft_entry__ as entry

        entry.load_package()
        _device_ops = importlib.import_module(entry.PKG_NAME + ".device_ops")
    return _device_ops

# q heads, kv heads, head size, layers and vocabulary of the benchmark's model shapes
SHAPES = {
    "tinyllama": dict(q_heads=32, kv_heads=4, dim=64, layers=22, vocab=32000),
    "smollm3": dict(q_heads=16, kv_heads=4, dim=128, layers=36, vocab=128256),
    "qwen3": dict(q_heads=32, kv_heads=8, dim=128, layers=36, vocab=151936),
    "gemma2": dict(q_heads=16, kv_heads=8, dim=256, layers=42, vocab=256000),
    "qwen3moe": dict(q_heads=32, kv_heads=4, dim=128, layers=48, vocab=151936),
}


def attention_case(name, shape, lanes, rows, shared, low, high, dtype="f16", ragged=False, window=0, softcap=0.0, page=16):
    s = SHAPES[shape]
    return dict(name=name, op="attention", lanes=lanes, rows=rows, shared=shared, low=low, high=high, dtype=dtype, ragged=ragged, window=window,
                softcap=softcap, page=page, q_heads=s["q_heads"], kv_heads=s["kv_heads"], dim=s["dim"])


def verify_case(name, lanes, drafts, vocab, top_k, top_p, dtype="f32", given=False, greedy=0, ragged=False):
    return dict(name=name, op="verify", lanes=lanes, drafts=drafts, vocab=vocab, top_k=top_k, top_p=top_p, dtype=dtype, given=given, greedy=greedy,
                ragged=ragged)


def copy_case(name, shape, pages, copies, tails, page=16, dtype="f16"):
    s = SHAPES[shape]
    return dict(name=name, op="copy", pages=pages, copies=copies, tails=tails, page=page, dtype=dtype, layers=s["layers"], kv_heads=s["kv_heads"], dim=s["dim"])


def gather_case(name, shape, lanes, context, low, high, first, page=16, dtype="f16"):
    s = SHAPES[shape]
    return dict(name=name, op="gather", lanes=lanes, context=context, low=low, high=high, first=first, page=page, dtype=dtype, layers=s["layers"],
                kv_heads=s["kv_heads"], dim=s["dim"])


def listed():
    return [
        # four samples of one short prompt, a few tokens in: launches and latency are everything
        attention_case("samples-4", "tinyllama", 4, 1, 512, 1, 60),
        # the benchmark's prefix workload in the middle of its decoding: 32 requests behind 2048 shared tokens
        attention_case("prefix-32", "qwen3", 32, 1, 2048, 17, 500),
        # a batch of agents behind one long set of instructions, four drafts each being verified, some with fewer
        attention_case("drafts-24", "smollm3", 24, 5, 16384, 100, 1500, dtype="bf16", ragged=True),
        # wide heads with capped scores, own parts as long as the shared one
        attention_case("capped-40", "gemma2", 40, 1, 2048, 300, 4000, softcap=50.0),
        # many questions to one long document
        attention_case("document-128", "qwen3", 128, 1, 32768, 20, 700),
        # one user's chat with drafts looked up in the prompt: a single lane
        verify_case("lookup-1", 1, 4, 32000, 40, 0.95),
        # a batch of looked-up drafts, lanes with fewer of them, every eighth lane greedy
        verify_case("lookup-40", 40, 6, 128256, 64, 0.9, greedy=8, ragged=True),
        # drafts of a smaller model with their whole distributions, nothing cut off
        verify_case("draft-model-64", 64, 4, 151936, 0, 1.0, given=True),
        # samples forked in the middle of a page: each gets its own copy of the rows that are filled
        copy_case("fork-8", "tinyllama", 400, 8, True),
        # the pool's live pages moved together
        copy_case("move-600", "qwen3", 1400, 600, False),
        # a lane keeps the drafted branch that was accepted
        gather_case("branch-2", "tinyllama", 2, 200, 4, 6, 180),
        # long contexts thinned out to their first, last and most attended tokens
        gather_case("thin-16", "smollm3", 16, 2000, 500, 700, 0),
    ]


def spread(low, high, n):
    """n whole numbers from low to high, even over their logarithm."""
    if n == 1:
        return [int(round(math.sqrt(low * high)))]
    return [int(round(low * (high / low) ** (i / (n - 1)))) for i in range(n)]


def log_int(rng, low, high):
    return int(round(low * (high / low) ** rng.random()))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "verify", "verify", "copy", "gather"])
    shape = rng.choice(sorted(SHAPES))
    if op == "attention":
        page = rng.choice([16, 16, 32, 64])
        c = attention_case("", shape, log_int(rng, 1, 128), rng.choice([1, 1, 2, 3, 5, 8]), 0, 1, log_int(rng, 1, 3000), dtype=rng.choice(["f16", "bf16"]),
                           ragged=rng.random() < 0.4, window=rng.choice([0, 0, 0, 1000, 4096]), softcap=rng.choice([0.0, 0.0, 50.0]), page=page)
        c["shared"] = log_int(rng, 1, 32768 // page) * page if rng.random() < 0.95 else 0
        c["low"] = log_int(rng, 1, c["high"])
        if work(c)["flops"] > 0.9 * work(listed()[4])["flops"]:
            c["lanes"], c["rows"] = max(1, c["lanes"] // 4), max(1, c["rows"] // 4)
        while c["lanes"] * c["rows"] * (c["high"] + page) * c["kv_heads"] * c["dim"] > 4e8:  # what the plain form lays out
            c["lanes"] = max(1, c["lanes"] // 2)
            c["high"] = max(1, c["high"] // 2)
            c["low"] = min(c["low"], c["high"])
    elif op == "verify":
        vocab = rng.choice([SHAPES[shape]["vocab"], SHAPES[shape]["vocab"], log_int(rng, 500, 256000)])
        top_k = rng.choice([0, 1, 10, 40, 200, 1000])
        c = verify_case("", log_int(rng, 1, 64), rng.choice([1, 2, 3, 4, 6, 8]), vocab, min(top_k, vocab), rng.choice([1.0, 0.9, 0.5]) if top_k else 1.0,
                        dtype=rng.choice(["f32", "f32", "bf16", "f16"]), given=rng.random() < 0.5, greedy=rng.choice([0, 0, 3]), ragged=rng.random() < 0.4)
        while c["lanes"] > 1 and work(c)["bytes"] > work(listed()[7])["bytes"]:
            c["lanes"] //= 2
    elif op == "copy":
        copies = log_int(rng, 1, 500)
        c = copy_case("", shape, 2 * copies + rng.randrange(100), copies, rng.random() < 0.5, page=rng.choice([16, 32, 64]), dtype=rng.choice(["f16", "bf16", "f32"]))
        while c["copies"] > 1 and work(c)["bytes"] > 0.9 * work(listed()[9])["bytes"]:
            c["copies"] = max(1, c["copies"] // 2)
            c["pages"] = 2 * c["copies"] + 50
    else:
        context = log_int(rng, 20, 3000)
        high = log_int(rng, 1, context // 2)
        c = gather_case("", shape, log_int(rng, 1, 32), context, rng.randrange(1, high + 1), high, rng.randrange(0, context // 3), page=rng.choice([16, 32, 64]),
                        dtype=rng.choice(["f16", "bf16", "f32"]))
        while c["lanes"] > 1 and gather_pool_bytes(c) > 3e9:
            c["lanes"] //= 2
        while gather_pool_bytes(c) > 3e9:
            c["layers"] //= 2
    del c["name"]
    return c


# ---- inputs ----------------------------------------------------------------------------------------------------------


def own_lengths(case):
    return spread(case["low"], case["high"], case["lanes"])


def row_counts(case):
    """Rows of each lane, by its place among the lengths."""
    if not case["ragged"]:
        return [case["rows"]] * case["lanes"]
    return [1 + (i * 7 + 3) % case["rows"] for i in range(case["lanes"])]


def random(g, *shape):
    return torch.randn(*shape, generator=g, device=DEVICE)


def pool(g, dtype, *shape):
    """Values of a cache: drawn once for a part of it and repeated with a shift, which is quick for gigabytes."""
    n = math.prod(shape)
    part = random(g, min(n, 1 << 24) + 1).to(dtype)
    out = torch.empty(n, dtype=dtype, device=DEVICE)
    for i, at in enumerate(range(0, n, part.numel() - 1)):
        m = min(part.numel() - 1, n - at)
        out[at:at + m] = part[i % 2:i % 2 + m]
    return out.view(*shape)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(1000003 * (seed + 1))
    dtype = DTYPES[case["dtype"]]
    s = dict(case=case)
    if case["op"] == "attention":
        lanes, page, shared = case["lanes"], case["page"], case["shared"]
        order = torch.randperm(lanes, generator=g, device=DEVICE).tolist()
        lengths, counts = own_lengths(case), row_counts(case)
        lengths, counts = [lengths[i] for i in order], [counts[i] for i in order]
        own_pages = [-(-n // page) for n in lengths]
        pages = shared // page + sum(own_pages)
        width = shared // page + max(own_pages)
        ids = torch.randperm(pages + 8, generator=g, device=DEVICE)[:pages].to(torch.int32)
        tables = torch.full((lanes, width), -1, dtype=torch.int32, device=DEVICE)
        tables[:, :shared // page] = ids[:shared // page]
        at = shared // page
        for i, n in enumerate(own_pages):
            tables[i, shared // page:shared // page + n] = ids[at:at + n]
            at += n
        total = sum(counts)
        s["q"] = (2 * random(g, total, case["q_heads"], case["dim"])).to(dtype)
        s["k"] = pool(g, dtype, pages + 8, case["kv_heads"], page, case["dim"])
        s["v"] = pool(g, dtype, pages + 8, case["kv_heads"], page, case["dim"])
        s["tables"] = tables
        s["lengths"] = torch.tensor([shared + n for n in lengths], dtype=torch.int32, device=DEVICE)
        s["cu"] = torch.tensor([sum(counts[:i]) for i in range(lanes + 1)], dtype=torch.int32, device=DEVICE) if case["ragged"] else None
        s["scale"] = case["dim"] ** -0.5
    elif case["op"] == "verify":
        lanes, n, vocab = case["lanes"], case["drafts"], case["vocab"]
        # a target model's logits: a broad bell and a few likely tokens above it
        logits = 2.2 * random(g, lanes, n + 1, vocab)
        hot = torch.randint(0, vocab, (lanes, n + 1, 8), generator=g, device=DEVICE)
        logits.scatter_(2, hot, 9.0 + 2.0 * random(g, lanes, n + 1, 8))
        s["logits"] = logits.to(dtype)
        s["temperature"] = 0.6 + 0.6 * torch.rand(lanes, generator=g, device=DEVICE)
        s["top_k"] = torch.full((lanes,), case["top_k"], dtype=torch.int32, device=DEVICE)
        s["top_p"] = torch.full((lanes,), case["top_p"], device=DEVICE)
        if case["greedy"]:
            s["temperature"][::case["greedy"]] = 0.0
        s["u"] = torch.rand(lanes, n + 1, generator=g, device=DEVICE)
        if case["given"]:  # a smaller model agrees in part
            s["probs"] = torch.softmax(0.7 * logits[:, :n] + 1.2 * random(g, lanes, n, vocab), -1)
            s["drafts"] = torch.multinomial(s["probs"].view(lanes * n, vocab), 1, generator=g).view(lanes, n).to(torch.int32)
        else:  # looked-up drafts are often the likeliest token
            s["probs"] = None
            other = torch.randint(0, vocab, (lanes, n), generator=g, device=DEVICE)
            s["drafts"] = torch.where(torch.rand(lanes, n, generator=g, device=DEVICE) < 0.8, logits[:, :n].argmax(-1), other).to(torch.int32)
        if case["ragged"]:
            have = torch.randint(0, n + 1, (lanes, 1), generator=g, device=DEVICE)
            s["drafts"] = torch.where(torch.arange(n, device=DEVICE) < have, s["drafts"], -1).to(torch.int32)
    elif case["op"] == "copy":
        for x in "kv":
            s[x] = pool(g, dtype, case["layers"], case["pages"], case["kv_heads"], case["page"], case["dim"])
        ids = torch.randperm(case["pages"], generator=g, device=DEVICE)[:2 * case["copies"]].view(2, -1)
        rows = torch.full_like(ids[0], case["page"])
        if case["tails"]:
            ids[0] = ids[0, torch.arange(case["copies"], device=DEVICE) // 4 * 4]  # four samples of a prompt
            rows = 1 + (ids[0] * 5 + 1) % (case["page"] - 1)
        s["copies"] = torch.stack([ids[0], ids[1], rows], 1).to(torch.int32)
    else:
        lanes, page, context = case["lanes"], case["page"], case["context"]
        pages, new = -(-context // page), -(-(case["first"] + case["high"]) // page)
        for x in "kv":
            s[x] = pool(g, dtype, case["layers"], lanes * (pages + new), case["kv_heads"], page, case["dim"])
        ids = torch.randperm(lanes * (pages + new), generator=g, device=DEVICE).to(torch.int32)
        s["src"], s["dst"] = ids[:lanes * pages].view(lanes, pages), ids[lanes * pages:].view(lanes, new)
        counts = kept(case)
        keep = torch.full((lanes, case["high"]), -1, dtype=torch.int32, device=DEVICE)
        for i, n in enumerate(counts):
            free = context - case["first"]
            keep[i, :n] = case["first"] + torch.randperm(free, generator=g, device=DEVICE)[:n].sort()[0].to(torch.int32)
        s["keep"] = keep
        s["counts"] = torch.tensor(counts, dtype=torch.int32, device=DEVICE)
        s["first"] = torch.full((lanes,), case["first"], dtype=torch.int32, device=DEVICE)
    return s


def kept(case):
    n = min(case["high"], case["context"] - case["first"])
    return [min(n, x) for x in spread(case["low"], case["high"], case["lanes"])]


def gather_pool_bytes(c):
    pages = c["lanes"] * (-(-c["context"] // c["page"]) - (-(c["first"] + c["high"]) // c["page"]))
    return c["layers"] * pages * c["kv_heads"] * c["page"] * c["dim"] * (4 if c["dtype"] == "f32" else 2)


# ---- one pass --------------------------------------------------------------------------------------------------------


def run(s):
    return {"attention": run_attention, "verify": run_verify, "copy": run_copy, "gather": run_gather}[s["case"]["op"]](s)


def run_attention(s):
    c = s["case"]
    if own:
        return framework().shared_attention(s["q"], s["k"], s["v"], s["tables"], s["lengths"], c["shared"], scale=s["scale"], cu_seqlens=s["cu"],
                                            max_rows=c["rows"], softcap=c["softcap"], window=c["window"])
    q, tables, lengths = s["q"].float(), s["tables"], s["lengths"]
    total, heads, dim = q.shape
    page, shared, kvh = c["page"], c["shared"], c["kv_heads"]
    t = torch.arange(total, device=q.device)
    if s["cu"] is None:
        lane = t // c["rows"]
        pos = lengths[lane] - c["rows"] + t % c["rows"]
    else:
        lane = torch.searchsorted(s["cu"], t, right=True) - 1
        pos = lengths[lane] - s["cu"][lane + 1] + t
    q = q.view(total, kvh, heads // kvh, dim)

    def capped(x):
        return c["softcap"] * torch.tanh(x / c["softcap"]) if c["softcap"] else x

    def masked(x, key):  # key: [1 or total][keys]
        see = key <= pos[:, None]
        if c["window"]:
            see &= pos[:, None] - key < c["window"]
        return x.masked_fill(~see[:, None, None], -math.inf)

    def rows_of(cache, pages):  # [...][keys][kv heads][dim]
        x = cache[pages.clamp_min(0)].float()
        return x.transpose(-3, -2).reshape(*pages.shape[:-1], pages.shape[-1] * page, kvh, dim)

    first = tables[0, :shared // page]
    mine = tables[:, shared // page:][lane]
    k0, v0, k1, v1 = rows_of(s["k"], first), rows_of(s["v"], first), rows_of(s["k"], mine), rows_of(s["v"], mine)
    a = masked(capped(torch.einsum("thgd,khd->thgk", q, k0) * s["scale"]), torch.arange(shared, device=q.device)[None])
    b = masked(capped(torch.einsum("thgd,tkhd->thgk", q, k1) * s["scale"]), shared + torch.arange(k1.shape[1], device=q.device)[None])
    top = torch.maximum(a.amax(-1, keepdim=True) if shared else b.amax(-1, keepdim=True), b.amax(-1, keepdim=True)).clamp_min(-1e30)
    a, b = torch.exp(a - top), torch.exp(b - top)
    den = a.sum(-1, keepdim=True) + b.sum(-1, keepdim=True)
    out = torch.einsum("thgk,khd->thgd", a, v0) + torch.einsum("thgk,tkhd->thgd", b, v1)
    return (out / den.clamp_min(1e-30)).reshape(total, heads, dim).to(s["q"].dtype)


def run_verify(s):
    c = s["case"]
    if own:
        return framework().verify_drafts(s["logits"], s["drafts"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], draft_probs=s["probs"])
    x, drafts, n = s["logits"].double(), s["drafts"].long(), c["drafts"]
    # the target's distributions: the top_k best (the lower token first among equals), scaled, and of those the head that adds up to top_p
    hot = s["temperature"] > 0
    z = (x - x.amax(-1, keepdim=True)) / torch.where(hot, s["temperature"], 1.0).double()[:, None, None]
    p = torch.exp(z)
    if c["top_k"]:
        order = torch.sort(x, dim=-1, descending=True, stable=True)[1]
        head = torch.exp(z.gather(-1, order)) * (torch.arange(c["vocab"], device=x.device) < s["top_k"][:, None, None])
        head = head / head.sum(-1, keepdim=True)
        head = head * (torch.cumsum(head, -1) - head < s["top_p"].double()[:, None, None])
        p = torch.zeros_like(x).scatter_(-1, order, head)
    p = p / p.sum(-1, keepdim=True)
    best = torch.zeros_like(p).scatter_(-1, x.argmax(-1, keepdim=True), 1.0)  # the first of equals
    p = torch.where(hot[:, None, None], p, best)
    # a draft stays while u * q < p; the first that does not is replaced from max(p - q, 0), or one more is drawn from p
    there = torch.cumprod((drafts >= 0).int(), -1).bool()
    token = drafts.clamp_min(0)[:, :, None]
    pd = p[:, :n].gather(-1, token)[:, :, 0]
    qd = s["probs"].gather(-1, token)[:, :, 0].double() if s["probs"] is not None else torch.ones_like(pd)
    accepted = torch.cumprod(((s["u"][:, :n].double() * qd < pd) & there).int(), -1).sum(-1)
    at = accepted[:, None, None]
    p = p.gather(1, at.expand(-1, 1, c["vocab"]))[:, 0]
    refused = accepted < there.sum(-1)
    row = accepted.clamp_max(n - 1)[:, None]
    if s["probs"] is not None:
        q = s["probs"].gather(1, row[:, :, None].expand(-1, 1, c["vocab"]))[:, 0].double()
    else:
        q = torch.zeros_like(p).scatter_(-1, token[:, :, 0].gather(1, row), 1.0)
    rest = torch.where(refused[:, None], (p - q).clamp_min(0), p)
    rest = torch.where(rest.sum(-1, keepdim=True) > 0, rest, p)
    up_to = torch.cumsum(rest, -1)
    picked = (up_to <= s["u"][:, n:].double() * up_to[:, -1:]).sum(-1)
    i = torch.arange(n + 1, device=x.device)
    padded = torch.nn.functional.pad(drafts, (0, 1), value=-1)
    tokens = torch.where(i < at[:, 0], padded, torch.where(i == at[:, 0], picked[:, None], -1))
    return tokens.to(torch.int32), accepted.to(torch.int32)


def run_copy(s):
    if own:
        framework().copy_pages(s["k"], s["v"], s["copies"])
        return s["k"], s["v"]
    src, dst, rows = s["copies"].long().unbind(1)
    filled = (torch.arange(s["case"]["page"], device=rows.device) < rows[:, None])[None, :, None, :, None]
    s["k"][:, dst] = torch.where(filled, s["k"][:, src], s["k"][:, dst])
    s["v"][:, dst] = torch.where(filled, s["v"][:, src], s["v"][:, dst])
    return s["k"], s["v"]


def run_gather(s):
    if own:
        framework().gather_tokens(s["k"], s["v"], s["src"], s["keep"], s["counts"], s["dst"], s["first"])
        return s["k"], s["v"]
    page = s["case"]["page"]
    j = torch.arange(s["keep"].shape[1], device=s["keep"].device)
    lane, j = torch.nonzero(j < s["counts"][:, None], as_tuple=True)
    frm, to = s["keep"][lane, j].long(), s["first"][lane] + j
    a, b = s["src"][lane, frm // page].long(), s["dst"][lane, to // page].long()
    s["k"][:, b, :, to % page] = s["k"][:, a, :, frm % page]
    s["v"][:, b, :, to % page] = s["v"][:, a, :, frm % page]
    return s["k"], s["v"]


# ---- what a pass cannot do without -----------------------------------------------------------------------------------


def work(c):
    size = 4 if c["dtype"] == "f32" else 2
    if c["op"] == "attention":
        keys = seen = 0  # keys of own parts that some row sees; pairs of rows and keys
        for n, rows in zip(own_lengths(c), row_counts(c)):
            for r in range(rows):
                p = c["shared"] + n - rows + r
                seen += min(p + 1, c["window"]) if c["window"] else max(0, p + 1)
            keys += min(n, c["window"] + rows - 1) if c["window"] else n
        first = c["shared"] if not c["window"] else max(0, min(c["shared"], c["window"] - c["low"] + max(row_counts(c)) - 1))
        total = sum(row_counts(c))
        return {"bytes": 2 * size * (keys + first) * c["kv_heads"] * c["dim"] + 2 * size * total * c["q_heads"] * c["dim"],
                "flops": 4 * seen * c["q_heads"] * c["dim"]}
    if c["op"] == "verify":
        rows = c["lanes"] * (c["drafts"] + 1) * c["vocab"]
        # of a draft's distribution the drafted token and the row that the last draw may take are read
        return {"bytes": size * rows + (4 * c["lanes"] * c["vocab"] if c["given"] and not c["top_k"] else 0), "flops": 4 * rows}
    row = c["layers"] * c["kv_heads"] * c["dim"] * size
    if c["op"] == "copy":
        tokens = c["copies"] * (c["page"] // 2 if c["tails"] else c["page"])
    else:
        tokens = sum(kept(c))
    return {"bytes": 2 * 2 * tokens * row, "flops": 0}


# ---- the definition, in 64 bits --------------------------------------------------------------------------------------


def exact(case, seed):
    if case["op"] != "attention":
        return None  # whole numbers, and copies
    s = prepare(case, seed)
    q, page, group = s["q"].double(), case["page"], case["q_heads"] // case["kv_heads"]
    counts = [case["rows"]] * case["lanes"] if s["cu"] is None else (s["cu"][1:] - s["cu"][:-1]).tolist()
    out, at = torch.zeros_like(q), 0
    for lane, (length, rows) in enumerate(zip(s["lengths"].tolist(), counts)):
        ids = s["tables"][lane, :-(-length // page)].long()
        k, v = (s[x][ids].double().permute(1, 0, 2, 3).flatten(1, 2)[:, :length].repeat_interleave(group, 0) for x in "kv")  # [heads][keys][dim]
        position = torch.arange(length - rows, length, device=DEVICE)[:, None]
        key = torch.arange(length, device=DEVICE)[None]
        hidden = key > position
        if case["window"]:
            hidden |= key <= position - case["window"]
        x = q[at:at + rows].transpose(0, 1) @ k.transpose(1, 2) * s["scale"]
        if case["softcap"]:
            x = case["softcap"] * torch.tanh(x / case["softcap"])
        x = torch.softmax(x.masked_fill(hidden, -math.inf), -1).nan_to_num(0.0)  # a row that sees nothing: zeros
        out[at:at + rows] = (x @ v).transpose(0, 1)
        at += rows
    return out
