"""Operators over device buffers for caches of keys and values in 4 or 8 bits and for scoring given tokens, as cases whose time is measured.

Four of them: rows of keys and values quantised into pages, rows of such pages read back, attention over the pages as they are, and log
probabilities of given tokens with entropy, rank and the likeliest alternatives.  Head layouts, vocabularies, pages and lengths are those of
the benchmark's model shapes and workloads, and longer contexts, which such a cache is for.

`run` computes them in elementary torch operations, or, where `own` is true, through the framework's entry points.  `exact` states them
again in 64 bits, lane by lane.
"""
import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
GROUP = 64  # neighbouring values of a head's row that share a step and a lowest value

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


# q heads, kv heads, head size and vocabulary of the benchmark's model shapes
SHAPES = {
    "tinyllama": dict(q_heads=32, kv_heads=4, dim=64, vocab=32000),
    "smollm3": dict(q_heads=16, kv_heads=4, dim=128, vocab=128256),
    "qwen3": dict(q_heads=32, kv_heads=8, dim=128, vocab=151936),
    "gemma2": dict(q_heads=16, kv_heads=8, dim=256, vocab=256000),
    "qwen3moe": dict(q_heads=32, kv_heads=4, dim=128, vocab=151936),
}


def lanes_case(name, op, shape, lanes, rows, low, high, bits=4, dtype="f16", ragged=False, window=0, softcap=0.0, page=16):
    s = SHAPES[shape]
    return dict(name=name, op=op, lanes=lanes, rows=rows, low=low, high=high, bits=bits, dtype=dtype, ragged=ragged, window=window, softcap=softcap,
                page=page, q_heads=s["q_heads"], kv_heads=s["kv_heads"], dim=s["dim"])


def score_case(name, rows, vocab, top, dtype="f32", masked=False):
    return dict(name=name, op="score", rows=rows, vocab=vocab, top=top, dtype=dtype, masked=masked)


def listed():
    return [
        # a few short chats, one token each: launches and latency are everything
        lanes_case("chat-3", "attention", "tinyllama", 3, 1, 40, 301),
        # a tick of a server's batch in the middle of its answers
        lanes_case("batch-48", "attention", "qwen3", 48, 1, 200, 6000),
        # a few users with whole books in their contexts
        lanes_case("books-3", "attention", "smollm3", 3, 1, 20000, 120001, dtype="bf16", page=64),
        # drafted tokens being verified over a cache of 8 bits, wide heads with capped scores, some lanes with fewer drafts
        lanes_case("drafts-20", "attention", "gemma2", 20, 5, 700, 8000, bits=8, ragged=True, softcap=50.0),
        # portions of long prompts behind what is already in the cache
        lanes_case("portions-4", "attention", "qwen3moe", 4, 1000, 2500, 12000, dtype="bf16", ragged=True),
        # the new tokens of a tick, written to the cache and read as the cache has them
        lanes_case("tick-64", "write", "qwen3", 64, 1, 17, 3000),
        # whole prompts written, and read as the cache has them
        lanes_case("prompts-5", "write", "qwen3", 5, 4096, 4096, 4096, dtype="bf16", ragged=True),
        # the tail of one chat, read back for an inspection
        lanes_case("tail-1", "read", "smollm3", 1, 37, 519, 519, bits=8, page=32),
        # contexts read back whole, to go on in 16 bits
        lanes_case("whole-12", "read", "qwen3", 12, 8000, 8000, 8000),
        # a chat's next tokens, with the few likeliest beside each
        score_case("answers-5", 5, 32000, 5),
        # a tick's tokens of a batch, as a service that reports 20 alternatives asks for, some tokens masked
        score_case("tick-40", 40, 151936, 20, masked=True),
        # a text scored under a model: the entropy and the tokens' own log probabilities
        score_case("text-2000", 2000, 128256, 0, dtype="bf16"),
    ]


def spread(low, high, n):
    """n whole numbers from low to high, even over their logarithm."""
    if n == 1:
        return [int(round(math.sqrt(low * high)))]
    return [int(round(low * (high / low) ** (i / (n - 1)))) for i in range(n)]


def log_int(rng, low, high):
    return int(round(low * (high / low) ** rng.random()))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "attention", "write", "read", "score", "score"])
    shape = rng.choice(sorted(SHAPES))
    most = {c["name"]: work(c) for c in listed()}
    if op == "score":
        vocab = rng.choice([SHAPES[shape]["vocab"], SHAPES[shape]["vocab"], log_int(rng, 300, 256000)])
        top = rng.choice([0, 0, 1, 5, 20, 64])
        c = score_case("", log_int(rng, 1, 2000), vocab, top, dtype=rng.choice(["f32", "bf16", "f16"]), masked=rng.random() < 0.3)
        limit = most["text-2000"]["bytes"] if not top else 0.25 * most["text-2000"]["bytes"]
        while c["rows"] > 1 and work(c)["bytes"] > limit:
            c["rows"] //= 2
    else:
        rows = {"attention": rng.choice([1, 1, 1, 2, 4, 7, log_int(rng, 8, 1500)]), "write": log_int(rng, 1, 4096), "read": log_int(rng, 1, 8000)}[op]
        high = log_int(rng, max(rows, 8), 100000 if rows < 8 else 12000)
        c = lanes_case("", op, shape, log_int(rng, 1, 100), rows, 1, high, bits=rng.choice([4, 4, 8]), dtype=rng.choice(["f16", "bf16"]), ragged=rng.random() < 0.4,
                       page=rng.choice([16, 16, 32, 64]))
        c["low"] = log_int(rng, min(rows, high), high)
        if op == "attention":
            c["window"] = rng.choice([0, 0, 0, 1000, 4096])
            c["softcap"] = rng.choice([0.0, 0.0, 50.0])
        name = {"attention": "portions-4", "write": "prompts-5", "read": "whole-12"}[op]
        size = c["kv_heads"] * c["dim"] * 8  # of a token's keys and values in 32 bits, as the plain forms lay them out
        while c["lanes"] > 1 and (work(c)["flops"] > 0.9 * most[name]["flops"] or work(c)["bytes"] > 0.9 * max(most[name]["bytes"], most["books-3"]["bytes"])
                                  or c["lanes"] * c["high"] * size > 6e9 or c["lanes"] * c["rows"] * c["q_heads"] * c["high"] * 4 > 8e9):
            c["lanes"] //= 2
        while c["rows"] > 1 and (work(c)["flops"] > 0.9 * most[name]["flops"] or work(c)["bytes"] > 0.9 * max(most[name]["bytes"], most["books-3"]["bytes"])):
            c["rows"] //= 2
    del c["name"]
    return c


# ---- inputs ----------------------------------------------------------------------------------------------------------


def lengths_of(case):
    return spread(case["low"], case["high"], case["lanes"])


def row_counts(case):
    """Rows of each lane, by its place among the lengths."""
    if not case["ragged"]:
        return [case["rows"]] * case["lanes"]
    return [max(1, case["rows"] - (i * 7 + 3) % 11 * case["rows"] // 16) for i in range(case["lanes"])]


def random(g, *shape):
    return torch.randn(*shape, generator=g, device=DEVICE)


def keys_and_values(g, case, tokens):
    """[2][tokens][kv heads][dim]: keys with channels that are far from 0 for every token, as rotated keys have them, and values."""
    x = random(g, 2, tokens, case["kv_heads"], case["dim"])
    x[0] += 2 * random(g, case["kv_heads"], case["dim"])
    return x.to(DTYPES[case["dtype"]])


def repeated(x, n):
    """x over and over along its first dimension, shifted by one each time, n in all."""
    out = torch.empty(n, *x.shape[1:], dtype=x.dtype, device=x.device)
    m = max(1, len(x) - 1)
    for i, at in enumerate(range(0, n, m)):
        k = min(m, n - at)
        begin = i % 2 if len(x) > 1 else 0
        out[at:at + k] = x[begin:begin + k]
    return out


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(1000003 * (seed + 1))
    dtype = DTYPES[case["dtype"]]
    s = dict(case=case)
    if case["op"] == "score":
        rows, vocab = case["rows"], case["vocab"]
        # a model's logits: a broad bell and a few likely tokens above it
        logits = 2.2 * random(g, rows, vocab)
        hot = torch.randint(0, vocab, (rows, 8), generator=g, device=DEVICE)
        logits.scatter_(1, hot, 9.0 + 2.0 * random(g, rows, 8))
        other = torch.randint(0, vocab, (rows,), generator=g, device=DEVICE)
        s["tokens"] = torch.where(torch.rand(rows, generator=g, device=DEVICE) < 0.7, hot[:, 0], other).to(torch.int32)
        if case["masked"]:  # a grammar or a list of banned words leaves part of the vocabulary
            logits.masked_fill_(torch.rand(vocab, generator=g, device=DEVICE) < 0.4, -math.inf)
            logits[:, vocab // 2] = 3.0
        s["logits"] = logits.to(dtype)
        return s
    lanes, page, bits, dim, heads = case["lanes"], case["page"], case["bits"], case["dim"], case["kv_heads"]
    order = torch.randperm(lanes, generator=g, device=DEVICE).tolist()
    lengths, counts = lengths_of(case), row_counts(case)
    lengths, counts = [lengths[i] for i in order], [counts[i] for i in order]
    own_pages = [-(-n // page) for n in lengths]
    pages, width, total = sum(own_pages) + 8, max(own_pages), sum(counts)
    ids = torch.randperm(pages, generator=g, device=DEVICE).to(torch.int32)
    s["tables"] = torch.full((lanes, width), -1, dtype=torch.int32, device=DEVICE)
    at = 0
    for i, n in enumerate(own_pages):
        s["tables"][i, :n] = ids[at:at + n]
        at += n
    s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=DEVICE)
    s["cu"] = torch.tensor([sum(counts[:i]) for i in range(lanes + 1)], dtype=torch.int32, device=DEVICE) if case["ragged"] else None
    s["total"] = total
    # codes of keys and of values, (step, lowest value) of each group of keys and of values
    if case["op"] == "write":
        s["pools"] = tuple(torch.zeros(pages, heads, page, n, dtype=torch.uint8, device=DEVICE) for n in 2 * (dim * bits // 8,)) + tuple(
            torch.zeros(pages, heads, page, dim // GROUP, 2, dtype=dtype, device=DEVICE) for _ in range(2))
        s["k"], s["v"] = keys_and_values(g, case, total)
    else:
        some = min(pages, max(1, (1 << 23) // (page * heads * dim)))
        codes, scales = packed(keys_and_values(g, case, some * page).view(2, some, page, heads, dim).transpose(2, 3), bits)
        s["pools"] = tuple(repeated(x, pages) for x in (codes[0], codes[1], scales[0], scales[1]))
    if case["op"] == "attention":
        s["q"] = (2 * random(g, total, case["q_heads"], dim)).to(dtype)
        s["scale"] = dim ** -0.5
    return s


# ---- one pass --------------------------------------------------------------------------------------------------------


def run(s):
    return {"attention": run_attention, "write": run_write, "read": run_read, "score": run_score}[s["case"]["op"]](s)


def packed(x, bits):
    """Codes and (step, lowest value) of the groups of x's rows."""
    top = 2 ** bits - 1
    g = x.float().unflatten(-1, (-1, GROUP))
    low, high = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    fine = torch.isfinite(high - low)
    step = torch.where(fine, ((high - low) / top).to(x.dtype).float(), math.nan)
    low = torch.where(fine, low, math.nan)
    code = torch.where(step > 0, torch.round((g - low) / step).clamp(0, top), 0.0).to(torch.uint8).flatten(-2)
    if bits == 4:
        code = code[..., ::2] | code[..., 1::2] << 4
    return code, torch.cat([step, low], -1).to(x.dtype)


def stands_for(code, scales, bits, wide=torch.float32):
    """The values of codes [..., bytes] with scales [..., groups, 2]."""
    if bits == 4:
        code = torch.stack([code & 15, code >> 4], -1).flatten(-2)
    scales = scales.to(wide)
    return (scales[..., 1:] + scales[..., :1] * code.to(wide).unflatten(-1, (-1, GROUP))).flatten(-2)


def places(s):
    """(lane, position) of each row: a lane's rows are the last of its tokens."""
    t = torch.arange(s["total"], device=s["lengths"].device)
    if s["cu"] is None:
        rows = s["case"]["rows"]
        lane = t // rows
        return lane, s["lengths"][lane] - rows + t % rows
    lane = torch.searchsorted(s["cu"], t, right=True) - 1
    return lane, s["lengths"][lane] - s["cu"][lane + 1] + t


def run_write(s):
    c = s["case"]
    if own:
        dops = framework()
        dops.quantize_rows(s["k"], s["v"], s["pools"], s["tables"], s["lengths"], cu_seqlens=s["cu"])
        return dops.dequantize_rows(s["pools"], s["tables"], s["lengths"], s["total"], cu_seqlens=s["cu"])
    lane, pos = places(s)
    page = s["tables"][lane, pos // c["page"]].long()
    for x, codes, scales in zip((s["k"], s["v"]), s["pools"][:2], s["pools"][2:]):
        codes[page, :, pos % c["page"]], scales[page, :, pos % c["page"]] = packed(x, c["bits"])
    return run_read(s)


def run_read(s):
    c = s["case"]
    if own:
        return framework().dequantize_rows(s["pools"], s["tables"], s["lengths"], s["total"], cu_seqlens=s["cu"])
    lane, pos = places(s)
    page = s["tables"][lane, pos // c["page"]].long()
    return tuple(stands_for(codes[page, :, pos % c["page"]], scales[page, :, pos % c["page"]], c["bits"]).to(scales.dtype)
                 for codes, scales in zip(s["pools"][:2], s["pools"][2:]))


def run_attention(s):
    c = s["case"]
    if own:
        return framework().quantized_attention(s["q"], s["pools"], s["tables"], s["lengths"], scale=s["scale"], cu_seqlens=s["cu"], max_rows=c["rows"],
                                               softcap=c["softcap"], window=c["window"])
    lanes, rows, heads, kvh, dim = c["lanes"], c["rows"], c["q_heads"], c["kv_heads"], c["dim"]
    lane, pos = places(s)
    first = s["cu"][lane] if s["cu"] is not None else lane * rows
    row = torch.arange(s["total"], device=lane.device) - first
    q = torch.zeros(lanes, rows, heads, dim, device=lane.device)
    q[lane, row] = s["q"].float()
    at = torch.full((lanes, rows), -1, dtype=torch.int64, device=lane.device)
    at[lane, row] = pos.long()
    q = q.view(lanes, rows, kvh, heads // kvh, dim).permute(0, 2, 1, 3, 4).flatten(2, 3)
    pages = s["tables"].clamp_min(0).long()
    k, v = (stands_for(codes[pages], scales[pages], c["bits"]).transpose(1, 2).flatten(2, 3) for codes, scales in zip(s["pools"][:2], s["pools"][2:]))
    x = (q @ k.transpose(2, 3)).mul_(s["scale"]).view(lanes, kvh, rows, heads // kvh, -1)
    if c["softcap"]:
        x = x.div_(c["softcap"]).tanh_().mul_(c["softcap"])
    key = torch.arange(k.shape[2], device=lane.device)
    hidden = key > at[:, :, None]
    if c["window"]:
        hidden |= key <= at[:, :, None] - c["window"]
    x.masked_fill_(hidden[:, None, :, None], -math.inf)
    x = x.sub_(x.amax(-1, keepdim=True).clamp_min(-1e30)).exp_()
    den = x.sum(-1, keepdim=True)
    out = (x.flatten(2, 3) @ v).view(lanes, kvh, rows, heads // kvh, dim) / den.clamp_min(1e-30)
    return out.permute(0, 2, 1, 3, 4).reshape(lanes, rows, heads, dim)[lane, row].to(s["q"].dtype)


def run_score(s):
    c = s["case"]
    if own:
        return tuple(framework().token_logprobs(s["logits"], s["tokens"], top=c["top"]))
    x, t = s["logits"].float(), s["tokens"].long()[:, None]
    z = x - x.amax(-1, keepdim=True)
    p = torch.exp(z)
    mass = p.sum(-1, keepdim=True)
    log_mass = torch.log(mass)
    entropy = log_mass[:, 0] - (p * z.clamp_min(-1e30)).sum(-1) / mass[:, 0]
    mine = x.gather(1, t)
    rank = 1 + (x > mine).sum(-1) + ((x == mine) & (torch.arange(c["vocab"], device=x.device) < t)).sum(-1)
    value, token = torch.sort(x, dim=-1, descending=True, stable=True) if c["top"] else (x, t)
    value, token = value[:, :c["top"]], token[:, :c["top"]]
    return ((z.gather(1, t) - log_mass)[:, 0], entropy, rank.to(torch.int32), token.to(torch.int32), value - x.amax(-1, keepdim=True) - log_mass)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------


def work(c):
    if c["op"] == "score":
        size = 4 if c["dtype"] == "f32" else 2
        return {"bytes": c["rows"] * (size * c["vocab"] + 16 + 8 * c["top"]), "flops": 6 * c["rows"] * c["vocab"]}
    token = 2 * c["kv_heads"] * (c["dim"] * c["bits"] // 8 + c["dim"] // GROUP * 4)  # bytes of a token's keys and values in the cache
    wide = 2 * c["kv_heads"] * c["dim"] * 2
    if c["op"] == "attention":
        keys = seen = 0  # keys that some row sees; pairs of rows and keys
        for n, rows in zip(lengths_of(c), row_counts(c)):
            for p in range(n - rows, n):
                seen += max(0, min(p + 1, c["window"]) if c["window"] else p + 1)
            keys += min(n, c["window"] + rows - 1) if c["window"] else n
        return {"bytes": keys * token + 2 * 2 * sum(row_counts(c)) * c["q_heads"] * c["dim"], "flops": 4 * seen * c["q_heads"] * c["dim"]}
    total = sum(row_counts(c))
    if c["op"] == "write":  # rows read, the cache's form written, and the values of that written as rows
        return {"bytes": total * (wide + token + wide), "flops": 8 * total * c["kv_heads"] * c["dim"]}
    return {"bytes": total * (token + wide), "flops": 4 * total * c["kv_heads"] * c["dim"]}


# ---- the definition, in 64 bits --------------------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "score":
        own_log, entropy, tops = [], [], []
        for x, t in zip(s["logits"].split(200), s["tokens"].split(200)):
            x = x.double()
            log_p = torch.log_softmax(x, -1)
            own_log.append(log_p.gather(1, t.long()[:, None])[:, 0])
            entropy.append(torch.special.entr(torch.softmax(x, -1)).sum(-1))
            tops.append(torch.topk(log_p, case["top"], -1)[0])
        return torch.cat(own_log), torch.cat(entropy), None, None, torch.cat(tops)
    page, bits, counts = case["page"], case["bits"], [case["rows"]] * case["lanes"] if s["cu"] is None else (s["cu"][1:] - s["cu"][:-1]).tolist()
    if case["op"] == "write":
        return tuple(rounded(x, bits) for x in (s["k"], s["v"]))

    def tokens_of(lane, kind, n):  # [n][kv heads][dim]
        ids = s["tables"][lane, :-(-n // page)].long()
        return stands_for(s["pools"][kind][ids], s["pools"][2 + kind][ids], bits, torch.float64).transpose(1, 2).flatten(0, 1)[:n]

    if case["op"] == "read":
        return tuple(torch.cat([tokens_of(lane, kind, n)[n - rows:] for lane, (n, rows) in enumerate(zip(s["lengths"].tolist(), counts))]) for kind in (0, 1))
    q, group = s["q"].double(), case["q_heads"] // case["kv_heads"]
    out, at = torch.zeros_like(q), 0
    for lane, (length, rows) in enumerate(zip(s["lengths"].tolist(), counts)):
        k, v = (tokens_of(lane, kind, length).transpose(0, 1) for kind in (0, 1))  # [kv heads][keys][dim]
        position = torch.arange(length - rows, length, device=DEVICE)[:, None]
        key = torch.arange(length, device=DEVICE)[None]
        hidden = key > position
        if case["window"]:
            hidden |= key <= position - case["window"]
        for h in range(case["q_heads"]):
            x = q[at:at + rows, h] @ k[h // group].t() * s["scale"]
            if case["softcap"]:
                x = case["softcap"] * torch.tanh(x / case["softcap"])
            x = torch.softmax(x.masked_fill(hidden, -math.inf), -1).nan_to_num(0.0)  # a row that sees nothing: zeros
            out[at:at + rows, h] = x @ v[h // group]
        at += rows
    return out


def rounded(x, bits):
    """x as a cache of so many bits holds it: to the nearest of the even steps from a group's lowest value to its highest."""
    g = x.double().view(*x.shape[:-1], -1, GROUP)
    low = g.min(-1, keepdim=True)[0]
    step = ((g.max(-1, keepdim=True)[0] - low) / (2 ** bits - 1)).to(x.dtype).double()
    return (low + step * torch.where(step > 0, torch.round((g - low) / step), 0.0).clamp(max=2 ** bits - 1)).view(x.shape)
