"""Log probabilities of given tokens against plain implementations in 64 bits."""
import importlib
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def dops(mk):
    capi = importlib.import_module("macllm_infer_b200._capi")
    if capi.lib().mk_device_count() <= 0:
        pytest.fail("this test needs a CUDA device: the library has no CPU fallback")
    return importlib.import_module("macllm_infer_b200.device_ops")


def generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def model_logits(g, rows, vocab, dtype, spread=2.2):
    x = spread * torch.randn(rows, vocab, generator=g, device="cuda")
    hot = torch.randint(0, vocab, (rows, min(8, vocab)), generator=g, device="cuda")
    x.scatter_(1, hot, 9 + 2 * torch.randn(rows, hot.shape[1], generator=g, device="cuda"))
    return x.to(dtype), hot[:, 0].to(torch.int32)


def check(logits, tokens, got, top):
    x, t = logits.double(), tokens.long()[:, None]
    log_p = torch.log_softmax(x, -1)
    p = torch.exp(log_p)
    # 32-bit differences from the maximum (2^-24 of them), 2^-22 of each exponential and of the sums of partial sums, and logarithms' 2^-22
    span = (x.amax(-1) - x.masked_fill(x == -math.inf, math.inf).amin(-1)).clamp_max(200)
    bound = 2 ** -21 * (1 + span) + 1e-6
    mine = log_p.gather(1, t)[:, 0]
    off = torch.where(mine == got.logprobs.double(), 0.0, (got.logprobs.double() - mine).abs())
    # the difference from the maximum and that from ln Z are rounded to 32 bits
    assert (off <= bound + 2 * 2 ** -24 * mine.abs()).all(), float((off - bound).max())
    entropy = torch.special.entr(p).sum(-1)
    assert ((got.entropy.double() - entropy).abs() <= bound * (1 + entropy)).all()
    value = x.gather(1, t)
    rank = 1 + (x > value).sum(-1) + ((x == value) & (torch.arange(x.shape[1], device="cuda") < t)).sum(-1)
    assert torch.equal(got.ranks.long(), rank)
    assert got.top_tokens.shape == got.top_logprobs.shape == (len(x), top)
    order = torch.sort(x, dim=-1, descending=True, stable=True)[1][:, :top]
    assert torch.equal(got.top_tokens.long(), order)
    want = log_p.gather(1, order)
    off = torch.where(want == got.top_logprobs.double(), 0.0, (got.top_logprobs.double() - want).abs())
    assert (off <= bound[:, None] + 2 * 2 ** -24 * want.abs()).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows, vocab", [(1, 1), (3, 2), (2, 33), (5, 1000), (1, 4097), (7, 32000), (2, 151936), (40, 50257), (1, 500003), (300, 2051), (1500, 700)])
@pytest.mark.parametrize("top", [0, 1, 5, 20, 64])
def test_types_sizes_and_tops(dops, dtype, rows, vocab, top):
    top = min(top, vocab)
    g = generator(rows + vocab + top)
    logits, tokens = model_logits(g, rows, vocab, dtype)
    tokens = torch.where(torch.rand(rows, generator=g, device="cuda") < 0.5, tokens, torch.randint(0, vocab, (rows,), generator=g, device="cuda")).to(torch.int32)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = dops.token_logprobs(logits, tokens, top=top, status=status)
    assert status.item() == 0
    check(logits, tokens, got, top)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("vocab", [70, 5000, 128256])
@pytest.mark.parametrize("kind", ["equal", "two", "rounded", "steps", "masked", "lowest", "alone", "ascending", "crowd"])
def test_ties_masks_and_extremes(dops, dtype, vocab, kind):
    """Thousands of equal logits, most of the vocabulary out of reach, one token with everything."""
    g = generator(vocab)
    x, tokens = model_logits(g, 4, vocab, dtype)
    if kind == "equal":
        x.fill_(1.5)
    elif kind == "two":
        x = (torch.rand(4, vocab, generator=g, device="cuda") < 0.5).to(dtype)
    elif kind == "rounded":
        x = x.float().round().to(dtype)
    elif kind == "steps":
        x = (torch.arange(vocab, device="cuda") // 7 % 50).to(dtype).expand(4, vocab).contiguous()
    elif kind == "masked":   # fewer are left than are asked for
        keep = torch.randint(0, vocab, (4, 10), generator=g, device="cuda")
        x = torch.full_like(x, -math.inf).scatter(1, keep, x.gather(1, keep))
        tokens = torch.where(torch.arange(4, device="cuda") < 2, keep[:, 3], (keep[:, 0] + 1) % vocab).to(torch.int32)
    elif kind == "lowest":
        x[:, ::2] = torch.finfo(dtype).min
    elif kind == "alone":
        x.fill_(-30 if dtype == F16 else -1e4)
        x[:, vocab - 1] = 60
        tokens.fill_(vocab - 1)
    elif kind == "ascending":
        x = torch.linspace(-8, 8, vocab, device="cuda").to(dtype).expand(4, vocab).contiguous()
    elif kind == "crowd":   # the best ones next to one another
        x[:, vocab // 2:vocab // 2 + 60] += 20
    check(x, tokens, dops.token_logprobs(x, tokens, top=min(64, vocab)), min(64, vocab))
    check(x, tokens, dops.token_logprobs(x, tokens, top=3), 3)


def test_far_logits_and_odd_strides(dops):
    g = generator(1)
    for dtype, scale in ((F32, 1e30), (BF16, 1e30), (F16, 6000.0), (F32, 1e-30)):
        x = (scale * torch.randn(3, 4001, generator=g, device="cuda")).to(dtype)
        tokens = x.float().argmax(-1).to(torch.int32)
        got = dops.token_logprobs(x, tokens, top=4)
        assert torch.equal(got.ranks.long(), torch.tensor([1, 1, 1], device="cuda")) and torch.equal(got.top_tokens[:, 0], tokens)
        check(x, tokens, got, 4)
    for dtype in (F32, F16, BF16):
        for gap, begin in ((1, 0), (3, 5), (8, 8)):
            wide = model_logits(g, 6, 3001 + gap + begin, dtype)[0]
            x = wide[:, begin:begin + 3001]
            tokens = torch.arange(6, dtype=torch.int32, device="cuda") * 500
            check(x, tokens, dops.token_logprobs(x, tokens, top=10), 10)
        x = model_logits(g, 1, 999, dtype)[0].expand(5, 999)
        tokens = torch.arange(5, dtype=torch.int32, device="cuda")
        check(x.contiguous(), tokens, dops.token_logprobs(x.contiguous(), tokens, top=2), 2)


def test_rows_beyond_two_to_the_31(dops):
    rows, vocab = 9000, 250000   # 2.25e9 values
    logits = torch.zeros(rows, vocab, dtype=F16, device="cuda")
    g = generator(2)
    some = torch.tensor([0, 1, 4500, 8588, 8589, 8590, 8999], device="cuda")
    logits[some] = model_logits(g, len(some), vocab, F16)[0]
    tokens = torch.randint(0, vocab, (rows,), generator=g, device="cuda").to(torch.int32)
    got = dops.token_logprobs(logits, tokens, top=2)
    check(logits[some], tokens[some], type(got)(*(t[some] for t in got)), 2)
    rest = torch.tensor([2, 8000, 8998], device="cuda")
    check(logits[rest], tokens[rest], type(got)(*(t[rest] for t in got)), 2)


@pytest.mark.parametrize("vocab", [50, 3000, 128256])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_tokens_and_rows_that_are_none(dops, vocab, dtype):
    g = generator(3)
    x, tokens = model_logits(g, 9, vocab, dtype)
    x[1, vocab // 2], x[2, vocab - 1], x[3] = math.nan, math.inf, -math.inf
    x[7, 0] = math.nan
    tokens[4], tokens[5], tokens[6], tokens[7] = -1, vocab, 2 ** 31 - 1, -5
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = dops.token_logprobs(x, tokens, top=5, status=status)
    assert status.item() == dops.BAD_RANGE | dops.BAD_ROW
    for r in (1, 2, 3, 7):
        assert math.isnan(got.entropy[r]) and got.ranks[r] == 0 and (got.top_tokens[r] == -1).all() and torch.isnan(got.top_logprobs[r]).all()
        assert math.isnan(got.logprobs[r]) or r == 7
    assert got.logprobs[4] == 0 and got.ranks[4] == 0 and got.logprobs[7] == 0 and torch.isnan(got.logprobs[5:7]).all() and (got.ranks[5:7] == 0).all()
    fine = torch.tensor([0, 8], device="cuda")
    check(x[fine], tokens[fine], type(got)(*(t[fine] for t in got)), 5)
    swapped = tokens.clone()
    swapped[4:7] = 0
    for r in (4, 5, 6):   # the rest of such a row is as ever
        one = torch.tensor([r], device="cuda")
        again = dops.token_logprobs(x[one], swapped[one], top=5)
        assert torch.equal(again.entropy[0], got.entropy[r]) or abs(float(again.entropy[0] - got.entropy[r])) < 1e-5
        assert torch.equal(again.top_tokens[0], got.top_tokens[r])


def test_captured_and_repeated(dops):
    g = generator(4)
    logits, tokens = model_logits(g, 12, 40000, F32)
    first = dops.token_logprobs(logits, tokens, top=20)
    assert all(all(torch.equal(a, b) for a, b in zip(dops.token_logprobs(logits, tokens, top=20), first)) for _ in range(10))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = dops.token_logprobs(logits, tokens, top=20)
    for seed in (5, 6):
        x, t = model_logits(generator(seed), 12, 40000, F32)
        logits.copy_(x)
        tokens.copy_(t)
        graph.replay()
        check(logits, tokens, held, 20)
    assert dops.token_logprobs(logits[:0], tokens[:0], top=3).top_tokens.shape == (0, 3)
