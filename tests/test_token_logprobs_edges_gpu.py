"""Log probabilities of given tokens where a row's maximum is at the end of its type's numbers."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_token_logprobs_gpu import BF16, F16, F32, check, dops, generator, model_logits  # noqa: E402, F401 (dops is a fixture)

# a thread's first and its later batches, a row's ends in single values, a CTA and clusters
SIZES = [(3, 1), (3, 9), (2, 257), (5, 4099), (200, 20001), (2, 128256), (1, 1000003)]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows, vocab", SIZES)
@pytest.mark.parametrize("place", [0.0, 0.001, 0.37, 0.93, 1.0])
def test_one_lowest_number_among_tokens_that_cannot_be(dops, dtype, rows, vocab, place):  # noqa: F811
    """The one token that can be has all of the probability, however low its logit is."""
    x = torch.full((rows, vocab + 3), -math.inf, dtype=dtype, device="cuda")[:, :vocab]
    at = int(place * (vocab - 1))
    x[:, at] = torch.finfo(dtype).min
    tokens = torch.full((rows,), at, dtype=torch.int32, device="cuda")
    if rows > 1:
        tokens[1] = (at + 1) % vocab   # one that cannot be
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = dops.token_logprobs(x, tokens, top=min(2, vocab), status=status)
    assert status.item() == 0
    assert got.logprobs[0] == 0 and (got.entropy == 0).all() and got.ranks[0] == 1 and (got.top_tokens[:, 0] == at).all() and (got.top_logprobs[:, 0] == 0).all()
    check(x, tokens, got, min(2, vocab))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows, vocab", SIZES)
def test_low_numbers_among_tokens_that_cannot_be(dops, dtype, rows, vocab):  # noqa: F811
    """Several of the lowest numbers, and of those just above them, spread over a row that is -inf for the rest."""
    g = generator(vocab)
    x = torch.full((rows, vocab), -math.inf, dtype=dtype, device="cuda")
    keep = torch.randint(0, vocab, (rows, 40), generator=g, device="cuda")
    low = torch.finfo(dtype).min * (1 - torch.finfo(dtype).eps * torch.randint(0, 6, (rows, 40), generator=g, device="cuda").double())
    x.scatter_(1, keep, low.to(dtype))
    tokens = keep[:, 7].to(torch.int32).contiguous()
    check(x, tokens, dops.token_logprobs(x, tokens, top=min(30, vocab)), min(30, vocab))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows, vocab", SIZES[2:])
def test_lowest_numbers_in_front_of_ordinary_ones(dops, dtype, rows, vocab):  # noqa: F811
    """A thread that has met nothing above the lowest number until its last vectors."""
    g = generator(vocab + 1)
    x = model_logits(g, rows, vocab, dtype)[0]
    x[:, :vocab - 5] = -math.inf
    x[:, 3:vocab - 5:11] = torch.finfo(dtype).min
    tokens = torch.full((rows,), vocab - 2, dtype=torch.int32, device="cuda")
    check(x, tokens, dops.token_logprobs(x, tokens, top=3), 3)
    x[:, -5:] = -math.inf
    tokens.fill_(14)
    check(x, tokens, dops.token_logprobs(x, tokens, top=3), 3)
