"""Operators over device buffers against plain implementations in 64 bits, at the sizes and masks where they can go wrong."""
import importlib
import itertools
import math

import numpy as np
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


# ---- attention of lanes that share their first pages ------------------------------------------------------------------------------------


class Batch:
    """Lanes of the given own lengths (beyond shared; negative: shorter than that) and rows over a pool in which everything that no lane may read is NaN."""

    def __init__(self, dtype, q_heads, kv_heads, dim, page, shared, own, rows, seed=0, spread=1.0, page_gap=0, q_gap=0):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        lanes = len(own)
        lengths = [max(0, shared + n) for n in own]
        pages = [max(0, -(-n // page) - shared // page) for n in lengths]
        total_pages = shared // page + sum(pages)
        width = shared // page + max(pages, default=0)
        pool = torch.full((2, total_pages + 3, kv_heads * page * dim + page_gap), math.nan, dtype=dtype, device="cuda")
        self.pools = [pool[i, :, :kv_heads * page * dim].view(-1, kv_heads, page, dim) if page_gap == 0 else
                      pool[i].as_strided((total_pages + 3, kv_heads, page, dim), (kv_heads * page * dim + page_gap, page * dim, dim, 1), pool[i].storage_offset()) for i in (0, 1)]
        ids = (torch.randperm(total_pages + 2, generator=g, device="cuda")[:total_pages] + 1).to(torch.int32)
        self.tables = torch.full((lanes, width + 1), 1 << 30, dtype=torch.int32, device="cuda")[:, :width]   # entries behind a lane's are no pages
        self.tables[:, :shared // page] = ids[:shared // page]
        at = shared // page
        for i, n in enumerate(pages):
            self.tables[i, shared // page:shared // page + n] = ids[at:at + n]
            at += n
        for x in self.pools:
            for p in ids[:shared // page].tolist():
                x[p] = torch.randn(kv_heads, page, dim, generator=g, device="cuda").to(dtype)
            for i, n in enumerate(lengths):
                for b in range(shared // page, -(-n // page)):
                    m = min(page, n - b * page)
                    x[int(self.tables[i, b])][:, :m] = torch.randn(kv_heads, m, dim, generator=g, device="cuda").to(dtype)
        self.lengths = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        self.rows = rows if isinstance(rows, list) else [rows] * lanes
        total = sum(self.rows)
        q = torch.full((total, q_heads * dim + q_gap), math.nan, dtype=dtype, device="cuda")
        self.q = q[:, :q_heads * dim].view(total, q_heads, dim) if q_gap == 0 else q.as_strided((total, q_heads, dim), (q_heads * dim + q_gap, dim, 1))
        self.q.copy_(spread * torch.randn(total, q_heads, dim, generator=g, device="cuda"))
        self.cu = torch.tensor([0, *itertools.accumulate(self.rows)], dtype=torch.int32, device="cuda") if isinstance(rows, list) else None
        self.shared, self.page, self.scale = shared, page, dim ** -0.5

    def run(self, dops, **more):
        return dops.shared_attention(self.q, *self.pools, self.tables, self.lengths, self.shared, scale=self.scale, cu_seqlens=self.cu, max_rows=max(self.rows, default=0), **more)

    def check(self, got, window=0, softcap=0.0):
        dtype, dim = self.q.dtype, self.q.shape[2]
        group = self.q.shape[1] // self.pools[0].shape[1]
        half = torch.finfo(dtype).eps / 2
        at = 0
        for lane, (n, rows) in enumerate(zip(self.lengths.tolist(), self.rows)):
            ids = self.tables[lane, :-(-n // self.page)].long()
            k, v = (x[ids].double().permute(1, 0, 2, 3).flatten(1, 2)[:, :n].repeat_interleave(group, 0) for x in self.pools)
            q = self.q[at:at + rows].double().transpose(0, 1)
            p = torch.arange(n - rows, n, device="cuda")[:, None]
            key = torch.arange(n, device="cuda")[None]
            hidden = (key > p) | ((key <= p - window) if window else torch.zeros_like(key, dtype=torch.bool))
            x = q @ k.transpose(1, 2) * self.scale
            size = q.abs() @ k.abs().transpose(1, 2) * self.scale
            if softcap:
                x = softcap * torch.tanh(x / softcap)
            w = torch.softmax(x.masked_fill(hidden, -math.inf), -1).nan_to_num(0.0)
            want, mean = w @ v, w @ v.abs()
            # weights and results are rounded to the type once each; a score is off by its products' 32-bit sums (each of them rounded: dim of them at the largest
            # intermediate value), its scaling and logarithm, 2^-21 for the exponential, and a few 1e-7 of the cap; each moves a weight by as much, relative, and the sum too
            score = (size.max() if size.numel() else torch.tensor(0.0)).item() * (dim + 8) * 2 ** -24 + 2 ** -21 + 1e-6 * softcap
            bound = half * (mean + want.abs()) * (1 + half) + 2 * score * (mean + want.abs()) + 1e-7 * (dtype == F16)
            off = (got[at:at + rows].double().transpose(0, 1) - want).abs()
            assert torch.isfinite(off).all(), lane
            assert (off <= bound).all(), (lane, float((off - bound).max()), float((off / bound.clamp_min(1e-30)).max()))
            at += rows


@pytest.mark.parametrize("dim, q_heads, kv_heads, page, dtype", [
    (64, 32, 4, 16, F16), (128, 16, 4, 16, F16), (128, 32, 8, 16, BF16), (256, 16, 8, 16, F16), (64, 3, 3, 32, BF16), (128, 5, 1, 64, F16), (256, 8, 8, 128, BF16), (128, 40, 2, 16, F16),
    (64, 71, 1, 16, F16), (256, 24, 2, 16, F16), (128, 128, 1, 16, BF16),
])
def test_head_layouts_types_and_pages(dops, dim, q_heads, kv_heads, page, dtype):
    shared = 3 * 128 + 64 if page < 128 else 4 * page
    b = Batch(dtype, q_heads, kv_heads, dim, page, shared // page * page, [1, 15, 16, 17, 40, 130, 0, 3], 1)
    b.check(b.run(dops))
    b = Batch(dtype, q_heads, kv_heads, dim, page, shared // page * page, [2, 70, 33], [2, 4, 3], seed=1)
    b.check(b.run(dops))


@pytest.mark.parametrize("shared", [0, 16, 32, 112, 128, 144, 1024, 5008])
@pytest.mark.parametrize("own", [[1], [0], [700], [1, 700, 31, 512, 513], [0, 0, 2000]])
def test_lengths(dops, shared, own):
    b = Batch(F16, 8, 2, 128, 16, shared, own, 1, seed=2)
    b.check(b.run(dops))


@pytest.mark.parametrize("lanes, rows", [(1, 1), (1, 5), (1, 40), (2, 100), (17, 1), (33, 3), (130, 1), (70, 8)])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_numbers_of_rows(dops, lanes, rows, dim):
    b = Batch(F16, 8, 2, dim, 16, 304, [rows + (i * 13) % 90 for i in range(lanes)], rows, seed=3)
    b.check(b.run(dops))


def test_lanes_of_different_rows_some_without(dops):
    b = Batch(BF16, 8, 2, 128, 16, 256, [9, 20, 300, 1, 40], [4, 0, 9, 1, 0], seed=4)
    b.check(b.run(dops))


def test_rows_at_and_before_the_first_key(dops):
    """Lanes shorter than their rows, without tokens, and shorter than the shared part: what they see is what is there, and nothing becomes zeros."""
    b = Batch(F16, 8, 2, 64, 16, 0, [2, 0, 5, 1], [4, 2, 5, 3], seed=5)
    got = b.run(dops)
    b.check(got)
    assert (got[0:2] == 0).all() and (got[4:6] == 0).all() and (got[11:13] == 0).all()
    b = Batch(F16, 8, 2, 64, 16, 320, [-320, -319, -200, -1, 7, 1], [1, 1, 3, 2, 3, 4], seed=6)
    got = b.run(dops)
    b.check(got)
    assert (got[0] == 0).all()


@pytest.mark.parametrize("dim, kv_heads", [(64, 4), (128, 8), (256, 2)])
@pytest.mark.parametrize("shared", [16, 320, 368, 576, 640])
@pytest.mark.parametrize("lanes", [1, 5, 40])
def test_few_keys(dops, dim, kv_heads, shared, lanes):
    """Around the numbers of keys and lanes from which the shared ones are read once; lanes shorter than them and without rows among them."""
    own = [16, 3, -7, 0, 15][:lanes] * max(1, lanes // 5)
    rows = [2, 1, 2, 0, 4][:lanes] * max(1, lanes // 5)
    b = Batch(BF16, 2 * kv_heads, kv_heads, dim, 16, shared, own, rows, seed=30)
    for window, softcap in ((0, 0.0), (100, 30.0)):
        b.check(b.run(dops, window=window, softcap=softcap), window, softcap)


@pytest.mark.parametrize("window", [1, 5, 64, 300, 2000])
@pytest.mark.parametrize("softcap", [0.0, 20.0])
@pytest.mark.parametrize("dim", [128, 256])
def test_windows_and_caps(dops, window, softcap, dim):
    b = Batch(F16, 16, 8, dim, 16, 640, [4, 30, 290, 700, 1300], [3, 4, 1, 2, 4], seed=7, spread=3.0)
    b.check(b.run(dops, window=window, softcap=softcap), window, softcap)


def test_large_scores(dops):
    """The maximum grows along the keys, again and again, and weights far below it vanish."""
    b = Batch(F16, 8, 2, 128, 16, 2048, [100, 900], 2, seed=8, spread=12.0)
    ramp = torch.linspace(0.2, 3.0, 2048, device="cuda").view(-1, 16, 1).to(F16)
    ids = b.tables[0, :128].long()
    b.pools[0][ids] = b.pools[0][ids] * ramp[:, None]
    b.check(b.run(dops))


def test_strided_queries_results_pages_and_tables(dops):
    b = Batch(F16, 8, 2, 128, 16, 160, [40, 3, 77], [2, 1, 5], seed=9, page_gap=2 * 128 * 24, q_gap=64)
    wide = torch.full((10, 8 * 128 + 24), 7.0, dtype=F16, device="cuda")
    out = wide[1:9, :1024].view(8, 8, 128)
    assert b.run(dops, out=out) is out
    b.check(out)
    assert (wide[0] == 7).all() and (wide[9] == 7).all() and (wide[:, 1024:] == 7).all()


def test_rows_of_no_lane_stay(dops):
    b = Batch(F16, 8, 2, 128, 16, 160, [40, 3], [2, 3], seed=10)
    q = torch.cat([b.q, b.q])
    out = torch.full_like(q, 5.0)
    dops.shared_attention(q, *b.pools, b.tables, b.lengths, b.shared, scale=b.scale, cu_seqlens=b.cu, max_rows=3, out=out)
    b.check(out[:5])
    assert (out[5:] == 5).all()
    b = Batch(F16, 8, 2, 128, 16, 160, [2000, 3], [2, 3], seed=10)   # a lane's keys shared out
    q = torch.cat([b.q, b.q])
    out = torch.full_like(q, 5.0)
    dops.shared_attention(q, *b.pools, b.tables, b.lengths, b.shared, scale=b.scale, cu_seqlens=b.cu, max_rows=3, out=out)
    b.check(out[:5])
    assert (out[5:] == 5).all()


def test_sharing_changes_nothing_but_roundings(dops):
    b = Batch(BF16, 32, 8, 128, 16, 1600, [17, 200, 90, 1], 2, seed=11)
    for shared in (0, 16, 800, 1600):
        b.shared = shared
        b.check(b.run(dops))


def test_the_same_call_gives_the_same_bits(dops):
    b = Batch(F16, 16, 4, 128, 16, 4096, [600, 20, 1500, 3, 77, 300], 3, seed=12)
    first = b.run(dops)
    for _ in range(5):
        assert torch.equal(first, b.run(dops))


def test_bad_pages_and_lengths_are_told(dops):
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    capi = importlib.import_module("macllm_infer_b200._capi")
    for shared in (0, 160):
        b = Batch(F16, 8, 2, 128, 16, shared, [40, 3], 1, seed=13)
        b.run(dops, status=status)
        dops.check_status(status)
        good = b.tables.clone()
        for lane, column, value in ((0, 0, -5), (1, 0, 10 ** 6), (0, shared // 16 + 1, -1)):
            if shared and lane == 1:
                continue   # the shared pages are read through lane 0's table
            b.tables.copy_(good)
            b.tables[lane, column] = value
            b.run(dops, status=status)
            with pytest.raises(capi.MkError, match="page number"):
                dops.check_status(status)
        b.tables.copy_(good)
        for length in (-3, b.tables.shape[1] * 16 + 1, 2 ** 31 - 1):
            b.lengths[1] = length
            b.run(dops, status=status)
            with pytest.raises(capi.MkError, match="length"):
                dops.check_status(status)
        b.lengths[1] = shared + 3
        for cu in ([0, 3, 2], [-1, 1, 2], [0, 1, 5], [5, 6, 7]):
            dops.shared_attention(b.q, *b.pools, b.tables, b.lengths, shared, scale=1.0, cu_seqlens=torch.tensor(cu, dtype=torch.int32, device="cuda"), max_rows=2, status=status)
            with pytest.raises(capi.MkError, match="range"):
                dops.check_status(status)
        b.check(b.run(dops, status=status))
        dops.check_status(status)


# ---- verification of drafts ---------------------------------------------------------------------------------------------------


def verify_plain(logits, drafts, u, temperature, top_k, top_p, probs):
    """Lane by lane in 64 bits; also the smallest distance of a decision from going the other way."""
    tokens, accepted, margin = np.full(u.shape, -1, np.int32), np.zeros(len(u), np.int32), np.inf

    def distribution(x, lane):
        nonlocal margin
        x = x.astype(np.float64)
        if not temperature[lane] > 0:
            return np.eye(1, len(x), int(np.argmax(x)))[0]
        e = np.exp((x - x.max()) / np.float64(temperature[lane]))
        if top_k[lane] > 0:
            order = np.argsort(-x, kind="stable")[:top_k[lane]]
            head = e[order] / e[order].sum()
            before = np.cumsum(head) - head
            if top_p[lane] < 1:
                margin = min(margin, np.abs(before[1:] - np.float64(top_p[lane])).min(initial=np.inf))
                head = np.where((before < np.float64(top_p[lane])) | (np.arange(len(head)) == 0), head, 0.0)
            e = np.zeros_like(e)
            e[order] = head
        return e / e.sum()

    for lane in range(len(u)):
        n = drafts.shape[1]
        for i in range(n + 1):
            p = distribution(logits[lane, i], lane)
            d = drafts[lane, i] if i < n else -1
            rest = p
            if d >= 0:
                q = probs[lane, i].astype(np.float64) if probs is not None else np.eye(1, len(p), d)[0]
                t = np.float64(u[lane, i]) * q[d]
                if p[d] > 0 and q[d] > 0 and temperature[lane] > 0:
                    margin = min(margin, abs(t - p[d]) / p[d])
                if t < p[d]:
                    tokens[lane, i] = d
                    accepted[lane] += 1
                    continue
                rest = np.maximum(p - q, 0)
                if not rest.sum() > 0:
                    rest = p
            upto = np.cumsum(rest)
            target = np.float64(u[lane, n]) * upto[-1]
            pick = int((upto <= target).sum())
            live = rest > 0
            margin = min(margin, np.abs(upto[live][:-1] - target).min(initial=np.inf) / upto[-1])
            tokens[lane, i] = min(pick, int(np.nonzero(live)[0][-1]))
            break
    return tokens, accepted, margin


def verify_case(seed, lanes, n, vocab, dtype=F32, given=False, spread=2.5, ragged=False):
    rng = np.random.default_rng(seed)
    logits = torch.tensor(spread * rng.standard_normal((lanes, n + 1, vocab)), dtype=F32).to(dtype)
    logits[:, :, :: max(1, vocab // 7)] += 4
    x = logits.double().numpy()
    probs = None
    if given:
        z = 0.8 * x[:, :n] + rng.standard_normal((lanes, n, vocab))
        probs = np.exp(z - z.max(-1, keepdims=True))
        probs = (probs / probs.sum(-1, keepdims=True)).astype(np.float32)
        drafts = np.array([[rng.choice(vocab, p=r.astype(np.float64) / r.astype(np.float64).sum()) for r in lane] for lane in probs], dtype=np.int32).reshape(lanes, n)
    else:
        drafts = np.where(rng.random((lanes, n)) < 0.7, x[:, :n].argmax(-1), rng.integers(0, vocab, (lanes, n))).astype(np.int32)
    if ragged:
        drafts = np.where(np.arange(n) < rng.integers(0, n + 1, (lanes, 1)), drafts, -1).astype(np.int32)
    return logits, drafts, rng.random((lanes, n + 1)).astype(np.float32), probs


def verify_check(dops, logits, drafts, u, probs, temperature, top_k, top_p):
    lanes = len(u)
    t, k, p = (np.broadcast_to(np.asarray(v, dtype=d), (lanes,)).copy() for v, d in ((temperature, np.float32), (top_k, np.int32), (top_p, np.float32)))
    want, count, margin = verify_plain(logits.float().numpy(), drafts, u, t, k, p, probs)
    # a decision's sides are sums of 64-bit numbers in 64 bits, of 32-bit weights (2^-22 each) where the whole vocabulary counts; whoever draws the inputs keeps clear of both
    assert margin > 1e-7
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    cuda = [torch.from_numpy(np.ascontiguousarray(v)).cuda() for v in (drafts, u, t, k, p)]
    tokens, accepted = dops.verify_drafts(logits.cuda(), cuda[0], cuda[1], temperature=cuda[2], top_k=cuda[3], top_p=cuda[4],
                                          draft_probs=None if probs is None else torch.from_numpy(probs).cuda(), status=status)
    assert np.array_equal(accepted.cpu().numpy(), count), (accepted.cpu().numpy(), count)
    assert np.array_equal(tokens.cpu().numpy(), want), np.nonzero(tokens.cpu().numpy() != want)
    dops.check_status(status)
    return count


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("given", [False, True])
@pytest.mark.parametrize("top_k, top_p", [(0, 1.0), (1, 1.0), (5, 0.7), (40, 0.95), (1000, 0.8)])
def test_verification(dops, dtype, given, top_k, top_p):
    verify_check(dops, *verify_case(1, 9, 4, 4100, dtype, given), [0.7, 1.0, 1.3] * 3, top_k, top_p)


@pytest.mark.parametrize("given", [False, True])
@pytest.mark.parametrize("top_k, top_p", [(0, 1.0), (50, 0.99)])
def test_verification_of_peaked_rows(dops, given, top_k, top_p):
    """Rows that bear out some drafts and not others."""
    verify_check(dops, *verify_case(12, 32, 5, 30000, given=given, spread=7.0), [0.5, 1.0] * 16, top_k, top_p)


@pytest.mark.parametrize("vocab", [1, 2, 7, 500, 1023, 32000, 50257, 128256])
@pytest.mark.parametrize("top_k", [0, 64])
def test_vocabularies(dops, vocab, top_k):
    verify_check(dops, *verify_case(2, 3, 3, vocab, given=vocab < 2000), 0.9, min(top_k, vocab), 0.9 if top_k else 1.0)


@pytest.mark.parametrize("lanes, n", [(1, 0), (1, 1), (1, 31), (5, 0), (70, 2), (3, 9)])
def test_numbers_of_drafts(dops, lanes, n):
    verify_check(dops, *verify_case(3, lanes, n, 900), 0.8, 20, 0.9)


@pytest.mark.parametrize("top_k", [16, 126, 127, 128, 129, 200, 511, 512, 513, 700, 1023, 1024])
@pytest.mark.parametrize("vocab", [3001, 70000])
def test_numbers_of_candidates(dops, top_k, vocab):
    """Around what is compared with one another, and sorted by one, two and four to a thread."""
    verify_check(dops, *verify_case(13, 4, 3, vocab, F16, given=top_k % 2 == 0), [0.8, 1.5] * 2, top_k, [0.99, 1.0] * 2)


@pytest.mark.parametrize("lanes", [47, 49, 97, 300])
@pytest.mark.parametrize("given", [False, True])
def test_numbers_of_lanes(dops, lanes, given):
    """Eight, four and two CTAs to a lane, all kinds of lanes beside one another."""
    t, k, p = (np.resize(v, lanes) for v in ([0.9, 0.9, 0.0, 1.2, 0.7], [0, 20, 0, 200, 0], [1.0, 0.9, 1.0, 1.0, 1.0]))
    verify_check(dops, *verify_case(14, lanes, 4, 901, given=given, ragged=True), t, k, p)


def test_greedy_ragged_and_mixed_lanes(dops):
    verify_check(dops, *verify_case(4, 24, 5, 3000, ragged=True), [0.0, 0.8, 1.0] * 8, [0, 7, 0, 100] * 6, [1.0, 0.6, 1.0, 0.9] * 6)
    verify_check(dops, *verify_case(5, 24, 5, 3000, given=True, ragged=True), [0.0, 0.8, 1.0] * 8, [3, 0, 50, 0] * 6, [0.5, 1.0, 0.9, 1.0] * 6)


def test_equal_logits_go_to_the_lower_token(dops):
    logits, drafts, u, _ = verify_case(6, 8, 3, 2000)
    logits = (logits * 2).round() / 2   # many equals at every border, zeros of both signs among them
    logits[::2] = logits[::2] * (torch.rand(logits[::2].shape) < 0.5) * -1
    verify_check(dops, logits, drafts, u, None, 0.9, [10, 300, 64, 1] * 2, 1.0)
    flat = torch.zeros_like(logits)
    verify_check(dops, flat, np.array([[1, 5, 900]] * 8, np.int32), u, None, [1.0, 0.0] * 4, [10, 1000, 1, 64] * 2, [1.0, 0.45, 1.0, 0.77] * 2)


def test_masked_tokens_have_no_share(dops):
    logits, drafts, u, probs = verify_case(7, 8, 3, 3000, given=True)
    logits[:, :, ::3] = -math.inf
    logits[:, :, 1::3] = -3.0e38
    logits[0, :, 5:] = -math.inf   # fewer tokens left than top_k
    verify_check(dops, logits, drafts, u, probs, 0.9, [50, 0] * 4, [0.9, 1.0] * 4)


def test_a_draft_distribution_equal_to_the_targets_is_always_kept(dops):
    logits, _, u, _ = verify_case(8, 6, 4, 1000)
    probs = torch.softmax(logits.double(), -1)[:, :4]
    drafts = probs.argmax(-1).int()
    u = torch.from_numpy(u).cuda()
    one = torch.ones(6, device="cuda")
    # the draft's 32-bit probabilities are off by at most 2^-24, so u below 1 - 2^-22 keeps every draft
    tokens, accepted = dops.verify_drafts(logits.cuda(), drafts.cuda(), u.clamp_max(0.999), temperature=one, top_k=torch.zeros(6, dtype=torch.int32, device="cuda"), top_p=one,
                                          draft_probs=probs.float().cuda())
    assert (accepted == 4).all() and torch.equal(tokens[:, :4].cpu(), drafts)


def test_draws_follow_the_target(dops):
    """Whatever the drafts are drawn from, the first token is distributed as the target says: a chi-square over 40000 lanes."""
    lanes, vocab = 40000, 12
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    row, other = 1.5 * torch.randn(vocab, generator=g, device="cuda"), torch.softmax(torch.randn(vocab, generator=g, device="cuda"), 0)
    drafts = torch.multinomial(other, lanes, replacement=True, generator=g).int().view(lanes, 1)
    u = torch.rand(lanes, 2, generator=g, device="cuda")
    for k, top_k, given in ((vocab, 0, True), (5, 5, True), (vocab, 0, False)):
        full = torch.full((lanes,), 1.0, device="cuda")
        tokens, _ = dops.verify_drafts(row.expand(lanes, 2, vocab).contiguous(), drafts, u, temperature=full, top_k=torch.full((lanes,), top_k, dtype=torch.int32, device="cuda"), top_p=full,
                                       draft_probs=other.expand(lanes, 1, vocab).contiguous() if given else None)
        p = torch.softmax(row.double(), 0)
        p = torch.where(p >= p.topk(k)[0][-1], p, 0.0)
        p = p / p.sum()
        if not given:   # looked-up drafts stand for themselves: kept with p(d), else drawn from the others - also p
            pass
        seen = torch.bincount(tokens[:, 0].long(), minlength=vocab).double()
        assert seen[p == 0].sum() == 0
        live = p > 0
        chi = ((seen - lanes * p)[live] ** 2 / (lanes * p[live])).sum().item()
        freedom = int(live.sum()) - 1
        assert chi < freedom + 6 * math.sqrt(2 * freedom) + 18, chi   # six standard deviations and the tail's skew


def test_rows_without_a_distribution_and_settings_out_of_range(dops):
    capi = importlib.import_module("macllm_infer_b200._capi")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    one = torch.ones(4, device="cuda")
    base, drafts, u, _ = verify_case(9, 4, 2, 700)
    drafts[:] = base[:, :2].argmax(-1).numpy()
    u[:, :2] = 0.0

    def run(logits, d=drafts, top_k=0, top_p=1.0):
        return dops.verify_drafts(logits.cuda(), torch.from_numpy(d).cuda(), torch.from_numpy(u).cuda(), temperature=one, top_k=torch.full((4,), top_k, dtype=torch.int32, device="cuda"),
                                  top_p=top_p * one, status=status)

    for value in (math.nan, math.inf, None):
        for top_k in (0, 9):
            x = base.clone()
            if value is None:
                x[1, 1] = -math.inf
            else:
                x[1, 1, 650] = value
            tokens, accepted = run(x, top_k=top_k)
            assert accepted.tolist() == [2, 1, 2, 2] and tokens[1].tolist() == [drafts[1, 0], -1, -1]
            with pytest.raises(capi.MkError, match="no distribution"):
                dops.check_status(status)
    wrong = drafts.copy()
    wrong[2, 0] = 700
    assert run(base, wrong)[1].tolist() == [2, 2, 0, 2]
    with pytest.raises(capi.MkError, match="range"):
        dops.check_status(status)
    for top_k, top_p in ((0, 0.5), (5000, 1.0)):
        run(base, top_k=top_k, top_p=top_p)
        with pytest.raises(capi.MkError, match="range"):
            dops.check_status(status)


@pytest.mark.parametrize("top_k", [0, 30])
def test_temperatures_without_measure(dops, top_k):
    """The lowest leave the best token, the highest make all alike; nothing between overflows."""
    logits, drafts, u, _ = verify_case(13, 4, 2, 1000)
    logits[:, :, 5] = -math.inf
    k = torch.full((4,), top_k, dtype=torch.int32, device="cuda")
    one = torch.ones(4, device="cuda")
    args = [logits.cuda(), torch.from_numpy(drafts).cuda(), torch.from_numpy(u).cuda()]
    greedy = dops.verify_drafts(*args, temperature=0 * one, top_k=k, top_p=one)
    for t in (1e-45, 1e-38, 1e-31, 1e-28, 1e-20):
        assert all(torch.equal(a, b) for a, b in zip(greedy, dops.verify_drafts(*args, temperature=t * one, top_k=k, top_p=one))), t
    hot = [dops.verify_drafts(*args, temperature=t * one, top_k=k, top_p=one) for t in (1e25, 1e35, math.inf)]
    assert all(torch.equal(a, b) for other in hot[1:] for a, b in zip(hot[0], other))
    drawn = hot[0][0][torch.arange(4), hot[0][1].long()]
    assert ((drawn >= 0) & (drawn != 5)).all()


def test_padded_rows_of_logits(dops):
    logits, drafts, u, _ = verify_case(10, 5, 3, 1001)
    wide = torch.full((5, 4, 1030), math.nan, device="cuda")
    wide[:, :, 3:1004] = logits.cuda()
    one = torch.ones(5, device="cuda")
    want, count, margin = verify_plain(logits.numpy(), drafts, u, np.ones(5), np.full(5, 30), np.full(5, 0.9, np.float32), None)
    assert margin > 1e-7
    tokens, accepted = dops.verify_drafts(wide[:, :, 3:1004], torch.from_numpy(drafts).cuda(), torch.from_numpy(u).cuda(), temperature=one, top_k=(30 * one).int(), top_p=0.9 * one)
    assert np.array_equal(tokens.cpu().numpy(), want) and np.array_equal(accepted.cpu().numpy(), count)


# ---- copies and moves -----------------------------------------------------------------------------------------------------------


def pools(layers, pages, heads, page, dim, dtype, seed=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return [torch.randn(layers, pages, heads, page, dim, generator=g, device="cuda").to(dtype) for _ in range(2)]


@pytest.mark.parametrize("layers, heads, page, dim, dtype", [(1, 1, 1, 1, F16), (3, 2, 16, 64, F16), (2, 8, 16, 128, BF16), (2, 3, 5, 7, F32), (5, 4, 64, 256, F16), (1, 2, 16, 33, BF16), (40, 1, 16, 2, F16)])
def test_copies_of_pages(dops, layers, heads, page, dim, dtype):
    k, v = pools(layers, 30, heads, page, dim, dtype)
    order = np.random.default_rng(1).permutation(30)
    rows = [page, 1, max(1, page - 1), 0, max(1, page // 2), page]
    copies = [(order[i % 3], order[10 + i], r) for i, r in enumerate(rows)] + [(order[20], order[20], page)]
    want = [k.clone(), v.clone()]
    for x in want:
        for s, d, r in copies:
            x[:, d, :, :r] = x[:, s, :, :r]
    dops.copy_pages(k, v, torch.tensor(np.array(copies), dtype=torch.int32, device="cuda"))
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])


def test_copies_of_many_pages_and_none(dops):
    k, v = pools(2, 2000, 2, 16, 64, F16)
    order = torch.randperm(2000, device="cuda")[:1800].view(2, 900)
    copies = torch.stack([order[0], order[1], torch.full_like(order[0], 16)], 1).int()
    want = [k.clone(), v.clone()]
    for x in want:
        x[:, order[1]] = x[:, order[0]]
    dops.copy_pages(k, v, copies)
    dops.copy_pages(k, v, copies[:0])
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])


def test_copies_of_bad_pages_are_told_and_left_out(dops):
    capi = importlib.import_module("macllm_infer_b200._capi")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    k, v = pools(2, 10, 2, 16, 64, F16)
    want = k.clone()
    want[:, 5] = want[:, 4]
    dops.copy_pages(k, v, torch.tensor([[-1, 1, 16], [1, 10, 16], [4, 5, 16], [2, 3, 17], [2, 3, -1]], dtype=torch.int32, device="cuda"), status=status)
    assert torch.equal(k, want)
    with pytest.raises(capi.MkError, match="page number"):
        dops.check_status(status)


def gather_plain(x, from_tables, keep, counts, to_tables, first, page):
    out = x.clone()
    for lane, n in enumerate(counts.tolist()):
        for j in range(n):
            s, d = int(keep[lane, j]), int(first[lane]) + j
            out[:, int(to_tables[lane, d // page]), :, d % page] = x[:, int(from_tables[lane, s // page]), :, s % page]
    return out


@pytest.mark.parametrize("layers, heads, page, dim, dtype", [(1, 1, 16, 64, F16), (3, 2, 16, 128, BF16), (2, 3, 5, 7, F32), (2, 4, 64, 256, F16), (1, 2, 16, 33, F16), (70, 1, 16, 64, F16)])
@pytest.mark.parametrize("same_pages", [False, True])
def test_kept_tokens_move_together(dops, layers, heads, page, dim, dtype, same_pages):
    rng = np.random.default_rng(2)
    lanes, context = 5, 300
    width = -(-context // page)
    k, v = pools(layers, 2 * lanes * width, heads, page, dim, dtype)
    ids = torch.from_numpy(rng.permutation(2 * lanes * width)).int().cuda()
    from_tables = ids[:lanes * width].view(lanes, width)
    to_tables = from_tables if same_pages else ids[lanes * width:].view(lanes, width)
    counts, first = [0, 1, 130, 299, 40], [3, 7, 20, 1, 100]
    keep = torch.full((lanes, 299), -1, dtype=torch.int32)
    for i, n in enumerate(counts):
        low = first[i]
        keep[i, :n] = torch.from_numpy(np.sort(rng.permutation(np.arange(low, context))[:n])).int()
    keep, counts, first = keep.cuda(), torch.tensor(counts, dtype=torch.int32, device="cuda"), torch.tensor(first, dtype=torch.int32, device="cuda")
    want = [gather_plain(x, from_tables, keep, counts, to_tables, first, page) for x in (k, v)]
    dops.gather_tokens(k, v, from_tables, keep, counts, to_tables, first)
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])


def test_a_long_lane_is_moved_by_one(dops):
    """In place, every token into its neighbour's row."""
    page, context = 16, 5000
    k, v = pools(1, 313, 2, page, 64, F16)
    table = torch.randperm(313, device="cuda").int().view(1, 313)
    keep = torch.arange(1, context, device="cuda").int().view(1, -1)
    n, zero = torch.tensor([context - 1], dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    want = [gather_plain(x, table, keep, n, table, zero, page) for x in (k, v)]
    dops.gather_tokens(k, v, table, keep, n, table, zero)
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])


def test_bad_positions_are_told_and_left_out(dops):
    capi = importlib.import_module("macllm_infer_b200._capi")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    k, v = pools(2, 10, 2, 16, 64, F16)
    before = k.clone()
    table = torch.tensor([[1, 2], [3, 40]], dtype=torch.int32, device="cuda")
    one = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    for keep, counts, first, message in (([[5, 32], [5, 6]], (2, 0), (0, 0), "range"), ([[-1, 6], [5, 6]], (1, 0), (0, 0), "range"), ([[5, 6], [5, 6]], (3, 0), (0, 0), "range"),
                                         ([[5, 6], [5, 6]], (-1, 0), (0, 0), "range"), ([[5, 6], [5, 6]], (2, 0), (31, 0), "range"), ([[5, 6], [5, 6]], (2, 0), (-1, 0), "range"),
                                         ([[5, 6], [17, 20]], (0, 2), (0, 0), "page number"), ([[5, 6], [5, 6]], (0, 2), (0, 20), "page number")):
        dops.gather_tokens(k, v, table, one(*keep), one(*counts), table, one(*first), status=status)
        with pytest.raises(capi.MkError, match=message):
            dops.check_status(status)
    assert torch.equal(k[:, 4:], before[:, 4:]) and torch.equal(k[:, 0], before[:, 0])


# ---- together -------------------------------------------------------------------------------------------------------------------


def test_operators_in_a_captured_graph_and_on_another_stream(dops):
    """What a graph reads is what the buffers hold when it is replayed; two graphs share nothing."""
    b = Batch(F16, 8, 2, 128, 16, 640, [40, 300, 700], 2, seed=20)
    c = Batch(F16, 8, 2, 128, 16, 320, [5, 900], 3, seed=21)
    logits, drafts, u, _ = verify_case(11, 3, 2, 2000)
    args = [torch.from_numpy(x).cuda() for x in (drafts, u)]
    logits, one, k = logits.cuda(), torch.ones(3, device="cuda"), torch.full((3,), 20, dtype=torch.int32, device="cuda")
    b.run(dops)
    dops.verify_drafts(logits, *args, temperature=one, top_k=k, top_p=0.9 * one)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    graphs, outs = [], []
    with torch.cuda.stream(side):
        for x in (b, c):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                outs.append((x.run(dops), dops.verify_drafts(logits, *args, temperature=one, top_k=k, top_p=0.9 * one)))
            graphs.append(graph)
    first = [x.run(dops) for x in (b, c)]
    for seed in (1, 2):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        for x in (b, c):
            x.q.copy_(torch.randn(x.q.shape, generator=g, device="cuda"))
        b.lengths[1] = 640 + 100 + seed
        args[1].uniform_(generator=g)
        torch.cuda.synchronize()
        for _ in range(3):
            for graph in graphs:
                graph.replay()
        torch.cuda.synchronize()
        want = dops.verify_drafts(logits, *args, temperature=one, top_k=k, top_p=0.9 * one)
        for x, (out, verified) in zip((b, c), outs):
            x.check(out)
            assert torch.equal(out, x.run(dops)) and all(torch.equal(p, q) for p, q in zip(verified, want))
    with torch.cuda.stream(side):
        again = [x.run(dops) for x in (b, c)]
    side.synchronize()
    for x, out in zip((b, c), again):
        x.check(out)
    assert not torch.equal(first[0], again[0])


def test_samples_of_one_prompt_from_fork_to_verification(dops):
    """Three samples forked inside a page, two ticks of drafted rows for each, the second behind what the first kept; an accepted branch is moved together.  The attention of every
    tick is checked against the cache as it then is, and lanes never see one another's rows."""
    layers, heads, kv_heads, dim, page, prompt = 2, 8, 2, 64, 16, 16 * 9 + 5
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    k, v = pools(layers, 64, kv_heads, page, dim, F16, seed=6)
    shared = prompt // page * page
    tables = torch.zeros(3, 14, dtype=torch.int32, device="cuda")
    tables[:, :10] = torch.arange(10, device="cuda").int()
    dops.copy_pages(k, v, torch.tensor([[9, 20, prompt - shared], [9, 21, prompt - shared]], dtype=torch.int32, device="cuda"))
    tables[1, 9], tables[2, 9] = 20, 21
    for lane in range(3):
        tables[lane, 10:] = torch.arange(30 + 4 * lane, 34 + 4 * lane, device="cuda").int()
    assert torch.equal(k[:, 20, :, :5], k[:, 9, :, :5])
    lengths = torch.full((3,), prompt, dtype=torch.int32, device="cuda")
    vocab, n = 300, 3
    one = torch.ones(3, device="cuda")
    for tick in range(2):
        rows = n + 1
        position = lengths.long()[:, None] + torch.arange(rows, device="cuda")
        for x in (k, v):   # the new rows' keys and values are written before attention
            x[:, torch.gather(tables.long(), 1, position // page), :, position % page] = torch.randn(3, rows, layers, kv_heads, dim, generator=g, device="cuda").half()
        q = torch.randn(3 * rows, heads, dim, generator=g, device="cuda").half()
        for layer in range(layers):
            out = dops.shared_attention(q, k[layer], v[layer], tables, lengths + rows, shared, scale=0.125)
            for lane in range(3):
                m = int(lengths[lane]) + rows
                kk, vv = (x[layer][tables[lane].long()].double().permute(1, 0, 2, 3).flatten(1, 2)[:, :m].repeat_interleave(4, 0) for x in (k, v))
                s = q[lane * rows:(lane + 1) * rows].double().transpose(0, 1) @ kk.transpose(1, 2) * 0.125
                s = s.masked_fill(torch.arange(m, device="cuda")[None] > torch.arange(m - rows, m, device="cuda")[:, None], -math.inf)
                want = (torch.softmax(s, -1) @ vv).transpose(0, 1)
                assert (out[lane * rows:(lane + 1) * rows].double() - want).abs().max() < 4 * 2 ** -11 * vv.abs().max()
        logits = 2 * torch.randn(3, rows, vocab, generator=g, device="cuda")
        drafts = logits[:, :n].argmax(-1).int()
        tokens, accepted = dops.verify_drafts(logits, drafts, torch.rand(3, rows, generator=g, device="cuda"), temperature=0.5 * one, top_k=torch.full((3,), 40, dtype=torch.int32, device="cuda"),
                                              top_p=0.95 * one)
        assert ((tokens >= 0).sum(1) == accepted + 1).all()
        # as for a tree of drafts: the row in front and every other one behind it stay, in the first rows
        keep = torch.stack([lengths, lengths + 2], 1).int()
        before = [x.clone() for x in (k, v)]
        dops.gather_tokens(k, v, tables, keep, torch.full((3,), 2, dtype=torch.int32, device="cuda"), tables, lengths)
        for x, y in zip((k, v), before):
            assert torch.equal(x, gather_plain(y, tables, keep, torch.full((3,), 2), tables, lengths, page))
        lengths += 2
