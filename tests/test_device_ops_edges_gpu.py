"""Operators over device buffers at the edges of what their calls allow: draws at the ends of the unit interval, settings and rows that end a lane, large caps, and the
forms of the attention that few sizes reach."""
import ctypes
import importlib
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
from test_device_ops_gpu import BF16, F16, F32, Batch, dops, pools, verify_case, verify_check, verify_plain  # noqa: E402,F401 (dops is a fixture)

pytestmark = pytest.mark.gpu


def verify(dops, logits, drafts, u, probs, temperature, top_k, top_p=1.0, status=None):
    lanes = len(u)
    settings = [torch.from_numpy(np.broadcast_to(np.asarray(v, dtype=d), (lanes,)).copy()) for v, d in ((temperature, np.float32), (top_k, np.int32), (top_p, np.float32))]
    tokens, accepted = dops.verify_drafts(logits.cuda(), torch.from_numpy(drafts).cuda(), torch.from_numpy(u).cuda(), temperature=settings[0].cuda(), top_k=settings[1].cuda(),
                                          top_p=settings[2].cuda(), draft_probs=None if probs is None else torch.from_numpy(probs).cuda(), status=status)
    return tokens.cpu().numpy(), accepted.cpu().numpy(), [x.numpy() for x in settings]


def masked_case(mask, kind, lanes, dtype, seed=40, vocab=9000, live=60):
    """Rows in which `live` tokens in the middle count and all others are masked: no draft, a looked-up one or one of a distribution, both on a masked token, and a
    distribution that covers the target's."""
    rng = np.random.default_rng(seed)
    logits = torch.full((lanes, 2, vocab), mask, dtype=F32)
    at = 5003 + 7 * np.arange(live)
    logits[:, :, at] = torch.tensor(rng.standard_normal((lanes, 2, live)), dtype=F32)
    if kind == "covers":
        logits[:, :, at[1:]] = mask
    if dtype != F32:
        logits = logits.clamp_min(torch.finfo(dtype).min if math.isfinite(mask) else -math.inf).to(dtype)
    drafts, probs = np.full((lanes, 1), -1 if kind == "none" else 3, np.int32), None
    if kind == "given":
        z = np.exp(rng.standard_normal((lanes, 1, vocab)))
        probs = (z / z.sum(-1, keepdims=True)).astype(np.float32)
    elif kind == "covers":
        probs = np.zeros((lanes, 1, vocab), np.float32)
        probs[:, :, at[0]] = 1.0
        probs[:, :, 3] = 1e-9
    return logits, drafts, probs


@pytest.mark.parametrize("mask", [-math.inf, -1e9, -3.0e38, -100.0])
@pytest.mark.parametrize("kind", ["none", "looked up", "given", "covers"])
@pytest.mark.parametrize("lanes, dtype", [(1, F32), (60, F32), (100, F32), (3, F16), (3, BF16)])
def test_whole_vocabulary_draws_at_the_ends_of_the_unit_interval(dops, mask, kind, lanes, dtype):
    """Masked tokens in front and behind: u = 0 draws the first token that has a weight in 64 bits (a mask of -100 leaves one), the highest u the last that counts."""
    logits, drafts, probs = masked_case(mask, kind, lanes, dtype)
    for end in (0.0, 1e-30, 2.0 ** -24, 1.0 - 2.0 ** -24):
        u = np.full((lanes, 2), 0.5, np.float32)
        u[:, 1] = end
        tokens, accepted, (t, k, p) = verify(dops, logits, drafts, u, probs, 0.9, 0)
        want, count, _ = verify_plain(logits.float().numpy(), drafts, u, t, k, p, probs)
        assert np.array_equal(accepted, count) and np.array_equal(tokens, want), (end, tokens[:3].tolist(), want[:3].tolist())


@pytest.mark.parametrize("kind", ["none", "looked up", "given", "covers"])
@pytest.mark.parametrize("vocab", [32000, 128256])
def test_a_draw_of_zero_behind_a_long_mask(dops, kind, vocab):
    logits, drafts, probs = masked_case(-math.inf, kind, 2, F32, vocab=vocab)
    u = np.zeros((2, 2), np.float32)
    tokens, _, _ = verify(dops, logits, drafts, u, probs, 1.0, 0)
    assert (tokens[:, 0] == 5003).all()


@pytest.mark.parametrize("vocab, lanes, dtype", [(1000, 40, F32), (20001, 60, F16), (20001, 100, BF16), (128256, 3, F32)])
@pytest.mark.parametrize("off", [0.0, 3e-5])
def test_a_remainder_of_roundings_is_drawn_from_as_it_is(dops, vocab, lanes, dtype, off):
    """A draft's distribution that is the target's but for the drafted token, and for 32-bit roundings or a little more: what is left of p - q then is less than what 32-bit weights round."""
    rng = np.random.default_rng(48)
    logits = torch.tensor(2.0 * rng.standard_normal((lanes, 2, vocab)), dtype=F32).to(dtype)
    p = torch.softmax(logits.double() / 0.875, -1)[:, :1].numpy()
    drafts = p.argmax(-1).astype(np.int32)
    probs = p * (1.0 + off * rng.standard_normal(p.shape))
    np.put_along_axis(probs, drafts[:, :, None], np.take_along_axis(p, drafts[:, :, None], -1) * 1.01, -1)
    probs = probs.astype(np.float32)
    u = np.full((lanes, 2), 0.999, np.float32)
    u[:, 1] = rng.random(lanes)
    tokens, accepted, settings = verify(dops, logits, drafts, u, probs, 0.875, 0)
    want, count, _ = verify_plain(logits.float().numpy(), drafts, u, *settings, probs)
    assert not count.any() and np.array_equal(accepted, count)
    # p - q is 2^-26 of p or more on average, in numbers of 2^-52 of p each: sums of them are off by less than 2^-24 of the whole, 416000 of them by chance; a border is met about that often
    assert (tokens != want).any(1).sum() <= lanes // 50, (tokens[:5].tolist(), want[:5].tolist())


@pytest.mark.parametrize("mask", [-math.inf, -1e9, -100.0, -45.0])
@pytest.mark.parametrize("kind", ["none", "looked up", "given", "covers"])
@pytest.mark.parametrize("top_k", [50, 70, 128, 129, 1000])
def test_draws_among_candidates_at_the_ends_of_the_unit_interval(dops, mask, kind, top_k):
    """A top_k beyond the tokens that count takes masked ones in: where they have a weight in 64 bits, they have their share of the draw."""
    logits, drafts, probs = masked_case(mask, kind, 5, F32, seed=41)
    if mask > -1e6 and top_k != 129:   # no two alike
        logits -= (logits == mask) * 5 * torch.rand(logits.shape, generator=torch.Generator().manual_seed(42))
    for end in (0.0, 1e-30, 2.0 ** -24, 1.0 - 2.0 ** -24):
        u = np.full((5, 2), 0.5, np.float32)
        u[:, 1] = end
        tokens, accepted, (t, k, p) = verify(dops, logits, drafts, u, probs, 0.9, top_k)
        want, count, _ = verify_plain(logits.numpy(), drafts, u, t, k, p, probs)
        assert np.array_equal(accepted, count) and np.array_equal(tokens, want), (end, tokens.tolist(), want.tolist())


@pytest.mark.parametrize("vocab, top_k", [(2, 2), (3, 3), (17, 17), (257, 129), (700, 700)])
@pytest.mark.parametrize("t, low", [(1.0, -60.0), (0.3, -20.0), (50.0, -30000.0), (1.0, -40.0)])
def test_a_light_token_beside_a_heavy_one_has_its_share(dops, vocab, top_k, t, low):
    """Sums of a thread's two candidates are not taken apart again, where the lighter one would be lost in the other."""
    logits = torch.full((3, 1, vocab), low)
    logits[0, 0, 1], logits[1, 0, vocab - 1], logits[2, 0, vocab // 2] = 1.0, 1.0, 1.0
    logits[:, :, ::2] -= torch.arange((vocab + 1) // 2) * t / 16   # no two alike
    drafts = np.empty((3, 0), np.int32)
    for u in (0.0, 1e-45, 1e-30, 0.5, 1.0 - 2.0 ** -24):
        tokens, accepted, settings = verify(dops, logits, drafts, np.full((3, 1), u, np.float32), None, t, top_k)
        want, _, _ = verify_plain(logits.numpy(), drafts, np.full((3, 1), u, np.float32), *settings, None)
        assert np.array_equal(tokens, want), (u, tokens.tolist(), want.tolist())


@pytest.mark.parametrize("temperature, top_k", [(1.0, 0), (1.0, 9), (1.0, 200), (0.0, 0)])
def test_rows_that_a_lane_does_not_reach_are_not_told_of(dops, temperature, top_k):
    logits, drafts, u, _ = verify_case(42, 4, 3, 700)
    drafts[:] = logits[:, :3].argmax(-1).numpy()
    u[:, :3] = 0.0
    logits[1, 0, drafts[1, 0]] = -math.inf   # refused at once
    logits[1, 2, 30], logits[1, 3] = math.nan, -math.inf
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    _, accepted, _ = verify(dops, logits, drafts, u, None, temperature, top_k, status=status)
    assert accepted.tolist() == [3, 0, 3, 3]
    dops.check_status(status)


@pytest.mark.parametrize("top_k, top_p", [(0, 0.9), (-1, 0.5), (1025, 1.0), (5000, 0.9)])
def test_a_setting_that_the_call_does_not_have_ends_its_lane(dops, top_k, top_p):
    """No token is drawn from another distribution than the one asked for; greedy lanes have no use for either setting, and the other lanes get what they get alone."""
    capi = importlib.import_module("macllm_infer_b200._capi")
    logits, drafts, u, _ = verify_case(43, 6, 2, 3000)
    t, k, p = [0.8, 0.8, 0.0, 0.8, 1.1, 0.0], np.array([20, top_k, top_k, 0, 5, 0]), np.array([0.9, top_p, top_p, 1.0, 1.0, 1.0])
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    tokens, accepted, settings = verify(dops, logits, drafts, u, None, t, k, p, status=status)
    with pytest.raises(capi.MkError, match="range"):
        dops.check_status(status)
    assert accepted[1] == 0 and tokens[1].tolist() == [-1, -1, -1]
    rest = [0, 2, 3, 4, 5]
    want, count, margin = verify_plain(logits[rest].numpy(), drafts[rest], u[rest], *(x[rest] for x in settings), None)
    assert margin > 1e-7 and np.array_equal(tokens[rest], want) and np.array_equal(accepted[rest], count)


@pytest.mark.parametrize("rows", [17, -1])
def test_a_number_of_rows_that_a_page_has_not_is_out_of_range(dops, rows):
    capi = importlib.import_module("macllm_infer_b200._capi")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    k, v = pools(2, 10, 2, 16, 64, F16)
    before = k.clone()
    dops.copy_pages(k, v, torch.tensor([[2, 3, rows]], dtype=torch.int32, device="cuda"), status=status)
    assert torch.equal(k, before) and int(status) == dops.BAD_RANGE
    with pytest.raises(capi.MkError, match="length, count"):
        dops.check_status(status)


@pytest.mark.parametrize("cap", [3e4, 1e9, 3e38])
@pytest.mark.parametrize("dim, shared, rows", [(128, 160, 1), (64, 1600, 2), (256, 1600, 2), (128, 1600, 2), (128, 1600, 40)])
def test_caps_far_above_the_scores(dops, cap, dim, shared, rows):
    """cap tanh(x / cap) = x - x^3 / (3 cap^2) + ..: scores stay below 60 here, so a cap of 3e4 moves them by less than 60^3 / (3 * 9e8) = 8e-5, which is less than what the bound below
    has for a score's 32-bit sums: (dim + 8) 2^-24 of the largest sum of |scale q k|, above 20 here, is 8e-5 at heads of 64 and more at wider ones."""
    b = Batch(F16, 8, 2, dim, 16, shared, [rows, 40 + rows, 300], rows, seed=45, spread=4.0)
    b.check(b.run(dops, softcap=cap))


@pytest.mark.parametrize("shared, rows", [(160, 1), (1600, 2), (1600, 140)])
def test_one_head_with_any_stride(dops, shared, rows):
    """A dimension of one element has any stride: queries, pools and results say so, and what is written is where the rows are."""
    b = Batch(F16, 1, 1, 128, 16, shared, [rows, 40 + rows, 300], rows, seed=46, q_gap=128)
    n, pages = b.q.shape[0], b.pools[0].shape[0]
    b.q = b.q.as_strided((n, 1, 128), (256, 9, 1))
    b.pools = [b.pools[0], b.pools[1].as_strided((pages, 1, 16, 128), (2048, 3, 128, 1), b.pools[1].storage_offset())]
    b.check(b.run(dops))
    wide = torch.full((n, 384), 7.0, dtype=F16, device="cuda")
    out = wide.as_strided((n, 1, 128), (384, 5, 1))
    b.run(dops, out=out)
    b.check(out)
    assert (wide[:, 128:] == 7).all()


# ---- forms of the attention -----------------------------------------------------------------------------------------------------
#
# With few keys altogether every lane reads the shared ones itself, in one launch without parts; else the shared keys' kernel is there, and a lane's own go through the small
# products (up to 24 items; joined by the lane's CTA or by a kernel of its own) or the tall ones.  Which of them a call takes shows in its workspace, so that the sizes below stay what
# they are for.
FORMS = {
    "one launch": dict(heads=(8, 2, 128), shared=160, own=[40, 3], rows=1),
    "joined by lanes": dict(heads=(8, 2, 128), shared=1024, own=[40, 3], rows=2),
    "two groups, joined": dict(heads=(8, 2, 128), shared=1024, own=[40, 13], rows=4),
    "three groups, joined": dict(heads=(8, 2, 64), shared=1024, own=[40, 13], rows=6),
    "two groups, wide heads": dict(heads=(8, 2, 256), shared=1024, own=[40, 13], rows=4),
    "shares of own keys": dict(heads=(8, 2, 128), shared=1024, own=[1900, 13], rows=1),
    "tall, 128 items": dict(heads=(8, 2, 128), shared=1024, own=[400, 23], rows=10),
    "tall, 256 items": dict(heads=(8, 2, 64), shared=1024, own=[900, 83], rows=40),
    "tall, wide heads": dict(heads=(8, 2, 256), shared=1024, own=[700, 43], rows=20),
    "tall alone": dict(heads=(8, 2, 128), shared=0, own=[1500, 43], rows=20),
}


def form(name, dtype=F16, seed=50, **more):
    """A batch of that form; its workspace says that it is one."""
    f = FORMS[name]
    capi = importlib.import_module("macllm_infer_b200._capi")
    heads, kv_heads, dim = f["heads"]
    b = Batch(dtype, heads, kv_heads, dim, 16, f["shared"], f["own"], f["rows"], seed=seed, **more)
    lanes, rows, width = len(f["own"]), f["rows"], b.tables.shape[1]

    def parts(width, shared):
        need = ctypes.c_int64()
        capi.check(capi.lib().mk_k_shared_attention_workspace(heads, kv_heads, dim, 16, width, lanes, rows, lanes * rows, shared, 0, ctypes.byref(need)))
        return need.value // (lanes * rows * heads * (dim * 4 + 8))

    own = parts(width - f["shared"] // 16, 0)
    assert (own > 0) == (name.startswith("tall") or name == "shares of own keys")
    assert (parts(width, f["shared"]) > own) == (name not in ("one launch", "tall alone"))
    return b


@pytest.mark.parametrize("name", FORMS)
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("window, softcap", [(0, 0.0), (1, 0.0), (5, 20.0), (64, 0.0), (300, 300.0), (1000, 0.0), (1200, 200.0), (5000, 0.0)])
def test_windows_and_caps_in_every_form(dops, name, dtype, window, softcap):
    b = form(name, dtype, spread=2.0)
    b.check(b.run(dops, window=window, softcap=softcap), window, softcap)


@pytest.mark.parametrize("name", FORMS)
def test_lanes_of_different_rows_in_every_form(dops, name):
    """Rows that no lane has, lanes without rows and ones that are shorter than the shared part or than their rows."""
    f = FORMS[name]
    heads, kv_heads, dim = f["heads"]
    rows = [f["rows"], 0, 1, max(1, f["rows"] - 1), f["rows"]]
    own = [f["own"][0], 7, -f["shared"] // 2, f["own"][1], -f["shared"] + f["rows"] // 2]
    b = Batch(BF16, heads, kv_heads, dim, 16, f["shared"], own, rows, seed=51)
    q = torch.cat([b.q, b.q[:3]])
    for window in (0, 40):
        out = torch.full_like(q, 5.0)
        dops.shared_attention(q, *b.pools, b.tables, b.lengths, b.shared, scale=b.scale, cu_seqlens=b.cu, max_rows=f["rows"], out=out, window=window)
        b.check(out[:-3], window)
        assert (out[-3:] == 5).all()


@pytest.mark.parametrize("name", FORMS)
def test_strides_in_every_form(dops, name):
    b = form(name, seed=52, page_gap=256 * 24, q_gap=64)
    n, heads, dim = b.q.shape
    wide = torch.full((n + 2, heads * dim + 24), 7.0, dtype=F16, device="cuda")
    out = wide[1:n + 1, :heads * dim].view(n, heads, dim)
    assert b.run(dops, out=out) is out
    b.check(out)
    assert (wide[0] == 7).all() and (wide[n + 1] == 7).all() and (wide[:, heads * dim:] == 7).all()


@pytest.mark.parametrize("name", FORMS)
def test_bad_pages_lengths_and_rows_are_told_in_every_form(dops, name):
    """Whatever the index arrays hold is told of and read nowhere; the call after that is as if nothing had been."""
    capi = importlib.import_module("macllm_infer_b200._capi")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    b = form(name, seed=53)
    first = b.run(dops, status=status)
    b.check(first)
    dops.check_status(status)
    tables, lengths, rows = b.tables.clone(), b.lengths.clone(), FORMS[name]["rows"]
    places = [(0, b.shared // 16, -1), (1, b.shared // 16, 1 << 30), (1, int(lengths[1] - 1) // 16, -(1 << 31))]
    for lane, column, value in places + ([(0, 0, -5), (0, b.shared // 16 - 1, 10 ** 6)] if b.shared else []):
        b.tables[lane, column] = value
        b.run(dops, status=status)
        with pytest.raises(capi.MkError, match="page number"):
            dops.check_status(status)
        b.tables.copy_(tables)
    for length in (-3, -(1 << 31), b.tables.shape[1] * 16 + 1, 2 ** 31 - 1):
        b.lengths[1] = length
        b.run(dops, status=status)
        with pytest.raises(capi.MkError, match="length"):
            dops.check_status(status)
        b.lengths.copy_(lengths)
    n = 2 * rows
    for cu in ([0, n + 1, n], [-1, rows, n], [0, rows, n + 3], [n + 1, n + 2, n + 3], [0, 0, 2 ** 31 - 1], [0, -(1 << 31), n], [rows, rows + 1, 0]):
        dops.shared_attention(b.q, *b.pools, b.tables, b.lengths, b.shared, scale=b.scale, cu_seqlens=torch.tensor(cu, dtype=torch.int32, device="cuda"), max_rows=rows, status=status)
        with pytest.raises(capi.MkError, match="range"):
            dops.check_status(status)
    assert torch.equal(b.run(dops, status=status), first)
    dops.check_status(status)


@pytest.mark.parametrize("name", FORMS)
def test_every_form_in_two_graphs_and_on_two_streams(dops, name):
    """Replayed beside one another on streams of their own, and again: workspaces are each call's, and nothing is kept."""
    batches = [form(name, seed=54 + i) for i in range(2)]
    want = [b.run(dops) for b in batches]
    for b, x in zip(batches, want):
        b.check(x)
    streams, graphs, outs = [torch.cuda.Stream() for _ in batches], [], []
    torch.cuda.synchronize()
    for b, s in zip(batches, streams):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            outs.append(b.run(dops))
        graphs.append(graph)
    for _ in range(3):
        for x in outs:
            x.fill_(3.0)
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(outs, want))


# ---- large vocabularies ---------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("vocab", [256000, 416000])
@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("top_k", [0, 64, 1024])
def test_the_largest_vocabularies_from_odd_addresses(dops, vocab, dtype, top_k):
    """The most runs and the most shared memory that the kernels are cut for; rows begin off 16 bytes."""
    logits, drafts, u, _ = verify_case(47, 1, 2, vocab, dtype)
    want, count, margin = verify_plain(logits.float().numpy(), drafts, u, np.full(1, 0.9, np.float32), np.full(1, top_k, np.int32), np.ones(1, np.float32), None)
    assert margin > 1e-7
    wide = torch.full((1, 3, vocab + 13), math.nan, dtype=dtype, device="cuda")
    wide[:, :, 5:vocab + 5] = logits.cuda()
    one = torch.ones(1, device="cuda")
    tokens, accepted = dops.verify_drafts(wide[:, :, 5:vocab + 5], torch.from_numpy(drafts).cuda(), torch.from_numpy(u).cuda(), temperature=0.9 * one, top_k=(top_k * one).int(), top_p=one)
    assert np.array_equal(tokens.cpu().numpy(), want) and np.array_equal(accepted.cpu().numpy(), count)


def test_a_vocabulary_beyond_the_largest_is_refused(dops):
    capi = importlib.import_module("macllm_infer_b200._capi")
    one = torch.ones(1, device="cuda")
    with pytest.raises(capi.MkError, match="at most 416000"):
        dops.verify_drafts(torch.zeros(1, 1, 416001, device="cuda"), torch.zeros(1, 0, dtype=torch.int32, device="cuda"), one[:, None], temperature=one, top_k=one.int(), top_p=one)
