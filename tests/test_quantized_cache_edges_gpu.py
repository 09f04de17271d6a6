"""Caches in 4 and 8 bits at the edges of what their calls allow: what is not finite, what some rows do not see, magnitudes far apart, rows behind the last."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_quantized_cache_gpu import BF16, F16, INT, Cache, attend, check_attention, codes_and_scales, dops, generator, ints, queries, unpacked  # noqa: E402, F401 (dops is a fixture)


# ---- what is not finite under a cap -------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("rows", [1, 3, 40])
@pytest.mark.parametrize("softcap", [50.0, 1000.0])
def test_what_is_not_finite_stays_so_under_a_cap(dops, rows, softcap):  # noqa: F811
    """A key or a query that is not a number has no score, capped or not; what a row does not see has no say."""
    c = Cache(F16, 4, 2, 128, 16, [200, 90, 70], rows, seed=30).fill()
    q = queries(c, 8)
    c.pools[2][int(c.tables[0, 3])][0, 5, 1, 1] = math.nan          # a key of head 0 that every row of lane 0 sees
    c.pools[3][int(c.tables[1, 1])][1, 2, 0, 0] = math.nan          # a value's first half, of head 1, lane 1
    c.pools[2][int(c.tables[2, 69 // 16])][:, 69 % 16] = math.nan   # the last key of lane 2, which only its last row sees
    if rows > 1:
        q[2 * rows, 3, 7] = math.nan
    got = attend(dops, c, q, softcap=softcap)
    plain = attend(dops, c, q)
    want = torch.zeros_like(got, dtype=torch.bool)
    want[:rows, :4] = True
    want[rows:2 * rows, 4:, :64] = True
    want[3 * rows - 1] = True
    if rows > 1:
        want[2 * rows, 3] = True
    assert torch.equal(torch.isnan(got), want) and torch.equal(torch.isnan(plain), want)


@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("softcap", [50.0, 1000.0])
def test_infinite_scores_reach_the_cap(dops, rows, softcap):  # noqa: F811
    """Scores far beyond the cap are the cap, of either sign."""
    c = Cache(BF16, 8, 1, 64, 16, [40], rows, seed=31)
    x = torch.ones(40, 1, 64, device="cuda", dtype=BF16)
    x[::2] *= -1
    dops.quantize_rows(x * 1e10, x, c.pools, c.tables, c.lengths, cu_seqlens=ints([0, 40]))
    q = torch.full((c.total, 2, 64), 1e10, dtype=BF16, device="cuda")
    got = attend(dops, c, q, softcap=softcap)
    assert (got[-1] == 1).all()   # e^(-2 softcap) is nothing


@pytest.mark.parametrize("own, rows, heads", [([40, 90], 1, (8, 2, 128)), ([700, 90], 1, (8, 2, 128)), ([300, 200], 40, (8, 2, 128)), ([300, 200], 40, (4, 1, 256)), ([500] * 40, 1, (8, 2, 64))])
@pytest.mark.parametrize("softcap", [50.0, 1000.0])
def test_keys_that_are_no_numbers_under_a_cap_in_16_bits(dops, own, rows, heads, softcap):  # noqa: F811
    """The same of shared_attention, whose caps are the same function."""
    from test_device_ops_gpu import Batch
    for shared in (0, 256):
        b = Batch(F16, *heads, 16, shared, own, rows, seed=32)
        n = int(b.lengths[0])
        place = (n - rows) // 2
        b.pools[0][int(b.tables[0, place // 16])][:, place % 16] = math.nan
        seen_by = [i for i in range(len(own)) if i == 0 or place < shared]
        want = torch.zeros(len(own), rows, dtype=torch.bool, device="cuda")
        want[seen_by] = True
        for cap in (0.0, softcap):
            got = torch.isnan(b.run(dops, softcap=cap)).flatten(1)
            assert torch.equal(got.all(1), want.flatten()) and torch.equal(got.any(1), want.flatten())


# ---- rows behind the last one -------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("total", [3, 4097, 4098, 40001, 40003])
@pytest.mark.parametrize("bits, dtype", [(4, F16), (8, BF16)])
def test_rows_behind_the_last_are_left_alone(dops, bits, dtype, total):  # noqa: F811
    """One, two and four rows to a warp: rows in front of the last one are right, and nothing behind it is read or written, whatever the list of rows says."""
    counts = [total // 3, 0, total - total // 3 - total // 4, total // 4]
    lengths = [n + 5 for n in counts]
    c = Cache(dtype, bits, 2, 64, 64, lengths, counts, seed=33)
    guard = 8
    x = torch.full((2, total + guard, 2, 64), 777.0, dtype=dtype, device="cuda")
    x[:, :total] = torch.randn(2, total, 2, 64, generator=c.g, device="cuda").to(dtype)
    back = torch.full_like(x, 555.0)
    status = torch.zeros(1, dtype=INT, device="cuda")

    def both(cu, lengths):
        dops.quantize_rows(x[0, :total], x[1, :total], c.pools, c.tables, lengths, cu_seqlens=cu, status=status)
        dops.dequantize_rows(c.pools, c.tables, lengths, total, cu_seqlens=cu, k=back[0, :total], v=back[1, :total], status=status)
        assert (back[:, total:] == 555).all()

    both(c.cu, c.lengths)
    assert status.item() == 0
    code, scale = codes_and_scales(x[:, :total], bits)
    want = (scale[..., 1:] + scale[..., :1] * code.unflatten(-1, (-1, 64))).flatten(-2)
    eps = torch.finfo(dtype).eps
    assert ((back[:, :total].double() - want).abs() <= eps / 2 * want.abs() * (1 + 2 ** -10) + torch.finfo(dtype).smallest_normal * eps * 0.51).all()
    # a list that ends behind the last row: its last lane has no rows that could be trusted, the others have theirs
    before = [p.clone() for p in c.pools]
    good = back.clone()
    for beyond in (1, 2, 3, 7, 1 << 20, 2 ** 31 - 1 - total):
        cu = c.cu.clone()
        cu[-1] += beyond
        status.zero_()
        both(cu, c.lengths)
        assert status.item() == (dops.BAD_RANGE if counts[-1] else 0)   # a lane all of whose rows lie behind has none
        first = total - counts[-1]
        assert torch.equal(back[:, :first], good[:, :first]) and (back[:, first:total] == 0).all()
        assert all(torch.equal(p.float().nan_to_num(-1), q.float().nan_to_num(-1)) for p, q in zip(c.pools, before))
    for wrong, told in (([-1, 1, 2, 3, total], dops.BAD_RANGE), ([0, 1, 2, total - 1, total + 1], dops.BAD_RANGE), ([0, 2, 1, 3, total], 0), ([0, 0, 0, total, total + 5], 0)):
        status.zero_()
        both(ints(wrong), ints([total + 9] * 4))
        assert status.item() & told == told


# ---- shares -------------------------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("length", [60, 6000])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_a_value_that_is_not_finite_reaches_every_row_that_sees_it(dops, rows, length, dim):  # noqa: F811
    """However small its weight is, and whether or not the lane's keys are shared out."""
    c = Cache(BF16, 4, 1, dim, 16, [length + rows], rows, seed=34)
    n = length + rows
    x = torch.ones(n, 1, dim, dtype=BF16, device="cuda")
    x[: n // 3] = -1   # keys whose scores are below the others' by 2 * 32 * dim^0.5, 2^-739 and less
    v = torch.randn(n, 1, dim, generator=c.g, device="cuda").to(BF16)
    v[5, 0, dim - 64:] = math.nan
    dops.quantize_rows(x, v, c.pools, c.tables, c.lengths, cu_seqlens=ints([0, n]))
    q = torch.full((c.total, 4, dim), 32.0, dtype=BF16, device="cuda")
    got = attend(dops, c, q)
    assert torch.isnan(got[..., dim - 64:]).all() and torch.isfinite(got[..., :dim - 64]).all()


@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("shared", [0, 256])
@pytest.mark.parametrize("heads", [(8, 2, 64), (4, 1, 128), (4, 1, 256)])
def test_a_value_that_is_not_finite_reaches_every_row_that_sees_it_in_16_bits(dops, rows, shared, heads):  # noqa: F811
    """The same of shared_attention, whose lanes are shared out alike."""
    from test_device_ops_gpu import Batch
    b = Batch(F16, *heads, 16, shared, [5000, 90], rows, seed=44)
    n = int(b.lengths[0])
    ids = b.tables[0, :-(-n // 16)].long()
    b.pools[0][ids] = 1.0
    b.pools[0][b.tables[0, :n // 48].long()] = -1.0   # keys whose scores are below the others' by 2 * 32 * dim^0.5, 2^-739 and less
    b.pools[1][int(b.tables[0, 0])][:, 5, :heads[2] // 2] = math.nan
    b.q.fill_(32.0)
    got = torch.isnan(b.run(dops))
    assert got[:rows, :, :heads[2] // 2].all() and not got[:rows, :, heads[2] // 2:].any()


# ---- magnitudes far apart -----------------------------------------------------------------------------------------------------------------


def put(c, lane, position, kind, x):
    """One token's keys (kind 0) or values (1), [kv heads][dim], by the definition."""
    code, scale = codes_and_scales(x.to(c.dtype), c.bits)
    code = code.to(torch.uint8)
    page, at = int(c.tables[lane, position // c.page]), position % c.page
    c.pools[kind][page][:, at] = code[..., ::2] | code[..., 1::2] << 4 if c.bits == 4 else code
    c.pools[2 + kind][page][:, at] = scale.to(c.dtype)


HUGE = [(F16, 6e4), (BF16, 1e10), (BF16, 1e30)]


@pytest.mark.parametrize("dtype, huge", HUGE)
@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("dim, bits", [(64, 8), (128, 4), (256, 8)])
@pytest.mark.parametrize("rows", [2, 5, 12, 40, 90])
def test_what_later_rows_see_has_no_say(dops, dtype, huge, kind, dim, bits, rows):  # noqa: F811
    """A last token whose keys or values are far above all others': the rows before it, which do not see it, are as exact as ever."""
    c = Cache(dtype, bits, 1, dim, 16, [rows + 60, rows + 1, 3 * rows], rows, seed=35).fill()
    q = queries(c, 4)
    for lane, n in enumerate(c.lengths_list):
        x = torch.randn(1, dim, generator=c.g, device="cuda")
        put(c, lane, n - 1, kind, x / x.abs().max() * huge)
    got = attend(dops, c, q)
    keep = [i for i in range(c.total) if (i + 1) % rows]   # all but each lane's last row
    clean = Cache(dtype, bits, 1, dim, 16, [n - 1 for n in c.lengths_list], rows - 1, seed=35)
    clean.pools, clean.tables = c.pools, c.tables
    check_attention(clean, q[keep], got[keep])


@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("dim, bits", [(64, 4), (128, 8), (256, 8)])
@pytest.mark.parametrize("rows", [2, 12, 40])
def test_sizes_at_both_ends_of_the_type(dops, kind, dim, bits, rows):  # noqa: F811
    """Keys or values of 1e-20 beside ones of 1e30 that only later rows see."""
    c = Cache(BF16, bits, 1, dim, 16, [rows + 60, rows + 1, 3 * rows], rows, seed=42).fill()
    c.pools[2 + kind].copy_((c.pools[2 + kind].float() * 2.0 ** -66).to(BF16))
    q = queries(c, 4)
    if kind == 0:
        q *= 2.0 ** 66
    for lane, n in enumerate(c.lengths_list):
        x = torch.randn(1, dim, generator=c.g, device="cuda")
        put(c, lane, n - 1, kind, x / x.abs().max() * 1e30)
    got = attend(dops, c, q)
    keep = [i for i in range(c.total) if (i + 1) % rows]
    clean = Cache(BF16, bits, 1, dim, 16, [n - 1 for n in c.lengths_list], rows - 1, seed=42)
    clean.pools, clean.tables = c.pools, c.tables
    check_attention(clean, q[keep], got[keep])


@pytest.mark.parametrize("dtype, huge", HUGE)
@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("dim, bits", [(64, 4), (128, 8), (256, 4)])
@pytest.mark.parametrize("rows", [1, 6, 40])
def test_what_is_in_front_of_the_window_has_no_say(dops, dtype, huge, kind, dim, bits, rows):  # noqa: F811
    window = 100
    c = Cache(dtype, bits, 1, dim, 16, [rows + 300, rows + 117], rows, seed=36).fill()
    q = queries(c, 4)
    for lane, n in enumerate(c.lengths_list):
        for position in (n - rows - window - 9, n - rows - window):   # the latter is the last that no row sees
            x = torch.randn(1, dim, generator=c.g, device="cuda")
            put(c, lane, position, kind, x / x.abs().max() * huge)
    check_attention(c, q, attend(dops, c, q, window=window), window=window)
    x = torch.randn(1, dim, generator=c.g, device="cuda")
    if rows > 1:   # the first row sees one more, the others do not
        put(c, 0, c.lengths_list[0] - rows - window + 1, kind, x / x.abs().max() * huge)
        got = attend(dops, c, q, window=window)
        check_attention(Tail(c), q[1:rows], got[1:rows], window=window)


class Tail(Cache):
    """Lane 0 of a cache without its first row."""

    def __init__(self, c):
        self.__dict__.update(c.__dict__)
        self.lengths_list, self.rows = c.lengths_list[:1], [c.rows[0] - 1]


@pytest.mark.parametrize("dtype, huge", HUGE)
@pytest.mark.parametrize("dim, bits", [(64, 4), (128, 8), (256, 8)])
@pytest.mark.parametrize("rows, length", [(1, 90), (6, 1500), (40, 90), (40, 1500)])
def test_a_huge_value_with_no_weight_has_no_say(dops, dtype, huge, dim, bits, rows, length):  # noqa: F811
    """Its weight times its size is far below what the others have, in front of them, among them and behind most."""
    c = Cache(dtype, bits, 1, dim, 16, [length + rows], rows, seed=37).fill()
    n = length + rows
    q = torch.ones(c.total, 4, dim, dtype=dtype, device="cuda") + (0.5 * torch.randn(c.total, 4, dim, generator=c.g, device="cuda")).to(dtype)
    low = torch.full((1, dim), -160.0 / dim ** 0.5, device="cuda")   # a score of about -160 where the others' are between -10 and 10
    for position in (0, 3, n // 2, n - rows - 2):
        put(c, 0, position, 0, low)
        put(c, 0, position, 1, torch.linspace(-huge, huge, dim, device="cuda")[None])
    check_attention(c, q, attend(dops, c, q))


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("rows, ratio", [(1, 1e10), (7, 1e30), (40, 1e5)])
def test_groups_of_one_head_far_apart(dops, bits, dim, rows, ratio):  # noqa: F811
    """Values of one group of 64 channels far above another's: each channel is as exact as its own group allows.  Above 32 items numbers have 11 bits down to 2^-21 of a token's largest."""
    c = Cache(BF16, bits, 2, dim, 16, [rows + 700, rows + 50], rows, seed=38).fill()
    c.pools[3][..., 0, :] = (c.pools[3][..., 0, :].float() * ratio).to(BF16)
    q = queries(c, 4 if rows < 40 else 8)
    check_attention(c, q, attend(dops, c, q))


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("rows", [1, 40])
def test_tokens_whose_sizes_rise_and_fall(dops, bits, dim, rows):  # noqa: F811
    """Keys and values of every size from 2^-20 to 2^20 in one context, in runs and mixed."""
    c = Cache(BF16, bits, 1, dim, 16, [rows + 1200, rows + 80], rows, seed=39).fill()
    for kind in (2, 3):
        by = torch.exp2(torch.randint(-20, 21, c.pools[kind].shape[:3], generator=c.g, device="cuda").float())
        by[1::2] = by[1::2, :, :1]   # every other page: all of its tokens alike
        if kind == 2:
            by = by.clamp(max=1)
        c.pools[kind].copy_((c.pools[kind].float() * by[..., None, None]).to(BF16))
    q = queries(c, 4)
    check_attention(c, q, attend(dops, c, q))


@pytest.mark.parametrize("seed", range(6))
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dim, dtype, span", [(128, F16, 6), (128, BF16, 30), (256, BF16, 12)])
@pytest.mark.parametrize("rows, window", [(1, 1000), (3, 0)])
def test_a_few_tokens_of_other_sizes(dops, dim, dtype, span, bits, rows, window, seed):  # noqa: F811
    """One token in fifty, and groups, of other sizes: the items of a warp have met different ones when the next come, so that its threads judge them differently."""
    c = Cache(dtype, bits, 3, dim, 32, [501, 1433, 90], rows, seed=43 + seed).fill()
    for kind in (2, 3):
        scales = c.pools[kind]
        f = torch.randint(-span, span + 1, scales.shape[:3], generator=c.g, device="cuda").float() * (torch.rand(scales.shape[:3], generator=c.g, device="cuda") < 0.02)
        f = f[..., None] + torch.randint(-3, 4, scales.shape[:4], generator=c.g, device="cuda").float()
        scales.copy_((scales.float() * torch.exp2(f.clamp(max=0) if kind == 2 else f)[..., None]).to(dtype))
    q = queries(c, 15)
    check_attention(c, q, attend(dops, c, q, window=window), window=window)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows", [1, 40])
def test_many_light_keys_behind_a_heavy_one(dops, dtype, rows):  # noqa: F811
    """One key has nearly all of the weight and a value of 0; 8000 have 2^-25.5 of it each and the value 1, and together the result."""
    n = 8000 + rows
    c = Cache(dtype, 4, 1, 64, 16, [n], rows, seed=40)
    k = torch.full((n, 1, 64), -25.5 * math.log(2) / 8, device="cuda").to(dtype)
    v = torch.ones(n, 1, 64, dtype=dtype, device="cuda")
    k[3], v[3] = 0, 0
    dops.quantize_rows(k, v, c.pools, c.tables, c.lengths, cu_seqlens=ints([0, n]))
    q = torch.ones(c.total, 4, 64, dtype=dtype, device="cuda")
    got = attend(dops, c, q)
    check_attention(c, q, got)
    assert (got > 2 ** -14).all()


# ---- codes --------------------------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("bits", [4, 8])
def test_codes_are_the_nearest_where_sizes_are_far_apart(dops, dtype, bits):  # noqa: F811
    """Values a hair above or below a half between two codes, where the lowest value is so far from them that 32 bits do not hold the difference."""
    g = generator(41)
    total, tiny = 300, 2.0 ** -24
    step = 2.0 ** torch.randint(-2, 3, (total, 1, 1), generator=g, device="cuda").double()
    # with low = -step / 2 (code 0) halves lie at 0 and at whole steps; the highest value makes the step a power of two
    low = -step / 2
    top = 2 ** bits - 1
    high = low + step * top * (1 + 2.0 ** -9 if dtype is BF16 else 1)
    half = step * torch.randint(0, 3, (total, 1, 64), generator=g, device="cuda").double()   # a code and a half
    off = torch.randint(-1, 2, (total, 1, 64), generator=g, device="cuda").double() * tiny
    x = torch.where(half == 0, off, half)
    x[..., :1], x[..., 1:2] = low, high
    x = x.to(dtype)
    code, scale = codes_and_scales(x, bits)
    c = Cache(dtype, bits, 1, 64, 16, [total], total, seed=41)
    dops.quantize_rows(x, x, c.pools, c.tables, c.lengths)
    for t, (page, at) in enumerate(c.slots()):
        for kind in (0, 1):
            assert torch.equal(unpacked(c.pools[kind][page][:, at], bits).double(), code[t]), (t, scale[t])
            assert torch.equal(c.pools[2 + kind][page][:, at].double(), scale[t])
