"""Caches of keys and values in 4 or 8 bits against plain implementations in 64 bits: rows written and read back, attention over the codes, and both as they are used together."""
import importlib
import itertools
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
INT = torch.int32


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


def ints(values):
    return torch.tensor(values, dtype=INT, device="cuda")


def codes_and_scales(x, bits):
    """The format's definition in 64 bits: codes [..., d] and (step, lowest value) [..., groups, 2] of rows x [..., d]."""
    top = 2 ** bits - 1
    g = x.double().unflatten(-1, (-1, 64))
    low, high = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    fine = torch.isfinite(high - low) & ((high - low) < 2.0 ** 128)   # a range in 32 bits
    step = torch.where(fine, ((high - low) / top).to(x.dtype).double(), math.nan)
    low = torch.where(fine, low, math.nan)
    code = torch.where(step > 0, torch.round((g - low) / step).clamp(0, top), 0.0).flatten(-2)
    return code, torch.cat([step, low], -1)


def unpacked(codes, bits):
    return torch.stack([codes & 15, codes >> 4], -1).flatten(-2) if bits == 4 else codes


def values(codes, scales, bits):
    s = scales.double()
    return (s[..., 1:] + s[..., :1] * unpacked(codes, bits).double().unflatten(-1, (-1, 64))).flatten(-2)


class Cache:
    """Lanes of the given lengths and rows over pools in whose other places codes are all ones and scales NaN; pages `gap` bytes further apart than they are long."""

    def __init__(self, dtype, bits, kv_heads, dim, page, lengths, rows, seed=0, gap=0, more_pages=3):
        g = generator(seed)
        self.g, self.dtype, self.bits, self.kv_heads, self.dim, self.page = g, dtype, bits, kv_heads, dim, page
        lanes = len(lengths)
        each = [-(-n // page) for n in lengths]
        pages, width = sum(each) + more_pages, max(each, default=0)

        def paged(row, of_dtype, fill, step):
            n = kv_heads * page * row
            return torch.full((pages, n + step), fill, dtype=of_dtype, device="cuda")[:, :n].view(pages, kv_heads, page, row)

        size = dim * bits // 8
        self.pools = [paged(size, torch.uint8, 255, gap) for _ in range(2)] + [paged(dim // 32, dtype, math.nan, gap).unflatten(-1, (-1, 2)) for _ in range(2)]
        ids = (torch.randperm(pages - 1, generator=g, device="cuda")[:pages - more_pages] + 1).to(INT)
        self.tables = torch.full((lanes, width + 1), 1 << 30, dtype=INT, device="cuda")[:, :width]   # entries behind a lane's are no pages
        at = 0
        for i, n in enumerate(each):
            self.tables[i, :n] = ids[at:at + n]
            at += n
        self.lengths_list, self.lengths = list(lengths), ints(lengths)
        self.rows = rows if isinstance(rows, list) else [rows] * lanes
        self.cu = ints([0, *itertools.accumulate(self.rows)]) if isinstance(rows, list) else None
        self.total = sum(self.rows)

    def fill(self, spread=1.0):
        """Whole contexts written by the definition."""
        for i, n in enumerate(self.lengths_list):
            for b in range(-(-n // self.page)):
                m = min(self.page, n - b * self.page)
                for kind in (0, 1):
                    x = spread * torch.randn(self.kv_heads, m, self.dim, generator=self.g, device="cuda")
                    if kind == 0:
                        x += torch.linspace(-2, 2, self.dim, device="cuda") * spread
                    code, scale = codes_and_scales(x.to(self.dtype), self.bits)
                    code = code.to(torch.uint8)
                    page = int(self.tables[i, b])
                    self.pools[kind][page][:, :m] = code[..., ::2] | code[..., 1::2] << 4 if self.bits == 4 else code
                    self.pools[2 + kind][page][:, :m] = scale.to(self.dtype)
        return self

    def tokens(self, lane, kind, n):
        """[n][kv heads][dim] in 64 bits."""
        ids = self.tables[lane, :-(-n // self.page)].long()
        return values(self.pools[kind][ids], self.pools[2 + kind][ids], self.bits).transpose(1, 2).flatten(0, 1)[:n]

    def slots(self):
        """(page, place in the page) of each row, None where it has none."""
        for lane, (n, rows) in enumerate(zip(self.lengths_list, self.rows)):
            for p in range(n - rows, n):
                yield (int(self.tables[lane, p // self.page]), p % self.page) if p >= 0 else None


# ---- rows into pages, and back ------------------------------------------------------------------------------------------------------------


def odd_rows(dtype, total, heads, dim, g):
    """Rows with groups that are constant, tiny, huge, one-sided, and with values that are not finite."""
    x = torch.randn(total, heads, dim, generator=g, device="cuda")
    flat = x.view(-1, 64)
    n = len(flat)
    big = torch.finfo(dtype).max
    small = torch.finfo(dtype).tiny
    for i, change in enumerate([lambda r: r.mul_(0), lambda r: r.fill_(-3.25), lambda r: r.mul_(small / 4), lambda r: r.mul_(0.01).add_(100), lambda r: r[5:6].fill_(math.nan),
                                lambda r: r[63:].fill_(math.inf), lambda r: r[:1].fill_(-math.inf), lambda r: (r[:1].fill_(big), r[1:2].fill_(0.45 * -big)), lambda r: r.round_(), lambda r: r.abs_(),
                                lambda r: r.mul_(0.25).round_().mul_(4), lambda r: (r.fill_(0), r[7:8].fill_(1.0)), lambda r: (r[:1].fill_(big), r[1:2].fill_(-big))]):
        change(flat[(3 + 5 * i) % n])
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dim, kv_heads, page", [(64, 4, 16), (64, 3, 32), (128, 1, 16), (128, 8, 64), (256, 5, 16), (256, 8, 128)])
def test_rows_written_and_read_back(dops, dtype, bits, dim, kv_heads, page):
    c = Cache(dtype, bits, kv_heads, dim, page, [70, 1, 16, 0, 33, 5, 200], [70, 1, 9, 0, 2, 5, 130], seed=dim + bits)
    x = [odd_rows(dtype, c.total, kv_heads, dim, c.g) for _ in range(2)]
    before = [p.clone() for p in c.pools]
    status = torch.zeros(1, dtype=INT, device="cuda")
    dops.quantize_rows(*x, tuple(c.pools), c.tables, c.lengths, cu_seqlens=c.cu, status=status)
    got = dops.dequantize_rows(c.pools, c.tables, c.lengths, c.total, cu_seqlens=c.cu, status=status)
    assert status.item() == 0
    want = [codes_and_scales(r, bits) for r in x]
    for t, (at, place) in enumerate(c.slots()):
        for kind in (0, 1):
            code, scale = want[kind]
            assert torch.equal(unpacked(c.pools[kind][at][:, place], bits).double(), code[t])
            assert torch.equal(c.pools[2 + kind][at][:, place].double().nan_to_num(1e300), scale[t].nan_to_num(1e300))
            for p in (kind, 2 + kind):
                before[p][at][:, place] = c.pools[p][at][:, place]
    for p, q in zip(c.pools, before):   # and nothing else
        assert torch.equal(p.float().nan_to_num(-1), q.float().nan_to_num(-1))
    for kind in (0, 1):
        code, scale = want[kind]
        exact = (scale[..., 1:] + scale[..., :1] * code.unflatten(-1, (-1, 64))).flatten(-2).clamp(max=torch.finfo(dtype).max)
        assert torch.equal(torch.isnan(got[kind]), torch.isnan(exact))
        # a value is rounded to 32 bits and then to the type
        bound = torch.finfo(dtype).eps / 2 * exact.abs() * (1 + 2 ** -10) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps * 0.51
        assert ((got[kind].double() - exact).abs() <= bound)[~torch.isnan(exact)].all()
        # and is within half a step of what was written; the step is off by half of the type's, L times over, at the group's far end
        step = scale[..., :1].expand(*scale.shape[:-1], 64).flatten(-2)
        away = (exact - x[kind].double()).abs()
        fine = ~torch.isnan(exact) & (step > 0) & (x[kind].double().abs() < 0.4 * torch.finfo(dtype).max)
        slack = step * (0.5 + (2 ** bits - 1) * torch.finfo(dtype).eps / 2) + (2 ** bits) * torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
        assert (away <= slack)[fine].all()


def test_strided_rows(dops):
    """Keys and values as slices of a fused projection, and with the heads in front."""
    c = Cache(BF16, 4, 4, 128, 16, [20, 7, 40], 5, seed=1)
    fused = torch.randn(c.total, 24, 128, generator=c.g, device="cuda").to(BF16)
    k, v = fused[:, 16:20], torch.randn(4, c.total, 128, generator=c.g, device="cuda").to(BF16).transpose(0, 1)
    dops.quantize_rows(k, v, c.pools, c.tables, c.lengths)
    plain = Cache(BF16, 4, 4, 128, 16, [20, 7, 40], 5, seed=1)
    dops.quantize_rows(k.contiguous(), v.contiguous(), plain.pools, c.tables, c.lengths)
    for p, q in zip(c.pools, plain.pools):
        assert torch.equal(p.float().nan_to_num(-1), q.float().nan_to_num(-1))
    into = torch.zeros(c.total, 24, 128, dtype=BF16, device="cuda")
    back = torch.zeros(4, c.total, 128, dtype=BF16, device="cuda")
    got = dops.dequantize_rows(c.pools, c.tables, c.lengths, c.total, k=into[:, 16:20], v=back.transpose(0, 1))
    want = dops.dequantize_rows(c.pools, c.tables, c.lengths, c.total)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(back, want[1].transpose(0, 1))
    assert (into[:, :16] == 0).all() and (into[:, 20:] == 0).all()
    one = torch.randn(1, 4, 128, generator=c.g, device="cuda").to(BF16).expand(c.total, 4, 128)   # a row for all
    dops.quantize_rows(one, one, c.pools, c.tables, c.lengths)
    a, b = dops.dequantize_rows(c.pools, c.tables, c.lengths, c.total)
    assert torch.equal(a, b) and (a == a[:1]).all()


def test_rows_without_a_place(dops):
    """Rows in front of the first token, of no lane, with a page or a length out of range: what they say, and what they leave."""
    c = Cache(F16, 4, 2, 64, 16, [3, 40, 20, 10], 6, seed=2)
    x = torch.randn(c.total, 2, 64, generator=c.g, device="cuda").to(F16)
    status = torch.zeros(1, dtype=INT, device="cuda")
    dops.quantize_rows(x, x, c.pools, c.tables, c.lengths, status=status)
    k, v = dops.dequantize_rows(c.pools, c.tables, c.lengths, c.total, status=status)
    assert status.item() == 0 and (k[:3] == 0).all() and (v[:3] == 0).all() and (k[3:] != 0).any(-1).all()
    cu = ints([2, 5, 5, 9, 10])
    k, v = torch.full_like(x, 7), torch.full_like(x, 7)
    dops.dequantize_rows(c.pools, c.tables, c.lengths, c.total, cu_seqlens=cu, k=k, v=v, status=status)
    assert status.item() == 0 and (k[:2] == 7).all() and (v[10:] == 7).all() and (k[2:10] != 7).any(-1).all()
    for lengths, tables, bit in ((ints([3, 1000, -1, 10]), c.tables, dops.BAD_RANGE), (c.lengths, c.tables.clone().fill_(-1), dops.BAD_PAGE),
                                 (c.lengths, torch.full_like(c.tables, len(c.pools[0])), dops.BAD_PAGE)):
        before = [p.clone() for p in c.pools]
        status.zero_()
        dops.quantize_rows(x, x, c.pools, tables, lengths, status=status)
        assert status.item() == bit
        status.zero_()
        k, v = dops.dequantize_rows(c.pools, tables, lengths, c.total, status=status)
        assert status.item() == bit and (k[6:12] == 0).all() and (v[6:18] == 0).all()
        if bit == dops.BAD_PAGE:
            assert all(torch.equal(p.float().nan_to_num(-1), q.float().nan_to_num(-1)) for p, q in zip(c.pools, before))
    for cu in ([5, 3, 1, 0, -4], [1 << 30, 0, 0, 0, 0], [-5, -4, 100, 200, 300], [0, 0, 0, 0, 0]):   # what no such list should hold leads nowhere else
        dops.quantize_rows(x, x, c.pools, c.tables, c.lengths, cu_seqlens=ints(cu))
        dops.dequantize_rows(c.pools, c.tables, c.lengths, c.total, cu_seqlens=ints(cu))
    torch.cuda.synchronize()


@pytest.mark.parametrize("lanes", [1, 2, 31, 32, 33, 65, 1000, 1025, 3000])
def test_lanes_of_rows_are_found(dops, lanes):
    rows = [(i * 7 + lanes) % 4 for i in range(lanes)]
    c = Cache(F16, 4, 1, 64, 16, [4 + i % 3 for i in range(lanes)], rows, seed=3)
    x = torch.randn(c.total, 1, 64, generator=c.g, device="cuda").to(F16)
    dops.quantize_rows(x, x, c.pools, c.tables, c.lengths, cu_seqlens=c.cu)
    k, v = dops.dequantize_rows(c.pools, c.tables, c.lengths, c.total, cu_seqlens=c.cu)
    code, scale = codes_and_scales(x, 4)
    want = (scale[..., 1:] + scale[..., :1] * code.unflatten(-1, (-1, 64))).flatten(-2)
    assert torch.equal(k, v)
    assert ((k.double() - want).abs() <= 2 ** -11 * want.abs() * 1.001 + 2 ** -25).all()


# ---- attention -----------------------------------------------------------------------------------------------------------------------------


def attend(dops, c, q, **more):
    return dops.quantized_attention(q, c.pools, c.tables, c.lengths, scale=c.dim ** -0.5, cu_seqlens=c.cu, max_rows=max(c.rows, default=0), **more)


def check_attention(c, q, got, window=0, softcap=0.0, pools=None):
    """Against the definition in 64 bits.

    Rounded: the result, to the type (half = eps / 2).  In 32 bits: the products' sums, d of them at the largest intermediate value, which in the form step (q . c) + low sum(q) is
    sum |q| (step c + |low|); values likewise, as step c and low
    apart, where they cancel too; the tensor cores cut a product's sum by its exponent fields, which for codes as f16 subnormals are up to 2^10 above the value: 2^-14 of step c at the most.
    2^-21 for the exponential; a few 1e-7 of the cap.  Where a lane has many rows, keys, values and weights are rounded to f16 once each (2^-11): a
    score moves by 2^-11 sum |q| |k|, a weight by as much (relative), twice, since the sum moves too.  Weights that underflow f16 are below 2^-24 of the largest."""
    dtype, scale = q.dtype, c.dim ** -0.5
    group = q.shape[1] // c.kv_heads
    half = torch.finfo(dtype).eps / 2
    many = max(c.rows, default=0) * group > 32
    at = 0
    for lane, (n, rows) in enumerate(zip(c.lengths_list, c.rows)):
        k, v = (c.tokens(lane, kind, n).transpose(0, 1).repeat_interleave(group, 0) for kind in (0, 1))
        ids = c.tables[lane, :-(-n // c.page)].long()
        low, low_v = (c.pools[kind][ids][..., 1].double().repeat_interleave(64, -1).transpose(1, 2).flatten(0, 1)[:n].abs().transpose(0, 1).repeat_interleave(group, 0) for kind in (2, 3))
        x64 = q[at:at + rows].double().transpose(0, 1)
        p = torch.arange(n - rows, n, device="cuda")[:, None]
        key = torch.arange(n, device="cuda")[None]
        hidden = (key > p) | ((key <= p - window) if window else torch.zeros_like(key, dtype=torch.bool))
        x = x64 @ k.transpose(1, 2) * scale
        if softcap:
            x = softcap * torch.tanh(x / softcap)
        w = torch.softmax(x.masked_fill(hidden, -math.inf), -1).nan_to_num(0.0)
        want, mean, parts = w @ v, w @ v.abs(), w @ (v.abs() + 2 * low_v)
        size = (x64.abs() @ (k.abs() + 2 * low).transpose(1, 2) * scale).masked_fill(hidden, 0.0)
        score = (size.amax(-1, keepdim=True) if n else torch.zeros_like(mean[..., :1])) * ((c.dim + 8) * 2 ** -24 + (2 ** -11 if many else 0)) + 2 ** -21 + 1e-6 * softcap
        bound = half * want.abs() * (1 + half) + (2 * score + (2 * 2 ** -11 if many else 0)) * (mean + want.abs()) + 2 ** -14 * parts + 1e-7 * (dtype == F16)
        off = (got[at:at + rows].double().transpose(0, 1) - want).abs()
        assert torch.isfinite(off).all(), lane
        assert (off <= bound).all(), (lane, float((off - bound).max()), float((off / bound.clamp_min(1e-30)).max()))
        if want.numel() and want.norm() > 0:   # roundings of many values add up like a random walk: a fourth of the sum of the bounds' parts is far
            assert float((off.norm() / want.norm())) < 4 * half + (2 ** -9 if many else 2 ** -16)
        at += rows


def queries(c, heads, spread=2.0, gap=0):
    x = torch.full((c.total, heads * c.dim + gap), math.nan, dtype=c.dtype, device="cuda")
    q = x[:, :heads * c.dim].view(c.total, heads, c.dim) if gap == 0 else x.as_strided((c.total, heads, c.dim), (heads * c.dim + gap, c.dim, 1))
    q.copy_(spread * torch.randn(c.total, heads, c.dim, generator=c.g, device="cuda"))
    return q


LAYOUTS = [(64, 32, 4, 16, F16), (128, 16, 4, 16, F16), (128, 32, 8, 16, BF16), (256, 16, 8, 16, F16), (64, 3, 3, 32, BF16), (128, 5, 1, 64, F16), (256, 8, 8, 128, BF16), (128, 40, 2, 16, F16),
           (64, 71, 1, 16, F16), (256, 24, 2, 16, F16), (128, 128, 1, 16, BF16), (256, 2, 2, 16, F16), (64, 7, 1, 16, BF16)]


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dim, q_heads, kv_heads, page, dtype", LAYOUTS)
def test_head_layouts_types_and_pages(dops, bits, dim, q_heads, kv_heads, page, dtype):
    c = Cache(dtype, bits, kv_heads, dim, page, [1, 15, 16, 17, 40, 530, 0, 3], 1, seed=1).fill()
    q = queries(c, q_heads)
    check_attention(c, q, attend(dops, c, q))
    c = Cache(dtype, bits, kv_heads, dim, page, [2, 370, 33], [2, 4, 3], seed=2, gap=64).fill()
    q = queries(c, q_heads, gap=16)
    check_attention(c, q, attend(dops, c, q))


@pytest.mark.parametrize("lengths", [[1], [0], [31], [32], [33], [700], [2047, 2048, 2049], [9000, 5, 700], [0, 0, 4100], [130] * 40, [20000]])
@pytest.mark.parametrize("dim, q_heads, dtype", [(64, 4, F16), (128, 8, BF16), (256, 2, F16)])
def test_lengths(dops, lengths, dim, q_heads, dtype):
    c = Cache(dtype, 4, 2, dim, 16, lengths, 1, seed=3).fill()
    q = queries(c, q_heads)
    check_attention(c, q, attend(dops, c, q))


@pytest.mark.parametrize("lanes, rows", [(1, 1), (1, 5), (1, 40), (2, 100), (17, 2), (33, 3), (130, 1), (20, 8), (5, 9), (1, 300), (3, 129)])
@pytest.mark.parametrize("dim, bits", [(64, 8), (128, 4), (256, 4)])
def test_numbers_of_rows(dops, lanes, rows, dim, bits):
    c = Cache(F16 if dim < 256 else BF16, bits, 2, dim, 16, [rows + (i * 13) % 90 + 60 * (i % 3) for i in range(lanes)], rows, seed=4).fill()
    q = queries(c, 8)
    check_attention(c, q, attend(dops, c, q))


def test_lanes_of_different_rows_some_without(dops):
    for rows in ([4, 0, 9, 1, 0], [40, 0, 200, 1, 0]):
        c = Cache(BF16, 4, 2, 128, 16, [60, 20, 300, 1, 40], rows, seed=5).fill()
        q = queries(c, 8)
        check_attention(c, q, attend(dops, c, q))


@pytest.mark.parametrize("more", [0, 60])
def test_rows_in_front_of_the_first_token(dops, more):
    """Lanes shorter than their rows: zeros, also where all of a lane's rows are."""
    c = Cache(F16, 4, 2, 64, 16, [2, 0, 5, 1], [4 + more, 2 + more, 5, 3], seed=6).fill()
    q = queries(c, 8)
    got = attend(dops, c, q)
    check_attention(c, q, got)
    at = 0
    for n, rows in zip(c.lengths_list, c.rows):
        assert (got[at:at + max(0, rows - n)] == 0).all()
        at += rows


@pytest.mark.parametrize("window", [1, 2, 16, 17, 100, 1000])
@pytest.mark.parametrize("rows", [1, 3, 50])
def test_windows(dops, window, rows):
    c = Cache(F16, 4, 2, 128, 16, [rows, 120 + rows, 700, 2500], rows, seed=7).fill()
    q = queries(c, 8)
    check_attention(c, q, attend(dops, c, q, window=window), window=window)


@pytest.mark.parametrize("softcap", [0.5, 30.0, 50.0, 1000.0, 3e38])
@pytest.mark.parametrize("rows", [1, 40])
def test_capped_scores(dops, softcap, rows):
    c = Cache(F16, 4, 2, 64, 16, [60, 700], rows, seed=8).fill()
    q = queries(c, 4, spread=4.0)
    check_attention(c, q, attend(dops, c, q, softcap=softcap), softcap=min(softcap, 1e5))


@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("dtype, spread", [(F16, 1e-4), (F16, 200.0), (BF16, 1e-30), (BF16, 1e15)])
def test_small_and_large_values(dops, rows, dtype, spread):
    """Keys and values far from 1: weights and steps are scaled before they are rounded, so that nothing underflows or overflows on the way."""
    c = Cache(dtype, 4, 2, 128, 16, [60, 700], rows, seed=9).fill(spread)
    q = queries(c, 8, spread=min(2.0 / spread, 8000.0))   # the queries themselves are finite
    check_attention_scaled(c, q, attend(dops, c, q), spread)


def check_attention_scaled(c, q, got, spread):
    """f16's own smallest steps count where values are that small."""
    floor = 2 ** -24 if c.dtype == F16 and spread < 1e-2 else 0.0
    if floor:
        keep = got.double()
        want = torch.cat([reference(c, q, lane) for lane in range(len(c.rows))])
        assert ((keep - want).abs() <= floor + 2 ** -6 * want.abs().clamp_min(spread)).all()
    else:
        check_attention(c, q, got)


def reference(c, q, lane, window=0):
    """A lane's result in 64 bits."""
    n, rows, at = c.lengths_list[lane], c.rows[lane], sum(c.rows[:lane])
    group = q.shape[1] // c.kv_heads
    k, v = (c.tokens(lane, kind, n).transpose(0, 1).repeat_interleave(group, 0) for kind in (0, 1))
    p = torch.arange(n - rows, n, device="cuda")[:, None]
    key = torch.arange(n, device="cuda")[None]
    hidden = (key > p) | ((key <= p - window) if window else torch.zeros_like(key, dtype=torch.bool))
    x = (q[at:at + rows].double().transpose(0, 1) @ k.transpose(1, 2) * c.dim ** -0.5).masked_fill(hidden, -math.inf)
    w = torch.softmax(x, -1).nan_to_num(0.0)
    return torch.where(hidden[None, :, :, None], 0.0, w[..., None] * v[:, None]).sum(2).transpose(0, 1)   # what is hidden may be NaN


@pytest.mark.parametrize("rows", [1, 3, 40])
def test_what_a_row_does_not_see_may_be_anything(dops, rows):
    """NaN in front of the window, behind a row's own position and in the value of a key that is seen."""
    c = Cache(F16, 4, 1, 128, 16, [200, 90], rows, seed=10).fill()
    q = queries(c, 4)
    window = 64
    before = 200 - rows - window
    for pos in (0, 7, before - 1):
        for kind in (2, 3):
            c.pools[kind][int(c.tables[0, pos // 16])][:, pos % 16] = math.nan
    if rows > 1:   # the last token's, which only the last row sees
        c.pools[3][int(c.tables[0, 199 // 16])][0, 199 % 16, 1] = math.nan
    got = attend(dops, c, q, window=window)
    want = reference(c, q, 0, window)
    assert torch.equal(torch.isnan(got[:rows]), torch.isnan(want))
    if rows > 1:
        assert torch.isnan(got[rows - 1][:, 64:]).all() and torch.isfinite(got[rows - 1][:, :64]).all() and torch.isfinite(got[:rows - 1]).all()
    fine = ~torch.isnan(want)
    assert ((got[:rows].double() - want).abs()[fine] <= 2 ** -6).all()
    c.pools[2][int(c.tables[1, 2])][0, 3, 0] = math.nan   # a key that every row of lane 1 sees
    got = attend(dops, c, q, window=window)
    assert torch.isnan(got[rows:]).all() and torch.equal(torch.isnan(got[:rows]), torch.isnan(want))


@pytest.mark.parametrize("rows", [1, 40])
def test_pages_in_front_of_the_window_may_be_gone(dops, rows):
    c = Cache(F16, 4, 2, 128, 16, [2000, 300], rows, seed=21).fill()
    q = queries(c, 8)
    want = attend(dops, c, q, window=200)
    for lane, n in enumerate(c.lengths_list):
        c.tables[lane, :(n - rows - 199) // 16] = -1
    status = torch.zeros(1, dtype=INT, device="cuda")
    assert torch.equal(attend(dops, c, q, window=200, status=status), want) and status.item() == 0


def test_queries_that_are_not_finite(dops):
    for rows in (1, 40):
        c = Cache(BF16, 4, 2, 64, 16, [100, 100], rows, seed=11).fill()
        q = queries(c, 4)
        q[0, 0, 5], q[0, 3, 9] = math.nan, math.inf
        got = attend(dops, c, q)
        assert torch.isnan(got[0, 0]).all() and torch.isnan(got[0, 3]).all()
        assert torch.isfinite(got[0, 1:3]).all() and torch.isfinite(got[1:]).all()


def test_rows_of_no_lane_and_given_results(dops):
    for rows in (2, 50):
        c = Cache(F16, 8, 2, 64, 16, [100, 200], rows, seed=12).fill()
        q = queries(c, 8)
        cu = ints([1, 1 + rows - 1, 2 * rows - 2])
        out = torch.full((c.total, 10, 64), 5.0, dtype=F16, device="cuda")
        got = dops.quantized_attention(q, c.pools, c.tables, c.lengths, scale=0.125, cu_seqlens=cu, max_rows=rows, out=out[:, 1:9])
        assert got.data_ptr() == out[:, 1:9].data_ptr()
        assert (out[:, 0] == 5).all() and (out[:, 9] == 5).all() and (out[0] == 5).all() and (out[2 * rows - 2:] == 5).all() and (out[1:2 * rows - 2, 1:9] != 5).any(-1).all()


def test_what_the_device_sees(dops):
    for rows in (1, 50):
        c = Cache(F16, 4, 2, 128, 16, [100, 200, 300], rows, seed=13).fill()
        q = queries(c, 8)
        for lengths, tables, bit in ((ints([100, 100000, 300]), c.tables, dops.BAD_RANGE), (ints([100, -7, 300]), c.tables, dops.BAD_RANGE)):
            status = torch.zeros(1, dtype=INT, device="cuda")
            got = dops.quantized_attention(q, c.pools, tables, lengths, scale=0.1, status=status)
            assert status.item() & bit
            assert torch.equal(got[:rows], dops.quantized_attention(q, c.pools, c.tables, c.lengths, scale=0.1)[:rows])
            assert torch.equal(got[2 * rows:], dops.quantized_attention(q, c.pools, c.tables, c.lengths, scale=0.1)[2 * rows:])
        status = torch.zeros(1, dtype=INT, device="cuda")
        dops.quantized_attention(q, c.pools, torch.full_like(c.tables, -1), c.lengths, scale=0.1, status=status)
        assert status.item() == dops.BAD_PAGE
        for cu in ([5, 3, 1, 0], [1 << 30, 0, 0, 0], [-5, -4, 100, 200], [0, 0, 0, 1 << 30]):
            status.zero_()
            dops.quantized_attention(q, c.pools, c.tables, c.lengths, scale=0.1, cu_seqlens=ints(cu), max_rows=rows, status=status)
            assert status.item() & dops.BAD_RANGE
    torch.cuda.synchronize()


def test_pools_beyond_four_gigabytes(dops):
    pages = 290000   # codes of 4.75 GB
    pools = [torch.empty(pages, 8, 16, 128, dtype=torch.uint8, device="cuda") for _ in range(2)] + [torch.empty(pages, 8, 16, 4, 2, dtype=F16, device="cuda") for _ in range(2)]
    c = Cache(F16, 4, 8, 256, 16, [500, 60], 30, seed=14)
    far = {int(p): pages - 1 - i for i, p in enumerate(c.tables[0].tolist() + c.tables[1, :4].tolist())}
    tables = c.tables.clone()
    for i, n in ((0, 32), (1, 4)):
        tables[i, :n] = ints([far[int(p)] for p in c.tables[i, :n].tolist()])
    c.fill()
    for p, to in far.items():
        for a, b in zip(pools, c.pools):
            a[to] = b[p]
    x = torch.randn(c.total, 8, 256, generator=c.g, device="cuda").to(F16)
    dops.quantize_rows(x, x, pools, tables, c.lengths)
    dops.quantize_rows(x, x, c.pools, c.tables, c.lengths)
    for a, b in zip(dops.dequantize_rows(pools, tables, c.lengths, c.total), dops.dequantize_rows(c.pools, c.tables, c.lengths, c.total)):
        assert torch.equal(a, b)
    for rows in (1, 30):
        q = queries(c, 16)[:2 * rows]
        assert torch.equal(dops.quantized_attention(q, pools, tables, c.lengths, scale=0.06), dops.quantized_attention(q, c.pools, c.tables, c.lengths, scale=0.06))


def spread_lengths(lanes, most, seed):
    return [1 + (i * 7919 + seed * 131) % 97 * most // 96 * (1 if i % 5 else 0) + i % 3 for i in range(lanes)]


@pytest.mark.parametrize("lanes, most", [(2, 9000), (31, 3000), (32, 2500), (33, 2500), (70, 2000), (130, 1500)])
@pytest.mark.parametrize("dim, q_heads, kv_heads, window", [(64, 8, 2, 0), (128, 4, 1, 0), (128, 4, 4, 700), (256, 6, 2, 0)])
def test_keys_of_many_lanes_are_shared_out(dops, lanes, most, dim, q_heads, kv_heads, window):
    """Lanes of very different lengths, more of them than threads of a warp: which CTA has which keys is found on the device."""
    c = Cache(F16, 4, kv_heads, dim, 64, spread_lengths(lanes, most, dim), 1, seed=18).fill()
    q = queries(c, q_heads)
    check_attention(c, q, attend(dops, c, q, window=window), window=window)


@pytest.mark.parametrize("lanes, rows, most", [(3, 20, 5000), (33, 20, 1500), (40, 9, 1200), (260, 6, 100), (300, 33, 60)])
@pytest.mark.parametrize("dim, kv_heads, dtype", [(64, 1, F16), (128, 2, BF16), (256, 1, BF16)])
def test_lanes_of_many_rows(dops, lanes, rows, most, dim, kv_heads, dtype):
    lengths = [rows + n for n in spread_lengths(lanes, most, rows)]
    counts = [max(0, rows - i % 7 * rows // 4) for i in range(lanes)]
    c = Cache(dtype, 4, kv_heads, dim, 16, lengths, counts, seed=19).fill()
    q = queries(c, 4 * kv_heads)
    check_attention(c, q, attend(dops, c, q))


def test_repeated_calls_give_the_same_bits(dops):
    for rows, lengths in ((1, [5000, 300, 20000]), (60, [5000, 300, 2000])):
        c = Cache(F16, 4, 2, 128, 16, lengths, rows, seed=15).fill()
        q = queries(c, 8)
        first = attend(dops, c, q)
        assert all(torch.equal(attend(dops, c, q), first) for _ in range(20))


def test_captured_and_on_two_streams(dops):
    """Captured calls replayed with other contents, and two streams at once, each with a workspace of its own."""
    for rows in (1, 50):
        c = Cache(BF16, 4, 2, 128, 16, [3000, 100, 64], rows, seed=16).fill()
        q = queries(c, 8)
        x = torch.randn(c.total, 2, 128, generator=c.g, device="cuda").to(BF16)
        out, k, v = torch.zeros_like(q), torch.zeros_like(x), torch.zeros_like(x)

        def step():
            dops.quantize_rows(x, x, c.pools, c.tables, c.lengths)
            dops.dequantize_rows(c.pools, c.tables, c.lengths, c.total, k=k, v=v)
            dops.quantized_attention(q, c.pools, c.tables, c.lengths, scale=0.1, out=out)

        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        for seed in range(3):
            g = generator(seed)
            q.copy_(2 * torch.randn(q.shape, generator=g, device="cuda"))
            x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
            c.lengths.copy_(ints([2990 + 3 * seed, 90 + seed, 60]))
            graph.replay()
            got = [t.clone() for t in (out, k, v)]
            step()
            assert all(torch.equal(a, b) for a, b in zip(got, (out, k, v)))
        streams = [torch.cuda.Stream() for _ in range(2)]
        torch.cuda.synchronize()
        results = [[], []]
        for _ in range(10):
            for s, r in zip(streams, results):
                with torch.cuda.stream(s):
                    r.append(dops.quantized_attention(q, c.pools, c.tables, c.lengths, scale=0.1))
        torch.cuda.synchronize()
        assert all(torch.equal(a, out) for r in results for a in r)


@pytest.mark.parametrize("bits, dim, dtype", [(4, 64, F16), (8, 128, BF16), (4, 256, BF16)])
def test_a_thinned_context(dops, bits, dim, dtype):
    """Kept tokens of a lane moved together, codes and scales alike: what is read back is what was there."""
    c = Cache(dtype, bits, 2, dim, 16, [150, 70], 1, seed=20).fill()
    keep = ints([[0, 1, 2, 17, 40, 41, 99, 149], [3, 5, 64, 69, -1, -1, -1, -1]])
    counts, first = ints([8, 4]), ints([0, 2])
    before = [[c.tokens(lane, kind, n) for kind in (0, 1)] for lane, n in enumerate(c.lengths_list)]
    for k, v in ((c.pools[0], c.pools[1]), (c.pools[2].flatten(3), c.pools[3].flatten(3))):
        dops.gather_tokens(k[None], v[None], c.tables, keep, counts, c.tables, first)
    for lane, (n, f) in enumerate(zip((8, 4), (0, 2))):
        for kind in (0, 1):
            now = c.tokens(lane, kind, f + n)
            assert torch.equal(now[f:], before[lane][kind][keep[lane, :n].long()])
    got = dops.dequantize_rows(c.pools, c.tables, ints([8, 6]), 2)
    for kind in (0, 1):
        want = torch.stack([before[lane][kind][p] for lane, p in ((0, 149), (1, 69))])
        assert ((got[kind].double() - want).abs() <= torch.finfo(dtype).eps / 2 * want.abs() * (1 + 2 ** -10) + 2 ** -25).all()


def test_a_text_behind_a_forked_prompt(dops):
    """A prompt into a 4-bit cache, its half-filled last page copied for a second answer, both answers token by token, and their log probabilities: as they are used."""
    g = generator(17)
    heads, kv, dim, page, vocab, prompt = 8, 2, 128, 16, 1000, 57
    pools = dops.quantized_pools(12, kv, page, dim, bits=4, dtype=BF16)
    head = torch.randn(heads * dim, vocab, generator=g, device="cuda") * 0.05
    rows = [torch.randn(prompt + 6, n, dim, generator=g, device="cuda").to(BF16) for n in (kv, kv)]
    tables = ints([[4, 9, 1, 7, 2], [4, 9, 1, 11, 3]])
    dops.quantize_rows(rows[0][:prompt], rows[1][:prompt], pools, tables[:1], ints([prompt]))
    copies = ints([[7, 11, prompt % page]])
    dops.copy_pages(pools.k_codes[None], pools.v_codes[None], copies)
    dops.copy_pages(pools.k_scales.flatten(3)[None], pools.v_scales.flatten(3)[None], copies)
    seen = [torch.cat([r[:prompt], r[:prompt]]).view(2, prompt, kv, dim) for r in rows]
    for step in range(6):
        new = [torch.stack([r[prompt + step], -r[prompt + step]]) for r in rows]
        lengths = ints([prompt + step + 1] * 2)
        dops.quantize_rows(*new, pools, tables, lengths)
        seen = [torch.cat([a, b[:, None]], 1) for a, b in zip(seen, new)]
        q = torch.randn(2, heads, dim, generator=g, device="cuda").to(BF16)
        out = dops.quantized_attention(q, pools, tables, lengths, scale=dim ** -0.5)
        logits = out.flatten(1).float() @ head
        tokens = ints([step, 999 - step])
        scored = dops.token_logprobs(logits, tokens, top=3)
        k, v = ((lambda cs: (cs[1][..., 1:] + cs[1][..., :1] * cs[0].unflatten(-1, (-1, 64))).flatten(-2))(codes_and_scales(x, 4)) for x in seen)
        x = torch.einsum("lhgd,lkhd->lhgk", q.double().view(2, kv, heads // kv, dim), k) * dim ** -0.5
        want = torch.einsum("lhgk,lkhd->lhgd", torch.softmax(x, -1), v).reshape(2, heads, dim)
        # bfloat16 keeps 8 bits, so a rounding is off by 2^-8 of the value at most
        assert ((out.double() - want).abs() <= 2 ** -8 * want.abs() * 1.01 + 1e-4).all()
        log_p = torch.log_softmax(logits.double(), -1)
        assert ((scored.logprobs - log_p.gather(1, tokens.long()[:, None])[:, 0]).abs() < 1e-5).all()
        assert torch.equal(scored.top_tokens.long(), log_p.topk(3, -1)[1])
        back = dops.dequantize_rows(pools, tables, lengths, 2)
        assert all(((b.double() - x[:, -1]).abs() <= 2 ** -8 * x[:, -1].abs() * 1.001).all() for b, x in zip(back, (k, v)))
