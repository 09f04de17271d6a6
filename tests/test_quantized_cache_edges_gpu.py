"""Caches in 4 and 8 bits at the edges of what their calls allow: what is not finite, what some rows do not see, magnitudes far apart, rows behind the last."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_quantized_cache_gpu import BF16, F16, INT, Cache, codes_and_scales, dops, generator, ints  # noqa: E402, F401 (dops is a fixture)


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
