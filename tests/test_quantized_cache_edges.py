"""The kernels of caches in 4 and 8 bits as they are written: what no device can be made to show."""
import importlib
import re

import pytest

from test_dependent_launches import CSRC, kernels


def body_of(name):
    return next(b for _, n, _, b in kernels() if n == name)


def test_products_end_before_their_memory_is_given_back():
    """Behind its loop, however that ended, a warp that issues products waits for all of them: for a barrier of its own, to which only the last commit arrives."""
    body = body_of("many_items_kernel")
    products = body[body.index("f16_idesc(kItemTile, kKeyTile, false)"):body.index("f16_idesc(kItemTile, D, true)")] + body[body.index("f16_idesc(kItemTile, D, true)"):]
    products = products[:products.index("} else if (warp < 4 * subs)")]
    assert products.count("commit(&drained[sub])") == 1 and products.count("bar_wait(&drained[sub], 0)") == 1
    last = products[products.rindex("commit(&v_empty[st]);"):]
    assert last.index("commit(&drained[sub])") < last.index("bar_wait(&drained[sub], 0)")
    assert not re.search(r"if \(!?ok[^)]*\)\s*\{", last) and not re.search(r"if \(ok\) *(if|commit)", last)   # also where only the others gave up
    assert re.search(r"bar_init\(&drained\[i\], 1\)", body)
    # a barrier of each tile of items, behind the others
    assert "bars[2 * KST + 2 * VST + 8 * SUBS]" in body and "*drained = q_full + SUBS" in body
    # tensor memory is given back behind the barrier of all threads that follows
    end = body[body.rindex("__syncthreads()"):]
    assert "tmem_dealloc(tmem, 512)" in end and body.count("tmem_dealloc(") == 1


def test_shares_are_counted_alike_in_every_kernel():
    """How many shares a lane has is found by the attention and by the kernel that joins them: from products, quotients and differences that are rounded where they stand, so that none is made
    one with its neighbour in one kernel alone."""
    text = re.sub(r"//[^\n]*", "", (CSRC / "quantized_attention.cu").read_text())
    text = text[text.index("Piece piece_of("):text.index("struct Shares")]
    for wanted in ("__frcp_rn(", "__fdiv_rn(warp_sum(total), c.want)", "__fmul_rn(", "__fsub_rn(n, 1e-3f)"):
        assert text.count(wanted) == 1, wanted
    for wrong in ("* per_share", "/ c.want", "n - 1e", "1.0f /"):
        assert wrong not in text, wrong
    assert re.search(r"total \+= \(float\)keys_of", text)   # whole numbers, added


def test_whole_warps_exchange_what_they_have():
    """An exchange among all threads of a warp stands behind nothing that some of them may find and others not: a thread that leaves it out leaves the others waiting."""
    uniform = ("!keys &&", "t > 0 &&", "ok && n_tiles > 0", "n_tiles > 0 &&")   # known to whole warps alike
    for name in ("quantized_attention.cu", "quantized_kv.cu", "token_logprobs.cu"):
        text = re.sub(r"//[^\n]*", "", (CSRC / name).read_text())
        for statement in re.split(r"[;{}]", text):
            first = re.search(r"&&|\|\|", statement)
            exchange = r"_sync\(|\bwarp_max\(|\bwarp_sum\(|\bof_item\("
            if first and re.search(exchange, statement[first.end():]) and not re.search(exchange, statement[:first.start()]):
                assert any(u in statement for u in uniform), (name, statement.strip())


@pytest.mark.parametrize("beyond", [1 << 31, (1 << 32) + 5, (1 << 63) + 7])
def test_numbers_that_lose_their_upper_bits_on_the_way_are_refused(mk, beyond):
    """A window of 2^32 + 5 was one of 5."""
    torch = pytest.importorskip("torch")
    dops = importlib.import_module("macllm_infer_b200.device_ops")
    pools = dops.quantized_pools(10, 2, 16, 64, device="cpu")
    pool = torch.zeros(10, 2, 16, 64, dtype=torch.float16)
    q, row = torch.zeros(3, 8, 64, dtype=torch.float16), torch.zeros(1, 2, 64, dtype=torch.float16)
    tables, lengths, cu = torch.zeros(3, 4, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), torch.zeros(4, dtype=torch.int32)
    calls = [lambda: dops.quantized_attention(q, pools, tables, lengths, scale=1.0, window=beyond),
             lambda: dops.quantized_attention(q, pools, tables, lengths, scale=1.0, cu_seqlens=cu, max_rows=beyond),
             lambda: dops.shared_attention(q, pool, pool, tables, lengths, 0, scale=1.0, window=beyond),
             lambda: dops.shared_attention(q, pool, pool, tables, lengths, 0, scale=1.0, cu_seqlens=cu, max_rows=beyond),
             lambda: dops.shared_attention(q, pool, pool, tables, lengths, beyond, scale=1.0),
             lambda: dops.dequantize_rows(pools, tables, lengths, beyond, cu_seqlens=cu)]
    if beyond < 1 << 40:
        many = row.expand(beyond, 2, 64)
        calls.append(lambda: dops.quantize_rows(many, many, pools, tables, lengths, cu_seqlens=cu))
    for call in calls:
        with pytest.raises(ValueError, match="at most 2\\^31 - 1"):
            call()
