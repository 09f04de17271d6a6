"""Operators over device buffers at the edges of what their calls allow, without a device."""
import importlib
import re

import pytest

from test_dependent_launches import kernels
from test_device_ops import ATTENTION, COPY, GATHER, VERIFY, A, capi  # noqa: F401 (capi is a fixture)

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def dops(mk):
    return importlib.import_module("macllm_infer_b200.device_ops")

# more than 860 threads and 180 KB of shared memory: no CTA that wants tensor memory fits beside one of these
ALONE_ON_AN_SM = {"qstream_tc_kernel"}


def test_kernels_have_their_tensor_memory_before_the_next_may_start():
    """The next kernel may take tensor memory and wait for this one's end: if this one still waited for that memory, neither would end."""
    seen = set()
    for file, name, _, body in kernels():
        takes = [m.start() for m in re.finditer(r"tmem_alloc\(|tcgen05\.alloc", body)]
        if takes and "pdl_trigger()" in body and name not in ALONE_ON_AN_SM:
            seen.add(name)
            assert takes[-1] < body.index("pdl_trigger()"), (file, name)
    assert {"shared_keys_kernel", "attn_umma_kernel", "hgemm_tc_kernel", "latent_umma_kernel"} <= seen


def test_a_loader_outlasts_its_last_copies():
    """Behind its loop the loader of shared_keys_kernel waits for the copies of the last tiles that it asked for, stage u % ST in parity u / ST & 1.  A wait in a parity is over when the
    barrier's present phase has the other one, and a tile is asked for only when the stage's copy before has landed: so no wait is over ahead of its copy, and none lasts beyond it."""
    body = next(b for _, name, _, b in kernels() if name == "shared_keys_kernel")
    loader = body[body.index("bar_wait(&v_empty[st], ph)"):body.index("f16_idesc(kItems, KEYS, false)")]
    assert re.search(r"for \(int u = max\(0, t - ST\); u <= t && u < n_tiles; \+\+u\)", loader) and loader.count("bar_wait(&k_full[u % ST], u / ST & 1)") == 1
    assert not re.search(r"if \(!ok\)\s*\{", loader)   # also where only the others gave up
    for stages in range(2, 7):
        for asked in range(1, 20):
            for under_way in range(0, min(stages, asked) + 1):   # of the last copies
                landed = [sum(1 for u in range(asked - under_way) if u % stages == st) for st in range(stages)]
                for u in range(max(0, asked - stages), asked):
                    over = (landed[u % stages] & 1) != (u // stages & 1)
                    assert over == (u < asked - under_way)


def test_copies_of_any_shape_but_a_table_are_refused(dops):
    pool = torch.zeros(2, 10, 2, 16, 64)
    for copies in (torch.tensor(3, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), torch.zeros(2, 3, 1, dtype=torch.int32)):
        with pytest.raises(ValueError, match="copies"):
            dops.copy_pages(pool, pool, copies)


def test_strides_of_one_head_or_one_page_do_not_matter(dops):
    """Dense tensors whose dimensions of one element have any stride pass every check but that for a device."""
    q, pool = torch.zeros(4, 1, 64, dtype=torch.float16), torch.zeros(10, 1, 16, 64, dtype=torch.float16)
    tables, lengths = torch.zeros(4, 4, dtype=torch.int32), torch.zeros(4, dtype=torch.int32)
    odd_q, odd_pool = q.as_strided((4, 1, 64), (64, 7, 1)), pool.as_strided((10, 1, 16, 64), (1024, 5, 64, 1))
    one_page = [pool[:1], pool.as_strided((1, 1, 16, 64), (3, 5, 64, 1))]
    for args, out in (((odd_q, pool, pool), None), ((q, odd_pool, odd_pool), None), ((q, pool, odd_pool), None), ((q, *one_page), None), ((q, pool, pool), odd_q)):
        with pytest.raises(ValueError, match="CUDA device"):
            dops.shared_attention(*args, tables, lengths, 0, scale=1.0, out=out)
    for args, message in (((q, pool, pool.as_strided((5, 1, 16, 64), (2048, 1024, 64, 1))), "strided alike"), ((q, pool[:5], pool.as_strided((5, 1, 16, 64), (2048, 1024, 64, 1))), "strided alike"),
                          ((q.as_strided((2, 1, 64), (64, 64, 2)), pool, pool), "dense"), ((torch.zeros(4, 2, 64, dtype=torch.float16).as_strided((4, 2, 64), (64, 7, 1)), pool, pool), "dense")):
        with pytest.raises(ValueError, match=message):
            dops.shared_attention(*args, tables[:args[0].shape[0]], lengths[:args[0].shape[0]], 0, scale=1.0)


def test_arrays_that_are_no_words_and_sizes_without_a_place_are_refused(capi):  # noqa: F811
    lib = capi.lib()
    for call, good, names, message in ((lib.mk_k_shared_attention_dev, ATTENTION, ("tables", "lengths", "cu", "status"), "aligned to 4"),
                                       (lib.mk_k_verify_drafts_dev, VERIFY, ("drafts_", "probs", "u", "temperature", "top_k", "top_p", "tokens", "accepted", "status"), "aligned to 4"),
                                       (lib.mk_k_copy_pages_dev, COPY, ("copies", "status"), "aligned to 4"),
                                       (lib.mk_k_gather_tokens_dev, GATHER, ("frm", "keep", "counts", "to", "first", "status"), "aligned to 4")):
        for name in names:
            assert name in good
            with pytest.raises(capi.MkError, match=message):
                capi.check(call(*{**good, name: A + 2}.values()))
    with pytest.raises(capi.MkError, match="null pointer"):
        capi.check(lib.mk_k_shared_attention_workspace(8, 2, 128, 16, 100, 3, 1, 3, 32, 0, None))
    with pytest.raises(capi.MkError, match="null pointer"):
        capi.check(lib.mk_k_verify_drafts_workspace(0, 3, 4, 1000, None))
