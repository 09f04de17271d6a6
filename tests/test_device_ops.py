"""Operators over device buffers, without a device: what the C entry points and their Python wrappers refuse, how calls are cut, and that nothing valid is refused before
a device is asked for."""
import ctypes as C
import importlib

import pytest

torch = pytest.importorskip("torch")

A = 1 << 20   # an address that is never followed


@pytest.fixture(scope="module")
def capi(mk):
    return importlib.import_module("macllm_infer_b200._capi")


@pytest.fixture(scope="module")
def dops(mk):
    return importlib.import_module("macllm_infer_b200.device_ops")


ATTENTION = dict(type=1, q=A, q_stride=1024, k_pool=A, v_pool=A, pool_pages=100, page_stride=2 * 16 * 128, q_heads=8, kv_heads=2, head_dim=128, block_tokens=16, tables=A,
                 table_stride=100, table_width=100, lengths=A, cu=None, lanes=3, rows=1, total=3, shared_len=32, scale=0.1, softcap=0.0, window=0, out=A, out_stride=1024,
                 workspace=A, workspace_bytes=1 << 30, status=None, stream=None)




@pytest.mark.parametrize("change, message", [
    (dict(type=0), "f16 or bf16"),
    (dict(head_dim=96, page_stride=2 * 16 * 96), "64, 128 or 256"),
    (dict(q_heads=7), "multiple of kv_heads"),
    (dict(q_heads=258, kv_heads=2), "at most 128 query heads"),
    (dict(block_tokens=24), "power of two"),
    (dict(block_tokens=8), "power of two"),
    (dict(shared_len=40), "whole pages"),
    (dict(shared_len=1616), "whole pages"),
    (dict(shared_len=-16), "whole pages"),
    (dict(total=4), "same number of rows"),
    (dict(rows=-1), "negative"),
    (dict(q=A + 8), "multiples of 16 bytes"),
    (dict(q_stride=1028), "multiples of 16 bytes"),
    (dict(out_stride=1000), "rows overlap"),
    (dict(table_stride=99), "rows overlap"),
    (dict(page_stride=2 * 16 * 128 - 128), "pages overlap"),
    (dict(page_stride=2 * 16 * 128 + 64), "pages overlap"),
    (dict(pool_pages=0), "pages overlap"),
    (dict(pool_pages=1 << 27), "2\\^31 - 1 rows"),
    (dict(table_width=1 << 27, table_stride=1 << 27), "2\\^30 positions"),
    (dict(k_pool=None), "null pointer"),
    (dict(lengths=None), "null pointer"),
    (dict(tables=None), "null pointer"),
    (dict(softcap=-1.0), "not negative"),
    (dict(window=-1), "not negative"),
    (dict(scale=0.0), "positive"),
    (dict(scale=float("nan")), "positive"),
    (dict(workspace=None), "workspace"),
    (dict(workspace_bytes=16), "workspace"),
    (dict(workspace=A + 4), "workspace"),
    ({}, "no usable CUDA device"),
])
def test_shared_attention_refuses(capi, change, message):
    if not change and capi.lib().mk_device_count() > 0:
        pytest.skip("a device is there")
    with pytest.raises(capi.MkError, match=message):
        capi.check(capi.lib().mk_k_shared_attention_dev(*{**ATTENTION, **change}.values()))


def test_an_empty_call_is_no_error(capi):
    capi.check(capi.lib().mk_k_shared_attention_dev(*{**ATTENTION, "lanes": 0, "total": 0}.values()))
    capi.check(capi.lib().mk_k_shared_attention_dev(*{**ATTENTION, "rows": 0, "total": 0}.values()))
    capi.check(capi.lib().mk_k_copy_pages_dev(None, None, 2, 10, 2, 16, 256, None, 0, None, None))
    capi.check(capi.lib().mk_k_gather_tokens_dev(None, None, 2, 10, 2, 16, 256, None, 4, 4, None, 4, 4, None, None, 4, 4, None, 0, None, None))
    capi.check(capi.lib().mk_k_verify_drafts_dev(0, None, 100, 0, 3, 100, *([None] * 8), None, 0, None, None))


def test_the_workspace_covers_every_size(capi):
    need = C.c_int64()
    for heads, kv, dim in ((32, 4, 64), (16, 4, 128), (32, 8, 128), (16, 8, 256), (71, 1, 64)):
        for page, width in ((16, 0), (16, 1), (16, 700), (64, 600), (16, 8192)):
            for lanes, rows in ((1, 1), (3, 7), (64, 1), (128, 5), (500, 16)):
                for pages in {0, width // 2, width}:
                    capi.check(capi.lib().mk_k_shared_attention_workspace(heads, kv, dim, page, width, lanes, rows, lanes * rows, pages * page, 0, C.byref(need)))
                    parts, rest = divmod(need.value, lanes * rows * heads * (dim * 4 + 8))
                    assert rest == 0 and 0 <= parts <= 2 + width * page // 64


VERIFY = dict(type=0, logits=A, stride=1000, lanes=3, drafts=4, vocab=1000, drafts_=A, probs=None, u=A, temperature=A, top_k=A, top_p=A, tokens=A, accepted=A, workspace=A,
              workspace_bytes=1 << 24, status=None, stream=None)


@pytest.mark.parametrize("change, message", [
    (dict(type=8), "f32, f16 or bf16"),
    (dict(vocab=0), "negative sizes"),
    (dict(stride=999), "rows overlap"),
    (dict(lanes=-1), "negative sizes"),
    (dict(lanes=1 << 26), "too many rows"),
    (dict(drafts=2 ** 31 - 1), "too many rows"),
    (dict(vocab=416001, stride=416001), "at most 416000"),
    (dict(logits=A + 2), "aligned"),
    (dict(drafts_=None), "null pointer"),
    (dict(u=None), "null pointer"),
    (dict(accepted=None), "null pointer"),
    (dict(workspace_bytes=8), "workspace"),
    (dict(workspace=A + 2), "workspace"),
])
def test_verify_drafts_refuses(capi, change, message):
    with pytest.raises(capi.MkError, match=message):
        capi.check(capi.lib().mk_k_verify_drafts_dev(*{**VERIFY, **change}.values()))


COPY = dict(k=A, v=A, layers=2, pages=10, heads=2, page=16, row=256, copies=A, n=3, status=None, stream=None)
GATHER = dict(k=A, v=A, layers=2, pages=10, heads=2, page=16, row=256, frm=A, ld_from=4, from_width=4, keep=A, ld_keep=8, keep_width=8, counts=A, to=A, ld_to=3, to_width=3, first=A, lanes=2,
              status=None, stream=None)


@pytest.mark.parametrize("change, message", [
    (dict(layers=-1), "negative or empty"), (dict(heads=0), "negative or empty"), (dict(n=-1), "negative or empty"), (dict(row=255), "even number of bytes"),
    (dict(row=1 << 17), "even number of bytes"), (dict(page=1 << 24), "2 GiB"), (dict(k=None), "null pointer"), (dict(copies=None), "null pointer"), (dict(v=A + 1), "even addresses"),
])
def test_copy_pages_refuses(capi, change, message):
    with pytest.raises(capi.MkError, match=message):
        capi.check(capi.lib().mk_k_copy_pages_dev(*{**COPY, **change}.values()))


@pytest.mark.parametrize("change, message", [
    (dict(page=0), "negative or empty"), (dict(lanes=-1), "negative or empty"), (dict(row=0), "even number of bytes"), (dict(ld_from=3), "overlap"), (dict(ld_to=2), "overlap"),
    (dict(ld_keep=7), "overlap"), (dict(from_width=1 << 28, ld_from=1 << 28), "too many positions"), (dict(keep=None), "null pointer"), (dict(first=None), "null pointer"),
    (dict(k=A + 1), "even addresses"),
])
def test_gather_tokens_refuses(capi, change, message):
    with pytest.raises(capi.MkError, match=message):
        capi.check(capi.lib().mk_k_gather_tokens_dev(*{**GATHER, **change}.values()))


def test_wrappers_refuse_by_shape_type_and_place(dops):
    q, pool = torch.zeros(3, 8, 64, dtype=torch.float16), torch.zeros(10, 2, 16, 64, dtype=torch.float16)
    tables, lengths = torch.zeros(3, 4, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)

    def attend(**change):
        a = dict(q=q, k_pool=pool, v_pool=pool, tables=tables, lengths=lengths, shared_len=0)
        a.update(change)
        return dops.shared_attention(a.pop("q"), a.pop("k_pool"), a.pop("v_pool"), a.pop("tables"), a.pop("lengths"), a.pop("shared_len"), scale=1.0, **a)

    for change, message in ((dict(q=q.float()), "float16 or bfloat16"), (dict(k_pool=pool.bfloat16()), "q's type"), (dict(k_pool=pool[:5]), "q's type"),
                            (dict(k_pool=pool.transpose(1, 2), v_pool=pool.transpose(1, 2)), "dense"), (dict(tables=tables.long()), "int32"), (dict(lengths=lengths[:2]), "int32"),
                            (dict(tables=tables[:2]), "same number of rows"), (dict(cu_seqlens=torch.zeros(4, dtype=torch.int32)), "max_rows"), (dict(out=q[:2]), "like q"),
                            (dict(q=torch.zeros(3, 64, 8, dtype=torch.float16).transpose(1, 2)), "dense"), (dict(status=torch.zeros(1)), "status"), ({}, "CUDA device")):
        with pytest.raises(ValueError, match=message):
            attend(**change)
    x, d, f = torch.zeros(2, 4, 50), torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2)
    good = dict(temperature=f, top_k=f.int(), top_p=f)
    for args, more, message in (((x[0], d, x), {}, "logits"), ((x.double(), d, x), {}, "logits"), ((x, d.long(), x[:, :, 0]), {}, "drafts"), ((x, d, x[:, :3, 0].contiguous()), {}, "u is"),
                                ((x.transpose(0, 1), d, x), {}, "evenly apart"), ((x, d, x[:, :, 0].contiguous()), dict(top_k=f), "top_k"),
                                ((x, d, x[:, :, 0].contiguous()), dict(draft_probs=x), "draft_probs"), ((x, d, x[:, :, 0].contiguous()), {}, "CUDA device")):
        with pytest.raises(ValueError, match=message):
            dops.verify_drafts(*args, **{**good, **more})
    pools = torch.zeros(2, 10, 2, 16, 64)
    for k, c, message in ((pools.double(), d, "type"), (pools[:, :5], d, "contiguous"), (pools, d[:, :2], "copies"), (pools, d.long(), "copies"), (pools, d, "CUDA device")):
        with pytest.raises(ValueError, match=message):
            dops.copy_pages(k, pools if k.shape != pools.shape or k.dtype != pools.dtype else k, c)
    for keep, counts, message in ((d[0], f.int(), "lanes"), (d.float(), f.int(), "keep"), (d, f, "counts"), (d, f.int(), "CUDA device")):
        with pytest.raises(ValueError, match=message):
            dops.gather_tokens(pools, pools, d, keep, counts, d, f.int())
