"""Caches in 4 or 8 bits and log probabilities of given tokens, without a device: what the C entry points and their Python wrappers refuse, and that nothing valid is refused before a
device is asked for."""
import ctypes as C
import importlib

import pytest

torch = pytest.importorskip("torch")

A = 1 << 20   # an address that is never followed
F16 = torch.float16


@pytest.fixture(scope="module")
def capi(mk):
    return importlib.import_module("macllm_infer_b200._capi")


@pytest.fixture(scope="module")
def dops(mk):
    return importlib.import_module("macllm_infer_b200.device_ops")


POOLS = dict(type=1, bits=4, k_codes=A, v_codes=A, k_scales=A, v_scales=A, pages=100, codes_stride=2 * 16 * 64, scales_stride=2 * 16 * 4, kv_heads=2, head_dim=128, block_tokens=16)
LANES = dict(tables=A, table_stride=100, table_width=100, lengths=A, cu=None, lanes=3)
ROWS = dict(k=A, k_row=256, k_head=128, v=A, v_row=256, v_head=128)
LAST = dict(status=None, stream=None)
WRITE = {**ROWS, **POOLS, **LANES, "total": 3, **LAST}
READ = {**POOLS, **LANES, "total": 3, **ROWS, **LAST}
ATTEND = {**dict(q=A, q_stride=1024, q_heads=8), **POOLS, **LANES, **dict(rows=1, total=3, scale=0.1, softcap=0.0, window=0, out=A, out_stride=1024, workspace=A, workspace_bytes=1 << 30), **LAST}

OF_POOLS = [
    (dict(type=0), "f16 or bf16"), (dict(bits=5), "4 or 8 bits"), (dict(head_dim=96), "64, 128 or 256"), (dict(kv_heads=0), "KV heads"), (dict(kv_heads=65536), "KV heads"),
    (dict(block_tokens=24), "power of two"), (dict(block_tokens=8), "power of two"), (dict(block_tokens=65536, kv_heads=4096), "too many rows"), (dict(pages=0), "1 to 2\\^31 - 1 pages"),
    (dict(codes_stride=2 * 16 * 64 - 16), "pages overlap"), (dict(scales_stride=2 * 16 * 4 - 8), "pages overlap"), (dict(codes_stride=2 * 16 * 64 + 8), "multiples of 16"),
    (dict(scales_stride=2 * 16 * 4 + 4), "multiples of 16"), (dict(codes_stride=1 << 60), "too far apart"), (dict(scales_stride=1 << 60), "too far apart"), (dict(bits=8), "pages overlap"),
    (dict(k_codes=None), "null pointer"), (dict(v_scales=None), "null pointer"), (dict(v_codes=A + 8), "multiples of 16"), (dict(k_scales=A + 4), "multiples of 16"),
    (dict(lengths=None), "null pointer"), (dict(tables=None), "null pointer"), (dict(table_stride=99), "table rows overlap"), (dict(table_width=1 << 27, table_stride=1 << 27), "2\\^30 positions"),
    (dict(lengths=A + 2), "aligned to 4"), (dict(status=A + 1), "aligned to 4"), (dict(lanes=-1), "negative"), (dict(total=-3), "negative"), (dict(total=4), "same number of rows"),
]
DEVICE = ({}, "no usable CUDA device")


def refuses(capi, name, arguments, change, message):
    if not change and capi.lib().mk_device_count() > 0:
        pytest.skip("a device is there")
    with pytest.raises(capi.MkError, match=message):
        capi.check(getattr(capi.lib(), name)(*{**arguments, **change}.values()))


@pytest.mark.parametrize("change, message", OF_POOLS + [
    (dict(k=None), "null pointer"), (dict(v=A + 8), "multiples of 16"), (dict(k_row=260), "multiples of 16"), (dict(v_head=132), "multiples of 16"), (dict(k_row=-8), "strides out of range"),
    (dict(v_head=1 << 60), "strides out of range"), (dict(k_row=0), "no usable CUDA device"), DEVICE])
def test_quantize_rows_refuses(capi, change, message):
    refuses(capi, "mk_k_quantize_rows_dev", WRITE, change, message)


@pytest.mark.parametrize("change, message", OF_POOLS + [
    (dict(k=None), "null pointer"), (dict(k=A + 8), "multiples of 16"), (dict(k_row=0), "rows overlap"), (dict(v_row=128), "rows overlap"), (dict(v_head=64), "rows overlap"),
    (dict(k_row=128, k_head=384), "no usable CUDA device"), DEVICE])
def test_dequantize_rows_refuses(capi, change, message):
    refuses(capi, "mk_k_dequantize_rows_dev", READ, change, message)


@pytest.mark.parametrize("change, message", OF_POOLS + [
    (dict(q=None), "null pointer"), (dict(out=None), "null pointer"), (dict(q_heads=7), "multiple of kv_heads"), (dict(q_heads=258), "at most 128 query heads"), (dict(rows=-1), "negative"),
    (dict(window=-1), "not negative"), (dict(softcap=-1.0), "not negative"), (dict(softcap=float("nan")), "not negative"), (dict(scale=0.0), "positive"), (dict(scale=float("inf")), "positive"),
    (dict(q=A + 8), "multiples of 16"), (dict(out_stride=1028), "multiples of 16"), (dict(q_stride=1000), "rows overlap"), (dict(rows=1 << 21, total=3 << 21), "too many rows"), DEVICE])
def test_quantized_attention_refuses(capi, change, message):
    refuses(capi, "mk_k_quantized_attention_dev", ATTEND, change, message)


def test_a_workspace_that_is_too_small(capi):
    long = dict(table_width=20000, table_stride=20000)
    need = C.c_int64()
    capi.check(capi.lib().mk_k_quantized_attention_workspace(4, 8, 2, 128, 16, 20000, 3, 1, 3, 0, C.byref(need)))
    if need.value == 0:
        pytest.skip("no workspace is needed")
    for change in (dict(workspace=None), dict(workspace_bytes=need.value - 1), dict(workspace=A + 8)):
        refuses(capi, "mk_k_quantized_attention_dev", ATTEND, {**long, **change}, "workspace")


def test_the_workspace_is_bounded(capi):
    """At most a part for each 128 keys that the tables hold."""
    need = C.c_int64()
    for heads, kv, dim in ((32, 4, 64), (16, 4, 128), (32, 8, 128), (16, 8, 256), (71, 1, 64)):
        for page, width in ((16, 0), (16, 1), (16, 700), (64, 600), (16, 8192), (16, 1 << 20)):
            for lanes, rows in ((1, 1), (3, 7), (64, 1), (128, 5), (500, 16), (2, 3000)):
                for bits in (4, 8):
                    for window in (0, 500):
                        capi.check(capi.lib().mk_k_quantized_attention_workspace(bits, heads, kv, dim, page, width, lanes, rows, lanes * rows, window, C.byref(need)))
                        assert 0 <= need.value <= (1 + width * page // 128) * lanes * rows * heads * (dim * 4 + 8)
    with pytest.raises(capi.MkError, match="null pointer"):
        capi.check(capi.lib().mk_k_quantized_attention_workspace(4, 8, 2, 128, 16, 10, 1, 1, 1, 0, None))


LOGPROBS = dict(type=0, logits=A, stride=1000, rows=3, vocab=1000, tokens=A, top=5, logprobs=A, entropy=A, ranks=A, top_tokens=A, top_logprobs=A, status=None, stream=None)


@pytest.mark.parametrize("change, message", [
    (dict(type=8), "f32, f16 or bf16"), (dict(rows=-1), "1 to 2\\^24"), (dict(vocab=0), "1 to 2\\^24"), (dict(vocab=(1 << 24) + 1), "1 to 2\\^24"), (dict(top=-1), "at most 64"), (dict(top=65), "at most 64"),
    (dict(vocab=4), "at most the vocabulary"), (dict(stride=999), "rows overlap"), (dict(stride=1 << 61), "too far apart"), (dict(logits=None), "null pointer"), (dict(tokens=None), "null pointer"),
    (dict(ranks=None), "null pointer"), (dict(top_tokens=None), "null pointer"), (dict(logits=A + 2), "aligned to their type"), (dict(type=1, logits=A + 1), "aligned to their type"),
    (dict(tokens=A + 2), "aligned to 4"), (dict(top_logprobs=A + 1), "aligned to 4"), (dict(top=0, top_tokens=None, top_logprobs=None), "no usable CUDA device"), DEVICE])
def test_token_logprobs_refuses(capi, change, message):
    refuses(capi, "mk_k_token_logprobs_dev", LOGPROBS, change, message)


def test_empty_calls_are_no_errors(capi):
    lib = capi.lib()
    capi.check(lib.mk_k_quantize_rows_dev(*{**WRITE, "total": 0}.values()))
    capi.check(lib.mk_k_dequantize_rows_dev(*{**READ, "lanes": 0, "total": 0}.values()))
    capi.check(lib.mk_k_quantized_attention_dev(*{**ATTEND, "lanes": 0, "total": 0}.values()))
    capi.check(lib.mk_k_quantized_attention_dev(*{**ATTEND, "rows": 0, "total": 0}.values()))
    capi.check(lib.mk_k_token_logprobs_dev(*{**LOGPROBS, "rows": 0}.values()))


def test_wrappers_refuse_by_shape_type_and_place(dops):
    pools = dops.quantized_pools(10, 2, 16, 64, device="cpu")
    assert [tuple(p.shape) for p in pools] == [(10, 2, 16, 32)] * 2 + [(10, 2, 16, 1, 2)] * 2
    assert dops.quantized_pools(10, 2, 16, 128, bits=8, dtype=torch.bfloat16, device="cpu").k_codes.shape == (10, 2, 16, 128)
    for wrong in (dict(bits=3), dict(dtype=torch.float32)):
        with pytest.raises(ValueError, match="4 or 8 bits"):
            dops.quantized_pools(10, 2, 16, 64, device="cpu", **wrong)
    rows, q = torch.zeros(3, 2, 64, dtype=F16), torch.zeros(3, 8, 64, dtype=F16)
    tables, lengths = torch.zeros(3, 4, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    bad_pools = [
        (pools._replace(k_codes=pools.k_codes.to(torch.int8)), "uint8"), (pools._replace(k_codes=pools.k_codes[..., :24]), "half a byte"), (pools._replace(v_codes=pools.v_codes[:9]), "alike"),
        (pools._replace(k_scales=pools.k_scales.float()), "float16 or bfloat16"), (pools._replace(v_scales=pools.v_scales.bfloat16()), "alike"), (pools._replace(k_scales=pools.k_scales[..., 0]), "scales"),
        (pools._replace(k_codes=pools.k_codes.transpose(1, 2).contiguous().transpose(1, 2)), "dense"), (pools._replace(v_codes=torch.zeros(20, 2, 16, 32, dtype=torch.uint8)[::2]), "equally far apart"),
    ]
    calls = [lambda **a: dops.quantize_rows(**{**dict(k=rows, v=rows, pools=pools, tables=tables, lengths=lengths), **a}),
             lambda **a: dops.dequantize_rows(**{**dict(pools=pools, tables=tables, lengths=lengths, total=3), **a}),
             lambda **a: dops.quantized_attention(**{**dict(q=q, pools=pools, tables=tables, lengths=lengths, scale=1.0), **a})]
    for call in calls:
        for changed, message in bad_pools:
            with pytest.raises(ValueError, match=message):
                call(pools=changed)
        for change, message in ((dict(tables=tables.long()), "int32"), (dict(lengths=lengths[:2]), "int32"), (dict(cu_seqlens=torch.zeros(3, dtype=torch.int32)), "cu_seqlens"),
                                (dict(status=torch.zeros(1)), "status|max_rows"), ({}, "CUDA device")):
            with pytest.raises(ValueError, match=message):
                call(**change)
    for change, message in ((dict(k=rows.bfloat16()), "k is"), (dict(v=rows[:2]), "v is"), (dict(k=rows[..., ::2]), "k is"), (dict(k=torch.zeros(3, 64, 2, dtype=F16).transpose(1, 2)), "dense heads")):
        with pytest.raises(ValueError, match=message):
            calls[0](**change)
    with pytest.raises(ValueError, match="v is"):
        calls[1](v=rows[:1])
    with pytest.raises(ValueError, match="total"):
        calls[1](total=-3)
    for change, message in ((dict(q=q.float()), "float16"), (dict(q=q[..., :32]), "64"), (dict(tables=tables[:2], lengths=lengths[:2]), "same number of rows"),
                            (dict(cu_seqlens=torch.zeros(4, dtype=torch.int32)), "max_rows"), (dict(out=q[:2]), "like q"), (dict(q=torch.zeros(3, 64, 8, dtype=F16).transpose(1, 2)[..., :64]), "64|dense")):
        with pytest.raises(ValueError, match=message):
            calls[2](**change)
    logits, tokens = torch.zeros(3, 100), torch.zeros(3, dtype=torch.int32)
    for a, message in (((logits.double(), tokens), "float32"), ((logits[0], tokens), "rows, vocabulary"), ((logits.t(), tokens), "dense"), ((logits, tokens.long()), "tokens"), ((logits, tokens[:2]), "tokens"),
                       ((logits, tokens), "CUDA device")):
        with pytest.raises(ValueError, match=message):
            dops.token_logprobs(*a)
    for top in (-1, 65, 101):
        with pytest.raises(ValueError, match="top is"):
            dops.token_logprobs(logits, tokens, top=top)
