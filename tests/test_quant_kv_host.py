"""8-bit KV caches without a GPU: what the records, the plans and the C ABI refuse, and the oracle's own arithmetic."""

import ctypes

import pytest
import torch

import stream_attention
import streamattn_b200 as sa
from oracle import quant_kv as oracle
from streamattn_b200 import native


def contig(layout="BHND", dtype=torch.int8, lens=True, **over):
    shape = (2, 4, 16, 64) if layout == "BHND" else (2, 16, 4, 64)
    fields = dict(key=torch.zeros(shape, dtype=torch.uint8).view(dtype), value=torch.zeros(shape, dtype=torch.uint8).view(dtype),
                  scales=torch.zeros(2, 4, 16, 2, dtype=torch.uint8), layout=layout,
                  sequence_lengths=torch.zeros(2, dtype=torch.int32) if lens else None)
    return sa.QuantKVCache(**{**fields, **over})


def paged(layout="HND", dtype=torch.int8, **over):
    shape = (6, 4, 16, 64) if layout == "HND" else (6, 16, 4, 64)
    fields = dict(key=torch.zeros(shape, dtype=torch.uint8).view(dtype), value=torch.zeros(shape, dtype=torch.uint8).view(dtype),
                  scales=torch.zeros(6, 4, 16, 2, dtype=torch.uint8), layout=layout,
                  page_table=torch.zeros(2, 3, dtype=torch.int32), sequence_lengths=torch.zeros(2, dtype=torch.int32))
    return sa.QuantPagedKVCache(**{**fields, **over})


def test_names_are_exported_under_both_import_names():
    for name in ("QuantKVCache", "QuantPagedKVCache", "quantize_kv", "dequantize_kv", "QuantizeKVPlan", "DequantizeKVPlan",
                 "QuantDecodePlan", "stream_attn_quant_decode"):
        assert getattr(stream_attention, name) is getattr(sa, name)
    from stream_attention.quant_kv import quantize_kv
    from stream_attention.quant_cache import QuantKVCache
    assert quantize_kv is sa.quantize_kv and QuantKVCache is sa.QuantKVCache


def test_empty_caches():
    c = sa.QuantKVCache.empty(2, 4, 13, 64, device="cpu", layout="bnhd")
    c.check()
    assert (c.batch_size, c.kv_heads, c.max_sequence_length, c.head_dim) == (2, 4, 16, 64)      # rounded up to 8 tokens
    assert c.key.dtype == torch.float8_e4m3fn and c.sequence_lengths.tolist() == [0, 0]
    p = sa.QuantPagedKVCache.empty(7, 16, 4, 64, batch=3, max_pages_per_request=2, dtype=torch.int8, layout="NHD", device="cpu")
    p.check()
    p.check_metadata()
    assert (p.num_pages, p.page_size, p.kv_heads, p.head_dim, p.batch_size, p.max_sequence_length) == (7, 16, 4, 64, 3, 32)
    assert p.page_table.tolist() == [[-1, -1]] * 3
    for bad in (dict(dtype=torch.bfloat16), dict(layout="HND")):
        with pytest.raises(ValueError):
            sa.QuantKVCache.empty(2, 4, 16, 64, device="cpu", **bad)
    with pytest.raises(ValueError, match="must be positive"):
        sa.QuantKVCache.empty(2, 0, 16, 64, device="cpu")


@pytest.mark.parametrize("over,match", [
    (dict(key=torch.zeros(2, 4, 16, 64)), "float8_e4m3fn or int8"),
    (dict(value=torch.zeros(2, 4, 16, 32, dtype=torch.int8)), "identical shape"),
    (dict(value=torch.zeros(2, 4, 16, 64, dtype=torch.uint8).view(torch.float8_e4m3fn)), "float8_e4m3fn or int8"),
    (dict(key=torch.zeros(4, 16, 64, dtype=torch.int8)), "rank 4"),
    (dict(scales=torch.zeros(2, 16, 4, 2, dtype=torch.uint8)), "capacity, 2"),
    (dict(scales=torch.zeros(2, 4, 16, 2)), "uint8 or float8_e8m0fnu"),
    (dict(scales=torch.zeros(2, 4, 2, 16, dtype=torch.uint8).transpose(2, 3)), "contiguous"),
    (dict(scales=torch.zeros(2, 4, 32, 2, dtype=torch.uint8)[:, :, ::2]), "contiguous"),
    (dict(scales=torch.zeros(2 * 4 * 32 + 1, dtype=torch.uint8)[1:].view(2, 4, 16, 2)), "straddle"),
    (dict(sequence_lengths=torch.zeros(3, dtype=torch.int32)), "sequence_lengths"),
    (dict(sequence_lengths=torch.zeros(2)), "sequence_lengths"),
    (dict(layout="HND"), "layout"),
])
def test_contiguous_records_are_checked(over, match):
    contig().check()
    with pytest.raises(ValueError, match=match):
        sa.quantize_kv(contig(**over), torch.zeros(2, 1, 4, 64), torch.zeros(2, 1, 4, 64))


@pytest.mark.parametrize("over,match", [
    (dict(key=torch.zeros(6, 4, 16, 64)), "float8_e4m3fn or int8"),
    (dict(scales=torch.zeros(6, 16, 4, 2, dtype=torch.uint8)), "page_size, 2"),
    (dict(page_table=torch.zeros(6, dtype=torch.int32)), "page_table must be"),
    (dict(page_table=torch.zeros(2, 3)), "int32 or int64"),
    (dict(sequence_lengths=torch.zeros(3, dtype=torch.int32)), "match batch"),
    (dict(page_table=torch.zeros(3, 2, dtype=torch.int32).t()), "contiguous"),
    (dict(layout="BHND"), "NHD or HND"),
])
def test_paged_records_are_checked(over, match):
    paged().check()
    with pytest.raises(ValueError, match=match):
        sa.dequantize_kv(paged(**over))


def test_metadata_of_paged_caches_is_checked_on_request():
    c = paged(sequence_lengths=torch.tensor([0, 48], dtype=torch.int32))
    c.check_metadata()
    for lens, match in (([0, 49], "exceed"), ([-1, 3], "negative")):
        with pytest.raises(ValueError, match=match):
            paged(sequence_lengths=torch.tensor(lens, dtype=torch.int32)).check_metadata()
    for bad in (-1, 6):
        with pytest.raises(ValueError, match="physical pages"):
            paged(sequence_lengths=torch.tensor([0, 17]), page_table=torch.tensor([[9, 9, 9], [0, bad, 0]])).check_metadata()


K = torch.zeros(2, 3, 4, 64, dtype=torch.bfloat16)


@pytest.mark.parametrize("kwargs,match", [
    (dict(key_new=K.to(torch.int8)), "bf16, fp16 or fp32"),
    (dict(value_new=K.half()), "share a dtype"),
    (dict(value_new=K[:, :2]), "identical shape"),
    (dict(key_new=K[:1], value_new=K[:1]), "batch, KV heads and head_dim"),
    (dict(new_layout="BHND"), "batch, KV heads and head_dim"),
    (dict(new_layout="NHD"), "BHND or BNHD"),
    (dict(key_new=K[:, :0], value_new=K[:, :0]), "non-empty"),
    (dict(positions=torch.zeros(3, dtype=torch.int32)), "one entry or one per batch row"),
    (dict(positions=torch.zeros(2)), "int32/int64"),
    (dict(positions=torch.zeros(2, dtype=torch.int64), advance_lengths=True), "dtype of the lengths"),
    (dict(counts=torch.zeros(1, dtype=torch.int32)), "counts"),
    (dict(counts=torch.zeros(2)), "counts"),
    (dict(cos=K[:, :, 0]), "given together"),
    (dict(cos=K[:, :, 0].float(), sin=K[:, :, 0].float()), "dtype of the new rows"),
    (dict(cos=K[:, :2, 0], sin=K[:, :2, 0]), "batch_or_1, tokens, dim"),
    (dict(cos=K[:, 0, 0], sin=K[:, 0, 0]), "batch_or_1, tokens, dim"),
    (dict(query_out=K), "needs query"),
    (dict(query=K, query_out=K), "must not alias"),
    (dict(query=K[:, :2]), "batch, tokens, head_dim"),
    (dict(query=K.half()), "batch, tokens, head_dim and dtype"),
    (dict(status=torch.zeros(1)), "int32"),
])
def test_writes_are_checked_before_anything_runs(kwargs, match):
    args = dict(key_new=K, value_new=K)
    args.update(kwargs)
    with pytest.raises(ValueError, match=match):
        sa.quantize_kv(contig(), args.pop("key_new"), args.pop("value_new"), **args)


def test_aliased_lengths_and_missing_lengths_are_refused():
    c = contig()
    with pytest.raises(ValueError, match="counts must not alias"):
        sa.quantize_kv(c, K, K, counts=c.sequence_lengths)
    with pytest.raises(ValueError, match="exclude each other"):
        sa.quantize_kv(c, K, K, lengths_out=torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="positions are required"):
        sa.quantize_kv(contig(lens=False), K, K)
    with pytest.raises(ValueError, match="needs a cache with sequence_lengths"):
        sa.quantize_kv(contig(lens=False), K, K, positions=torch.zeros(2, dtype=torch.int32), advance_lengths=True)
    with pytest.raises(ValueError, match="QuantKVCache"):
        sa.quantize_kv(K, K, K)
    shared = torch.zeros(1, 4, 16, 64, dtype=torch.int8).expand(2, 4, 16, 64)
    with pytest.raises(ValueError, match="must not share memory"):
        sa.quantize_kv(contig(key=shared, value=shared), K, K)


def test_overlapping_operands_are_refused():
    codes = torch.zeros(2, 4, 16, 64, dtype=torch.int8)
    with pytest.raises(ValueError, match="must not share memory"):
        sa.quantize_kv(contig(key=codes, value=codes), K, K)
    spread = torch.zeros(1, 3, 4, 64, dtype=torch.bfloat16).expand(2, 3, 4, 64)
    with pytest.raises(ValueError, match="query_out must not share memory"):
        sa.quantize_kv(contig(), K, K, query=K, query_out=spread)
    with pytest.raises(ValueError, match="value_out must not share memory"):
        sa.DequantizeKVPlan.build(contig(), spread, torch.zeros(1, 3, 4, 64, dtype=torch.bfloat16).expand(2, 3, 4, 64))
    with pytest.raises(ValueError, match="value_out must not share memory"):
        sa.DequantizeKVPlan.build(contig(), K, K)
    buffer = torch.zeros(5, dtype=torch.int32)
    with pytest.raises(ValueError, match="not a part of them"):
        sa.quantize_kv(contig(), K, K, positions=buffer[:2], lengths_out=buffer[1:3])
    with pytest.raises(ValueError, match="counts must not alias"):
        sa.quantize_kv(contig(), K, K, positions=buffer[:2], lengths_out=buffer[3:], counts=buffer[2:4])
    with pytest.raises(RuntimeError, match="CUDA"):                       # beside each other, or the same, is fine
        sa.quantize_kv(contig(), K, K, positions=buffer[:2], lengths_out=buffer[2:4])
    with pytest.raises(RuntimeError, match="CUDA"):
        sa.quantize_kv(contig(), K, K, positions=buffer[:2], lengths_out=buffer[:2])


@pytest.mark.parametrize("kwargs,match", [
    (dict(key_out=K.to(torch.int8)), "bf16, fp16 or fp32"),
    (dict(value_out=K.half()), "share a dtype"),
    (dict(value_out=K[:, :2]), "identical shape"),
    (dict(out_layout="BHND"), "batch, KV heads and head_dim"),
    (dict(starts=torch.zeros(3, dtype=torch.int32)), "starts"),
    (dict(counts=torch.zeros(2)), "counts"),
    (dict(status=torch.zeros(1)), "int32"),
])
def test_reads_are_checked_before_anything_runs(kwargs, match):
    args = dict(key_out=K, value_out=K)
    args.update(kwargs)
    with pytest.raises(ValueError, match=match):
        sa.DequantizeKVPlan.build(contig(), args.pop("key_out"), args.pop("value_out"), **args)
    with pytest.raises(ValueError, match="tokens must be positive"):
        sa.dequantize_kv(contig(), tokens=0)


Q = torch.zeros(2, 1, 8, 64, dtype=torch.bfloat16)


@pytest.mark.parametrize("query,kwargs,match", [
    (Q[:, 0], {}, "batch, 1, heads, dim"),
    (Q.to(torch.int8), {}, "bf16, fp16 or fp32"),
    (Q[:1], {}, "batch and head_dim"),
    (Q[..., :32], {}, "batch and head_dim"),
    (Q[:, :, :6], {}, "multiple of KV heads"),
    (Q, dict(splits=0), "splits"),
    (Q, dict(record_page_walk=True), "paged"),
])
def test_decode_calls_are_checked(query, kwargs, match):
    with pytest.raises(ValueError, match=match):
        sa.QuantDecodePlan.build(query, contig(), **kwargs)


def test_sixteen_bit_calls_refuse_8_bit_caches():
    with pytest.raises(ValueError, match="QuantDecodePlan"):
        sa.PagedExactDecodePlan.build(Q, paged())
    with pytest.raises((ValueError, RuntimeError)):
        sa.paged_append_kv(paged(), K[:, :1], K[:, :1])


def test_there_is_no_cpu_path():
    for call in (lambda: sa.quantize_kv(contig(), K, K), lambda: sa.dequantize_kv(paged()),
                 lambda: sa.stream_attn_quant_decode(Q, contig()), lambda: sa.QuantDecodePlan.build(Q, paged())):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


def _c_call(cache, **over):
    """sa_quantize_kv with host pointers: only for calls that are refused before anything is launched."""
    a = dict(k=1 << 20, v=1 << 20, tokens=3, strides=(768, 256, 64), pos=1 << 20, pos_dtype=0, num=2, counts=None, counts_dtype=0,
             lens=None, cos=None, sin=None, rope=(0, 0), q=None, qo=None, q_heads=0, qs=(0,) * 6, dtype=0)
    a.update(over)
    return native.load().sa_quantize_kv(
        ctypes.byref(cache) if cache is not None else None, a["k"], a["v"], a["tokens"], *a["strides"], a["pos"], a["pos_dtype"], a["num"],
        a["counts"], a["counts_dtype"], a["lens"], a["cos"], a["sin"], *a["rope"], a["q"], a["qo"], a["q_heads"], *a["qs"],
        a["dtype"], None, None)


@pytest.mark.parametrize("over,code", [
    (dict(k=None), 1), (dict(pos=None), 1), (dict(tokens=0), 1), (dict(tokens=-1), 1), (dict(tokens=1 << 40), 2), (dict(dtype=7), 1),
    (dict(pos_dtype=3), 1), (dict(num=3), 1), (dict(counts=1 << 20, counts_dtype=9), 1), (dict(cos=1 << 20), 1),
    (dict(q=1 << 20), 1), (dict(q=1 << 20, qo=1 << 20, q_heads=8), 1), (dict(q=1 << 20, qo=1 << 21, q_heads=6), 1),
    (dict(lens=1 << 20, num=1), 1), (dict(lens=1 << 21, counts=1 << 21), 1),
])
def test_c_abi_refuses_bad_writes(over, code):
    assert _c_call(contig().descriptor(), **over) == code
    assert native.last_error()


@pytest.mark.parametrize("field,value,code", [
    ("key", None, 1), ("scales", None, 1), ("code", 0, 1), ("code", 3, 1), ("batch", 0, 1), ("kv_heads", -1, 1), ("head_dim", 0, 1),
    ("head_dim", 257, 1), ("capacity", 0, 1), ("capacity", 1 << 31, 2), ("stride_n", 0, 1), ("stride_b", -1, 1), ("scale_stride_h", -2, 1),
    ("batch", 1 << 17, 2), ("scales", 3, 1),
])
def test_c_abi_refuses_bad_caches(field, value, code):
    desc = contig().descriptor()
    setattr(desc, field, value)
    assert _c_call(desc, num=1) == code
    assert _c_call(None) == 1


@pytest.mark.parametrize("field,value", [("page_size", 0), ("max_pages", 0), ("num_pages", 0), ("layout", 2), ("table_dtype", 5),
                                         ("max_pages", 1 << 30)])
def test_c_abi_refuses_bad_paged_caches(field, value):
    desc = paged().descriptor()
    setattr(desc, field, value)
    assert _c_call(desc) in (1, 2) and native.last_error()
    lib = native.load()
    assert lib.sa_dequantize_kv(ctypes.byref(desc), 1 << 20, 1 << 20, 3, 768, 256, 64, None, 0, None, 0, 0, None, None) in (1, 2)


def test_c_abi_refuses_bad_decode_calls():
    lib = native.load()

    def call(desc, **over):
        a = dict(q=1 << 20, out=1 << 20, ws=1 << 20, bytes=1 << 30, lens=1 << 20, lens_dtype=0, heads=8, dtype=0, mode=0, ctas=0, kernel=0)
        a.update(over)
        return lib.sa_quant_decode(a["q"], ctypes.byref(desc), a["out"], a["ws"], a["bytes"], a["lens"], a["lens_dtype"], None, a["heads"],
                                   512, 64, a["dtype"], a["mode"], a["ctas"], a["kernel"], None)

    desc = contig().descriptor()
    for over in (dict(q=None), dict(out=None), dict(ws=None), dict(heads=6), dict(heads=0), dict(dtype=5), dict(mode=2), dict(ctas=-1),
                 dict(kernel=9), dict(lens_dtype=4)):
        assert call(desc, **over) == 1, over
    assert call(paged().descriptor(), lens=None) == 1
    desc.code = 0
    assert call(desc) == 1 and "code type" in native.last_error()


def test_oracle_scales_and_codes():
    x = torch.tensor([[448.0, 1.0], [449.0, 1.0], [0.0, 0.0], [2.0 ** -140, 0.0], [float("inf"), 1.0]])
    codes, e = oracle.encode(x, torch.float8_e4m3fn)
    assert e.tolist() == [127, 128, 27, 27, 255]
    assert codes.float()[0].tolist() == [448.0, 1.0] and codes.float()[1].tolist() == [224.0, 0.5] and codes.float()[4].tolist() == [0.0, 0.0]
    codes, e = oracle.encode(torch.tensor([[127.0, 0.5], [127.5, 1.0], [-64.0, 1.5], [2.5, 63.5]]), torch.int8)
    assert e.tolist() == [127, 128, 127, 126]
    assert codes.tolist() == [[127, 0], [64, 0], [-64, 2], [5, 127]]
    # rounding: half a step of the value, or of the smallest step
    g = torch.Generator().manual_seed(0)
    y = torch.randn(500, 64, generator=g, dtype=torch.float64)
    for code, relative in ((torch.float8_e4m3fn, 2 ** -4), (torch.int8, 0.0)):
        c, e = oracle.encode(y, code)
        scale = torch.exp2(e.double() - 127).unsqueeze(-1)
        bound = torch.maximum(y.abs() * relative, scale * (0.5 if code == torch.int8 else 2 ** -10))
        assert bool(((oracle.decode(c, e) - y).abs() <= bound).all())
        again, e2 = oracle.encode(oracle.decode(c, e), code)
        assert torch.equal(oracle.decode(again, e2), oracle.decode(c, e))


def test_partly_overlapping_operands_are_refused():
    """Contiguous operands that share a part of their memory; slices of one buffer that interleave are fine."""
    buffer = torch.zeros(5, 3, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="must not alias query"):
        sa.quantize_kv(contig(), K, K, query=buffer[:2], query_out=buffer[1:3])
    with pytest.raises(ValueError, match="must not alias the new rows"):
        sa.quantize_kv(contig(), buffer[:2], K, query=K, query_out=buffer[1:3])
    with pytest.raises(ValueError, match="must not alias the new rows"):
        sa.quantize_kv(contig(), K, K, query=buffer[:2], query_out=K)
    with pytest.raises(ValueError, match="value_out must not share memory"):
        sa.DequantizeKVPlan.build(contig(), buffer[:2], buffer[1:3])
    codes = torch.zeros(3, 4, 16, 64, dtype=torch.int8)
    with pytest.raises(ValueError, match="must not share memory"):
        sa.quantize_kv(contig(key=codes[:2], value=codes[1:]), K, K)
    fused = torch.zeros(2, 3, 16, 64, dtype=torch.bfloat16)                # heads of K, V, the query and its result side by side
    k, v, q, out = fused.split(4, dim=2)
    with pytest.raises(RuntimeError, match="CUDA"):
        sa.quantize_kv(contig(), k, v, query=q, query_out=out)
    with pytest.raises(RuntimeError, match="CUDA"):
        sa.DequantizeKVPlan.build(contig(), k, v)
    with pytest.raises(RuntimeError, match="CUDA"):
        sa.quantize_kv(contig(), buffer[:2], buffer[2:4], query=K, query_out=torch.empty_like(K))
