"""8-bit KV caches on the GPU: writing rows, reading them back, and their errors, through the public calls.

Codes and scale bytes are whole numbers and must equal the 64-bit oracle's (``oracle/quant_kv.py``): a
division by a power of two is exact, so there is one right answer.  Read-back is exact too, up to the
one rounding into the target type.  Whole buffers are compared, so a byte written outside the rows
that were asked for is seen.
"""

import pytest
import torch

import streamattn_b200 as sa
from oracle import quant_kv as oracle
from streamattn_b200 import native

pytestmark = pytest.mark.gpu
CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a CUDA device; refusing to skip")
    return torch.device("cuda:0")


def make_cache(dev, kind, layout, code, batch, heads, dim, capacity, page=16, seed=0, table_dtype=torch.int32):
    """A cache filled with random bytes (what an unwritten row may hold), and the oracle's copy of it."""
    g = torch.Generator().manual_seed(seed)
    table = None
    if kind == "paged":
        per_row = -(-capacity // page)
        capacity = per_row * page
        pages = batch * per_row + 3
        shape = (pages, page, heads, dim) if layout == "NHD" else (pages, heads, page, dim)
        scale_shape = (pages, heads, page, 2)
        table = torch.randperm(pages, generator=g)[:batch * per_row].view(batch, per_row).to(table_dtype)
    else:
        shape = (batch, capacity, heads, dim) if layout == "BNHD" else (batch, heads, capacity, dim)
        scale_shape = (batch, heads, capacity, 2)
    key = torch.randint(0, 256, shape, generator=g, dtype=torch.uint8).view(CODES[code])
    value = torch.randint(0, 256, shape, generator=g, dtype=torch.uint8).view(CODES[code])
    scales = torch.randint(0, 256, scale_shape, generator=g, dtype=torch.uint8)
    mirror = dict(key=key, value=value, scales=scales, table=table, page=page, capacity=capacity,
                  heads_first=layout in ("HND", "BHND"))
    lens = torch.zeros(batch, dtype=torch.int32, device=dev)
    if kind == "paged":
        cache = sa.QuantPagedKVCache(key=key.to(dev), value=value.to(dev), scales=scales.to(dev), page_table=table.to(dev),
                                     sequence_lengths=lens, layout=layout)
    else:
        cache = sa.QuantKVCache(key=key.to(dev), value=value.to(dev), scales=scales.to(dev), sequence_lengths=lens,
                                layout=layout)
    return cache, mirror


def new_rows(shape, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * torch.exp(2.0 * torch.randn(shape[:-1] + (1,), generator=g))
    return x.to(dtype)


def angles(batch, tokens, dim, dtype, seed=5):
    a = torch.randn(batch, tokens, dim // 2, generator=torch.Generator().manual_seed(seed)) * 3
    a = torch.cat((a, a), dim=-1)
    return a.cos().to(dtype), a.sin().to(dtype)


def same_bytes(cache, mirror):
    for name in ("key", "value", "scales"):
        got, want = getattr(cache, name).cpu().view(torch.uint8), mirror[name].view(torch.uint8)
        if not torch.equal(got, want):
            at = (got != want).nonzero()
            raise AssertionError(f"{name}: {len(at)} bytes differ, first at {at[0].tolist()}: {got[tuple(at[0])]} != {want[tuple(at[0])]}")


WRITES = [
    # kind, layout, code, dtype, batch, heads, dim, tokens, page, rope
    ("paged", "HND", "e4m3", "bf16", 3, 2, 64, 1, 16, True),        # a decode step
    ("paged", "NHD", "int8", "fp16", 2, 8, 128, 1, 64, False),
    ("contig", "BHND", "e4m3", "bf16", 2, 2, 64, 70, 0, True),      # several CTAs a row
    ("contig", "BNHD", "int8", "bf16", 1, 3, 128, 33, 0, True),
    ("paged", "NHD", "e4m3", "fp16", 3, 1, 128, 65, 8, False),
    ("paged", "HND", "int8", "fp32", 2, 2, 64, 9, 1, True),         # pages of one token
    ("contig", "BHND", "e4m3", "fp32", 2, 4, 256, 5, 0, True),
    ("contig", "BNHD", "e4m3", "bf16", 2, 2, 80, 7, 0, True),       # 10 of 16 lanes hold the row
    ("paged", "HND", "int8", "bf16", 1, 2, 96, 40, 24, False),      # a page size that is no power of two
    ("contig", "BHND", "int8", "fp16", 2, 2, 40, 6, 0, True),       # rotation pairs that split a lane's piece
    ("contig", "BHND", "e4m3", "bf16", 2, 2, 7, 6, 0, False),       # one element at a time
    ("paged", "NHD", "int8", "fp32", 2, 3, 1, 17, 16, False),
    ("contig", "BNHD", "e4m3", "fp16", 1, 1, 8, 300, 0, False),
]


@pytest.mark.parametrize("ragged", [False, True], ids=["even", "ragged"])
@pytest.mark.parametrize("case", WRITES, ids=lambda c: "-".join(map(str, c)))
def test_write_gives_the_oracles_bytes_and_nothing_else(dev, case, ragged):
    kind, layout, code, dtype, B, H, D, T, page, rope = case
    dtype = TYPES[dtype]
    cache, mirror = make_cache(dev, kind, layout, code, B, H, D, T + 24, page=page or 16, seed=D + T)
    k, v = new_rows((B, T, H, D), dtype, 1), new_rows((B, T, H, D), dtype, 2)
    starts = [mirror["capacity"] - T, 0, 5][:B]
    counts = [T, 0, max(1, T // 2)][:B] if ragged else [T] * B
    kwargs, q = {}, None
    if rope:
        cos, sin = angles(B if T % 2 else 1, T, D, dtype)
        q = new_rows((B, T, 2 * H, D), dtype, 3)
        out = torch.full_like(q, 7.0).to(dev)
        kwargs = dict(cos=cos.to(dev), sin=sin.to(dev), query=q.to(dev), query_out=out)
    positions = torch.tensor(starts, dtype=torch.int32, device=dev)
    lengths = torch.full((B,), -9, dtype=torch.int32, device=dev)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    got = sa.quantize_kv(cache, k.to(dev), v.to(dev), positions=positions, lengths_out=lengths, status=status,
                         counts=torch.tensor(counts, device=dev) if ragged else None, **kwargs)
    torch.cuda.synchronize()
    oracle.write(mirror, oracle.rotate(k, cos, sin) if rope else k, v, starts, counts)
    same_bytes(cache, mirror)
    assert int(status) == 0 and lengths.tolist() == [s + n for s, n in zip(starts, counts)]
    assert positions.tolist() == starts and cache.sequence_lengths.tolist() == [0] * B
    if rope:
        assert got is out and torch.equal(got.cpu(), oracle.rotate(q, cos, sin).to(dtype))   # padding as well


@pytest.mark.parametrize("code", list(CODES))
@pytest.mark.parametrize("dim", [64, 20], ids=["vector", "scalar"])
def test_write_rows_at_the_edges_of_the_format(dev, code, dim):
    top, big = oracle.TOP[CODES[code]], torch.finfo(torch.float32).max
    rows = [torch.zeros(dim), torch.full((dim,), top), torch.full((dim,), top * 2.0 ** -40), torch.full((dim,), big),
            torch.full((dim,), 2.0 ** -149), torch.full((dim,), top * 2.0 ** -100), torch.full((dim,), top * 2.0 ** -103)]
    above = torch.full((dim,), 1.0)
    above[3] = torch.nextafter(torch.tensor(top), torch.tensor(big))      # one step above: the next scale
    ties = torch.arange(dim).float() + 0.5                                # halves, to even
    ties[-1] = top
    ties8 = (torch.arange(dim) % 8 + 8.5) * 2.0 ** (torch.arange(dim) // 8 - 12).float()
    ties8[-1] = -top
    inf, nan, minus = torch.ones(dim), torch.ones(dim), torch.ones(dim)
    inf[dim // 2], nan[dim - 1], minus[0] = float("inf"), float("nan"), -float("inf")
    rows += [above, ties, ties8, -ties8, inf, nan, minus]
    k = torch.stack(rows)[None, :, None]
    v = k.flip(1).contiguous()
    T = len(rows)
    cache, mirror = make_cache(dev, "contig", "BHND", code, 1, 1, dim, T + 3)
    sa.quantize_kv(cache, k.to(dev), v.to(dev))
    oracle.write(mirror, k, v, [0], [T])
    same_bytes(cache, mirror)
    assert cache.sequence_lengths.tolist() == [T]
    assert mirror["scales"][0, 0, T - 3:T, 0].tolist() == [255] * 3
    back, _ = sa.dequantize_kv(cache, dtype=torch.float32, tokens=T)
    want = oracle.rows(mirror, 0, 0, T)[0].float()
    assert torch.equal(torch.nan_to_num(back[0].cpu(), nan=123.0, posinf=1e9), torch.nan_to_num(want, nan=123.0, posinf=1e9))
    assert bool(torch.isnan(back[0, T - 3:]).all())
    # Row 3 is (2 - 2^-23) * 2^127 throughout.  The codes' steps at the top of that binade are 2^124 (e4m3)
    # and 2^122 (int8), so the nearest code stands for 2^128, which fp32 does not have: it reads back as
    # infinity.  Every other row is below half the largest fp32 value.
    assert bool(torch.isinf(back[0, 3]).all()) and bool(torch.isfinite(back[0, [t for t in range(T - 3) if t != 3]]).all())


def test_write_takes_any_strides(dev):
    B, T, H, D = 2, 6, 3, 64
    for pad in (8, 1):                                        # 16-byte pieces, and one element at a time
        cache, mirror = make_cache(dev, "contig", "BHND", "e4m3", B, H, D, 16)
        wide = new_rows((H, B, T, D + pad), torch.bfloat16, 4)
        k = wide.to(dev).permute(1, 2, 0, 3)[..., :D]
        v = new_rows((H, B, T, D + pad), torch.bfloat16, 6).to(dev).permute(1, 2, 0, 3)[..., :D]
        sa.quantize_kv(cache, k, v)
        oracle.write(mirror, k.cpu(), v.cpu(), [0] * B, [T] * B)
        same_bytes(cache, mirror)
        cache, mirror = make_cache(dev, "contig", "BNHD", "int8", B, H, D, 16)
        sa.quantize_kv(cache, k.transpose(1, 2), v.transpose(1, 2), new_layout="BHND")
        oracle.write(mirror, k.cpu(), v.cpu(), [0] * B, [T] * B)
        same_bytes(cache, mirror)
    # a cache that is a view of a larger one, scales too
    key, value = (torch.zeros(B, H, 16, D + 16, dtype=torch.uint8, device=dev).view(torch.int8)[..., :D] for _ in range(2))
    scales = torch.zeros(B, H + 1, 24, 2, dtype=torch.uint8, device=dev)[:, :H, :16]
    cache = sa.QuantKVCache(key=key, value=value, scales=scales, sequence_lengths=torch.zeros(B, dtype=torch.int64, device=dev))
    mirror = dict(key=key.cpu().contiguous(), value=value.cpu().contiguous(), scales=scales.cpu().contiguous(), table=None,
                  page=0, capacity=16, heads_first=True)
    sa.quantize_kv(cache, k, v)
    oracle.write(mirror, k.cpu(), v.cpu(), [0] * B, [T] * B)
    assert torch.equal(key.cpu(), mirror["key"]) and torch.equal(value.cpu(), mirror["value"]) and torch.equal(scales.cpu(), mirror["scales"])
    assert cache.sequence_lengths.tolist() == [T] * B


@pytest.mark.parametrize("tokens", [1, 200], ids=["one CTA a row", "several"])
def test_write_reports_rows_that_do_not_fit_and_pages_that_are_not_there(dev, tokens):
    B, H, D, page = 4, 2, 64, 16
    cache, mirror = make_cache(dev, "paged", "HND", "e4m3", B, H, D, 256, page=page)
    capacity = mirror["capacity"]
    mirror["table"][1, 2] = -1
    mirror["table"][3, 2] = mirror["scales"].shape[0]
    cache.page_table.copy_(mirror["table"])
    k, v = new_rows((B, tokens, H, D), torch.bfloat16, 1), new_rows((B, tokens, H, D), torch.bfloat16, 2)
    starts = [capacity - tokens + 1, 33, 20, 32]              # past the end; no page; good; page id past the pool
    cache.sequence_lengths.copy_(torch.tensor(starts))
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    sa.quantize_kv(cache, k.to(dev), v.to(dev), status=status)
    torch.cuda.synchronize()
    assert int(status) == native.SA_DEV_BAD_PAGE | native.SA_DEV_BAD_POSITION
    assert cache.sequence_lengths.tolist() == [starts[0], 33, 20 + tokens, 32]
    oracle.write(mirror, k, v, starts, [tokens] * B)
    same_bytes(cache, mirror)
    cache.sequence_lengths.copy_(torch.tensor([-1, 0, 0, 0]))
    before = cache.sequence_lengths.tolist()
    sa.quantize_kv(cache, k.to(dev), v.to(dev), status=status, advance_lengths=False)
    assert cache.sequence_lengths.tolist() == before
    # counts: clipped to what the call holds; a full row takes an empty update
    cache.sequence_lengths.copy_(torch.tensor([capacity, 0, 0, 0]))
    counts = torch.tensor([0, -5, 10 ** 9, 1], dtype=torch.int64, device=dev)
    status.zero_()
    sa.quantize_kv(cache, k.to(dev), v.to(dev), status=status, counts=counts)
    assert cache.sequence_lengths.tolist() == [capacity, 0, tokens, 1] and int(status) == 0


@pytest.mark.parametrize("kind,layout,code,dtype,D,page", [
    ("paged", "HND", "e4m3", "bf16", 64, 16), ("paged", "NHD", "int8", "fp16", 128, 64), ("contig", "BHND", "int8", "bf16", 80, 0),
    ("contig", "BNHD", "e4m3", "fp32", 256, 0), ("paged", "NHD", "int8", "fp32", 13, 5), ("contig", "BHND", "e4m3", "fp16", 8, 0)])
def test_read_back_any_range(dev, kind, layout, code, dtype, D, page):
    B, H, N, T = 3, 2, 90, 41
    cache, mirror = make_cache(dev, kind, layout, code, B, H, D, N, page=page or 16, seed=D)
    mirror["scales"].clamp_(100, 150)                         # random bytes make rows from 2^-27 up to 2^23
    if code == "e4m3":                                        # the code of NaN is no row's
        for name in ("key", "value"):
            b = mirror[name].view(torch.uint8)
            b[(b & 0x7f) == 0x7f] = 0x42
            getattr(cache, name).view(torch.uint8).copy_(b)
    cache.scales.copy_(mirror["scales"])
    starts, counts = [0, 17, mirror["capacity"] - 3], [T, 0, 3]
    for out_layout in ("BNHD", "BHND"):
        shape = (B, T, H, D) if out_layout == "BNHD" else (B, H, T, D)
        key = torch.full(shape, 3.0, dtype=TYPES[dtype], device=dev)
        value = torch.full(shape, 4.0, dtype=TYPES[dtype], device=dev)
        status = torch.zeros(1, dtype=torch.int32, device=dev)
        got = sa.DequantizeKVPlan.build(cache, key, value, starts=torch.tensor(starts, device=dev),
                                        counts=torch.tensor(counts, dtype=torch.int32, device=dev), out_layout=out_layout,
                                        status=status).run()
        assert got[0] is key and got[1] is value and int(status) == 0
        for b in range(B):
            k, v, held = oracle.rows(mirror, b, starts[b], counts[b])
            assert bool(held.all())
            for t, want, fill in ((key, k, 3.0), (value, v, 4.0)):
                t = (t if out_layout == "BNHD" else t.transpose(1, 2))[b].cpu()
                assert torch.equal(t[:counts[b]], want.to(TYPES[dtype])) and bool((t[counts[b]:] == fill).all())


def test_read_back_leaves_out_what_is_not_there(dev):
    cache, mirror = make_cache(dev, "paged", "NHD", "int8", 2, 1, 64, 64, page=16)
    mirror["scales"].clamp_(100, 150)
    cache.scales.copy_(mirror["scales"])
    mirror["table"][0, 1] = -1
    cache.page_table.copy_(mirror["table"])
    key = torch.full((2, 40, 1, 64), 9.0, device=dev)
    value = torch.full_like(key, 9.0)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    sa.DequantizeKVPlan.build(cache, key, value, starts=torch.tensor([0, 50], device=dev), status=status).run()
    assert int(status) == native.SA_DEV_BAD_PAGE | native.SA_DEV_BAD_POSITION
    for b, start in ((0, 0), (1, 50)):
        k, v, held = oracle.rows(mirror, b, start, 40)
        for got, want in ((key, k), (value, v)):
            assert torch.equal(got[b].cpu()[held], want[held].float()) and bool((got[b].cpu()[~held] == 9.0).all())
    assert not bool(held.all())


@pytest.mark.parametrize("code", list(CODES))
@pytest.mark.parametrize("dtype", list(TYPES))
def test_a_second_quantisation_changes_nothing(dev, code, dtype):
    """Read back and written again, a row has the values it had: power-of-two scales are exact in every type."""
    B, T, H, D = 2, 50, 2, 64
    first = sa.QuantKVCache.empty(B, H, T, D, dtype=CODES[code], device=dev)
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn(B, T, H, D, generator=g).to(dev) for _ in range(2))
    sa.quantize_kv(first, k, v)
    again = sa.QuantPagedKVCache.empty(B * 4, 16, H, D, batch=B, max_pages_per_request=4, dtype=CODES[code], device=dev)
    again.page_table.copy_(torch.arange(B * 4, device=dev).flip(0).view(B, 4))
    rows = sa.dequantize_kv(first, tokens=T, dtype=TYPES[dtype])
    sa.quantize_kv(again, *rows)
    for a, b in zip(rows, sa.dequantize_kv(again, tokens=T, dtype=TYPES[dtype])):
        assert torch.equal(a, b)
    assert again.sequence_lengths.tolist() == [T] * B


def test_update_replays_in_a_graph_and_runs_on_other_streams(dev):
    B, H, D = 2, 2, 64
    cache, mirror = make_cache(dev, "paged", "HND", "e4m3", B, H, D, 64)
    k, v = new_rows((B, 1, H, D), torch.bfloat16, 1).to(dev), new_rows((B, 1, H, D), torch.bfloat16, 2).to(dev)
    plan = sa.QuantizeKVPlan.build(cache, k, v)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        plan.run()
    torch.cuda.current_stream(dev).wait_stream(side)
    torch.cuda.synchronize()
    oracle.write(mirror, k.cpu(), v.cpu(), [0] * B, [1] * B)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.run()
    for step in range(1, 20):
        k.copy_(new_rows((B, 1, H, D), torch.bfloat16, 10 + step))
        graph.replay()
        torch.cuda.synchronize()
        oracle.write(mirror, k.cpu(), v.cpu(), [step] * B, [1] * B)
    same_bytes(cache, mirror)
    assert cache.sequence_lengths.tolist() == [20] * B


@pytest.mark.parametrize("batch,tokens,heads,dim,page", [(5000, 40, 2, 64, 16), (9, 5000, 8, 128, 64), (6, 8191, 4, 64, 8)])
@pytest.mark.parametrize("new_layout", ["BNHD", "BHND"])
def test_large_ragged_writes_give_the_bytes_of_even_ones(dev, batch, tokens, heads, dim, page, new_layout):
    """Threads that take several units: same bytes, nothing behind the counts, bad pages and lengths as ever."""
    g = torch.Generator(dev).manual_seed(batch)
    pages = -(-tokens // page)
    shape = (batch, tokens, heads, dim) if new_layout == "BNHD" else (batch, heads, tokens, dim)
    k, v, cos, sin = (torch.randn(s, generator=g, device=dev).bfloat16() for s in (shape, shape, (1, tokens, dim), (1, tokens, dim)))
    counts = torch.randint(0, tokens + 1, (batch,), generator=g, device=dev)
    counts[:2] = tokens
    even, ragged = (sa.QuantPagedKVCache.empty(batch * pages, page, heads, dim, batch=batch, max_pages_per_request=pages, device=dev)
                    for _ in range(2))
    for cache in (even, ragged):
        cache.page_table.copy_(torch.arange(batch * pages, device=dev).view(batch, pages))
    ragged.page_table[1, 0] = -1                                          # its first tokens have no page, the others do
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    sa.quantize_kv(even, k, v, cos=cos, sin=sin, new_layout=new_layout)
    sa.quantize_kv(ragged, k, v, cos=cos, sin=sin, new_layout=new_layout, counts=counts, status=status)
    assert int(status) == native.SA_DEV_BAD_PAGE and bool((even.sequence_lengths == tokens).all())
    want = counts.clone()
    want[1] = 0
    assert torch.equal(ragged.sequence_lengths.long(), want)
    written = torch.arange(pages * page, device=dev)[None] < counts[:, None]
    written[1, :page] = False
    written = written.view(batch * pages, 1, page, 1)
    for name in ("key", "value", "scales"):
        a, b = (getattr(c, name).view(torch.uint8) for c in (even, ragged))
        assert torch.equal(torch.where(written, a, torch.zeros_like(a)), b)


def test_many_ctas_advance_their_row_in_place_once(dev):
    """Lengths that are positions too: no CTA of a row may see the new value."""
    B, T, H, D = 5, 700, 4, 128
    cache = sa.QuantKVCache.empty(B, H, 4 * T, D, device=dev)
    k, v = torch.randn(B, T, H, D, device=dev).bfloat16(), torch.randn(B, T, H, D, device=dev).bfloat16()
    plan = sa.QuantizeKVPlan.build(cache, k, v)
    for _ in range(4):
        plan.run()
    assert cache.sequence_lengths.tolist() == [4 * T] * B
    key, value = sa.dequantize_kv(cache, dtype=torch.float32)
    for a, x in ((key, k), (value, v)):
        assert torch.equal(a[:, :T], a[:, 3 * T:])
        # a code is off by half a step: 2^-4 of the value, or half the smallest step 2^-9 * scale, scale <= max|x| / 224
        bound = torch.maximum(x.float().abs() * 2 ** -4, x.float().abs().amax(-1, keepdim=True) / 224 * 2 ** -10)
        assert bool(((a[:, :T] - x.float()).abs() <= bound).all())
