"""8-bit KV caches on the GPU: what a round trip keeps, and the one-element kernels at sizes where their loops run."""

import pytest
import torch

import streamattn_b200 as sa
from oracle import quant_kv as oracle
from tests.test_gpu_quant_kv import CODES, dev, make_cache, new_rows, same_bytes  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("code", list(CODES))
def test_a_round_trip_keeps_values_and_int8_keeps_bytes(dev, code):
    """Largest elements of 225 to 232 times a power of two are rounded to 224, which fits half the scale as 448."""
    B, T, H, D = 1, 64, 2, 64
    rows = new_rows((B, T, H, D), torch.float32, 3)
    tops = [224.0, 225.0, 231.0, 233.0, 448.0, 230.9]
    for t, top in enumerate(tops):
        rows[0, t] = torch.linspace(-1.0, 1.0, D) * top
    first, second = (sa.QuantKVCache.empty(B, H, T, D, dtype=CODES[code], device=dev) for _ in range(2))
    sa.quantize_kv(first, rows.to(dev), rows.to(dev))
    k, v = sa.dequantize_kv(first, dtype=torch.float32)
    sa.quantize_kv(second, k, v)
    again, _ = sa.dequantize_kv(second, dtype=torch.float32)
    assert torch.equal(again, k) and torch.equal(k, v)
    codes, scales = ([getattr(c, name).cpu() for c in (first, second)] for name in ("key", "scales"))
    changed = ((codes[0].view(torch.uint8) != codes[1].view(torch.uint8)).any(-1) | (scales[0] != scales[1]).any(-1))[0]     # [H, T]
    if code == "int8":
        assert not bool(changed.any())
    else:
        largest = codes[0].float().abs().amax(-1)[0]
        assert torch.equal(changed, largest == 224.0)
        assert [bool(x) for x in changed[0, :len(tops)]] == [False, True, True, False, False, True]
        at = changed.nonzero()[0].tolist()
        one, two = (c.float()[0, at[0], at[1]] for c in codes)
        assert torch.equal(two, 2 * one) and int(scales[1][0, at[0], at[1], 0]) == int(scales[0][0, at[0], at[1], 0]) - 1
    mirror = dict(key=first.key.cpu(), value=first.value.cpu(), scales=first.scales.cpu(), table=None, page=0, capacity=T, heads_first=True)
    want, _, _ = oracle.rows(mirror, 0, 0, T)
    assert torch.equal(k[0].cpu().double(), want)


@pytest.mark.parametrize("kind,layout,code,dtype,dim,page", [
    ("contig", "BHND", "e4m3", torch.bfloat16, 40, 0), ("contig", "BNHD", "int8", torch.float32, 13, 0),
    ("paged", "HND", "int8", torch.float16, 72, 24), ("paged", "NHD", "e4m3", torch.bfloat16, 8, 16)])
def test_many_ragged_rows_of_single_elements(dev, kind, layout, code, dtype, dim, page):
    """Head sizes that are no multiple of 16: a warp takes units in turn, and the lengths follow in a launch of their own."""
    B, T, H = 4, 300, 3
    cache, mirror = make_cache(dev, kind, layout, code, B, H, dim, T + 60, page=page or 16, seed=dim)
    k, v = new_rows((B, T, H, dim), dtype, 1), new_rows((B, T, H, dim), dtype, 2)
    starts, counts = [60, 0, 7, 33], [T, 0, 1, 213]
    cache.sequence_lengths.copy_(torch.tensor(starts))
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    plan = sa.QuantizeKVPlan.build(cache, k.to(dev), v.to(dev), counts=torch.tensor(counts, device=dev), status=status)
    plan.run()
    oracle.write(mirror, k, v, starts, counts)
    same_bytes(cache, mirror)
    assert cache.sequence_lengths.tolist() == [s + n for s, n in zip(starts, counts)] and int(status) == 0
    key, value = (torch.full((B, T, H, dim), 9.0, dtype=torch.float32, device=dev) for _ in range(2))
    sa.DequantizeKVPlan.build(cache, key, value, starts=torch.tensor(starts, device=dev), counts=torch.tensor(counts, device=dev)).run()
    for b, n in enumerate(counts):
        want_k, want_v, _ = oracle.rows(mirror, b, starts[b], n)
        assert torch.equal(key[b, :n].cpu().double(), want_k) and torch.equal(value[b, :n].cpu().double(), want_v)
        assert bool((key[b, n:] == 9.0).all()) and bool((value[b, n:] == 9.0).all())
    # a second run goes on behind the first where there is room (row 1 and 2), and leaves out rows whose tokens do not fit
    plan.run()
    held = [s + n for s, n in zip(starts, counts)]
    oracle.write(mirror, k, v, held, counts)
    same_bytes(cache, mirror)
    fits = [h + n <= mirror["capacity"] for h, n in zip(held, counts)]
    assert fits == [False, True, True, False]
    assert cache.sequence_lengths.tolist() == [h + n if ok else h for h, n, ok in zip(held, counts, fits)]


@pytest.mark.parametrize("kernel", ["auto", "generic"])
@pytest.mark.parametrize("kind", ["contig", "paged"])
@pytest.mark.parametrize("wide", [torch.int32, torch.int64])
def test_lengths_beyond_the_capacity_and_below_zero(dev, kernel, kind, wide):
    """They are clipped to the capacity, here of rows that are full, and to 0, which gives zeros; replayed as well."""
    B, H, D, N, page = 3, 2, 64, 512, 64
    k, v = (torch.randn(B, N, H, D, generator=torch.Generator().manual_seed(s)).to(dev) for s in (1, 2))
    if kind == "paged":
        cache = sa.QuantPagedKVCache.empty(B * N // page, page, H, D, batch=B, max_pages_per_request=N // page, device=dev)
        cache.page_table.copy_(torch.randperm(B * N // page, generator=torch.Generator().manual_seed(3)).view(B, -1))
    else:
        cache = sa.QuantKVCache.empty(B, H, N, D, device=dev)
    sa.quantize_kv(cache, k, v)
    fields = {name: getattr(cache, name) for name in cache.__dataclass_fields__}
    cache = type(cache)(**{**fields, "sequence_lengths": cache.sequence_lengths.to(wide)})
    q = torch.randn(B, 1, 8, D, generator=torch.Generator().manual_seed(4)).bfloat16().to(dev)
    plan = sa.QuantDecodePlan.build(q, cache, kernel=kernel)
    full = plan.run().clone()
    assert bool(full.any(-1).all())
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        plan.run()
    limits = torch.iinfo(wide)
    for lengths in ([N + 1, -3, N], [limits.max, limits.min, 0], [-1, N + page, 10 ** 6]):
        cache.sequence_lengths.copy_(torch.tensor(lengths))
        graph.replay()
        out = plan.output.clone()
        for b, n in enumerate(lengths):
            if n <= 0:
                assert not bool(out[b].any())
            else:  # full rows, in other groups: both rounded to bf16 (2^-9 each), p to fp16 beside values of mean size below 1
                assert bool(((out[b].float() - full[b].float()).abs() <= 2.0 ** -8 * full[b].float().abs() + 2.0 ** -10).all())
        assert plan.device_status() == 0
