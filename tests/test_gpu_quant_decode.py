"""One-token attention over 8-bit KV caches, against the 64-bit oracle over the values the codes stand for.

What may differ (all relative to sum_t p_t |v_t| unless said otherwise):
  * the result is rounded to its type once: half a step of the value;
  * p is rounded to fp16 before it meets the codes of V: 2^-11;
  * a score is a sum of D products in fp32, some 2^-23 each of sum_d |q_d k_d| / sqrt(D), and a few more
    roundings of that size; p = exp(score - max) carries the error of both, the denominator as well;
  * the sums over N tokens in fp32: 2^-23 a step, and 2^-20 for the exponential.
"""

import pytest
import torch

import streamattn_b200 as sa
from oracle import quant_kv as oracle
from streamattn_b200 import native
from tests.test_gpu_quant_kv import CODES, TYPES, dev, make_cache, new_rows  # noqa: F401

pytestmark = pytest.mark.gpu
KERNELS = ["auto", "generic"]


def tolerance(want, spread, reach, dtype, dim, tokens):
    step = torch.finfo(dtype).eps / 2
    inner = 2 ** -11 + 4 * (dim + 8) * 2 ** -23 * reach + tokens * 2 ** -23 + 2 ** -20
    return step * want.abs() + spread * (1 + step) * inner + torch.finfo(dtype).tiny


def check(got, q, mirror, lengths, rows=None):
    want, spread, reach = oracle.attend(q, mirror, lengths)
    tol = tolerance(want, spread, reach, q.dtype, q.shape[-1], max([int(n) for n in lengths] + [1]))
    off = (got.cpu().double() - want).abs() - tol
    rows = range(len(lengths)) if rows is None else rows
    for b in rows:
        assert bool((off[b] <= 0).all()), (b, int(lengths[b]), float(off[b].max()), float(want[b].abs().max()))


def filled(dev, kind, layout, code, batch, heads, dim, capacity, lengths, page=16, seed=0, table_dtype=torch.int32, lens_dtype=torch.int32):
    """A cache of random rows up to each row's length; behind it the codes and scales are random bytes, NaNs among them."""
    cache, mirror = make_cache(dev, kind, layout, code, batch, heads, dim, capacity, page=page, seed=seed, table_dtype=table_dtype)
    T = max(max(lengths), 1)
    k, v = new_rows((batch, T, heads, dim), torch.float32, seed + 1), new_rows((batch, T, heads, dim), torch.float32, seed + 2)
    k = k / k.square().mean(-1, keepdim=True).sqrt().clamp_min(1.0)        # scores of a few units
    oracle.write(mirror, k, v, [0] * batch, lengths)
    for name in ("key", "value", "scales"):
        getattr(cache, name).view(torch.uint8).copy_(mirror[name].view(torch.uint8))
    lens = torch.tensor(lengths, dtype=lens_dtype, device=dev)
    fields = dict(key=cache.key, value=cache.value, scales=cache.scales, sequence_lengths=lens, layout=layout)
    if kind == "paged":
        return sa.QuantPagedKVCache(page_table=cache.page_table, **fields), mirror
    return sa.QuantKVCache(**fields), mirror


CASES = [
    # kind, layout, code, dtype, kv_heads, group, dim, lengths, page
    ("contig", "BHND", "e4m3", "bf16", 2, 8, 64, [300, 1, 0, 64], 0),
    ("contig", "BNHD", "int8", "fp16", 2, 4, 128, [257, 65, 63], 0),
    ("contig", "BHND", "int8", "bf16", 1, 16, 128, [190], 0),
    ("contig", "BNHD", "e4m3", "fp16", 3, 1, 64, [129, 2], 0),
    ("contig", "BHND", "e4m3", "bf16", 1, 24, 64, [100, 70], 0),          # a group that is split in two
    ("paged", "HND", "e4m3", "bf16", 2, 8, 64, [300, 1, 0, 16, 17], 16),
    ("paged", "NHD", "int8", "fp16", 2, 4, 128, [200, 64, 65], 64),
    ("paged", "HND", "int8", "bf16", 1, 7, 128, [143, 9], 8),
    ("paged", "NHD", "e4m3", "fp16", 2, 16, 64, [260, 128], 128),
    ("paged", "HND", "e4m3", "fp16", 2, 2, 128, [130, 300], 32),
    # the generic kernel's own ground: sizes, pages and types that have no tensor-core form
    ("contig", "BHND", "int8", "fp32", 2, 2, 64, [70, 33], 0),
    ("contig", "BNHD", "e4m3", "bf16", 2, 3, 80, [70, 33], 0),
    ("contig", "BHND", "e4m3", "fp16", 1, 2, 256, [40], 0),
    ("paged", "HND", "int8", "bf16", 2, 2, 64, [70, 33, 5], 4),
    ("paged", "NHD", "e4m3", "fp32", 1, 2, 13, [70, 33, 5], 24),
]


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)).replace(" ", ""))
def test_decode_matches_the_oracle(dev, case, kernel):
    kind, layout, code, dtype, H, G, D, lengths, page = case
    B = len(lengths)
    cache, mirror = filled(dev, kind, layout, code, B, H, D, -(-max(lengths) // 8) * 8 + 8, lengths, page=page or 16, seed=D + G)
    q = new_rows((B, 1, H * G, D), TYPES[dtype], 9).clamp(-30, 30)
    plan = sa.QuantDecodePlan.build(q.to(dev), cache, kernel=kernel)
    out = plan.run()
    assert plan.device_status() == 0 and out is plan.output
    check(out, q, mirror, lengths)
    first = out.clone()
    assert torch.equal(plan.run(), first)                                 # the same bits from launch to launch
    for b, n in enumerate(lengths):
        if n == 0:
            assert not bool(out[b].any())


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("splits", [1, 3, 40])
def test_any_number_of_splits(dev, kernel, splits):
    lengths = [700, 64, 130]
    cache, mirror = filled(dev, "paged", "HND", "int8", 3, 2, 64, 1024, lengths, table_dtype=torch.int64, lens_dtype=torch.int64)
    q = new_rows((3, 1, 8, 64), torch.bfloat16, 3).clamp(-30, 30)
    plan = sa.QuantDecodePlan.build(q.to(dev), cache, splits=splits, kernel=kernel)
    check(plan.run(), q, mirror, lengths)
    check(plan.run(), q, mirror, lengths)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("code", list(CODES))
def test_scales_of_any_size(dev, kernel, code):
    """Rows from 2^-90 to 2^90 next to each other: none may overflow, underflow or hide another."""
    B, H, D, lengths = 2, 2, 64, [200, 130]
    cache, mirror = filled(dev, "contig", "BHND", code, B, H, D, 256, lengths, seed=4)
    g = torch.Generator().manual_seed(8)
    e = torch.randint(37, 218, (B, H, 256), generator=g)
    e[0, 0] = torch.randint(37, 60, (256,), generator=g)                   # a head of small values throughout
    mirror["scales"][..., 1] = e.to(torch.uint8)
    mirror["scales"][..., 0].clamp_(100, 120)
    cache.scales.copy_(mirror["scales"])
    q = new_rows((B, 1, 8, D), torch.bfloat16, 3).clamp(-2, 2)
    q[1, 0, 0] *= 2.0 ** -100
    q[1, 0, 1] *= 2.0 ** 40
    got = sa.QuantDecodePlan.build(q.to(dev), cache, kernel=kernel).run()
    check(got, q, mirror, lengths)


@pytest.mark.parametrize("kernel", KERNELS)
def test_nan_rows_reach_their_head_and_no_other(dev, kernel):
    B, H, G, D, lengths = 3, 2, 4, 64, [200, 130, 64]
    cache, mirror = filled(dev, "paged", "HND", "e4m3", B, H, D, 256, lengths, seed=6)
    bad = torch.full((1, 1, H, D), 1.0)
    bad[0, 0, 1, 5] = float("nan")                                         # K of head 1 of row 0, in the middle of the row
    oracle_at = mirror["scales"]
    page, slot = oracle.place(mirror, 0, 77)
    oracle_at[page, 1, slot, 0] = 255
    page, slot = oracle.place(mirror, 2, 63)
    oracle_at[page, 0, slot, 1] = 255                                      # V of head 0 of row 2, its last token
    page, slot = oracle.place(mirror, 1, 130)
    oracle_at[page, :, slot] = 255                                         # behind row 1's last token
    cache.scales.copy_(oracle_at)
    q = new_rows((B, 1, H * G, D), torch.bfloat16, 3).clamp(-30, 30)
    for splits in (None, 1, 5):
        out = sa.QuantDecodePlan.build(q.to(dev), cache, kernel=kernel, splits=splits).run().cpu().view(B, H, G, D)
        nan = torch.isnan(out)
        assert bool(nan[0, 1].all()) and bool(nan[2, 0].all())
        assert not bool(nan[0, 0].any()) and not bool(nan[2, 1].any()) and not bool(nan[1].any())
    mirror["scales"][mirror["scales"] == 255] = 120
    out = out.view(B, 1, H * G, D)
    want, spread, reach = oracle.attend(q, mirror, lengths)
    tol = tolerance(want, spread, reach, q.dtype, D, 200)
    for b, h in ((0, 0), (1, 0), (1, 1), (2, 1)):
        at = slice(h * G, (h + 1) * G)
        assert bool(((out[b, 0, at].double() - want[b, 0, at]).abs() <= tol[b, 0, at]).all())


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("code", list(CODES))
def test_nan_and_infinite_queries_make_their_head_nan(dev, kernel, code):
    B, H, G, D, lengths = 2, 1, 11, 64, [300, 0]
    cache, mirror = filled(dev, "contig", "BHND", code, B, H, D, 320, lengths, seed=6)
    q = new_rows((B, 1, H * G, D), torch.bfloat16, 3).clamp(-30, 30)
    q[0, 0, 2, 5], q[0, 0, 9, 63], q[0, 0, 10, 0], q[1, 0, 0, 0] = float("nan"), float("inf"), -float("inf"), float("nan")
    bad = [2, 9, 10]
    for splits in (None, 1, 4):
        plan = sa.QuantDecodePlan.build(q.to(dev), cache, kernel=kernel, splits=splits)
        out = plan.run().cpu()
        assert bool(torch.isnan(out[0, 0, bad]).all()) and not bool(out[1].any())      # a row of no tokens is zero
        good = [h for h in range(G) if h not in bad]
        want, spread, reach = oracle.attend(q[:, :, good], mirror, lengths)
        tol = tolerance(want, spread, reach, q.dtype, D, 300)
        assert bool(((out[:, :, good].double() - want).abs() <= tol).all())
    state = sa.QuantDecodePlan.build(q.to(dev), cache, kernel=kernel, return_state=True).run().cpu()
    assert bool(torch.isfinite(state[0, :, D:]).all()) and bool(torch.isnan(state[0, bad, :D]).all())


def test_offsets_beyond_32_bits(dev):
    """A row whose codes pass 2^32 bytes: written, attended to and read back at its far end."""
    H, D, N, T = 16, 128, 2 ** 21 + 128, 70
    cache = sa.QuantKVCache.empty(1, H, N, D, device=dev)                 # 4.3 GB each of K and V
    cache.scales.fill_(100)
    k = torch.full((1, T, H, D), 4.0, device=dev).bfloat16()
    v = torch.randn(1, T, H, D, generator=torch.Generator(dev).manual_seed(1), device=dev).bfloat16()
    start = torch.full((1,), N - T, dtype=torch.int64, device=dev)
    lens = torch.zeros(1, dtype=torch.int64, device=dev)
    sa.quantize_kv(cache, k, v, positions=start, lengths_out=lens)
    assert int(lens) == N
    key, value = sa.dequantize_kv(cache, tokens=T, starts=start, dtype=torch.float32)
    assert torch.equal(key, k.float())
    bound = torch.maximum(v.float().abs() * 2 ** -4, v.float().abs().amax(-1, keepdim=True) / 224 * 2 ** -10)
    assert bool(((value - v.float()).abs() <= bound).all())
    # q . k / sqrt(D) = 4 * D / sqrt(D) = 45 for the T last tokens and 0 for all others: e^-45 of 2^21 tokens is nothing
    q = torch.ones(1, 1, H * 4, D, device=dev).bfloat16()
    cache.sequence_lengths.fill_(N)
    out = sa.stream_attn_quant_decode(q, cache)
    want = value[0].double().mean(0).repeat_interleave(4, dim=0)
    spread = value[0].double().abs().mean(0).repeat_interleave(4, dim=0)
    assert bool(((out[0, 0].double() - want).abs() <= 2 ** -8 * want.abs() + spread * (2 ** -11 + 2 ** -15)).all())


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page", [8, 16, 64, 128])
def test_bad_pages_are_left_out_and_reported(dev, kernel, page, dim):
    B, H, lengths = 2, 2, [400, 300]
    cache, mirror = filled(dev, "paged", "HND", "e4m3", B, H, dim, 512, lengths, page=page, seed=page)
    pool = mirror["scales"].shape[0]
    mirror["table"][0, 1], mirror["table"][1, 0], mirror["table"][0, 0] = -1, pool, 2 ** 31 - 1
    mirror["table"][1, lengths[1] // page] = -(2 ** 31)
    cache.page_table.copy_(mirror["table"])
    with pytest.raises(ValueError, match="active page_table entries must reference physical pages"):
        sa.QuantDecodePlan.build(torch.zeros(B, 1, 4, dim, dtype=torch.bfloat16, device=dev), cache)
    q = new_rows((B, 1, 4, dim), torch.bfloat16, 3).clamp(-30, 30)
    plan = sa.QuantDecodePlan.build(q.to(dev), cache, kernel=kernel, validate_metadata=False)
    out = plan.run()
    assert plan.device_status() == native.SA_DEV_BAD_PAGE
    check(out, q, mirror, lengths)
    cache.page_table.fill_(-1)                                             # nothing is left: zeros, as for an empty row
    assert not bool(plan.run().any()) and plan.device_status() == native.SA_DEV_BAD_PAGE


@pytest.mark.parametrize("kernel", KERNELS)
def test_row_subsets_states_and_page_walk(dev, kernel):
    B, H, G, D, lengths = 4, 2, 4, 64, [200, 130, 64, 0]
    cache, mirror = filled(dev, "paged", "NHD", "int8", B, H, D, 256, lengths, page=16, seed=2)
    q = new_rows((B, 1, H * G, D), torch.bfloat16, 3).clamp(-30, 30)
    out = torch.full((B, 1, H * G, D), 5.0, dtype=torch.bfloat16, device=dev)
    rows = torch.tensor([2, 0, 2, 99], dtype=torch.int64, device=dev)
    plan = sa.QuantDecodePlan.build(q.to(dev), cache, output=out, kernel=kernel, row_indices=rows, record_page_walk=True)
    plan.run()
    check(out, q, mirror, lengths, rows=[0, 2])
    assert bool((out[[1, 3]] == 5.0).all())
    plan.set_row_indices(None)
    plan.run()
    check(out, q, mirror, lengths)
    walk = torch.full_like(mirror["table"], -1)
    for b, n in enumerate(lengths):
        walk[b, :-(-n // 16)] = mirror["table"][b, :-(-n // 16)]
    assert torch.equal(plan.trace.cpu(), walk)
    # states of the first 100 and of the other tokens merge to the whole
    want, spread, reach = oracle.attend(q, mirror, lengths)
    state = sa.QuantDecodePlan.build(q.to(dev), cache, kernel=kernel, return_state=True).run()
    assert tuple(state.shape) == (B, H * G, D + 2) and state.dtype == torch.float32
    o, l = state[..., :D].double().cpu(), state[..., D + 1].double().cpu()
    assert l[3].tolist() == [0.0] * (H * G) and torch.isinf(state[3, :, D]).all()
    tol = tolerance(want, spread, reach, torch.float32, D, 200)
    assert bool(((o[:3] / l[:3, :, None] - want[:3, 0]).abs() <= tol[:3, 0]).all())


@pytest.mark.parametrize("page,layout,dim,group", [(8, "HND", 64, 4), (32, "NHD", 128, 16), (64, "HND", 64, 12),
                                                   (128, "NHD", 128, 24), (256, "HND", 128, 9), (0, "BNHD", 128, 20)])
def test_wide_indices_subsets_and_walks_on_every_placement(dev, page, layout, dim, group):
    """Lengths 0 and 1, row subsets, 64-bit tables and lengths, groups of more than 8 and 16 heads."""
    B, H, lengths = 5, 2, [513, 0, 1, 320, 65]
    kind = "paged" if page else "contig"
    cache, mirror = filled(dev, kind, layout, "e4m3", B, H, dim, 768, lengths, page=page or 16, seed=page,
                           table_dtype=torch.int64, lens_dtype=torch.int64)
    q = new_rows((B, 1, H * group, dim), torch.bfloat16, 3).clamp(-30, 30)
    out = torch.full((B, 1, H * group, dim), 5.0, dtype=torch.bfloat16, device=dev)
    plan = sa.QuantDecodePlan.build(q.to(dev), cache, output=out, record_page_walk=bool(page))
    assert plan.kernel_name == "sm100_tma_mma_stream"
    plan.set_row_indices(torch.tensor([3, 1, 2], device=dev))
    plan.run()
    check(out, q, mirror, lengths, rows=[1, 2, 3])
    assert bool((out[[0, 4]] == 5.0).all()) and not bool(out[1].any())
    plan.set_row_indices(None)
    plan.run()
    check(out, q, mirror, lengths)
    assert plan.device_status() == 0
    if page:
        walk = torch.full(tuple(mirror["table"].shape), -1, dtype=torch.int32)
        for b, n in enumerate(lengths):
            walk[b, :-(-n // page)] = mirror["table"][b, :-(-n // page)].int()
        assert torch.equal(plan.trace.cpu(), walk)


@pytest.mark.parametrize("B,H,D", [(900, 2, 64), (3500, 1, 128)], ids=["warps' slices", "no room for them"])
def test_a_large_batch_of_one_token_rows(dev, B, H, D):
    """More rows than a CTA has threads, and more pairs than the grid has CTAs."""
    cache = sa.QuantPagedKVCache.empty(B, 16, H, D, batch=B, max_pages_per_request=3, device=dev)
    cache.page_table[:, 0] = torch.randperm(B, generator=torch.Generator().manual_seed(1)).int().to(dev)
    k, v = (torch.randn(B, 1, H, D, generator=torch.Generator(dev).manual_seed(i), device=dev).bfloat16() for i in (1, 2))
    q = torch.randn(B, 1, 4 * H, D, device=dev).bfloat16()
    moved = sa.quantize_kv(cache, k, v, query=q)
    assert torch.equal(moved, q) and bool((cache.sequence_lengths == 1).all())
    value = sa.dequantize_kv(cache, tokens=1, dtype=torch.float32)[1]
    out = sa.stream_attn_quant_decode(q, cache).view(B, H, 4, D).float()
    want = value[:, 0, :, None].expand_as(out)                            # a softmax of one token: its V row, rounded once
    assert bool(((out - want).abs() <= want.abs() * 2 ** -8).all())


@pytest.mark.parametrize("kernel", KERNELS)
def test_lengths_change_on_the_device_and_graphs_follow(dev, kernel):
    B, H, G, D = 2, 2, 4, 128
    cache, mirror = filled(dev, "contig", "BHND", "e4m3", B, H, D, 512, [511, 511], seed=3)
    q = new_rows((B, 1, H * G, D), torch.float16, 3).clamp(-30, 30)
    plan = sa.QuantDecodePlan.build(q.to(dev), cache, kernel=kernel)
    plan.run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.run()
    for lengths in ([500, 400], [0, 511], [1, 0], [-3, 10 ** 6], [64, 128]):
        cache.sequence_lengths.copy_(torch.tensor(lengths))
        graph.replay()
        clipped = [min(max(n, 0), 512) for n in lengths]
        if max(clipped) < 512:
            check(plan.output, q, mirror, clipped)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        plan.run()
    side.synchronize()
    check(plan.output, q, mirror, [64, 128])


def test_two_plans_at_once(dev):
    B, H, G, D = 4, 2, 8, 64
    lengths = [4000, 3000, 10, 2000]
    cache = sa.QuantKVCache.empty(B, H, 4096, D, device=dev)
    k, v = torch.randn(B, 4096, H, D, device=dev).bfloat16(), torch.randn(B, 4096, H, D, device=dev).bfloat16()
    sa.quantize_kv(cache, k, v, counts=torch.tensor(lengths, device=dev))
    qs = [torch.randn(B, 1, H * G, D, device=dev).bfloat16() for _ in range(2)]
    plans = [sa.QuantDecodePlan.build(q, cache) for q in qs]
    alone = [p.run().clone() for p in plans]
    streams = [torch.cuda.Stream(dev) for _ in plans]
    torch.cuda.synchronize()
    for _ in range(20):
        for p, s in zip(plans, streams):
            with torch.cuda.stream(s):
                p.run()
    torch.cuda.synchronize()
    for p, want in zip(plans, alone):
        assert torch.equal(p.output, want) and p.device_status() == 0


def test_pinned_query_and_output(dev):
    lengths = [200, 30]
    cache, mirror = filled(dev, "contig", "BNHD", "int8", 2, 2, 64, 256, lengths, seed=3)
    q = new_rows((2, 1, 8, 64), torch.bfloat16, 3).clamp(-30, 30).pin_memory()
    out = torch.zeros(2, 1, 8, 64, dtype=torch.bfloat16).pin_memory()
    plan = sa.QuantDecodePlan.build(q, cache, output=out)
    plan.run()
    torch.cuda.synchronize()
    check(out, q, mirror, lengths)


@pytest.mark.parametrize("batch,heads,capacity,low", [(40, 3, 256, 1), (63, 2, 1024, 100), (20, 8, 512, 0), (9, 8, 640, 400)])
@pytest.mark.parametrize("page", [0, 16, 64])
def test_many_short_rows(dev, batch, heads, capacity, low, page):
    """Around one CTA a (row, KV head) pair: aligned slices, one CTA each, and slices across pairs give the same."""
    D, G = 64, 4
    g = torch.Generator().manual_seed(batch)
    lengths = torch.randint(low, capacity + 1, (batch,), generator=g)
    cache = sa.QuantKVCache.empty(batch, heads, capacity, D, device=dev)
    k, v = (torch.randn(batch, capacity, heads, D, generator=g).bfloat16().to(dev) for _ in range(2))
    sa.quantize_kv(cache, k, v, counts=lengths.to(dev))
    key, value = (x.transpose(1, 2).double() for x in sa.dequantize_kv(cache, dtype=torch.float32))    # [B, H, N, D]
    if page:
        paged = sa.QuantPagedKVCache.empty(batch * capacity // page, page, heads, D, batch=batch,
                                           max_pages_per_request=capacity // page, device=dev)
        paged.page_table.copy_(torch.randperm(batch * capacity // page, generator=g).view(batch, -1))
        sa.quantize_kv(paged, k, v, counts=lengths.to(dev))
        cache = paged
    q = torch.randn(batch, 1, heads * G, D, generator=g).bfloat16().to(dev)
    qh = q[:, 0].double().view(batch, heads, G, D)
    scores = qh @ key.transpose(2, 3) / D ** 0.5
    mask = torch.arange(capacity, device=dev)[None, None, None] >= lengths.to(dev)[:, None, None, None]
    p = torch.softmax(scores.masked_fill(mask, -1e300), -1).masked_fill(mask, 0.0)
    want, spread = p @ value, p @ value.abs()
    reach = (qh.abs() @ key.abs().transpose(2, 3)).masked_fill(mask, 0.0).amax(-1, keepdim=True) / D ** 0.5
    tol = tolerance(want, spread, reach, q.dtype, D, capacity)
    for splits in (None, 1, 3):
        got = sa.QuantDecodePlan.build(q, cache, splits=splits).run().double().view_as(want)
        assert bool(((got - want).abs() <= tol).all()), (splits, float(((got - want).abs() - tol).max()))


@pytest.mark.parametrize("code,dtype,dim,batch,heads,group,capacity,low", [
    (torch.int8, torch.float16, 128, 30, 8, 4, 1024, 0), (torch.float8_e4m3fn, torch.bfloat16, 64, 3, 60, 8, 4096, 3000),
    (torch.float8_e4m3fn, torch.float16, 128, 21, 9, 1, 640, 1), (torch.int8, torch.bfloat16, 64, 50, 4, 12, 512, 0)])
@pytest.mark.parametrize("page", [0, 8, 64])
def test_more_pairs_than_ctas(dev, code, dtype, dim, batch, heads, group, capacity, low, page):
    """Slices that hold pairs, end in them and lie inside them; outputs and states; a subset of the rows."""
    g = torch.Generator().manual_seed(batch)
    lengths = torch.randint(low, capacity + 1, (batch,), generator=g)
    lengths[batch // 2] = capacity
    k, v = (torch.randn(batch, capacity, heads, dim, generator=g).to(dtype).to(dev) for _ in range(2))
    q = torch.randn(batch, 1, heads * group, dim, generator=g).to(dtype).to(dev)
    if page:
        cache = sa.QuantPagedKVCache.empty(batch * capacity // page, page, heads, dim, batch=batch, dtype=code, layout="NHD",
                                           max_pages_per_request=capacity // page, device=dev)
        cache.page_table.copy_(torch.randperm(batch * capacity // page, generator=g).view(batch, -1))
    else:
        cache = sa.QuantKVCache.empty(batch, heads, capacity, dim, device=dev, dtype=code)
    sa.quantize_kv(cache, k, v, counts=lengths.to(dev))
    key, value = (x.transpose(1, 2).double() for x in sa.dequantize_kv(cache, dtype=torch.float32))
    qh = q[:, 0].double().view(batch, heads, group, dim)
    mask = torch.arange(capacity, device=dev)[None, None, None] >= lengths.to(dev)[:, None, None, None]
    p = torch.softmax((qh @ key.transpose(2, 3) / dim ** 0.5).masked_fill(mask, -1e300), -1).masked_fill(mask, 0.0)
    want, spread = p @ value, p @ value.abs()
    reach = (qh.abs() @ key.abs().transpose(2, 3)).masked_fill(mask, 0.0).amax(-1, keepdim=True) / dim ** 0.5
    plan = sa.QuantDecodePlan.build(q, cache)
    got = plan.run().double().view_as(want)
    tol = tolerance(want, spread, reach, dtype, dim, capacity)
    assert bool(((got - want).abs() <= tol).all()), float(((got - want).abs() - tol).max())
    first = plan.output.clone()
    assert torch.equal(plan.run(), first) and plan.device_status() == 0
    plan.output.fill_(5.0)
    rows = torch.arange(0, batch, 2, device=dev)
    plan.set_row_indices(rows)
    got = plan.run().double().view_as(want)
    assert bool(((got - want).abs() <= tol)[rows].all()) and bool((got[1::2] == 5.0).all())
    state = sa.QuantDecodePlan.build(q, cache, return_state=True).run().double().view(batch, heads, group, dim + 2)
    some = (lengths > 0).to(dev)
    tol = tolerance(want, spread, reach, torch.float32, dim, capacity)
    assert bool(((state[..., :dim] / state[..., dim + 1:] - want).abs() <= tol)[some].all())
    assert bool((state[~some][..., dim + 1] == 0).all()) and bool(torch.isinf(state[~some][..., dim]).all())


def test_strided_query_and_views_of_larger_caches(dev):
    B, H, G, D, lengths = 2, 2, 4, 64, [90, 33]
    cache, mirror = filled(dev, "contig", "BHND", "e4m3", B, H, D, 96, lengths, seed=7)
    q = new_rows((B, 1, H * G, 3 * D), torch.bfloat16, 3).clamp(-30, 30)
    dq = q.to(dev)[..., D:2 * D]
    check(sa.stream_attn_quant_decode(dq, cache), q[..., D:2 * D], mirror, lengths)
    # odd capacity: rows of scales that start between the copies' boundaries
    wide = {n: torch.zeros(B, H, 97, *tail, dtype=torch.uint8, device=dev) for n, tail in (("key", (D,)), ("value", (D,)), ("scales", (2,)))}
    for n, t in wide.items():
        t[:, :, :96].copy_(getattr(cache, n).view(torch.uint8))
    odd = sa.QuantKVCache(key=wide["key"].view(torch.float8_e4m3fn), value=wide["value"].view(torch.float8_e4m3fn),
                          scales=wide["scales"].view(torch.float8_e8m0fnu), sequence_lengths=cache.sequence_lengths)
    check(sa.stream_attn_quant_decode(dq, odd), q[..., D:2 * D], mirror, lengths)


@pytest.mark.parametrize("code", list(CODES))
def test_serving_loop_prompt_steps_release_and_read_back(dev, code):
    """The operators together: ragged prompts, decode steps with rotation, a request replaced, the history read back."""
    B, H, G, D, page = 3, 2, 4, 64, 16
    cache = sa.QuantPagedKVCache.empty(24, page, H, D, batch=B, max_pages_per_request=8, dtype=CODES[code], device=dev)
    mirror = dict(key=cache.key.cpu(), value=cache.value.cpu(), scales=cache.scales.cpu(), table=None, page=page, capacity=8 * page,
                  heads_first=True)
    writer = sa.PagedKVWriter.attach(cache)
    dtype, held, T = torch.bfloat16, [0] * B, 70

    def update(tokens, counts, seed):
        k, v = new_rows((B, tokens, H, D), dtype, seed), new_rows((B, tokens, H, D), dtype, seed + 1)
        k = (k.float() / k.float().square().mean(-1, keepdim=True).sqrt().clamp_min(1.0)).to(dtype)
        q = torch.randn(B, tokens, H * G, D, generator=torch.Generator().manual_seed(seed)).to(dtype)
        at = torch.tensor(held)[:, None] + torch.arange(tokens)
        angle = at[..., None].double() * 10000.0 ** (-torch.arange(D // 2, dtype=torch.float64) / (D // 2))
        angle = torch.cat((angle, angle), -1)
        cos, sin = angle.cos().to(dtype), angle.sin().to(dtype)
        turned = writer.append(k.to(dev), v.to(dev), counts=counts, cos=cos.to(dev), sin=sin.to(dev), query=q.to(dev))
        counts = counts or [tokens] * B
        mirror["table"] = cache.page_table.cpu()
        oracle.write(mirror, oracle.rotate(k, cos, sin), v, held, counts)
        for b in range(B):
            held[b] += counts[b]
        want = oracle.rotate(q, cos, sin).to(dtype)
        assert torch.equal(turned.cpu(), want)
        return turned, want

    update(T, [70, 33, 0], 1)
    assert writer.lengths == held == cache.sequence_lengths.tolist()
    query = torch.empty(B, 1, H * G, D, dtype=dtype, device=dev)
    plan = sa.StreamAttnEngine().plan(query, cache, mode="exact_native")
    for step in range(20):
        turned, want = update(1, None, 10 + 2 * step)
        query.copy_(turned)
        out = plan.run(return_info=False)
        check(out, want, mirror, held)
    writer.release(1)
    held[1] = 0
    update(5, [0, 5, 0], 90)
    assert writer.lengths == held == cache.sequence_lengths.tolist()
    out, info = sa.decode(query, cache)
    check(out, query.cpu(), mirror, held)
    assert info.backend_used == plan.backend and info.plan_reason == "quant_kv_exact_only" and info.kv_len == max(held)
    key, value = sa.dequantize_kv(cache, dtype=dtype, tokens=96)
    for b in range(B):
        k, v, _ = oracle.rows(mirror, b, 0, held[b])
        assert torch.equal(key[b, :held[b]].cpu(), k.to(dtype)) and torch.equal(value[b, :held[b]].cpu(), v.to(dtype))
        assert not bool(key[b, held[b]:].any()) and not bool(value[b, held[b]:].any())
    # refused calls leave the writer, the table and the lengths as they were
    before = (list(writer.lengths), cache.page_table.clone(), cache.sequence_lengths.clone(), writer.pool.free_pages)
    k = torch.zeros(B, 100, H, D, dtype=dtype, device=dev)
    for kwargs in (dict(), dict(counts=[101, 0, 0]), dict(counts=[1, 2]), dict(positions=cache.sequence_lengths)):
        with pytest.raises(ValueError):
            writer.append(k, k, **kwargs)
    assert writer.lengths == before[0] and torch.equal(cache.page_table, before[1]) and torch.equal(cache.sequence_lengths, before[2])
    assert writer.pool.free_pages == before[3]


def test_engine_routes_over_contiguous_caches(dev):
    lengths = [200, 30]
    cache, mirror = filled(dev, "contig", "BNHD", "int8", 2, 2, 64, 256, lengths, seed=3)
    q = new_rows((2, 1, 8, 64), torch.bfloat16, 3).clamp(-30, 30)
    out, info = sa.decode(q.to(dev), cache, mode="exact_native")
    check(out, q, mirror, lengths)
    assert info.plan_reason == "explicit_quant_exact_native" and info.stats["code_dtype"] == "int8" and info.kv_len == 200
    with pytest.raises(ValueError, match="must be omitted"):
        sa.decode(q.to(dev), cache, cache.value)
    with pytest.raises(ValueError, match="8-bit KV"):
        sa.decode(q.to(dev), cache, mode="seed_only_native")
    full = sa.QuantKVCache(key=cache.key, value=cache.value, scales=cache.scales.clamp(100, 120), layout="BNHD")
    assert sa.decode(q.to(dev), full)[1].kv_len == 256
