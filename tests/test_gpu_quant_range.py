"""One-token attention over 8-bit KV caches where the inputs span a wide range, against the 64-bit oracle.

The bound is the one of ``tests/test_gpu_quant_decode.py``.  It has no term for the query: the kernels use it as it is
(fp16 after a power of two, in which the elements of these queries are exact).
"""

import pytest
import torch

import streamattn_b200 as sa
from oracle import quant_kv as oracle
from tests.test_gpu_quant_decode import KERNELS, check, tolerance
from tests.test_gpu_quant_kv import CODES, TYPES, dev, make_cache, new_rows  # noqa: F401

pytestmark = pytest.mark.gpu


def written(dev, kind, code, k, v, page=16):
    """A cache that holds the rows k, v [B, T, H, D], and the oracle's copy of it."""
    B, T, H, D = k.shape
    cache, mirror = make_cache(dev, kind, "HND" if kind == "paged" else "BHND", code, B, H, D, -(-T // 8) * 8 + 8, page=page)
    oracle.write(mirror, k, v, [0] * B, [T] * B)
    return cache, mirror


def upload(cache, mirror, lengths):
    for name in ("key", "value", "scales"):
        getattr(cache, name).view(torch.uint8).copy_(mirror[name].view(torch.uint8))
    cache.sequence_lengths.copy_(torch.tensor(lengths))


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("code", list(CODES))
@pytest.mark.parametrize("kind", ["contig", "paged"])
@pytest.mark.parametrize("dtype,dim,group,outlier,under", [
    ("fp16", 64, 4, 300.0, 0.05), ("fp16", 128, 12, 60000.0, 0.0), ("bf16", 128, 8, 5000.0, 0.002), ("bf16", 64, 16, 1e8, 0.0)])
def test_a_few_large_query_elements_leave_the_small_ones_exact(dev, kind, dtype, dim, group, outlier, under, code, kernel):
    """K is `under` times as large in the channels that meet the large elements, so that the others decide."""
    B, T, H = 2, 300, 2
    k, v = (torch.randn(B, T, H, dim, generator=torch.Generator().manual_seed(s)) for s in (1, 2))
    q = 2 * torch.randn(B, 1, H * group, dim, generator=torch.Generator().manual_seed(3))
    k[..., [5, dim - 1]] *= under
    q[..., 5], q[..., dim - 1] = outlier, -outlier
    q[:, :, 1] = 0.0                                                       # one head of the group has nothing but them
    q[:, :, 1, 5] = outlier
    q = q.to(TYPES[dtype])
    cache, mirror = written(dev, kind, code, k, v)
    upload(cache, mirror, [T, T - 33])
    plan = sa.QuantDecodePlan.build(q.to(dev), cache, kernel=kernel)
    check(plan.run(), q, mirror, [T, T - 33])
    assert plan.device_status() == 0


def shifted(dev, code, q, k, v, query, cache_k):
    """Query times 2^query, K rows times 2^cache_k (exactly, by their scale bytes): (device query, cache, query, mirror)."""
    cache, mirror = written(dev, "contig", code, k, v)
    bytes_ = mirror["scales"][..., 0].int() + cache_k
    mirror["scales"][..., 0] = torch.where(mirror["scales"][..., 0] == 0, 0, bytes_.clamp(27, 254)).to(torch.uint8)
    q = (q.float() * 2.0 ** query).to(q.dtype)
    upload(cache, mirror, [k.shape[1]] * k.shape[0])
    return q.to(dev), cache, q, mirror


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("code", list(CODES))
@pytest.mark.parametrize("dim,group", [(64, 5), (128, 16)])
@pytest.mark.parametrize("power", [-112, -100, -30, 60, 94])
def test_queries_and_keys_at_opposite_ends_of_the_range(dev, kernel, code, dim, group, power):
    """Scores of a few units from queries of 2^power and keys of 2^-power."""
    B, T, H = 1, 150, 2
    k, v = (torch.randn(B, T, H, dim, generator=torch.Generator().manual_seed(s)) for s in (1, 2))
    q = torch.randn(B, 1, H * group, dim, generator=torch.Generator().manual_seed(3)).bfloat16()
    q[q.abs() < 2.0 ** -10] = 0.0                                          # what is left is a normal number after the shift
    dq, cache, q, mirror = shifted(dev, code, q, k, v, power, -power)
    check(sa.QuantDecodePlan.build(dq, cache, kernel=kernel).run(), q, mirror, [T])


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("code", list(CODES))
@pytest.mark.parametrize("dim,group", [(64, 4), (128, 11)])
@pytest.mark.parametrize("power", [96, 112, 118])
def test_huge_keys_pick_their_token(dev, kernel, code, dim, group, power):
    """Keys up to 2^119 with ordinary queries: one token's score is twice the next, so its V row is the result."""
    B, T, H = 2, 200, 2
    size = 1.0 - 2.0 * (torch.arange(T) % 2)                               # the others: 1 and -1
    size[131] = 2.0
    k = size.view(1, T, 1, 1).expand(B, T, H, dim)
    v = torch.randn(B, T, H, dim, generator=torch.Generator().manual_seed(2))
    q = torch.randn(B, 1, H * group, dim, generator=torch.Generator().manual_seed(3)).abs().bfloat16()
    q[0, 0, 0] *= 2.0 ** -90                                               # next to small queries and one of zeros
    q[0, 0, 1] = 0.0
    dq, cache, q, mirror = shifted(dev, code, q, k, v, 0, power)
    got = sa.QuantDecodePlan.build(dq, cache, kernel=kernel).run().cpu().double().view(B, H, group, dim)
    value = oracle.decode(mirror["value"], mirror["scales"][..., 1])[:, :, :T]
    want = value[:, :, 131, None].expand(B, H, group, dim).clone()
    assert bool(((got - want).abs() <= 2.0 ** -8 * want.abs())[:, :, 2:].all())
    # the head of zeros weighs all tokens alike: the sum of T products in fp32, p rounded to fp16, the result to bf16
    mean, spread = value[0, 0].mean(0), value[0, 0].abs().mean(0)
    assert bool(((got[0, 0, 1] - mean).abs() <= 2.0 ** -8 * mean.abs() + spread * (2.0 ** -11 + T * 2.0 ** -23 + 2.0 ** -20) * 2).all())
    assert bool(((got[0, 0, 0] - want[0, 0, 0]).abs() <= 2.0 ** -8 * want[0, 0, 0].abs()).all())


def check_products(got, q, mirror, lengths):
    """As ``check``, and one term more: p times a row's V scale is rounded to fp16 in a unit of which the largest such product
    of the row is at least 2^6, so below 2^-14 the rounding is 2^-25: 2^-31 of the largest product for every token."""
    H, D = mirror["scales"].shape[1], q.shape[-1]
    for b, n in enumerate(lengths):
        k, v = (oracle.decode(mirror[name][b, :, :n], mirror["scales"][b, :, :n, i]) for i, name in enumerate(("key", "value")))
        x = q[b, 0].double().view(H, -1, D)
        p = torch.softmax(x @ k.mT / D ** 0.5, dim=-1)                     # [H, group, n]
        want, spread = p @ v, p @ v.abs()
        reach = (x.abs() @ k.abs().mT).amax(-1, keepdim=True) / D ** 0.5
        largest = (p * oracle.decode(torch.ones(H, n, 1), mirror["scales"][b, :, :n, 1])[:, None, :, 0]).amax(-1, keepdim=True)
        tol = tolerance(want, spread, reach, q.dtype, D, n) + n * 2.0 ** -31 * oracle.TOP[mirror["key"].dtype] * largest
        off = (got[b, 0].cpu().double().view_as(want) - want).abs() - tol
        assert bool((off <= 0).all()), (b, float(off.max()), float(want.abs().max()))


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("code", list(CODES))
@pytest.mark.parametrize("dim,group,splits", [(64, 4, None), (128, 3, 2), (64, 13, 1)])
@pytest.mark.parametrize("power", [20, 45, 100])
def test_large_value_rows_that_hardly_count_hide_no_others(dev, kernel, code, dim, group, splits, power):
    """A few V rows 2^power times the others, with scores far below: before, among and behind them."""
    B, T, H = 3, 330, 2
    k, v = (torch.randn(B, T, H, dim, generator=torch.Generator().manual_seed(s)) for s in (1, 2))
    q = torch.randn(B, 1, H * group, dim, generator=torch.Generator().manual_seed(3))
    q[..., 0] = 4.0 + torch.arange(H * group).float()                      # each head drops them by another amount
    k[..., 0] = 0.0
    cache, mirror = written(dev, "contig", code, k, v)
    big = [0, 1, 70, 200, T - 1]
    far = torch.zeros(B, T, H, dim)
    far[..., 0] = -power * 0.7 * dim ** 0.5 / 8.0                          # e^(0.7 power / 2) less for the first head, more for others
    far_mirror = written(dev, "contig", code, far, v)[1]
    for b, tokens in enumerate((big, big[1:3], big[3:])):
        for name in ("key", "scales"):
            view = mirror[name].view(torch.uint8)
            src = far_mirror[name].view(torch.uint8)
            if name == "key":
                view[b, :, tokens] = src[b, :, tokens]
            else:
                view[b, :, tokens, 0] = src[b, :, tokens, 0]
                view[b, :, tokens, 1] = (view[b, :, tokens, 1].int() + power).to(torch.uint8)
    q = q.to(torch.bfloat16)
    upload(cache, mirror, [T] * B)
    plan = sa.QuantDecodePlan.build(q.to(dev), cache, kernel=kernel, splits=splits)
    check_products(plan.run(), q, mirror, [T] * B)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("code", list(CODES))
@pytest.mark.parametrize("splits", [None, 1])
@pytest.mark.parametrize("case", ["rising scores, falling values", "falling scores, rising values", "steps", "anything"])
def test_scores_and_value_sizes_that_drift(dev, kernel, code, splits, case):
    B, T, H, group, dim = 2, 1700, 2, 6, 64
    g = torch.Generator().manual_seed(len(case))
    v = torch.randn(B, T, H, dim, generator=g)
    t = torch.arange(T).float()
    if case == "steps":                                                    # small steps, several a tile and one in many tiles
        size, power = torch.floor(t / 20), -torch.floor(t / 40) * 4
    elif case == "anything":
        size, power = 8 * torch.randn(T, generator=g), torch.randint(-90, 90, (T,), generator=g).float()
    else:
        sign = 1.0 if case.startswith("rising") else -1.0
        size, power = sign * t / 20, -sign * torch.floor(t / 18)
    k = torch.zeros(B, T, H, dim)
    k[..., 3] = size.view(1, T, 1)
    q = torch.randn(B, 1, H * group, dim, generator=g)
    q[..., 3] = torch.linspace(0.25, 12.0, H * group)                      # the score's natural logarithm a step of k
    cache, mirror = written(dev, "contig", code, k, v)
    e = mirror["scales"][:, :, :T, 1].int() + power.int().view(1, 1, T)
    mirror["scales"][:, :, :T, 1] = e.clamp(27, 250).to(torch.uint8)
    q = q.to(torch.bfloat16)
    upload(cache, mirror, [T, T - 700])
    plan = sa.QuantDecodePlan.build(q.to(dev), cache, kernel=kernel, splits=splits)
    out = plan.run().clone()
    check_products(out, q, mirror, [T, T - 700])
    assert torch.equal(plan.run(), out)
