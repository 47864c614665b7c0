"""One-token attention over 8-bit KV caches where the inputs span a wide range, against the 64-bit oracle.

The bound is the one of ``tests/test_gpu_quant_decode.py``.  It has no term for the query: the kernels use it as it is
(fp16 after a power of two, in which the elements of these queries are exact).
"""

import pytest
import torch

import streamattn_b200 as sa
from oracle import quant_kv as oracle
from tests.test_gpu_quant_decode import KERNELS, check
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
