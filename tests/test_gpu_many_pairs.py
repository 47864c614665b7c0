"""The generic decode kernel with more (row, query head) pairs than a grid has rows: 8-bit, fp32 and 16-bit caches."""

import pytest
import torch

import streamattn_b200 as sa
from tests.test_gpu_quant_kv import dev  # noqa: F401

pytestmark = pytest.mark.gpu
B, H, G, D, N = 520, 4, 32, 16, 8                                          # 66560 pairs, two slabs of the grid


@pytest.fixture(scope="module")
def operands(dev):  # noqa: F811
    g = torch.Generator(dev).manual_seed(1)
    k, v = (torch.randn(B, H, N, D, generator=g, device=dev) for _ in range(2))
    q = torch.randn(B, 1, H * G, D, generator=g, device=dev)
    lengths = torch.randint(0, N + 1, (B,), generator=torch.Generator().manual_seed(2)).to(dev)
    return q, k, v, lengths


def attend(q, k, v, lengths):
    """(result, sum of p |v|) in 64 bits."""
    qh = q[:, 0].double().view(B, H, G, D)
    off = torch.arange(N, device=q.device) >= lengths[:, None, None, None]
    p = torch.softmax((qh @ k.double().mT / D ** 0.5).masked_fill(off, -1e300), -1).masked_fill(off, 0.0)
    return ((p @ v.double()).view(B, 1, H * G, D), (p @ v.double().abs()).view(B, 1, H * G, D))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("cached", ["as the query", torch.float8_e4m3fn, torch.int8])
def test_every_pair_is_computed(dev, operands, dtype, cached):  # noqa: F811
    q, k, v, lengths = operands
    q, k, v = q.to(dtype), k.to(dtype), v.to(dtype)
    if cached == "as the query":
        plan = sa.ExactDecodePlan.build(q, k, v, seq_lens=lengths, kv_layout="BHND")
    else:
        cache = sa.QuantKVCache.empty(B, H, N, D, dtype=cached, device=dev)
        sa.quantize_kv(cache, k, v, counts=lengths, new_layout="BHND")
        k, v = (t.float() for t in sa.dequantize_kv(cache, dtype=torch.float32, out_layout="BHND"))
        plan = sa.QuantDecodePlan.build(q, cache)
    assert plan.kernel_name != "sm100_tma_mma_stream"
    plan.output.fill_(7.0)
    out = plan.run().double()
    want, spread = attend(q, k, v, lengths)
    # half a step of the output; products, exponentials and sums of 8 tokens x 16 elements in fp32
    tol = torch.finfo(dtype).eps / 2 * want.abs() + spread * 2.0 ** -17
    assert bool(((out - want).abs() <= tol).all())
