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
    codes = [c.key.view(torch.uint8) for c in (first, second)]
    changed = (codes[0] != codes[1]).any(-1)[0].cpu() | (first.scales != second.scales).any(-1)[0].cpu()     # [H, T]
    if code == "int8":
        assert not bool(changed.any())
    else:
        largest = first.key.float().abs().amax(-1)[0].cpu()
        assert torch.equal(changed, largest == 224.0)
        assert [bool(x) for x in changed[0, :len(tops)]] == [False, True, True, False, False, True]
        at = changed.nonzero()[0].tolist()
        one, two = (c.key.float()[0, at[0], at[1]].cpu() for c in (first, second))
        assert torch.equal(two, 2 * one) and int(second.scales[0, at[0], at[1], 0]) == int(first.scales[0, at[0], at[1], 0]) - 1
    mirror = dict(key=first.key.cpu(), value=first.value.cpu(), scales=first.scales.cpu(), table=None, page=0, capacity=T, heads_first=True)
    want, _, _ = oracle.rows(mirror, 0, 0, T)
    assert torch.equal(k[0].cpu().double(), want)
