"""8-bit KV cache restated with tensor operations in 64 bits, on the CPU (test infrastructure only).

The row format is the one documented in ``streamattn_b200/quant_cache.py``; nothing here imports it.
"""

from __future__ import annotations

import math

import torch

TOP = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def rotate(x, cos, sin):
    """x [B, T, heads, D]; cos/sin [B or 1, T, D].  Computed in float32, which is part of the definition."""
    x, cos, sin = x.float(), cos.float()[:, :, None], sin.float()[:, :, None]
    half = x.shape[-1] // 2
    turned = torch.cat((-x[..., half:], x[..., :half]), dim=-1)
    return x * cos + turned * sin


def encode(x, code):
    """x [..., D] -> (codes [..., D] of dtype `code`, scale bytes [...] uint8)."""
    x = x.double()
    top = x.abs().amax(dim=-1)
    bad = ~torch.isfinite(x).all(dim=-1)
    top = torch.where(bad, torch.zeros_like(top), top)
    mantissa, exponent = torch.frexp(top / TOP[code])            # top / TOP = mantissa * 2^exponent, mantissa in [0.5, 1)
    e = exponent - (mantissa == 0.5).to(exponent.dtype)          # smallest power of two not below it
    e = torch.where(top == 0, torch.full_like(e, -1000), e).clamp_min(-100) + 127
    y = x / torch.exp2((e - 127).double()).unsqueeze(-1)
    y = torch.where(bad.unsqueeze(-1), torch.zeros_like(y), y)
    codes = torch.round(y).to(torch.int8) if code == torch.int8 else y.float().to(code)
    return codes, torch.where(bad, torch.full_like(e, 255), e).to(torch.uint8)


def decode(codes, e):
    """The values of codes [..., D] with scale bytes [...], in float64 (NaN where the byte is 255, 0 where it is 0)."""
    scale = torch.exp2(e.double() - 127)
    scale = torch.where(e == 255, torch.full_like(scale, float("nan")), scale)
    scale = torch.where(e == 0, torch.zeros_like(scale), scale)
    return codes.double() * scale.unsqueeze(-1)


def place(cache, b, pos):
    """(outer, slot) of token `pos` of row b, or None where its page is out of range.  cache: see `write`."""
    if cache["table"] is None:
        return b, pos
    page = int(cache["table"][b, pos // cache["page"]])
    return (page, pos % cache["page"]) if 0 <= page < cache["scales"].shape[0] else None


def _cell(cache, name, spot, h):
    outer, slot = spot
    t = cache[name]
    return t[outer, h, slot] if cache["heads_first"] else t[outer, slot, h]


def write(cache, k, v, positions, counts):
    """cache: dict of key/value codes, scales, table (or None), page, capacity, heads_first; k/v [B, T, H, D] (rotated)."""
    code = cache["key"].dtype
    coded = {"key": encode(k, code), "value": encode(v, code)}
    for b in range(k.shape[0]):
        start, n = positions[b], counts[b]
        if start < 0 or start + n > cache["capacity"]:
            continue
        for t in range(n):
            spot = place(cache, b, start + t)
            if spot is None:
                continue
            for h in range(k.shape[2]):
                for i, name in enumerate(("key", "value")):
                    _cell(cache, name, spot, h).view(torch.uint8).copy_(coded[name][0][b, t, h].view(torch.uint8))
                    cache["scales"][spot[0], h, spot[1], i] = coded[name][1][b, t, h]


def rows(cache, b, start, count):
    """(K, V, held) of tokens [start, start + count) of row b: [count, H, D] float64, held [count] bool."""
    H, D = cache["scales"].shape[1], cache["key"].shape[-1]
    k, v = torch.zeros(count, H, D, dtype=torch.float64), torch.zeros(count, H, D, dtype=torch.float64)
    held = torch.zeros(count, dtype=torch.bool)
    for t in range(count):
        spot = place(cache, b, start + t) if 0 <= start + t < cache["capacity"] else None
        if spot is None:
            continue
        held[t] = True
        for h in range(H):
            for i, (out, name) in enumerate(((k, "key"), (v, "value"))):
                out[t, h] = decode(_cell(cache, name, spot, h), cache["scales"][spot[0], h, spot[1], i])
    return k, v, held


def attend(q, cache, lengths):
    """q [B, 1, Hq, D] -> (out float64 like q, spread): spread = sum_t p_t |v_t|, the size of what P's rounding touches."""
    B, _, Hq, D = q.shape
    out = torch.zeros(B, Hq, D, dtype=torch.float64)
    spread = torch.zeros_like(out)
    reach = torch.zeros(B, Hq, dtype=torch.float64)   # largest sum_d |q_d k_d| / sqrt(D) of a head
    for b in range(B):
        k, v, held = rows(cache, b, 0, min(int(lengths[b]), cache["capacity"]))
        k, v = k[held], v[held]
        if not len(k):
            continue
        group = Hq // k.shape[1]
        for h in range(Hq):
            kh, vh, x = k[:, h // group], v[:, h // group], q[b, 0, h].double()
            p = torch.softmax(kh @ x / math.sqrt(D), dim=0)
            out[b, h], spread[b, h] = p @ vh, p @ vh.abs()
            reach[b, h] = (kh.abs() @ x.abs()).max() / math.sqrt(D)
    return out.view(B, 1, Hq, D), spread.view(B, 1, Hq, D), reach.view(B, 1, Hq, 1)
