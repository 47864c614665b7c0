"""Cases of the 8-bit KV cache operators: writing rows into the cache, reading them back, and one-token
attention over it, for contiguous and paged caches.

A cache row (one token of one KV head, D values of K or V) is held as D codes of 8 bits, float8 e4m3 or
int8, and one power-of-two scale 2^(e - 127) held as the byte e:

    e       the smallest exponent with  max|x| <= top * 2^(e - 127),  top = 448 (e4m3) or 127 (int8), e >= 27
    code_d  x_d / 2^(e - 127) rounded to the code's type, halves to the even neighbour
    x_d'    code_d * 2^(e - 127)

Scales lie head-major whatever the codes' layout is, the K and V byte of a token side by side: [B, Hkv, N, 2]
or [pages, Hkv, page_size, 2].

    write    K (rotated by cos/sin where they are given) and V of T new tokens a row, at the row's position;
             the query of the same tokens rotated beside them
    read     the rows' tokens [start, start + count) as K and V of a dtype, padding left as it was
    decode   softmax(q K'^T / sqrt(D)) V' of one query token a row, over the row's tokens
"""

import math

import torch

own = False

_TOP = {"e4m3": 448.0, "int8": 127.0}
_CODE = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
_TYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_MIN_EXP = 27   # 2^-100: rows smaller than that are held at this scale


def listed():
    return [
        # -- write ---------------------------------------------------------------------------------------
        # the cache update of one decode step over the ragged paged cache of the repository's benchmark
        dict(name="write_step_paged", op="write", code="e4m3", dtype="bf16", batch=8, q_heads=16, kv_heads=2, dim=64,
             tokens=1, capacity=65536, page=16, layout="HND", rope=True, ragged=True),
        # a chunk of prompts going into the head-major contiguous cache of the same benchmark
        dict(name="write_chunk_contig", op="write", code="e4m3", dtype="bf16", batch=8, q_heads=16, kv_heads=2, dim=64,
             tokens=4096, capacity=65536, page=0, layout="BHND", rope=True, ragged=False),
        # a padded batch of prompts of different lengths into large token-major pages, no rotation (done before)
        dict(name="write_prompts_paged", op="write", code="int8", dtype="fp16", batch=13, q_heads=0, kv_heads=8, dim=128,
             tokens=8190, capacity=16384, page=64, layout="NHD", rope=False, ragged=True),
        # -- read ----------------------------------------------------------------------------------------
        # a short history for a model's own dense attention; odd length
        dict(name="read_short_paged", op="read", code="e4m3", dtype="bf16", batch=1, q_heads=0, kv_heads=8, dim=128,
             tokens=1003, capacity=2048, page=16, layout="HND", rope=False, ragged=False),
        # the whole ragged paged cache of the benchmark gathered into contiguous rows
        dict(name="read_ragged_paged", op="read", code="e4m3", dtype="bf16", batch=8, q_heads=0, kv_heads=2, dim=64,
             tokens=65536, capacity=65536, page=16, layout="HND", rope=False, ragged=True),
        # a token-major contiguous cache, int8, handed to half-precision code
        dict(name="read_contig", op="read", code="int8", dtype="fp16", batch=3, q_heads=0, kv_heads=8, dim=128,
             tokens=32768, capacity=32768, page=0, layout="BNHD", rope=False, ragged=False),
        # -- decode --------------------------------------------------------------------------------------
        # the smallest shape of the repository's configurations: latency counts
        dict(name="decode_short_contig", op="decode", code="e4m3", dtype="bf16", batch=2, q_heads=16, kv_heads=2, dim=64,
             tokens=4096, capacity=4096, page=0, layout="BHND", rope=False, ragged=False),
        # the benchmark's long contiguous cache
        dict(name="decode_long_contig", op="decode", code="e4m3", dtype="bf16", batch=8, q_heads=16, kv_heads=2, dim=64,
             tokens=65536, capacity=65536, page=0, layout="BHND", rope=False, ragged=False),
        # its paged one: ragged rows of 16K to 64K tokens in pages of 16
        dict(name="decode_ragged_paged", op="decode", code="e4m3", dtype="bf16", batch=8, q_heads=16, kv_heads=2, dim=64,
             tokens=65536, capacity=65536, page=16, layout="HND", rope=False, ragged=True),
        # serving: many rows of very different lengths, an odd number of them, token-major pages of 64
        dict(name="decode_batch_paged", op="decode", code="int8", dtype="fp16", batch=61, q_heads=32, kv_heads=8, dim=128,
             tokens=8191, capacity=8192, page=64, layout="NHD", rope=False, ragged=True),
        # one very long row, the repository's one-million-token configuration
        dict(name="decode_million", op="decode", code="int8", dtype="bf16", batch=1, q_heads=32, kv_heads=8, dim=128,
             tokens=1048576, capacity=1048576, page=0, layout="BHND", rope=False, ragged=False),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["write", "read", "decode", "decode"])
    dim = rng.choice([64, 128] if op == "decode" else [64, 128, 64, 128, 80, 96, 256])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    group = rng.choice([1, 2, 4, 7, 8, 16])
    rope = op == "write" and rng.random() < 0.5
    tokens = _log(rng, 1, {"write": 8192, "read": 32768, "decode": 131072}[op])
    # rows: at most 2^28 codes of K in all, a quarter of the largest listed case
    most = max(1, min(64, (1 << 28) // (tokens * kv_heads * dim)))
    batch = _log(rng, 1, most)
    page = rng.choice([0, 0, 8, 16, 32, 64, 128])
    layout = rng.choice(["NHD", "HND"] if page else ["BNHD", "BHND"])
    room = tokens + (_log(rng, 1, 4096) if op == "write" else rng.choice([0, 5, 64]))
    unit = page or 8
    return dict(op=op, code=rng.choice(["e4m3", "int8"]), dtype=rng.choice(["bf16", "fp16"]), batch=batch,
                q_heads=kv_heads * group if op == "decode" or rope else 0, kv_heads=kv_heads, dim=dim, tokens=tokens,
                capacity=-(-room // unit) * unit, page=page, layout=layout, rope=rope, ragged=rng.random() < 0.6)


# -- the rows' codes and scales, in 32 or 64 bits ------------------------------------------------------------

def _encode(x, code):
    """x [..., D], float32 or float64 -> (codes [..., D] as values of x's dtype, e [...] int32)."""
    mantissa, exponent = torch.frexp(x.abs().amax(dim=-1))           # amax = mantissa * 2^exponent, mantissa in [0.5, 1)
    top_mantissa, top_exponent = math.frexp(_TOP[code])
    e = exponent - top_exponent + (mantissa > top_mantissa).to(exponent.dtype) + 127
    e = e.clamp_min(_MIN_EXP)
    y = x * torch.exp2((127 - e).to(x.dtype)).unsqueeze(-1)           # exact: a power of two
    y = torch.round(y) if code == "int8" else y.to(torch.float8_e4m3fn).to(x.dtype)
    return y, e


def _values(codes, e, dtype):
    """codes [..., D], e [...] (bytes) -> the values they stand for."""
    return codes.to(dtype) * torch.exp2(e.to(dtype) - 127).unsqueeze(-1)


def _bytes(codes):
    return codes.view(torch.uint8)


# -- inputs --------------------------------------------------------------------------------------------------

def _rows_like(shape, generator, device):
    """K or V rows as a model makes them: normal values, rows of different sizes."""
    x = torch.randn(shape, generator=generator, device=device)
    return x * torch.exp(0.5 * torch.randn(shape[:-1] + (1,), generator=generator, device=device))


def prepare(case, seed):
    device = torch.device("cuda")
    g = torch.Generator(device=device).manual_seed(seed)
    c, dtype = case, _TYPE[case["dtype"]]
    B, H, D, N, page, T = c["batch"], c["kv_heads"], c["dim"], c["capacity"], c["page"], c["tokens"]
    state = {"case": case}
    # where the tokens lie
    if page:
        per_row = N // page
        shape = (B * per_row, page, H, D) if c["layout"] == "NHD" else (B * per_row, H, page, D)
        scale_shape = (B * per_row, H, page, 2)
        state["table"] = torch.randperm(B * per_row, generator=g, device=device).to(torch.int32).view(B, per_row)
    else:
        shape = (B, N, H, D) if c["layout"] == "BNHD" else (B, H, N, D)
        scale_shape = (B, H, N, 2)
    # how many tokens each row has, from a quarter of the longest up (the longest row is there)
    counts = torch.full((B,), T, dtype=torch.int64, device=device)
    if c["ragged"]:
        low = max(1, T // 4)
        counts = torch.randint(low, T + 1, (B,), generator=g, device=device)
        counts[0] = T
    if c["op"] == "write":
        key = torch.zeros(shape, dtype=torch.uint8, device=device).view(_CODE[c["code"]])
        state |= {"key": key, "value": torch.zeros_like(_bytes(key)).view(key.dtype),
                  "scales": torch.full(scale_shape, 127, dtype=torch.uint8, device=device)}
        state["new_key"] = _rows_like((B, T, H, D), g, device).to(dtype)
        state["new_value"] = _rows_like((B, T, H, D), g, device).to(dtype)
        room = N - T
        state["starts"] = (torch.rand(B, generator=g, device=device) * (room + 1)).long().clamp_max(room).to(torch.int32)
        state["held"] = state["starts"]
        state["lengths"] = torch.zeros(B, dtype=torch.int32, device=device)
        if c["rope"]:
            state["query"] = torch.randn(B, T, c["q_heads"], D, generator=g, device=device).to(dtype)
            state["query_out"] = torch.empty_like(state["query"])
            at = state["starts"].double()[:, None] + torch.arange(T, device=device)
            angle = at[..., None] * 10000.0 ** (-torch.arange(D // 2, dtype=torch.float64, device=device) / (D // 2))
            angle = torch.cat((angle, angle), dim=-1)
            state["cos"], state["sin"] = angle.cos().to(dtype), angle.sin().to(dtype)
    else:
        for name, at in (("key", 0), ("value", 1)):
            codes, e = _encode(_rows_like(shape, g, device), c["code"])
            state[name] = codes.to(_CODE[c["code"]])
            if "scales" not in state:
                state["scales"] = torch.empty(scale_shape, dtype=torch.uint8, device=device)
            state["scales"][..., at] = e if c["layout"] in ("HND", "BHND") else e.transpose(1, 2)
        if c["op"] == "read":
            state["starts"] = ((T - counts) // 2).to(torch.int32)     # any part of a row
            state["held"] = torch.full((B,), T, dtype=torch.int32, device=device)
            state["out_key"] = torch.zeros(B, T, H, D, dtype=dtype, device=device)
            state["out_value"] = torch.zeros_like(state["out_key"])
        else:
            state["query"] = torch.randn(B, 1, c["q_heads"], D, generator=g, device=device).to(dtype)
            state["output"] = torch.empty_like(state["query"])
    state["counts"] = counts.to(torch.int32)
    state.setdefault("held", state["counts"])                         # tokens that the rows hold before the call
    if own:
        _bind(state)
    return state


def _bind(state):
    """The cache and the plan that a program keeps."""
    import streamattn_b200 as sa

    c = state["case"]
    if c["page"]:
        cache = sa.QuantPagedKVCache(key=state["key"], value=state["value"], scales=state["scales"], page_table=state["table"],
                                     sequence_lengths=state["held"], layout=c["layout"])
    else:
        whole = c["op"] == "decode" and not c["ragged"] and c["tokens"] == c["capacity"]    # rows that fill the cache
        cache = sa.QuantKVCache(key=state["key"], value=state["value"], scales=state["scales"],
                                sequence_lengths=None if whole else state["held"], layout=c["layout"])
    if c["op"] == "write":
        state["plan"] = sa.QuantizeKVPlan.build(
            cache, state["new_key"], state["new_value"], positions=state["starts"],
            counts=state["counts"] if c["ragged"] else None, cos=state.get("cos"), sin=state.get("sin"),
            query=state.get("query"), query_out=state.get("query_out"), lengths_out=state["lengths"])
    elif c["op"] == "read":
        state["plan"] = sa.DequantizeKVPlan.build(cache, state["out_key"], state["out_value"], starts=state["starts"],
                                                  counts=state["counts"] if c["ragged"] else None)
    else:
        state["plan"] = sa.QuantDecodePlan.build(state["query"], cache, output=state["output"])


# -- one pass ------------------------------------------------------------------------------------------------

def run(state):
    if own:
        state["plan"].run()
    else:
        {"write": _write, "read": _read, "decode": _decode}[state["case"]["op"]](state)
    return _outputs(state)


def _outputs(state):
    op = state["case"]["op"]
    if op == "write":
        return {k: state[k] for k in ("key", "value", "scales", "lengths", "query_out") if k in state}
    if op == "read":
        return {"key": state["out_key"], "value": state["out_value"]}
    return state["output"]


def _rotate(x, cos, sin):
    """x [B, T, heads, D] turned by the angles of [B, T, D]: the halves of a row are the pairs' parts."""
    half = x.shape[-1] // 2
    turned = torch.cat((-x[..., half:], x[..., :half]), dim=-1)
    return x * cos[:, :, None] + turned * sin[:, :, None]


def _new_rows(state, dtype):
    k, v = state["new_key"].to(dtype), state["new_value"].to(dtype)
    if state["case"]["rope"]:
        k = _rotate(k, state["cos"].to(dtype), state["sin"].to(dtype))
    return k, v


def _places(state):
    """(batch rows, new tokens, positions) of the tokens that are written."""
    T = state["case"]["tokens"]
    row, t = (torch.arange(T, device="cuda")[None] < state["counts"][:, None]).nonzero(as_tuple=True)
    return row, t, state["starts"].long()[row] + t


def _write(state):
    c, page = state["case"], state["case"]["page"]
    row, t, at = _places(state)
    for index, (x, name) in enumerate(zip(_new_rows(state, torch.float32), ("key", "value"))):
        codes, e = _encode(x, c["code"])
        codes, e = _bytes(codes.to(_CODE[c["code"]]))[row, t], e[row, t].to(torch.uint8)     # [tokens, H, D], [tokens, H]
        to, outer, inner = _bytes(state[name]), row, at
        if page:
            outer, inner = state["table"].long()[row, at // page], at % page
        if c["layout"] in ("NHD", "BNHD"):
            to[outer, inner] = codes
        else:
            to[outer, :, inner] = codes
        state["scales"][outer, :, inner, index] = e
    state["lengths"].copy_(state["starts"] + state["counts"])
    if c["rope"]:
        q = _rotate(state["query"].float(), state["cos"].float(), state["sin"].float())
        state["query_out"].copy_(q)


def _tokens(state, name, at, dtype):
    """The values of `name` as [B, H, N, D], N the row's capacity."""
    c, codes, e = state["case"], state[name], state["scales"][..., at]
    if c["layout"] in ("NHD", "BNHD"):
        codes = codes.transpose(1, 2)
    if c["page"]:
        table = state["table"].long()
        codes = _bytes(codes)[table].view(codes.dtype).transpose(1, 2).flatten(2, 3)
        e = e[table].transpose(1, 2).flatten(2, 3)
    return _values(codes, e, dtype)


def _read_rows(state, dtype):
    """K and V of the tokens that are read, [B, T, H, D], and which of them a row has."""
    T = state["case"]["tokens"]
    t = torch.arange(T, device="cuda")[None]
    at = (state["starts"].long()[:, None] + t).clamp_max(state["case"]["capacity"] - 1)
    has = (t < state["counts"][:, None])[..., None, None]
    row = torch.arange(at.shape[0], device="cuda")[:, None]
    return [_tokens(state, name, i, dtype).transpose(1, 2)[row, at] for i, name in enumerate(("key", "value"))], has


def _read(state):
    rows, has = _read_rows(state, torch.float32)
    for x, name in zip(rows, ("out_key", "out_value")):
        state[name].copy_(torch.where(has, x, state[name].float()))


def _attend(state, dtype):
    c = state["case"]
    k, v = _tokens(state, "key", 0, dtype), _tokens(state, "value", 1, dtype)
    B, H, N, D = k.shape
    q = state["query"].to(dtype).view(B, H, c["q_heads"] // H, D)
    scores = (q @ k.transpose(2, 3)) / math.sqrt(D)
    has = torch.arange(N, device="cuda")[None] < state["counts"][:, None]
    scores = scores.masked_fill(~has[:, None, None], -math.inf)
    p = torch.exp(scores - scores.amax(dim=-1, keepdim=True))
    return ((p @ v) / p.sum(dim=-1, keepdim=True)).view(B, 1, c["q_heads"], D)


def _decode(state):
    state["output"].copy_(_attend(state, torch.float32))


# -- what a pass needs, and its answer in 64 bits --------------------------------------------------------------

def work(case):
    c, size = case, {"bf16": 2, "fp16": 2, "fp32": 4}[case["dtype"]]
    # ragged rows hold between a quarter and all of the longest: five eighths of it on average, and one row all
    mean = ((c["tokens"] + max(1, c["tokens"] // 4)) / 2 * (c["batch"] - 1) + c["tokens"]) / c["batch"] if c["ragged"] else c["tokens"]
    tokens = mean * c["batch"]
    rows = 2 * tokens * c["kv_heads"]                       # K and V rows
    cache = rows * (c["dim"] + 1) + (4 * tokens / c["page"] if c["page"] else 0)
    if c["op"] == "write":
        queries = 2 * c["batch"] * c["tokens"] * c["q_heads"] * c["dim"] * size if c["rope"] else 0
        angles = 2 * c["batch"] * c["tokens"] * c["dim"] * size if c["rope"] else 0
        return {"bytes": cache + rows * c["dim"] * size + queries + angles, "flops": 3 * rows * c["dim"]}
    if c["op"] == "read":
        return {"bytes": cache + rows * c["dim"] * size, "flops": rows * c["dim"]}
    io = 2 * c["batch"] * c["q_heads"] * c["dim"] * size
    return {"bytes": cache + io, "flops": 4 * tokens * c["q_heads"] * c["dim"]}


def exact(case, seed):
    """In 64 bits, from the definition at the head of this file (whole numbers are compared as they are)."""
    if case["op"] == "write" and case["code"] == "int8" and not case["rope"]:
        return None
    state = prepare(case, seed)
    wide = torch.float64
    if case["op"] == "read":
        rows, has = _exact_rows(state), (torch.arange(case["tokens"], device="cuda")[None] < state["counts"][:, None])
        has = has[..., None, None]
        return {name: torch.where(has, x, torch.zeros_like(x)) for name, x in zip(("key", "value"), rows)}
    if case["op"] == "decode":
        key, value = _exact_cache(state, "key", 0), _exact_cache(state, "value", 1)    # [B, N, H, D]
        group = case["q_heads"] // case["kv_heads"]
        q = state["query"].to(wide)[:, 0].unflatten(1, (case["kv_heads"], group))
        logits = torch.einsum("bhgd,bnhd->bhgn", q, key) * case["dim"] ** -0.5
        out = torch.arange(case["capacity"], device="cuda") >= state["counts"][:, None]
        weights = torch.softmax(logits.masked_fill(out[:, None, None], -math.inf), dim=-1)
        return torch.einsum("bhgn,bnhd->bhgd", weights, value).flatten(1, 2)[:, None]
    result = {"scales": None, "lengths": None}
    B, T, half = case["batch"], case["tokens"], case["dim"] // 2

    def turn(x):
        if not case["rope"]:
            return x
        cos, sin = state["cos"].to(wide)[:, :, None], state["sin"].to(wide)[:, :, None]
        a, b = x[..., :half], x[..., half:]
        return torch.cat((a * cos[..., :half] - b * sin[..., :half], b * cos[..., half:] + a * sin[..., half:]), dim=-1)

    here = torch.arange(T, device="cuda")[None] < state["counts"][:, None]
    where = (state["starts"][:, None] + torch.arange(T, device="cuda")).long()
    row = torch.arange(B, device="cuda")[:, None].expand(B, T)
    for name, x in (("key", turn(state["new_key"].to(wide))), ("value", state["new_value"].to(wide))):
        if case["code"] == "int8":
            result[name] = None
            continue
        # the grid of e4m3 below 448: steps of 2^(floor(log2 |y|) - 3), of 2^-9 below 2^-6
        top = x.abs().amax(dim=-1, keepdim=True).clamp_min(448.0 * 2.0 ** -100)
        m, power = torch.frexp(top / 448.0)                            # m in [0.5, 1): the power of two at or above it
        y = x / torch.exp2((power - (m == 0.5).int()).to(wide))
        step = torch.exp2((torch.frexp(y.abs().clamp_min(2.0 ** -6))[1] - 4).to(wide))
        y = torch.round(y / step) * step
        held = torch.zeros(state[name].shape, dtype=wide, device="cuda")
        outer, inner = row[here], where[here]
        if case["page"]:
            outer, inner = state["table"].long()[outer, inner // case["page"]], inner % case["page"]
        view = held if case["layout"] in ("NHD", "BNHD") else held.transpose(1, 2)
        view[outer, inner] = y[here]
        result[name] = held
    if case["rope"]:
        result["query_out"] = turn(state["query"].to(wide))
    return result


def _exact_cache(state, name, at):
    """[B, N, H, D] in 64 bits."""
    c, codes, e = state["case"], state[name], state["scales"][..., at].to(torch.int64)
    if c["layout"] in ("HND", "BHND"):
        codes = codes.transpose(1, 2)
    e = e.transpose(1, 2)
    if c["page"]:
        index = state["table"].long().flatten()
        codes = _bytes(codes).index_select(0, index).view(codes.dtype).reshape(c["batch"], -1, c["kv_heads"], c["dim"])
        e = e.index_select(0, index).reshape(c["batch"], -1, c["kv_heads"])
    return codes.to(torch.float64) * torch.exp2((e - 127).to(torch.float64))[..., None]


def _exact_rows(state):
    at = state["starts"].long()[:, None, None, None] + torch.arange(state["case"]["tokens"], device="cuda")[None, :, None, None]
    at = at.clamp_max(state["case"]["capacity"] - 1).expand(-1, -1, state["case"]["kv_heads"], state["case"]["dim"])
    return [torch.gather(_exact_cache(state, name, i), 1, at) for i, name in enumerate(("key", "value"))]
