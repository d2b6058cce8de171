"""The operators on smaller caches that this framework is timed on, at the sizes its users meet.

A restored prompt's cache is most of what a decode step reads and of what the memory holds.  Two
ways make it smaller: its rows are held in 4 bits (blocks of 32 channels with a power of two as
their scale), or the tokens that little attention falls on are evicted.  For the first, tokens
are appended to such a cache, read back from it and attended to in it; for the second, the
weights that queries give each cached token are added up, and the tokens with the largest
sums, and the newest, are moved to blocks of their own.  One case is one layer's call.  Head
counts, head sizes, block sizes, both cache orders and prefix lengths are those of the
repository's benchmark and tests; lengths of requests are ragged.

`run` computes an operator in elementary torch operations while `own` is false, and calls the
framework while it is true.
"""
from __future__ import annotations

import math
import random

import torch

own = False

_TYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16,
          "float8_e4m3fn": torch.float8_e4m3fn, "mxfp4": torch.uint8}
_EPS = 1e-6
_SPARE_BLOCKS = 5  # blocks of the cache that no request of the case has
_GROUP = 32  # channels with one scale
# powers of two that scales are limited to: float16 holds every product exactly
_LEAST_SCALE, _MOST_SCALE = -23, 13
# of a drawn case; the largest listed ones of the operator have more
_MOST_BYTES = {"append": 60_000_000, "read": 100_000_000, "attend": 250_000_000,
               "weigh": 120_000_000, "evict": 120_000_000}
_MOST_FLOPS = {"attend": 200_000_000_000, "weigh": 100_000_000_000}


def listed() -> list[dict]:
    wide = {"query_heads": 32, "heads": 8, "head_dim": 128, "block_size": 16,
            "dtype": "bfloat16", "cache": "kv_first"}
    append = {"op": "append", **wide, "cache_dtype": "mxfp4", "padding": 0, "norm": False,
              "rotary_dim": 128, "interleaved": False, "table": 40960}
    read = {"op": "read", **wide, "cache_dtype": "mxfp4", "padding": 0}
    attend = {"op": "attend", **wide, "cache_dtype": "mxfp4", "prefix": 0, "query_tokens": 1,
              "lengths_seed": 1}
    weigh = {"op": "weigh", **wide, "cache_dtype": "bfloat16", "query_tokens": 1,
             "lengths_seed": 1}
    evict = {"op": "evict", **wide, "cache_dtype": "bfloat16", "lengths_seed": 1}
    return [
        # A decode step of 64 places, 3 of them unused, into a 4-bit cache, and the rows as the
        # cache holds them; the 28 / 4 heads of the benchmark's ragged batch.
        {"name": "append_step", **append, "query_heads": 28, "heads": 4, "tokens": 64,
         "padding": 3, "cache": "blocks_first"},
        # A prompt's tokens after its prefix, queries and keys normalised per head; the rows as
        # held are what the prompt's own attention then sees.
        {"name": "append_prompt", **append, "tokens": 8192, "norm": True},
        # The benchmark's ragged request out of a 4-bit cache, to be saved or to be attended to by
        # a long prompt.
        {"name": "read_request", **read, "tokens": 32753},
        # A short request of an fp8 cache, half precision, heads of 64.
        {"name": "read_short", **read, "query_heads": 12, "heads": 12, "head_dim": 64,
         "dtype": "float16", "cache_dtype": "float8_e4m3fn", "tokens": 333, "padding": 5},
        # One request just after its restore: few rows, so latency counts.
        {"name": "attend_one", **attend, "requests": 1, "least": 1029, "most": 1029},
        # A decode step of requests that share nothing, the 4-bit cache's main use.
        {"name": "attend_batch", **attend, "requests": 32, "least": 1000, "most": 16384,
         "lengths_seed": 2},
        # A decode step of a full batch over the benchmark's 32768-token prefix.
        {"name": "attend_prefix", **attend, "requests": 64, "prefix": 32768, "least": 17,
         "most": 1024, "lengths_seed": 3, "cache": "blocks_first"},
        # Drafted tokens looked over in one pass: five queries a request, half precision.
        {"name": "attend_draft", **attend, "query_heads": 12, "heads": 12, "head_dim": 64,
         "dtype": "float16", "requests": 24, "prefix": 2000, "least": 5, "most": 600,
         "query_tokens": 5, "lengths_seed": 5},
        # A decode step's weights over the tokens that 16 requests have left.
        {"name": "weigh_step", **weigh, "requests": 16, "least": 2048, "most": 8192,
         "lengths_seed": 6},
        # Two prompts' weights from all of their own queries; the 28 / 4 heads, a 4-bit cache.
        {"name": "weigh_prompt", **weigh, "query_heads": 28, "heads": 4, "requests": 2,
         "cache_dtype": "mxfp4", "least": 3500, "most": 4096, "query_tokens": 4096,
         "lengths_seed": 7},
        # A batch goes back to its budget after some tens of tokens, fp8.
        {"name": "evict_step", **evict, "requests": 32, "least": 1024, "most": 1096,
         "keep": 1024, "recent": 128, "cache_dtype": "float8_e4m3fn", "lengths_seed": 8,
         "cache": "blocks_first"},
        # Four restored prompts to an eighth of the longest.
        {"name": "evict_prompt", **evict, "requests": 4, "least": 20000, "most": 32768,
         "keep": 4096, "recent": 512, "lengths_seed": 9},
    ]


def _spread(rng, least: int, most: int) -> int:
    """A whole number from [least, most], spread over its logarithm."""
    return max(least, min(most, int(round(math.exp(rng.uniform(math.log(least),
                                                               math.log(most)))))))


def draw(rng) -> dict:
    heads, group = rng.choice([(8, 4), (8, 1), (4, 7), (1, 8), (2, 4), (12, 1), (8, 5), (1, 16)])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16"])
    op = rng.choice(["append", "read", "attend", "attend", "attend", "weigh", "weigh", "evict",
                     "evict"])
    case = {"op": op, "query_heads": heads * group, "heads": heads,
            "head_dim": rng.choice([64, 128, 128, 128, 80, 256]),
            "block_size": rng.choice([16, 16, 32, 24]), "dtype": dtype,
            "cache_dtype": "mxfp4" if op in ("append", "attend") else
            rng.choice([dtype, "float8_e4m3fn", "mxfp4"]),
            "cache": rng.choice(["kv_first", "blocks_first"])}
    if op in ("append", "read"):
        tokens = _spread(rng, 1, 8192 if op == "append" else 32768)
        case.update(tokens=tokens, padding=rng.randint(0, tokens // 8))
        if op == "append":
            case.update(norm=rng.random() < 0.5, interleaved=rng.random() < 0.3, table=40960,
                        rotary_dim=rng.choice([case["head_dim"], case["head_dim"], 32]))
        while work(case)["bytes"] > _MOST_BYTES[op]:
            case["tokens"], case["padding"] = case["tokens"] // 2, case["padding"] // 2
        return case
    case["lengths_seed"] = rng.randint(0, 9999)
    if op == "evict":
        case.update(requests=_spread(rng, 1, 32), most=_spread(rng, 20, 32768))
        case["keep"] = _spread(rng, 1, case["most"])
        case["recent"] = rng.randint(0, case["keep"])
    else:
        kind = rng.choice(["decode", "decode", "draft", "extend"])
        case.update(requests=_spread(rng, 1, {"decode": 64, "draft": 32, "extend": 4}[kind]),
                    query_tokens={"decode": 1, "draft": rng.randint(2, 64),
                                  "extend": rng.randint(100, 1000)}[kind])
        if op == "attend":
            case["prefix"] = rng.choice([0, 0, _spread(rng, 100, 16384)])
        case["most"] = case["query_tokens"] + _spread(rng, 1, 16384 if kind == "decode" else 2048)
    case["least"] = rng.randint(1, case["most"])
    while (work(case)["bytes"] > _MOST_BYTES[op]
           or work(case)["flops"] > _MOST_FLOPS.get(op, math.inf)):
        if case["requests"] > 1:
            case["requests"] = -(-case["requests"] // 2)
        else:
            case["most"] = case["most"] // 2
            case["least"] = min(case["least"], case["most"])
            if "keep" in case:
                case["keep"], case["recent"] = -(-case["keep"] // 2), case["recent"] // 2
        if "prefix" in case:
            case["prefix"] //= 2
    return case


# -- inputs --------------------------------------------------------------------------------


def _row_bytes(head_dim: int) -> int:
    """Bytes of a row in 4 bits: the channels' values, and a byte for the scale of each 32 of
    them, filled up to whole dwords."""
    return head_dim // 2 + 4 * -(-head_dim // (4 * _GROUP))


def _lengths(case: dict) -> tuple[list[int], list[int]]:
    """(query tokens, tokens) of each request; a request's queries are the last of its tokens, one
    at least."""
    rng = random.Random(case["lengths_seed"])
    tokens = [rng.randint(case["least"], case["most"]) for _ in range(case["requests"])]
    return [min(t, case.get("query_tokens", 1)) for t in tokens], tokens


def _randn(gen, *shape) -> torch.Tensor:
    return torch.randn(*shape, generator=gen, device="cuda")


def _quantize(x: torch.Tensor) -> torch.Tensor:
    """Rows [.., D] of binary32 as rows of bytes in 4 bits."""
    D = x.shape[-1]
    groups = -(-D // _GROUP)
    g = torch.nn.functional.pad(x, (0, groups * _GROUP - D)).unflatten(-1, (groups, _GROUP))
    size = g.abs()
    # the least power of two at which no value is further from its 4 bits than half a step
    part, power = torch.frexp(size.amax(-1))
    power = (power - 3 + (part > 0.875)).clamp(_LEAST_SCALE, _MOST_SCALE)
    y = torch.ldexp(size, -power[..., None])
    code = ((y > 0.25).to(torch.uint8) + (y >= 0.75) + (y > 1.25) + (y >= 1.75) + (y > 2.5)
            + (y >= 3.5) + (y > 5.0))
    code = (code + 8 * torch.signbit(g)).to(torch.uint8).flatten(-2)[..., :D]
    out = torch.zeros(*x.shape[:-1], _row_bytes(D), dtype=torch.uint8, device=x.device)
    out[..., :D // 2] = code[..., 0::2] + 16 * code[..., 1::2]
    out[..., D // 2:D // 2 + groups] = (power + 127).to(torch.uint8)
    return out


def _dequantize(rows: torch.Tensor, head_dim: int) -> torch.Tensor:
    """The values, in binary32, that rows of bytes in 4 bits stand for."""
    values = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=rows.device)
    values = torch.cat((values, -values))
    half, groups = head_dim // 2, -(-head_dim // _GROUP)
    byte = rows[..., :half].int()
    x = values[torch.stack((byte & 15, byte >> 4), -1).flatten(-2)]
    scale = torch.ldexp(torch.ones((), device=rows.device),
                        rows[..., half:half + groups].int() - 127)
    return x * scale.repeat_interleave(_GROUP, -1)[..., :head_dim]


def _cache(case: dict, gen, blocks: int) -> tuple[torch.Tensor, float, float]:
    """A paged cache with keys whose channels differ in size, and values off zero; and the
    scales of an fp8 cache's entries."""
    H, D, bs = case["heads"], case["head_dim"], case["block_size"]
    kind, first = case["cache_dtype"], case["cache"] == "kv_first"
    row = _row_bytes(D) if kind == "mxfp4" else D
    cache = torch.empty((2, blocks, bs, H, row) if first else (blocks, 2, bs, H, row),
                        dtype=_TYPES[kind], device="cuda")
    scales = (0.03125, 0.0225) if kind == "float8_e4m3fn" else (1.0, 1.0)
    sizes = (torch.exp(0.5 * _randn(gen, H, D)), 0.25 * _randn(gen, H, D))
    for at in range(0, blocks, 4096):
        n = min(4096, blocks - at)
        for half in (0, 1):
            x = _randn(gen, n, bs, H, D)
            x = x * sizes[0] if half == 0 else 0.5 * x + sizes[1]
            if kind == "float8_e4m3fn":
                x = (x / scales[half]).clamp(-448, 448)
            x = _quantize(x) if kind == "mxfp4" else x.to(_TYPES[kind])
            if first:
                cache[half, at:at + n] = x
            else:
                cache[at:at + n, half] = x
    return cache, *scales


def _prepare_rows(case: dict, gen) -> dict:
    """Of appending and reading: the cache and the tokens' slots."""
    bs, T, real = case["block_size"], case["tokens"], case["tokens"] - case["padding"]
    blocks = -(-real // bs) + _SPARE_BLOCKS
    cache, k_scale, v_scale = _cache(case, gen, blocks)
    if T <= 64:  # one token of each request, in a block of its own
        used = torch.randperm(blocks * bs, generator=gen, device="cuda")[:real]
    else:  # a request's tokens, block after block
        count = torch.arange(real, device="cuda")
        used = torch.randperm(blocks, generator=gen, device="cuda")[count // bs] * bs + count % bs
    slots = torch.full((T,), -1, device="cuda")
    slots[:real] = used
    return {"cache": cache, "k_scale": k_scale, "v_scale": v_scale, "slots": slots, "real": real}


def _prepare_append(case: dict, gen) -> dict:
    Hq, H, D, T = case["query_heads"], case["heads"], case["head_dim"], case["tokens"]
    dtype, rot, table = _TYPES[case["dtype"]], case["rotary_dim"], case["table"]
    angle = (torch.arange(table, dtype=torch.float64, device="cuda")[:, None]
             * 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot))
    state = {**_prepare_rows(case, gen),
             # one row of a token: its queries, keys and values, as a projection leaves them
             "rows": _randn(gen, T, Hq + 2 * H, D).to(dtype),
             "cos_sin": torch.cat((angle.cos(), angle.sin()), 1).float(),
             "positions": torch.randint(0, table, (T,), generator=gen, device="cuda"),
             "query_norm": None, "key_norm": None}
    if case["norm"]:
        state["query_norm"] = (1 + 0.2 * _randn(gen, D)).to(dtype)
        state["key_norm"] = (1 + 0.2 * _randn(gen, D)).to(dtype)
    return state


def _prepare_attend(case: dict, gen) -> dict:
    """Of attending and of adding up weights: the cache, the requests' blocks and queries."""
    Hq, D, bs, B = case["query_heads"], case["head_dim"], case["block_size"], case["requests"]
    queries, tokens = _lengths(case)
    shared, width = -(-case.get("prefix", 0) // bs), -(-max(tokens) // bs)
    blocks = shared + sum(-(-t // bs) for t in tokens) + _SPARE_BLOCKS
    cache, k_scale, v_scale = _cache(case, gen, blocks)
    ids = torch.randperm(blocks, generator=gen, device="cuda")
    tables = torch.zeros(B, width, dtype=torch.int64, device="cuda")
    at = shared
    for r, t in enumerate(tokens):  # each request has the blocks that its tokens need
        n = -(-t // bs)
        tables[r, :n] = ids[at:at + n]
        at += n
    starts = torch.tensor([0, *queries]).cumsum(0)
    # queries that find some keys: scores with a spread of about two
    query = (2.0 * _randn(gen, sum(queries), Hq, D)).to(_TYPES[case["dtype"]])
    return {"query": query, "cache": cache, "k_scale": k_scale, "v_scale": v_scale,
            "prefix_ids": ids[:shared].contiguous() if shared else None, "tables": tables,
            "tokens": torch.tensor(tokens, device="cuda"),
            "starts": None if max(queries) == 1 else starts.cuda(),
            "most_queries": max(queries), "most_tokens": max(tokens)}


def _prepare_weigh(case: dict, gen) -> dict:
    state = {"case": case, **_prepare_attend(case, gen)}
    H, queries, tokens = case["heads"], *_lengths(case)
    # what the attention returned, and the sums of the steps before
    lse = torch.empty(state["query"].shape[:2], device="cuda")
    first = 0
    for r, n in enumerate(queries):
        score = _scores_of(state, r, first, n, tokens[r])
        lse[first:first + n] = torch.logsumexp(score, -1).flatten(0, 1).T
        first += n
    before = torch.rand(case["requests"], H, state["most_tokens"], generator=gen, device="cuda")
    return {**state, "lse": lse, "before": before.pow(4), "sums": torch.empty_like(before)}


def _prepare_evict(case: dict, gen) -> dict:
    bs, H, keep = case["block_size"], case["heads"], case["keep"]
    _, tokens = _lengths(case)
    width, kept = -(-max(tokens) // bs), -(-min(keep, max(tokens)) // bs)
    blocks = sum(-(-t // bs) for t in tokens) + case["requests"] * kept + _SPARE_BLOCKS
    cache, k_scale, v_scale = _cache(case, gen, blocks)
    ids = torch.randperm(blocks, generator=gen, device="cuda")
    tables = torch.zeros(case["requests"], width, dtype=torch.int64, device="cuda")
    at = case["requests"] * kept
    for r, t in enumerate(tokens):
        n = -(-t // bs)
        tables[r, :n] = ids[at:at + n]
        at += n
    # sums of weights: few large, many small, and tokens that no query has seen
    weights = torch.exp(3.0 * _randn(gen, case["requests"], H, max(tokens)) - 4.0)
    weights *= torch.rand(weights.shape, generator=gen, device="cuda") < 0.9
    return {"cache": cache, "k_scale": k_scale, "v_scale": v_scale, "tables": tables,
            "out_tables": ids[:case["requests"] * kept].view(case["requests"], kept),
            "tokens": torch.tensor(tokens, device="cuda"), "most_tokens": max(tokens),
            "weights": weights, "out_weights": torch.empty_like(weights)}


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    make = {"append": _prepare_append, "read": _prepare_rows, "attend": _prepare_attend,
            "weigh": _prepare_weigh, "evict": _prepare_evict}[case["op"]]
    return {"case": case, **make(case, gen)}


# -- the operators in elementary operations ------------------------------------------------


def _by_block(s: dict) -> torch.Tensor:
    """The cache's bits as [NB, 2, bs, H, row]."""
    cache = s["cache"]
    bits = cache.view(torch.uint8 if cache.element_size() == 1 else torch.int16)
    return bits.transpose(0, 1) if s["case"]["cache"] == "kv_first" else bits


def _widen(s: dict, bits: torch.Tensor, scale: float) -> torch.Tensor:
    """Rows of the cache's bits in binary32."""
    if s["case"]["cache_dtype"] == "mxfp4":
        return _dequantize(bits, s["case"]["head_dim"])
    return bits.view(s["cache"].dtype).float() * scale


def _rows_of(s: dict, ids: torch.Tensor, tokens: int, half: int) -> torch.Tensor:
    """Keys (half 0) or values of blocks [.., n] in binary32, [.., tokens, heads, dim]."""
    bits = _by_block(s)[ids, half].flatten(-4, -3)[..., :tokens, :, :]
    return _widen(s, bits, s["v_scale" if half else "k_scale"])


def _plain_read(s: dict):
    bs, slots = s["case"]["block_size"], s["slots"]
    inside = (slots >= 0)[:, None, None]
    at = slots.clamp(min=0)
    rows = _by_block(s)[at // bs, :, at % bs]
    return tuple((_widen(s, rows[:, half], s[name]) * inside).to(_TYPES[s["case"]["dtype"]])
                 for half, name in ((0, "k_scale"), (1, "v_scale")))


def _plain_norm(x: torch.Tensor, weight) -> torch.Tensor:
    if weight is None:
        return x
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + _EPS) * weight.float()


def _plain_rotate(x: torch.Tensor, cos_sin: torch.Tensor, interleaved: bool) -> torch.Tensor:
    rot = cos_sin.shape[-1]
    cos, sin = cos_sin[:, None].chunk(2, -1)
    turned, rest = x[..., :rot], x[..., rot:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = turned.chunk(2, -1)
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, rest), -1)


def _plain_append(s: dict):
    case, bs = s["case"], s["case"]["block_size"]
    Hq, H = case["query_heads"], case["heads"]
    rows, cos_sin = s["rows"].float(), s["cos_sin"][s["positions"]]
    query = _plain_rotate(_plain_norm(rows[:, :Hq], s["query_norm"]), cos_sin,
                          case["interleaved"])
    key = _plain_rotate(_plain_norm(rows[:, Hq:Hq + H], s["key_norm"]), cos_sin,
                        case["interleaved"])
    real = s["real"]  # the places in use come first
    pair = _quantize(torch.stack((key, rows[:, Hq + H:]), 1)[:real])
    slots = s["slots"][:real]
    _by_block(s)[slots // bs, :, slots % bs] = pair
    return query.to(s["rows"].dtype), *_plain_read(s)


def _plain_attend(s: dict) -> torch.Tensor:
    case, query = s["case"], s["query"]
    Hq, H, D = case["query_heads"], case["heads"], case["head_dim"]
    B, G, P, N = case["requests"], Hq // H, case["prefix"], query.shape[0]
    Q, L = s["most_queries"], s["most_tokens"]
    scale = D ** -0.5
    # each request's own tokens, its queries padded to the longest
    count = torch.arange(max(N, Q, L), device=query.device)
    starts = s["starts"]
    if starts is None:
        starts = torch.arange(B + 1, device=query.device)
    at = (starts[:B, None] + count[:Q]).clamp(max=N - 1)
    mine = query.float()[at].view(B, Q, H, G, D).permute(0, 2, 1, 3, 4).reshape(B, H, Q * G, D)
    mine = scale * (mine @ _rows_of(s, s["tables"], L, 0).permute(0, 2, 3, 1))  # [B, H, Q G, L]
    last = (s["tokens"] - (starts[1:] - starts[:B]))[:, None] + count[:Q]  # the last one seen
    mine = mine.view(B, H, Q, G, L).masked_fill(
        (count[:L] > last[..., None])[:, None, :, None], -math.inf)
    # one softmax over both; a query of the batch is number `i` of request `r`
    r = torch.searchsorted(starts[1:], count[:N], right=True)
    i = count[:N] - starts[r]
    top = mine.amax(-1)[r, :, i].transpose(0, 1)  # [H, N, G]
    if P:  # the prefix: every query of the batch against the same keys
        q = query.float().view(N, H, G, D).transpose(0, 1).reshape(H, N * G, D)
        near = (scale * (q @ _rows_of(s, s["prefix_ids"], P, 0).permute(1, 2, 0))).view(H, N, G, P)
        top = torch.maximum(near.amax(-1), top)
    e = torch.exp(mine - top[:, at].permute(1, 0, 2, 3)[..., None])
    total = e.sum(-1)[r, :, i].transpose(0, 1)
    out = (e.view(B, H, Q * G, L) @ _rows_of(s, s["tables"], L, 1).transpose(1, 2))
    out = out.view(B, H, Q, G, D)[r, :, i].transpose(0, 1)
    if P:
        e = torch.exp(near - top[..., None])
        total = e.sum(-1) + total
        near = e.view(H, N * G, P) @ _rows_of(s, s["prefix_ids"], P, 1).transpose(0, 1)
        out = near.view(H, N, G, D) + out
    out = out / total[..., None]
    return out.transpose(0, 1).reshape(N, Hq, D).to(query.dtype)


def _scores_of(s: dict, r: int, first: int, n: int, t: int) -> torch.Tensor:
    """Request r's scores [H, G, n, t] in binary32: its n queries from `first`, which are the last
    of its t tokens."""
    case = s["case"]
    H, D, bs = case["heads"], case["head_dim"], case["block_size"]
    k = _rows_of(s, s["tables"][r, :-(-t // bs)], t, 0)
    q = s["query"][first:first + n].float().view(n, H, -1, D).permute(1, 2, 0, 3)
    score = D ** -0.5 * (q.flatten(1, 2) @ k.permute(1, 2, 0)).unflatten(1, (-1, n))
    if n > 1:
        place = torch.arange(t, device=q.device)
        score = score.masked_fill(place > (place[t - n:, None]), -math.inf)
    return score


def _plain_weigh(s: dict) -> torch.Tensor:
    case, sums = s["case"], s["before"].clone()
    H, (queries, tokens) = case["heads"], _lengths(case)
    first = 0
    for r, n in enumerate(queries):
        lse = s["lse"][first:first + n].T.view(H, -1, n, 1)
        sums[r, :, :tokens[r]] += torch.exp(
            _scores_of(s, r, first, n, tokens[r]) - lse).sum((1, 2))
        first += n
    return sums


def _held(s: dict):
    """The cache's rows that the evicted requests have now, as the values they stand for where
    that takes 4 bits; else the whole cache."""
    case = s["case"]
    if case["cache_dtype"] != "mxfp4":
        return s["cache"]
    bs, n = case["block_size"], min(case["keep"], s["most_tokens"])
    place = torch.arange(n, device="cuda")
    slots = s["out_tables"][:, place // bs] * bs + place % bs
    slots = slots.masked_fill(place >= s["tokens"][:, None], -1).flatten()
    if own:
        from origami_amd.lossless import native_gpu

        return native_gpu.read_kv_cache(s["cache"], slots, dtype=_TYPES[case["dtype"]])
    return _plain_read({**s, "slots": slots})


def _plain_evict(s: dict):
    case, w = s["case"], s["weights"]
    keep, recent, bs, L = case["keep"], case["recent"], case["block_size"], s["most_tokens"]
    B, H = case["requests"], case["heads"]
    n = s["tokens"][:, None, None]
    place = torch.arange(L, device=w.device)
    # the newest come first, then by weight; a stable sort gives ties to the lowest place
    rank = torch.where(place >= n - recent, math.inf, w).masked_fill(place >= n, -math.inf)
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices
    many = min(keep, L)
    kept = order[..., :many]
    kept = torch.sort(kept.masked_fill(kept >= n, L), -1).values  # what is past the end, last
    there = kept < L
    safe = kept.clamp(max=L - 1)
    sums = torch.zeros_like(w)
    sums[..., :many] = torch.gather(w, -1, safe) * there
    # the rows of each head from the kept places to the first ones of the new blocks
    by_block, head = _by_block(s), torch.arange(H, device=w.device)[None, :, None]
    request = torch.arange(B, device=w.device)[:, None, None]
    rows = by_block[s["tables"][request, safe // bs], :, safe % bs, head]
    to = place[:many].expand(B, H, many)
    at = s["out_tables"][request, to // bs]
    head = head.expand(B, H, many)
    by_block[at[there], :, (to % bs)[there], head[there]] = rows[there]
    full = torch.full((B, H, keep), -1, device=w.device)
    full[..., :many] = kept.masked_fill(~there, -1)
    return full, sums, _held(s)


# -- one pass ------------------------------------------------------------------------------


def _own_read(s: dict):
    from origami_amd.lossless import native_gpu

    return native_gpu.read_kv_cache(s["cache"], s["slots"], dtype=_TYPES[s["case"]["dtype"]],
                                    k_scale=s["k_scale"], v_scale=s["v_scale"])


def _own_append(s: dict):
    from origami_amd.lossless import native_gpu

    Hq, H = s["case"]["query_heads"], s["case"]["heads"]
    rows = s["rows"]
    query = native_gpu.append_kv_cache(
        rows[:, Hq:Hq + H], rows[:, Hq + H:], s["cache"], s["slots"], query=rows[:, :Hq],
        positions=s["positions"], cos_sin=s["cos_sin"], interleaved=s["case"]["interleaved"],
        query_norm=s["query_norm"], key_norm=s["key_norm"], eps=_EPS)
    return query, *_own_read(s)


def _own_attend(s: dict) -> torch.Tensor:
    from origami_amd.lossless import native_gpu

    return native_gpu.shared_prefix_attention(
        s["query"], s["cache"], s["prefix_ids"], s["case"]["prefix"], s["tables"], s["tokens"],
        query_starts=s["starts"], max_query_tokens=s["most_queries"],
        max_own_tokens=s["most_tokens"])


def _own_weigh(s: dict) -> torch.Tensor:
    from origami_amd.lossless import native_gpu

    return native_gpu.accumulate_attention_weights(
        s["query"], s["cache"], s["tables"], s["tokens"], s["lse"], s["before"],
        query_starts=s["starts"], max_tokens=s["most_tokens"], k_scale=s["k_scale"],
        out=s["sums"])


def _own_evict(s: dict):
    from origami_amd.lossless import native_gpu

    kept, sums = native_gpu.evict_kv_cache(
        s["cache"], s["tables"], s["tokens"], s["weights"], s["out_tables"], s["case"]["keep"],
        recent=s["case"]["recent"], max_tokens=s["most_tokens"], out_weights=s["out_weights"])
    return kept, sums, _held(s)


def run(state: dict):
    op = state["case"]["op"]
    if own:
        return {"append": _own_append, "read": _own_read, "attend": _own_attend,
                "weigh": _own_weigh, "evict": _own_evict}[op](state)
    return {"append": _plain_append, "read": _plain_read, "attend": _plain_attend,
            "weigh": _plain_weigh, "evict": _plain_evict}[op](state)


# -- what a pass cannot do without -----------------------------------------------------------


def work(case: dict) -> dict:
    Hq, H, D, bs = case["query_heads"], case["heads"], case["head_dim"], case["block_size"]
    row = {"mxfp4": _row_bytes(D), "float8_e4m3fn": D}.get(case["cache_dtype"], 2 * D)
    if case["op"] in ("append", "read"):
        T, real = case["tokens"], case["tokens"] - case["padding"]
        moved = real * 2 * H * row + T * (2 * H * D * 2 + 8)  # the rows that are read back
        if case["op"] == "read":
            return {"bytes": moved, "flops": 0}
        rot = case["rotary_dim"]
        moved += (2 * T * Hq * D * 2 + real * 2 * H * (2 * D + row)
                  + min(T, case["table"]) * rot * 4 + T * 16)
        return {"bytes": moved,
                "flops": (T * Hq + real * H) * (3 * rot + (4 * D if case["norm"] else 0))}
    queries, tokens = _lengths(case)
    N, B, P = sum(queries), case["requests"], case.get("prefix", 0)
    ids = 8 * (-(-P // bs) + sum(-(-t // bs) for t in tokens) + 2 * B)
    seen = N * P + sum(n * t - n * (n - 1) // 2 for n, t in zip(queries, tokens))
    if case["op"] == "attend":
        return {"bytes": (P + sum(tokens)) * 2 * H * row + ids + 2 * N * Hq * D * 2,
                "flops": 4 * D * Hq * seen}
    if case["op"] == "weigh":
        return {"bytes": (sum(tokens) * H * row + ids + N * Hq * (2 * D + 4)
                          + 2 * B * H * max(tokens) * 4),
                "flops": 2 * D * Hq * seen}
    kept = sum(min(t, case["keep"]) for t in tokens)
    return {"bytes": (sum(tokens) * H * 4 + B * H * (8 * case["keep"] + 4 * max(tokens)) + ids
                      + 2 * kept * 2 * H * row),
            "flops": 0}


# -- the definition in 64 bits ---------------------------------------------------------------


def _exact_values(rows: torch.Tensor, D: int) -> torch.Tensor:
    """What rows of bytes in 4 bits stand for: sign, two bits of a power and one behind the
    point, times two to the power of the group's scale."""
    rows = rows.long()
    channel = torch.arange(D, device=rows.device)
    code = (rows[..., channel // 2] >> (4 * (channel % 2))) & 15
    power, bit = (code >> 1) & 3, (code & 1).double()
    size = torch.where(power == 0, 0.5 * bit, (1.0 + 0.5 * bit) * 2.0 ** (power - 1).double())
    scale = 2.0 ** (rows[..., D // 2 + channel // 32] - 127).double()
    return torch.where(code >= 8, -size, size) * scale


def _exact_rounded(x: torch.Tensor) -> torch.Tensor:
    """The values that rows become in 4 bits."""
    D = x.shape[-1]
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64,
                        device=x.device)
    out = torch.empty_like(x)
    for first in range(0, D, 32):
        g = x[..., first:first + 32]
        top = g.abs().amax(-1, keepdim=True)
        power = torch.full_like(top, -23.0)
        for e in range(-22, 14):
            power[top > 7.0 * 2.0 ** (e - 1)] = float(e)
        apart = (g.abs()[..., None] * 2.0 ** -power[..., None] - grid).abs()
        # the nearest; of two as near, the one of an even number
        apart = apart * 4.0 + 1e-13 * (torch.arange(8, device=x.device) % 2)
        out[..., first:first + 32] = torch.sign(g) * grid[apart.argmin(-1)] * 2.0 ** power
    return out


def _exact_cells(s: dict, half: int) -> torch.Tensor:
    """Keys or values of the whole cache, [NB, bs, H, D]."""
    case, cache = s["case"], s["cache"]
    part = cache[half] if case["cache"] == "kv_first" else cache[:, half]
    if case["cache_dtype"] == "mxfp4":
        return _exact_values(part, case["head_dim"])
    return part.double() * s["v_scale" if half else "k_scale"]


def _exact_rows(s: dict, half: int) -> torch.Tensor:
    flat = _exact_cells(s, half).flatten(0, 1)
    return torch.where((s["slots"] < 0)[:, None, None], 0.0, flat[s["slots"].clamp(min=0)])


def _exact_append(s: dict):
    case, D, rot = s["case"], s["case"]["head_dim"], s["case"]["rotary_dim"]
    Hq, H = case["query_heads"], case["heads"]
    cs = s["cos_sin"].double()[s["positions"]]
    place = torch.arange(rot, device="cuda")
    if case["interleaved"]:
        pair, partner, minus = place // 2, place ^ 1, place % 2 == 0
    else:
        pair, partner, minus = place % (rot // 2), (place + rot // 2) % rot, place < rot // 2

    def turned(x, weight):
        x = x.double()
        if weight is not None:
            x = weight.double() * x / (x.pow(2).sum(-1, keepdim=True) / D + _EPS).sqrt()
        y = x.clone()
        sign = 1.0 - 2.0 * minus.double()
        y[..., :rot] = (x[..., :rot] * cs[:, pair][:, None]
                        + sign * x[..., partner] * cs[:, rot // 2 + pair][:, None])
        return y

    gone = (s["slots"] < 0)[:, None, None]
    key = _exact_rounded(turned(s["rows"][:, Hq:Hq + H], s["key_norm"]))
    value = _exact_rounded(s["rows"][:, Hq + H:].double())
    return (turned(s["rows"][:, :Hq], s["query_norm"]), torch.where(gone, 0.0, key),
            torch.where(gone, 0.0, value))


def _exact_attend(s: dict) -> torch.Tensor:
    case, query = s["case"], s["query"].double()
    H, D, P, bs = case["heads"], case["head_dim"], case["prefix"], case["block_size"]
    G = case["query_heads"] // H
    out = torch.empty_like(query)
    queries, tokens = _lengths(case)
    keys, values = _exact_cells(s, 0), _exact_cells(s, 1)
    for h in range(H):
        def stored(cells, ids, n):
            return cells[:, :, h][ids[:-(-n // bs)]].reshape(-1, D)[:n]

        before = [stored(c, s["prefix_ids"], P) for c in (keys, values)] if P else []
        first = 0
        for r, (n, t) in enumerate(zip(queries, tokens)):
            k, v = (stored(c, s["tables"][r], t) for c in (keys, values))
            if P:
                k, v = torch.cat((before[0], k)), torch.cat((before[1], v))
            seen = P + t - n + 1 + torch.arange(n, device="cuda")
            hidden = torch.arange(P + t, device="cuda")[None] >= seen[:, None]
            for g in range(h * G, h * G + G):
                score = query[first:first + n, g] @ k.T / math.sqrt(D)
                score[hidden] = -math.inf
                out[first:first + n, g] = torch.softmax(score, 1) @ v
            first += n
    return out


def _exact_weigh(s: dict) -> torch.Tensor:
    case, query = s["case"], s["query"].double()
    H, D, bs = case["heads"], case["head_dim"], case["block_size"]
    G = case["query_heads"] // H
    sums, keys = s["before"].double(), _exact_cells(s, 0)
    queries, tokens = _lengths(case)
    first = 0
    for r, (n, t) in enumerate(zip(queries, tokens)):
        place = torch.arange(t, device="cuda")
        k = keys[s["tables"][r, place // bs], place % bs]
        hidden = place[None] - (t - n) > torch.arange(n, device="cuda")[:, None]
        for head in range(H * G):
            score = query[first:first + n, head] @ k[:, head // G].T / math.sqrt(D)
            score = score - s["lse"][first:first + n, head].double()[:, None]
            score[hidden] = -math.inf
            sums[r, head // G, :t] += score.exp().sum(0)
        first += n
    return sums


def _exact_evict(s: dict):
    case, w = s["case"], s["weights"].double().cpu()
    keep, recent, bs, H = case["keep"], case["recent"], case["block_size"], case["heads"]
    _, tokens = _lengths(case)
    kept = torch.full((case["requests"], H, keep), -1, dtype=torch.int64)
    sums = torch.zeros_like(w)
    for r, t in enumerate(tokens):
        for h in range(H):
            last = min(recent, keep, t)
            old = w[r, h, :t - last]
            best = torch.argsort(-old, stable=True)[:max(min(keep, t) - last, 0)]
            places = torch.cat((best.sort().values, torch.arange(t - last, t)))
            kept[r, h, :len(places)] = places
            sums[r, h, :len(places)] = w[r, h, places]
    kept = kept.cuda()
    cells = [_exact_cells(s, half) for half in (0, 1)]
    four = case["cache_dtype"] == "mxfp4"
    if four:
        n = min(keep, max(tokens))
        held = [torch.zeros(case["requests"], n, H, case["head_dim"], dtype=torch.float64,
                            device="cuda") for _ in (0, 1)]
    else:
        held = s["cache"].double()
        held = held if case["cache"] == "kv_first" else held.transpose(0, 1)
    for r, t in enumerate(tokens):
        m = min(keep, t)
        to = torch.arange(m, device="cuda")
        for h in range(H):
            places = kept[r, h, :m]
            block, offset = s["tables"][r, places // bs], places % bs
            for half in (0, 1):
                if four:
                    held[half][r, :m, h] = cells[half][block, offset, h]
                else:
                    scale = s["v_scale" if half else "k_scale"]
                    held[half][s["out_tables"][r, to // bs], to % bs, h] = (
                        cells[half][block, offset, h] / scale)
    if four:
        held = tuple(x.flatten(0, 1) for x in held)
    elif case["cache"] != "kv_first":
        held = held.transpose(0, 1)
    return kept, sums.cuda(), held


def exact(case: dict, seed: int):
    state = prepare(case, seed)
    if case["op"] == "read":
        return _exact_rows(state, 0), _exact_rows(state, 1)
    return {"append": _exact_append, "attend": _exact_attend, "weigh": _exact_weigh,
            "evict": _exact_evict}[case["op"]](state)
