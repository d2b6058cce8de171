"""The operators on the paged KV cache that this framework is timed on, at the sizes its users meet.

A serving engine that restores a prompt's prefix into its paged cache then runs the tokens
after it, layer by layer: their keys are rotated to their positions (and, in some model
families, normalised per head first), keys and values are appended to the cache, and the
queries attend to the prefix, which the whole batch shares, and to each request's own
tokens.  One case is one layer's call.  Head counts, head sizes, block sizes, both cache
orders and prefix lengths are those of the repository's benchmark and tests; lengths of
requests are ragged, since prompts and answers have any length.

`run` computes an operator in elementary torch operations while `own` is false, and calls
the framework while it is true.
"""
from __future__ import annotations

import math
import random

import torch

own = False

_TYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16,
          "float8_e4m3fn": torch.float8_e4m3fn}
_EPS = 1e-6
_MOST_BYTES = 205_000_000  # of a drawn case; the largest listed ones have more
_SPARE_BLOCKS = 5  # blocks of the cache that no request of the case has


def listed() -> list[dict]:
    wide = {"query_heads": 32, "heads": 8, "head_dim": 128, "block_size": 16,
            "dtype": "bfloat16", "cache_dtype": "bfloat16", "cache": "kv_first"}
    append = {"op": "append", **wide, "padding": 0, "norm": False, "rotary_dim": 128,
              "interleaved": False, "table": 40960}
    attend = {"op": "attend", **wide, "query_tokens": 1, "lengths_seed": 1}
    return [
        # One token of one request: the launch and the host path are nearly all there is.
        {"name": "append_one", **append, "tokens": 1},
        # A decode step of a captured batch of 64 with 3 unused places, queries and keys
        # normalised per head; the 28 / 4 heads of the benchmark's ragged batch.
        {"name": "append_step", **append, "query_heads": 28, "heads": 4, "tokens": 64,
         "padding": 3, "norm": True, "cache": "blocks_first"},
        # A prompt's tokens after its prefix, all at once.
        {"name": "append_prompt", **append, "tokens": 8192, "norm": True},
        # A ragged prompt into an fp8 cache, half of each head rotated in neighbouring pairs.
        {"name": "append_fp8", **append, "query_heads": 8, "heads": 8, "head_dim": 64,
         "tokens": 2053, "rotary_dim": 32, "interleaved": True,
         "cache_dtype": "float8_e4m3fn"},
        # One request just after its restore: few rows, so latency counts.
        {"name": "attend_one", **attend, "requests": 1, "prefix": 1000, "least": 29, "most": 29},
        # A small batch on a system prompt, answers of any length; the 28 / 4 heads, blocks first.
        {"name": "attend_ragged", **attend, "query_heads": 28, "heads": 4, "requests": 8,
         "prefix": 4104, "least": 1, "most": 2053, "cache": "blocks_first", "lengths_seed": 2},
        # A decode step of a full batch over the benchmark's 32768-token prefix.
        {"name": "attend_batch", **attend, "requests": 64, "prefix": 32768, "least": 17,
         "most": 1024, "lengths_seed": 3},
        # The fp8 batch of the benchmark: 16 requests, 16384 shared tokens, longer own parts.
        {"name": "attend_fp8", **attend, "cache_dtype": "float8_e4m3fn", "requests": 16,
         "prefix": 16384, "least": 200, "most": 4096, "lengths_seed": 4},
        # Drafted tokens looked over in one pass: five queries a request, one KV head per query
        # head of 64 channels, half precision.
        {"name": "attend_draft", **attend, "query_heads": 12, "heads": 12, "head_dim": 64,
         "dtype": "float16", "cache_dtype": "float16", "requests": 24, "prefix": 2000,
         "least": 5, "most": 600, "query_tokens": 5, "lengths_seed": 5},
        # Prompts that go on after a restored prefix: up to 1024 query tokens a request.
        {"name": "attend_extend", **attend, "requests": 4, "prefix": 8192, "least": 400,
         "most": 1024, "query_tokens": 1024, "lengths_seed": 6},
        # One tensor-parallel rank (one KV head) of the 131072-token layer.
        {"name": "attend_long", **attend, "query_heads": 8, "heads": 1, "requests": 16,
         "prefix": 131072, "least": 1, "most": 512, "lengths_seed": 7},
    ]


def _spread(rng, least: int, most: int) -> int:
    """A whole number from [least, most], spread over its logarithm."""
    return max(least, min(most, int(round(math.exp(rng.uniform(math.log(least),
                                                               math.log(most)))))))


def draw(rng) -> dict:
    heads, group = rng.choice([(8, 4), (8, 1), (4, 7), (1, 8), (2, 4), (12, 1), (8, 5), (1, 16)])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16"])
    case = {"op": rng.choice(["append", "attend", "attend"]), "query_heads": heads * group,
            "heads": heads, "head_dim": rng.choice([64, 128, 128, 128, 80, 256]),
            "block_size": rng.choice([16, 16, 32, 24]), "dtype": dtype,
            "cache_dtype": rng.choice([dtype, dtype, "float8_e4m3fn"]),
            "cache": rng.choice(["kv_first", "blocks_first"])}
    if case["op"] == "append":
        tokens = _spread(rng, 1, 8192)
        case.update(tokens=tokens, padding=rng.randint(0, tokens // 8),
                    norm=rng.random() < 0.5, interleaved=rng.random() < 0.3, table=40960,
                    rotary_dim=rng.choice([case["head_dim"], case["head_dim"], 32]))
        while work(case)["bytes"] > _MOST_BYTES:
            case["tokens"], case["padding"] = case["tokens"] // 2, case["padding"] // 2
        return case
    kind = rng.choice(["decode", "decode", "draft", "extend"])
    requests = _spread(rng, 1, {"decode": 64, "draft": 32, "extend": 4}[kind])
    case.update(requests=requests, lengths_seed=rng.randint(0, 9999),
                prefix=_spread(rng, 100, {"decode": 32768, "draft": 16384, "extend": 4096}[kind]),
                query_tokens={"decode": 1, "draft": rng.randint(2, 8),
                              "extend": rng.randint(100, 700)}[kind])
    case["most"] = case["query_tokens"] + _spread(rng, 1, 2048 if kind == "decode" else 512)
    case["least"] = rng.randint(1, case["most"])
    while work(case)["bytes"] > _MOST_BYTES:
        case["requests"], case["prefix"] = -(-case["requests"] // 2), case["prefix"] // 2
    return case


# -- inputs --------------------------------------------------------------------------------


def _lengths(case: dict) -> tuple[list[int], list[int]]:
    """(query tokens, own tokens) of each request; a request's queries are the last of its own
    tokens, one at least."""
    rng = random.Random(case["lengths_seed"])
    tokens = [rng.randint(case["least"], case["most"]) for _ in range(case["requests"])]
    return [min(t, case["query_tokens"]) for t in tokens], tokens


def _randn(gen, *shape) -> torch.Tensor:
    return torch.randn(*shape, generator=gen, device="cuda")


def _cache(case: dict, gen, blocks: int) -> tuple[torch.Tensor, float, float]:
    """A paged cache with keys whose channels differ in size, and values off zero; and the
    scales of an fp8 cache's entries."""
    H, D, bs = case["heads"], case["head_dim"], case["block_size"]
    k = _randn(gen, blocks, bs, H, D) * torch.exp(0.5 * _randn(gen, H, D))
    v = 0.5 * _randn(gen, blocks, bs, H, D) + 0.25 * _randn(gen, H, D)
    scales = (1.0, 1.0)
    if case["cache_dtype"] == "float8_e4m3fn":
        scales = (0.03125, 0.0225)
        k, v = (k / scales[0]).clamp(-448, 448), (v / scales[1]).clamp(-448, 448)
    cache = torch.stack((k, v), 0 if case["cache"] == "kv_first" else 1)
    return cache.to(_TYPES[case["cache_dtype"]]), *scales


def _prepare_append(case: dict, gen) -> dict:
    Hq, H, D, T = case["query_heads"], case["heads"], case["head_dim"], case["tokens"]
    bs, dtype, real = case["block_size"], _TYPES[case["dtype"]], case["tokens"] - case["padding"]
    blocks = -(-real // bs) + _SPARE_BLOCKS
    cache, k_scale, v_scale = _cache(case, gen, blocks)
    # one row of a token: its queries, keys and values, as a projection leaves them
    rows = _randn(gen, T, Hq + 2 * H, D).to(dtype)
    if T <= 64:  # one token of each request, in a block of its own
        used = torch.randperm(blocks * bs, generator=gen, device="cuda")[:real]
    else:  # a request's tokens, block after block
        count = torch.arange(real, device="cuda")
        used = torch.randperm(blocks, generator=gen, device="cuda")[count // bs] * bs + count % bs
    slots = torch.full((T,), -1, device="cuda")
    slots[:real] = used
    rot, table = case["rotary_dim"], case["table"]
    angle = (torch.arange(table, dtype=torch.float64, device="cuda")[:, None]
             * 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot))
    state = {"rows": rows, "cache": cache, "k_scale": k_scale, "v_scale": v_scale,
             "slots": slots, "real": real,
             "cos_sin": torch.cat((angle.cos(), angle.sin()), 1).float(),
             "positions": torch.randint(0, table, (T,), generator=gen, device="cuda"),
             "query_norm": None, "key_norm": None}
    if case["norm"]:
        state["query_norm"] = (1 + 0.2 * _randn(gen, D)).to(dtype)
        state["key_norm"] = (1 + 0.2 * _randn(gen, D)).to(dtype)
    return state


def _prepare_attend(case: dict, gen) -> dict:
    Hq, D, bs, B = case["query_heads"], case["head_dim"], case["block_size"], case["requests"]
    queries, tokens = _lengths(case)
    shared, width = -(-case["prefix"] // bs), -(-max(tokens) // bs)
    blocks = shared + B * width + _SPARE_BLOCKS
    cache, k_scale, v_scale = _cache(case, gen, blocks)
    ids = torch.randperm(blocks, generator=gen, device="cuda")
    tables = torch.empty(B, shared + width, dtype=torch.int64, device="cuda")
    tables[:, :shared] = ids[:shared]
    tables[:, shared:] = ids[shared:shared + B * width].view(B, width)
    starts = torch.tensor([0, *queries]).cumsum(0)
    # queries that find some keys: scores with a spread of about two
    query = (2.0 * _randn(gen, sum(queries), Hq, D)).to(_TYPES[case["dtype"]])
    return {"query": query, "cache": cache, "k_scale": k_scale, "v_scale": v_scale,
            "prefix_ids": tables[0, :shared].contiguous(), "tables": tables[:, shared:],
            "tokens": torch.tensor(tokens, device="cuda"),
            "starts": None if case["query_tokens"] == 1 else starts.cuda(),
            "most_queries": max(queries), "most_tokens": max(tokens)}


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    state = (_prepare_append if case["op"] == "append" else _prepare_attend)(case, gen)
    return {"case": case, **state}


# -- the operators in elementary operations ------------------------------------------------


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
    case, cache = s["case"], s["cache"]
    Hq, H, bs = case["query_heads"], case["heads"], case["block_size"]
    rows, cos_sin = s["rows"].float(), s["cos_sin"][s["positions"]]
    query = _plain_rotate(_plain_norm(rows[:, :Hq], s["query_norm"]), cos_sin,
                          case["interleaved"])
    key = _plain_rotate(_plain_norm(rows[:, Hq:Hq + H], s["key_norm"]), cos_sin,
                        case["interleaved"])
    pair = torch.stack((key / s["k_scale"], rows[:, Hq + H:] / s["v_scale"]), 1)
    if cache.dtype == torch.float8_e4m3fn:
        pair = pair.clamp(-448, 448)
    real = s["real"]  # the places in use come first
    slots, pair = s["slots"][:real], pair[:real].to(cache.dtype)
    store = cache.view(torch.uint8) if cache.dtype == torch.float8_e4m3fn else cache
    pair = pair.view(store.dtype)
    by_block = store.transpose(0, 1) if case["cache"] == "kv_first" else store
    by_block[slots // bs, :, slots % bs] = pair
    return query.to(s["rows"].dtype), cache


def _plain_attend(s: dict) -> torch.Tensor:
    case, cache, query = s["case"], s["cache"], s["query"]
    Hq, H, D, bs = case["query_heads"], case["heads"], case["head_dim"], case["block_size"]
    B, G, P, N = case["requests"], Hq // H, case["prefix"], query.shape[0]
    Q, L = s["most_queries"], s["most_tokens"]
    bits = cache.view(torch.uint8 if cache.element_size() == 1 else torch.int16)
    by_block = bits.transpose(0, 1) if case["cache"] == "kv_first" else bits

    def rows(ids, tokens, half):  # [.., blocks] -> [.., tokens, heads, dim]
        return by_block[ids, half].view(cache.dtype).flatten(-4, -3)[..., :tokens, :, :].float()

    scale = D ** -0.5 * s["k_scale"]
    # the prefix: every query of the batch against the same keys
    q = query.float().view(N, H, G, D).transpose(0, 1).reshape(H, N * G, D)
    near = (scale * (q @ rows(s["prefix_ids"], P, 0).permute(1, 2, 0))).view(H, N, G, P)
    # each request's own tokens, its queries padded to the longest
    count = torch.arange(max(N, Q, L), device=query.device)
    starts = s["starts"]
    if starts is None:
        starts = torch.arange(B + 1, device=query.device)
    at = (starts[:B, None] + count[:Q]).clamp(max=N - 1)
    mine = query.float()[at].view(B, Q, H, G, D).permute(0, 2, 1, 3, 4).reshape(B, H, Q * G, D)
    mine = scale * (mine @ rows(s["tables"], L, 0).permute(0, 2, 3, 1))  # [B, H, Q G, L]
    last = (s["tokens"] - (starts[1:] - starts[:B]))[:, None] + count[:Q]  # the last one seen
    mine = mine.view(B, H, Q, G, L).masked_fill(
        (count[:L] > last[..., None])[:, None, :, None], -math.inf)
    # one softmax over both; a query of the batch is number `i` of request `r`
    r = torch.searchsorted(starts[1:], count[:N], right=True)
    i = count[:N] - starts[r]
    top = torch.maximum(near.amax(-1), mine.amax(-1)[r, :, i].transpose(0, 1))  # [H, N, G]
    e = torch.exp(mine - top[:, at].permute(1, 0, 2, 3)[..., None])
    own_sum = e.sum(-1)
    own_out = (e.view(B, H, Q * G, L) @ rows(s["tables"], L, 1).transpose(1, 2)).view(B, H, Q, G, D)
    e = torch.exp(near - top[..., None])
    total = e.sum(-1) + own_sum[r, :, i].transpose(0, 1)
    out = e.view(H, N * G, P) @ rows(s["prefix_ids"], P, 1).transpose(0, 1)
    out = out.view(H, N, G, D) + own_out[r, :, i].transpose(0, 1)
    out = s["v_scale"] * out / total[..., None]
    return out.transpose(0, 1).reshape(N, Hq, D).to(query.dtype)


# -- one pass ------------------------------------------------------------------------------


def _own_append(s: dict):
    from origami_amd.lossless import native_gpu

    Hq, H = s["case"]["query_heads"], s["case"]["heads"]
    rows = s["rows"]
    query = native_gpu.append_kv_cache(
        rows[:, Hq:Hq + H], rows[:, Hq + H:], s["cache"], s["slots"], query=rows[:, :Hq],
        positions=s["positions"], cos_sin=s["cos_sin"], interleaved=s["case"]["interleaved"],
        query_norm=s["query_norm"], key_norm=s["key_norm"], eps=_EPS, k_scale=s["k_scale"],
        v_scale=s["v_scale"])
    return query, s["cache"]


def _own_attend(s: dict) -> torch.Tensor:
    from origami_amd.lossless import native_gpu

    return native_gpu.shared_prefix_attention(
        s["query"], s["cache"], s["prefix_ids"], s["case"]["prefix"], s["tables"], s["tokens"],
        query_starts=s["starts"], max_query_tokens=s["most_queries"],
        max_own_tokens=s["most_tokens"], k_scale=s["k_scale"], v_scale=s["v_scale"])


def run(state: dict):
    if own:
        return (_own_append if state["case"]["op"] == "append" else _own_attend)(state)
    return (_plain_append if state["case"]["op"] == "append" else _plain_attend)(state)


# -- what a pass cannot do without -----------------------------------------------------------


def work(case: dict) -> dict:
    Hq, H, D = case["query_heads"], case["heads"], case["head_dim"]
    cell = 1 if case["cache_dtype"] == "float8_e4m3fn" else 2
    if case["op"] == "append":
        T, real, rot = case["tokens"], case["tokens"] - case["padding"], case["rotary_dim"]
        read = T * Hq * D * 2 + real * 2 * H * D * 2 + min(T, case["table"]) * rot * 4 + T * 16
        written = T * Hq * D * 2 + real * 2 * H * D * cell
        flops = (T * Hq + real * H) * (3 * rot + (4 * D if case["norm"] else 0))
        return {"bytes": read + written, "flops": flops}
    queries, tokens = _lengths(case)
    N, P, bs = sum(queries), case["prefix"], case["block_size"]
    cells = (P + sum(tokens)) * 2 * H * D * cell
    ids = 8 * (-(-P // bs) + sum(-(-t // bs) for t in tokens))
    seen = N * P + sum(n * t - n * (n - 1) // 2 for n, t in zip(queries, tokens))
    return {"bytes": cells + ids + 2 * N * Hq * D * 2, "flops": 4 * D * Hq * seen}


# -- the definition in 64 bits ---------------------------------------------------------------


def _exact_append(s: dict):
    case, D, rot = s["case"], s["case"]["head_dim"], s["case"]["rotary_dim"]
    Hq, H, bs = case["query_heads"], case["heads"], case["block_size"]
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

    query = turned(s["rows"][:, :Hq], s["query_norm"])
    key = turned(s["rows"][:, Hq:Hq + H], s["key_norm"]) / s["k_scale"]
    value = s["rows"][:, Hq + H:].double() / s["v_scale"]
    if case["cache_dtype"] == "float8_e4m3fn":
        key, value = key.clamp(-448, 448), value.clamp(-448, 448)
    cache = s["cache"].double()
    keys, values = (cache[0], cache[1]) if case["cache"] == "kv_first" else (cache[:, 0], cache[:, 1])
    at = s["slots"] >= 0
    block, offset = s["slots"][at] // bs, s["slots"][at] % bs
    keys[block, offset] = key[at]
    values[block, offset] = value[at]
    return query, cache


def _exact_attend(s: dict) -> torch.Tensor:
    case, query = s["case"], s["query"].double()
    Hq, H, D, P = case["query_heads"], case["heads"], case["head_dim"], case["prefix"]
    G = Hq // H
    cache = (s["cache"] if case["cache"] == "kv_first" else s["cache"].transpose(0, 1)).double()
    out = torch.empty_like(query)
    queries, tokens = _lengths(case)
    for h in range(H):
        def stored(half, ids, n, scale):
            return scale * cache[half][:, :, h][ids].reshape(-1, D)[:n]

        kp, vp = (stored(i, s["prefix_ids"], P, s[x]) for i, x in ((0, "k_scale"), (1, "v_scale")))
        first = 0
        for r, (n, t) in enumerate(zip(queries, tokens)):
            k = torch.cat((kp, stored(0, s["tables"][r], t, s["k_scale"])))
            v = torch.cat((vp, stored(1, s["tables"][r], t, s["v_scale"])))
            seen = P + t - n + 1 + torch.arange(n, device="cuda")
            for g in range(h * G, h * G + G):
                score = query[first:first + n, g] @ k.T / math.sqrt(D)
                score[torch.arange(P + t, device="cuda")[None] >= seen[:, None]] = -math.inf
                out[first:first + n, g] = torch.softmax(score, 1) @ v
            first += n
    return out


def exact(case: dict, seed: int):
    state = prepare(case, seed)
    return (_exact_append if case["op"] == "append" else _exact_attend)(state)
