"""Plain 64-bit forms of the paged cache in 4 bits and of eviction, on any device."""
import math

import torch

GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
LEAST, MOST = -23, 13  # powers that appending keeps scales within
GROUP = 32


def row_bytes(D):
    return D // 2 + 4 * math.ceil(D / 128)


def two_to(power):
    """2 to whole numbers in float64, which pow on a device may miss by a unit."""
    return ((power.long() + 1023) << 52).view(torch.float64)


def powers(x):
    """The power of two of each group's scale, [.., groups], for rows [.., D] of numbers: the least
    at which the largest value is at most 7 times as large."""
    groups = [g.abs().amax(-1) for g in x.double().split(GROUP, -1)]
    top = torch.stack(groups, -1)
    power = torch.full_like(top, LEAST)
    for e in range(LEAST + 1, MOST + 1):
        power[top > 7.0 * 2.0 ** (e - 1)] = e
    return power


def pack(x):
    """Rows of bytes for rows [.., D] of numbers; a group with a NaN has the scale 255."""
    x = x.double()
    D, power = x.shape[-1], powers(x.nan_to_num(0.0, math.inf, -math.inf))
    grid = torch.tensor(GRID, dtype=torch.float64, device=x.device)
    y = x.nan_to_num(0.0, 1e30, -1e30).abs() / two_to(power.repeat_interleave(GROUP, -1)[..., :D])
    apart = (y.clamp(max=6.0)[..., None] - grid).abs()
    near = apart == apart.amin(-1, keepdim=True)
    # of two as near the one of an even number
    score = near.long() * (2 - torch.arange(8, device=x.device) % 2)
    code = score.argmax(-1) + 8 * torch.signbit(x)
    out = torch.zeros(*x.shape[:-1], row_bytes(D), dtype=torch.uint8, device=x.device)
    out[..., :D // 2] = (code[..., 0::2] + 16 * code[..., 1::2]).to(torch.uint8)
    odd = torch.stack([g.isnan().any(-1) for g in x.split(GROUP, -1)], -1)
    n = power.shape[-1]
    out[..., D // 2:D // 2 + n] = torch.where(odd, 255, power.long() + 127).to(torch.uint8)
    return out


def values(rows, D):
    """The numbers, in float64, that rows of bytes stand for."""
    channel = torch.arange(D, device=rows.device)
    code = (rows[..., channel // 2].long() >> (4 * (channel % 2))) & 15
    grid = torch.tensor(GRID, dtype=torch.float64, device=rows.device)
    x = torch.where(code >= 8, -grid[code & 7], grid[code & 7])
    s = rows[..., D // 2 + channel // GROUP].long()
    return torch.where(s == 255, math.nan, x * two_to(s - 127))


def halves(cache):
    return cache if cache.shape[0] == 2 else cache.transpose(0, 1)


def cells(cache, D, k_scale=1.0, v_scale=1.0):
    """A cache of any type as float64 [2, NB, bs, H, D], with its scales."""
    both = halves(cache)
    if cache.dtype == torch.uint8:
        return values(both, D)
    return torch.stack((both[0].double() * k_scale, both[1].double() * v_scale))


def weigh(query, kv, tables, tokens, lse, weights, starts=None, scale=None):
    """(sums, what one call adds, the largest sum of |q k| times the scale); kv as of cells()."""
    (N, Hq, D), (NB, bs, H) = query.shape, kv.shape[1:4]
    G = Hq // H
    scale = D ** -0.5 if scale is None else scale
    added = torch.zeros(weights.shape, dtype=torch.float64, device=query.device)
    starts = list(range(len(tokens) + 1)) if starts is None else starts.tolist()
    largest = 0.0
    for r, n in enumerate(tokens.tolist()):
        first, count = starts[r], starts[r + 1] - starts[r]
        t = torch.arange(min(n, weights.shape[2]), device=query.device)
        if not count or not len(t):
            continue
        block = tables[r][t // bs]
        good = (block >= 0) & (block < NB)
        k = kv[0][block.clamp(0, NB - 1), t % bs]  # [t, H, D]
        q = query[first:first + count].double().view(count, H, G, D)
        for h in range(H):
            s = scale * torch.matmul(q[:, h], k[:, h].T)  # [count, G, t]
            size = abs(scale) * torch.matmul(q[:, h].abs(), k[:, h].abs().T)
            if size[size.isfinite()].numel():
                largest = max(largest, float(size[size.isfinite()].max()))
            row = lse[first:first + count, h * G:h * G + G].double()[..., None]
            e = torch.exp(s - row)
            seen = t <= n - count + torch.arange(count, device=query.device)[:, None]
            e = torch.where(seen[:, None] & (row > -math.inf) & good, e, 0.0)
            added[r, h, :len(t)] = e.sum((0, 1))
    return weights.double() + added, added, largest


def weigh_tolerance(D, largest, lse, added, sums):
    """A binary32 score loses (D + 2) 2^-24 of sum |q k| scale; the difference from lse, the
    product with log2 e and the exponential lose 5 2^-24 of |score| + |lse| and two units more, all
    of which is relative to the weight.  The sum of a token's weights (trees of 16 and lanes, and
    sums that keep what they lose between them) loses 16 2^-24 of it, and the result is rounded."""
    most = float(lse[lse.isfinite()].abs().max()) if lse.isfinite().any() else 0.0
    rate = 2.0 ** -24 * ((D + 7) * largest + 5 * most + 4)
    return (math.expm1(rate) + 16 * 2.0 ** -24) * added + 2.0 ** -23 * sums.abs() + 2.0 ** -126


def kept_places(weights, tokens, keep, recent):
    """The places that each request's heads keep, lists of lists in order."""
    out = []
    for r, n in enumerate(tokens):
        n = min(n, weights.shape[2])
        last = min(recent, keep, n)
        heads = []
        for h in range(weights.shape[1]):
            w = [math.inf if math.isnan(x) else x for x in weights[r, h, :n - last].tolist()]
            odd = [math.isnan(x) for x in weights[r, h, :n - last].tolist()]
            order = sorted(range(n - last), key=lambda t: (not odd[t], -w[t], t))
            best = sorted(order[:max(min(keep, n) - last, 0)])
            heads.append(best + list(range(n - last, n)))
        out.append(heads)
    return out
