"""Plain 64-bit forms of the operators on the paged cache, and how far a correct result in
16 bits may be from them."""
import math

import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float8_e4m3fn: 2.0 ** -4}
# half of the smallest subnormal
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float8_e4m3fn: 2.0 ** -10}


def halves(cache):
    """The cache as [2, NB, bs, H, D], a view."""
    return cache if cache.shape[0] == 2 else cache.transpose(0, 1)


def cells(cache):
    """Float64 copy of the cache as [2, NB, bs, H, D] (fp8 through its bytes)."""
    return halves(cache).contiguous().double()


def rotate(x, cos_sin, positions, interleaved, weight=None, eps=1e-6):
    """Normalised and rotated rows [T, heads, D] in float64; rows placed outside the table are
    zero."""
    x = x.double()
    D = x.shape[-1]
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.double()
    if cos_sin is None:
        return x
    rot = cos_sin.shape[1]
    inside = (positions >= 0) & (positions < cos_sin.shape[0])
    cs = cos_sin.double()[positions.clamp(0, cos_sin.shape[0] - 1)]
    y = x.clone()
    for i in range(rot // 2):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
        cos, sin = cs[:, i, None], cs[:, rot // 2 + i, None]
        y[..., a] = x[..., a] * cos - x[..., b] * sin
        y[..., b] = x[..., b] * cos + x[..., a] * sin
    return torch.where(inside[:, None, None], y, torch.zeros((), dtype=y.dtype, device=y.device))


def attend(query, cache, prefix_ids, prefix, tables, own, starts=None, scale=None, k_scale=1.0,
           v_scale=1.0):
    """(output, lse, mean |v| under the weights, largest sum |q k|) in float64, row by row;
    rows of no request are NaN."""
    kv, (N, Hq, D) = cells(cache), query.shape
    NB, bs, H = kv.shape[1:4]
    G = Hq // H
    scale = (D ** -0.5 if scale is None else scale) * k_scale
    out = torch.full((N, Hq, D), math.nan, dtype=torch.float64, device=query.device)
    size, lse = out.clone(), out[..., 0].clone()
    largest = 0.0
    own = own.tolist()
    starts = list(range(len(own) + 1)) if starts is None else starts.tolist()

    def gathered(ids, n):
        t = torch.arange(n, device=query.device)
        block = ids[t // bs]
        good = (block >= 0) & (block < NB)
        return block.clamp(0, NB - 1), t % bs, good

    for r, n_own in enumerate(own):
        first, count = starts[r], starts[r + 1] - starts[r]
        parts = [gathered(tables[r], n_own)] if n_own else []
        if prefix:
            parts.insert(0, gathered(prefix_ids, prefix))
        for i in range(count):
            seen = prefix + min(max(n_own - count + i + 1, 0), n_own)
            if not seen:
                out[first + i], size[first + i], lse[first + i] = 0, 0, -math.inf
                continue
            block, offset, good = (torch.cat(x)[:seen] for x in zip(*parts))
            block, offset = block[good], offset[good]
            if not block.numel():
                out[first + i], size[first + i], lse[first + i] = 0, 0, -math.inf
                continue
            k, v = kv[0][block, offset], kv[1][block, offset] * v_scale  # [t, H, D]
            q = query[first + i].double().view(H, G, D)
            s = scale * torch.matmul(q, k.permute(1, 2, 0))
            w = torch.softmax(s, -1)
            out[first + i] = torch.matmul(w, v.transpose(0, 1)).reshape(Hq, D)
            size[first + i] = torch.matmul(w, v.abs().transpose(0, 1)).reshape(Hq, D)
            lse[first + i] = torch.logsumexp(s, -1).reshape(Hq)
            bound = abs(scale) * torch.matmul(q.abs(), k.abs().permute(1, 2, 0))
            largest = max(largest, float(bound[bound.isfinite()].max()) if bound.isfinite().any()
                          else 0.0)
    return out, lse, size, largest


def attend_tolerance(dtype, D, tokens, size, largest, ref):
    """The result is rounded once, to half a step of |ref|.  Each exponential is rounded to
    half a step for the product with the values: half a step of the weighted mean of |v|.  A
    score is a binary32 sum of D products (D 2^-24 sum |q k| scale), which changes numerator
    and sum alike (twice); sums over the tokens, the exponentials and the joins add
    (2 tokens + 64) 2^-24."""
    step = HALF_STEP[dtype]
    more = 2.0 ** -24 * (2 * D * largest + 2 * tokens + 64)
    return step * (1 + step) * ref.abs() + (step + more) * size + TINY[dtype]


def lse_tolerance(D, tokens, largest, ref):
    """The binary32 score and sum errors as above, and the logarithm's and the result's
    rounding."""
    return 2.0 ** -24 * (D * largest + tokens + 64 + 4 * ref.abs())


def rotate_tolerance(dtype, ref, x, weight, cos_sin):
    """One rounding to dtype; in binary32, the norm (a sum of D squares, a root, a division, two
    products) and the rotation (two products and a sum) of |x| <= the row's largest
    normalised size: (D / 2 + 8) 2^-24 of it each way."""
    D = x.shape[-1]
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-12) * weight.double()
    most = x.abs().amax(-1, keepdim=True)
    return HALF_STEP[dtype] * ref.abs() + (D / 2 + 8) * 2.0 ** -24 * 2 * most + TINY[dtype]
