"""accumulate_attention_weights and evict_kv_cache on the GPU against plain 64-bit forms
(tests/kv4ref.py)."""
import math

import pytest
import torch

from origami_amd.lossless import native_gpu
from tests import kv4ref

pytestmark = pytest.mark.gpu
BF16, F16, FP8, U8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn, torch.uint8


def make_cache(gen, cache_dtype, NB, bs, H, D, order, dev, scale=1.0):
    kv = torch.randn(2, NB, bs, H, D, generator=gen) * scale
    kv = kv if order == "kv_first" else kv.transpose(0, 1).contiguous()
    return (kv4ref.pack(kv) if cache_dtype == U8 else kv.to(cache_dtype)).to(dev)


class Weights:
    """A batch whose rows have been attended to (in 64 bits), and sums of weights so far."""

    def __init__(self, dev, *, heads=2, group=4, D=128, bs=16, dtype=BF16, cache_dtype=None,
                 order="kv_first", tokens=(5, 33), queries=None, seed=0, spare=7, peak=2.0):
        gen = torch.Generator().manual_seed(seed)
        B = len(tokens)
        self.D, self.bs, self.most = D, bs, max(tokens, default=0)
        self.k_scale = 0.5 if cache_dtype == FP8 else 1.0
        width = max(-(-max(tokens, default=0) // bs), 1)
        NB = B * width + 3
        self.cache = make_cache(gen, cache_dtype or dtype, NB, bs, heads, D, order, dev)
        self.tables = torch.randperm(NB, generator=gen)[:B * width].view(B, width).to(dev)
        self.tokens = torch.tensor(tokens, dtype=torch.int64, device=dev)
        self.starts, n = None, B
        if queries is not None:
            self.starts = torch.tensor([0, *queries]).cumsum(0).to(dev)
            n = sum(queries)
        self.query = (peak * torch.randn(n, heads * group, D, generator=gen)).to(dtype).to(dev)
        self.weights = torch.rand(B, heads, max(tokens, default=0) + spare, generator=gen).to(dev)
        # any number near the true one does: what matters is that it is subtracted
        self.lse = (3.0 + torch.rand(n, heads * group, generator=gen)).to(dev) * peak

    def run(self, **kw):
        return native_gpu.accumulate_attention_weights(
            self.query, self.cache, self.tables, self.tokens, self.lse,
            **{"weights": self.weights, "query_starts": self.starts, "k_scale": self.k_scale,
               "max_tokens": self.most, **kw})

    def check(self, got, weights=None, scale=None):
        weights = self.weights if weights is None else weights
        kv = kv4ref.cells(self.cache, self.D, self.k_scale)
        sums, added, largest = kv4ref.weigh(self.query, kv, self.tables, self.tokens, self.lse,
                                            weights, self.starts, scale)
        assert torch.equal(got.isnan(), sums.isnan())
        tol = kv4ref.weigh_tolerance(self.D, largest, self.lse, added, sums)
        off = (got.double() - sums).abs() - tol
        same = got.double() == torch.where(sums > torch.finfo(torch.float32).max, math.inf, sums)
        assert (same | (off <= 0) | sums.isnan()).all(), float(off.nan_to_num(0).max())
        return added


@pytest.mark.parametrize("dtype,cache_dtype", [(BF16, BF16), (F16, F16), (BF16, FP8), (F16, FP8),
                                               (BF16, U8), (F16, U8)])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("queries", [None, (1, 30, 16, 2, 33)])
def test_weights_types_and_sizes(cuda_device, dtype, cache_dtype, D, queries):
    for order in ("kv_first", "blocks_first"):
        w = Weights(cuda_device, D=D, dtype=dtype, cache_dtype=cache_dtype, order=order,
                    tokens=(1, 340, 16, 277, 33), queries=queries, seed=D)
        w.check(w.run())


@pytest.mark.parametrize("D", [8, 16, 24, 40, 72, 80, 96, 120, 136, 160, 192, 248])
@pytest.mark.parametrize("cache_dtype", [BF16, FP8, U8])
def test_weights_odd_head_sizes(cuda_device, D, cache_dtype):
    for queries in (None, (9, 70)):
        w = Weights(cuda_device, D=D, cache_dtype=cache_dtype, tokens=(300, 70), queries=queries,
                    seed=D, bs=24)
        w.check(w.run())


@pytest.mark.parametrize("heads,group", [(1, 1), (3, 1), (1, 7), (2, 16), (1, 17), (1, 48), (5, 8),
                                         (12, 1)])
@pytest.mark.parametrize("queries", [None, (2, 0, 5, 1)])
def test_weights_head_groups(cuda_device, heads, group, queries):
    w = Weights(cuda_device, heads=heads, group=group, D=64, tokens=(90, 3, 500, 1),
                queries=queries, seed=heads * group)
    w.check(w.run())


@pytest.mark.parametrize("bs", [1, 2, 5, 16, 24, 256])
@pytest.mark.parametrize("tokens,queries", [((0,), None), ((1,), None), ((0, 5, 0, 129), None),
                                            ((511, 513, 512), None), ((0, 700), (3, 700)),
                                            ((2, 40, 7), (6, 40, 0)), ((1030,), (257,))])
def test_weights_lengths(cuda_device, bs, tokens, queries):
    w = Weights(cuda_device, bs=bs, tokens=tokens, queries=queries, D=64, group=3)
    w.check(w.run())


def test_weights_of_long_prompts(cuda_device):
    w = Weights(cuda_device, tokens=(2500, 1777), queries=(2500, 64), heads=1, group=5, D=64)
    w.check(w.run())
    w = Weights(cuda_device, tokens=(9000, 20011), heads=2, group=4, cache_dtype=U8)
    w.check(w.run())


def test_weights_of_steep_scores(cuda_device):
    """Weights of one token, and far below it; sums of infinity where lse is too small."""
    for peak in (0.0, 12.0):
        w = Weights(cuda_device, tokens=(300, 40), queries=(5, 40), peak=peak)
        w.check(w.run())
    w.lse.fill_(-200.0)
    w.check(w.run())
    assert w.run()[0, :, 0].isinf().all()


def test_weights_places_and_results(cuda_device):
    """In place; without sums so far; into strided sums; places past the tokens."""
    w = Weights(cuda_device, tokens=(70, 300, 0), spare=200)
    want = w.run()
    w.check(want)
    assert torch.equal(want[0, :, 70:], w.weights[0, :, 70:])
    first = w.run(weights=None, max_tokens=None)
    assert first.shape[2] == w.tables.shape[1] * w.bs and (first[2] == 0).all()
    w.check(first, torch.zeros_like(first))
    B, H, S = w.weights.shape
    room = torch.full((H, B + 1, S + 5), 7.0, device=cuda_device)
    out = room[:, :B, 3:3 + S].transpose(0, 1)
    assert w.run(out=out).data_ptr() == out.data_ptr()
    assert torch.equal(out, want) and (room[:, B] == 7.0).all() and (room[..., :3] == 7.0).all()
    out.copy_(w.weights)
    w.run(weights=out, out=out)
    assert torch.equal(out, want)
    short = w.run(max_tokens=100)  # tokens past the bound get nothing, places stay the lengths'
    assert torch.equal(short[:, :, :100], want[:, :, :100])
    assert torch.equal(short[:, :, 100:], w.weights[:, :, 100:])


def test_weights_of_hidden_rows_and_tokens(cuda_device):
    """A row that saw nothing gives nothing; a NaN or infinite key is its own token's alone; blocks
    outside the cache get nothing."""
    w = Weights(cuda_device, tokens=(70, 300), queries=(20, 33), cache_dtype=BF16)
    w.lse[5] = -math.inf
    w.lse[30, 3] = -math.inf
    w.check(w.run())
    want = w.run()
    for value in (math.nan, math.inf):
        clean = w.cache.clone()
        t = 290  # of request 1, whose queries 23 on see it: keys of head 1
        w.cache[0, int(w.tables[1, t // w.bs]), t % w.bs, 1, 7] = value
        got = w.run()
        odd = torch.zeros_like(got, dtype=torch.bool)
        odd[1, 1, t] = True
        assert not got[odd].isfinite().any() or value == math.inf
        assert torch.equal(got[~odd], want[~odd])
        w.cache = clean
    w.tables[0, 1], w.tables[1, 0], w.tables[1, 2] = -1, 1 << 40, w.cache.shape[1]
    added = w.check(w.run())
    assert (added[0, :, 16:32] == 0).all() and (added[1, :, :16] == 0).all()


def test_weights_captured_and_on_another_stream(cuda_device):
    for queries in (None, (3, 9, 64)):
        w = Weights(cuda_device, tokens=(900, 40, 333), queries=queries, cache_dtype=U8)
        grown = w.tokens.clone()
        out = torch.empty_like(w.weights)
        kw = dict(out=out, max_tokens=900)
        w.run(**kw)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            w.run(**kw)
        for part in (0.1, 1.0, 0.5, 0.0):
            w.tokens.copy_((grown * part).long())
            graph.replay()
            w.check(out)
            assert torch.equal(out, w.run(max_tokens=900))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = w.run(max_tokens=900)
        side.synchronize()
        assert torch.equal(got, out)


class Eviction:
    def __init__(self, dev, *, heads=2, D=64, bs=16, cache_dtype=BF16, order="kv_first",
                 tokens=(50, 33), keep=20, recent=5, seed=0, spare=3):
        gen = torch.Generator().manual_seed(seed)
        B, most = len(tokens), max(tokens, default=0)
        self.bs, self.keep, self.recent, self.dev, self.most = bs, keep, recent, dev, most
        width, kept = max(-(-most // bs), 1), max(-(-min(keep, most) // bs), 1)
        NB = B * (width + kept) + 3
        self.cache = make_cache(gen, cache_dtype, NB, bs, heads, D, order, dev)
        ids = torch.randperm(NB, generator=gen)[:B * (width + kept)].to(dev)
        self.tables = ids[:B * width].view(B, width)
        self.out_tables = ids[B * width:].view(B, kept)
        self.tokens = torch.tensor(tokens, dtype=torch.int64, device=dev)
        self.weights = torch.rand(B, heads, most + spare, generator=gen).pow(6).to(dev)

    def run(self, **kw):
        return native_gpu.evict_kv_cache(
            self.cache, self.tables, self.tokens, self.weights, self.out_tables, self.keep,
            **{"recent": self.recent, "max_tokens": self.most, **kw})

    def check(self, **kw):
        before = kv4ref.halves(self.cache.view(U8) if self.cache.dtype != U8 else self.cache).clone()
        kept, sums = self.run(**kw)
        NB, want = before.shape[1], before.clone()
        lists = kv4ref.kept_places(self.weights.cpu(), self.tokens.tolist(), self.keep, self.recent)
        tables, new = self.tables.tolist(), self.out_tables.tolist()
        for r, heads in enumerate(lists):
            for h, places in enumerate(heads):
                n = len(places)
                assert kept[r, h].tolist() == places + [-1] * (self.keep - n)
                at = torch.tensor(places, dtype=torch.int64, device=self.dev)
                held = self.weights[r, h, at]
                assert torch.equal(sums[r, h, :n].nan_to_num(9.0), held.nan_to_num(9.0))
                assert (sums[r, h, n:] == 0).all()
                src = torch.tensor([tables[r][t // self.bs] for t in places], dtype=torch.int64)
                dst = torch.tensor([new[r][j // self.bs] for j in range(n)], dtype=torch.int64)
                src, dst = src.to(self.dev), dst.to(self.dev)
                rows = before[:, src.clamp(0, NB - 1), at % self.bs, h]
                rows = torch.where(((src >= 0) & (src < NB))[None, :, None], rows,
                                   torch.zeros_like(rows))
                to = torch.arange(n, device=self.dev) % self.bs
                inside = (dst >= 0) & (dst < NB)
                want[:, dst[inside], to[inside], h] = rows[:, inside]
        now = kv4ref.halves(self.cache.view(U8) if self.cache.dtype != U8 else self.cache)
        assert torch.equal(now, want)
        return kept, sums


@pytest.mark.parametrize("cache_dtype", [BF16, F16, FP8, U8])
@pytest.mark.parametrize("D", [8, 64, 80, 128, 200, 256])
@pytest.mark.parametrize("order", ["kv_first", "blocks_first"])
def test_evict_types_and_sizes(cuda_device, cache_dtype, D, order):
    Eviction(cuda_device, cache_dtype=cache_dtype, D=D, order=order, tokens=(50, 33, 7),
             seed=D).check()


@pytest.mark.parametrize("tokens", [(0,), (1,), (64, 65, 63, 1, 0), (1023, 1025), (5000,),
                                    (2048, 2049)])
@pytest.mark.parametrize("keep,recent", [(0, 0), (1, 0), (1, 1), (64, 0), (64, 64), (64, 100),
                                         (1000, 17), (1000, 999)])
def test_evict_lengths(cuda_device, tokens, keep, recent):
    Eviction(cuda_device, tokens=tokens, keep=keep, recent=recent, heads=3, D=16,
             seed=keep).check()


@pytest.mark.parametrize("bs", [1, 3, 16, 24, 128])
@pytest.mark.parametrize("heads", [1, 5, 12])
def test_evict_block_sizes_and_heads(cuda_device, bs, heads):
    Eviction(cuda_device, bs=bs, heads=heads, tokens=(300, 77, 5), keep=60, recent=9, D=32,
             seed=bs).check()


def test_evict_long(cuda_device):
    Eviction(cuda_device, tokens=(20011, 32768), keep=4096, recent=300, heads=2, D=64).check()
    Eviction(cuda_device, tokens=(70001,), keep=30000, recent=1, heads=1, D=8).check()


@pytest.mark.parametrize("most", [4096, 4097, 8191, 16384, 16385, 32768, 32769, 49155])
@pytest.mark.parametrize("keep,recent", [(0, 0), (700, 0), (700, 65), (5000, 4999)])
def test_evict_on_both_sides_of_a_lane_s_places(cuda_device, most, keep, recent):
    """Requests of all lengths in one call, with weights that are all different, few, or one."""
    e = Eviction(cuda_device, tokens=(most, most - 1, 0, 1, keep + 1, most // 2 + 1), keep=keep,
                 recent=recent, heads=3, D=8, seed=most + keep)
    e.weights[:, 1] = (e.weights[:, 1] * 8).round() - 3.0
    e.weights[:, 2] = -0.0
    e.check()


def test_evict_ties_and_odd_weights(cuda_device):
    """Equal weights go to the first places; both zeros are equal; NaN is larger than infinity;
    ranks that differ in their last bit."""
    for seed in range(3):
        e = Eviction(cuda_device, tokens=(3000, 700), keep=500, recent=10, seed=seed)
        w = e.weights
        w[0, 0] = 1.0
        w[0, 1] = torch.where(w[0, 1] > 0.5, 0.0, -0.0)
        w[1, 0] = (w[1, 0] * 4).round() / 4
        w[1, 1] = 1.0 + torch.randint(0, 700, w[1, 1].shape, device=cuda_device) * 2.0 ** -23
        e.check()
    w[0, 0, 5:40] = math.nan
    w[0, 0, 50:52] = -math.nan
    w[0, 0, 100:700] = math.inf
    w[0, 1, :] = -math.inf
    w[0, 1, 30:60] = -1.0
    w[0, 1, 70] = -1e-45
    w[1, 0] = 1e-45 * torch.randint(0, 100, w[1, 0].shape, device=cuda_device)
    e.check()


def test_evict_shared_and_missing_blocks(cuda_device):
    """Tables that share blocks; blocks outside the cache on both sides."""
    e = Eviction(cuda_device, tokens=(100, 90, 64), keep=40, recent=4)
    e.tables[1, :3] = e.tables[0, :3]
    e.check()
    e = Eviction(cuda_device, tokens=(100, 90, 64), keep=40, recent=4)
    e.tables[0, 2], e.tables[0, 6], e.tables[1, 0] = -1, 1 << 40, e.cache.shape[1]
    e.out_tables[0, 0], e.out_tables[2, 1] = -7, 1 << 50
    e.check()


def test_evict_places_and_results(cuda_device):
    e = Eviction(cuda_device, tokens=(100, 30), keep=40, recent=4, spare=20)
    kept, sums = e.check(max_tokens=100)
    assert sums.shape == e.weights.shape
    B, H, S = e.weights.shape
    room = torch.full((B, H + 1, 64), 7.0, device=cuda_device)
    out = room[:, :H, 5:50]
    _, got = e.check(out_weights=out)
    assert got.data_ptr() == out.data_ptr() and torch.equal(out[..., :40], sums[..., :40])
    assert (out[..., 40:] == 0).all() and (room[:, H] == 7.0).all() and (room[..., :5] == 7.0).all()
    # strided sums; the bound cuts the lengths
    wide = torch.zeros(H, B, S + 1, device=cuda_device)[..., 1:].transpose(0, 1)
    wide.copy_(e.weights)
    e.weights = wide
    kept2, _ = e.check()
    assert torch.equal(kept, kept2)
    kept3, _ = e.run(max_tokens=60)
    assert kept3[0].max() == 59 and (kept3[0] >= 56).sum() == 4 * H


def test_evict_captured_and_on_another_stream(cuda_device):
    e = Eviction(cuda_device, tokens=(900, 300), keep=200, recent=30, cache_dtype=U8, D=128)
    grown, start = e.tokens.clone(), e.cache.clone()
    sums = torch.empty_like(e.weights)
    kw = dict(out_weights=sums, max_tokens=900)
    e.run(**kw)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept, _ = e.run(**kw)
    for part in (1.0, 0.1, 0.5, 0.9):
        e.tokens.copy_((grown * part).long())
        e.weights.copy_(torch.rand_like(e.weights))
        e.cache.copy_(start)
        graph.replay()
        got = kept.clone(), sums.clone(), e.cache.clone()
        e.cache.copy_(start)
        want_kept, want = e.check(max_tokens=900)
        assert torch.equal(got[0], want_kept) and torch.equal(got[1], want)
        assert torch.equal(got[2], e.cache)
    e.cache.copy_(start)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kept2, sums2 = e.run(max_tokens=900)
    side.synchronize()
    assert torch.equal(kept2, want_kept) and torch.equal(sums2, want)
    assert torch.equal(e.cache, got[2])


@pytest.mark.parametrize("dtype,cache_dtype", [(BF16, BF16), (F16, FP8), (BF16, U8), (F16, U8)])
@pytest.mark.parametrize("order", ["kv_first", "blocks_first"])
def test_attend_weigh_evict_and_go_on(cuda_device, dtype, cache_dtype, order):
    """A prompt appended, attended to, weighed and evicted; then decode steps on what is left."""
    from tests import pagedref
    from tests.test_gpu_append import table_of

    dev, gen = cuda_device, torch.Generator().manual_seed(3)
    B, Hq, H, D, bs, keep, recent = 3, 8, 2, 128, 16, 48, 16
    counts, width, narrow = [150, 20, 77], 12, 5
    NB = B * (width + narrow) + 2
    cache = make_cache(gen, cache_dtype, NB, bs, H, D, order, dev)
    ids = torch.randperm(NB, generator=gen).to(dev)
    tables, small = ids[:B * width].view(B, width), ids[B * width:B * (width + narrow)].view(B, -1)
    cos_sin = table_of(1000, D, dev)
    scales = dict(k_scale=0.05, v_scale=0.04) if cache_dtype == FP8 else {}
    place = torch.tensor(counts, device=dev)  # the positions of what comes next

    def step(counts, tables, before):
        """Appends and attends; the sums of weights are checked against softmax's."""
        n, r = sum(counts), torch.repeat_interleave(torch.arange(B), torch.tensor(counts)).to(dev)
        i = torch.cat([torch.arange(c) for c in counts]).to(dev)
        at, tokens = before[r] + i, before + torch.tensor(counts, device=dev)
        rows = torch.randn(n, Hq + 2 * H, D, generator=gen).to(dtype).to(dev)
        rows[:, :Hq + H] *= 1.5
        query = native_gpu.append_kv_cache(
            rows[:, Hq:Hq + H], rows[:, Hq + H:], cache, tables[r, at // bs] * bs + at % bs,
            query=rows[:, :Hq], positions=place[r] - before[r] + at, cos_sin=cos_sin, **scales)
        starts = None if counts == [1] * B else torch.tensor([0, *counts]).cumsum(0).to(dev)
        out, lse = native_gpu.shared_prefix_attention(
            query, cache, None, 0, tables, tokens, query_starts=starts, return_lse=True, **scales)
        kv = kv4ref.cells(cache, D, *scales.values())
        ref, ref_lse, size, largest = pagedref.attend(query, kv, None, 0, tables, tokens, starts)
        tol = pagedref.attend_tolerance(dtype, D, int(tokens.max()), size, largest, ref)
        assert (out.double() - ref).abs().le(tol).all()
        return query, tokens, starts, lse

    query, tokens, starts, lse = step(counts, tables, torch.zeros_like(place))
    weights = native_gpu.accumulate_attention_weights(
        query, cache, tables, tokens, lse, query_starts=starts,
        **({"k_scale": 0.05} if scales else {}))
    # every query gives weights of 1 together, G of them to each cache head
    total = weights.double().sum(-1)
    assert torch.allclose(total, (tokens * (Hq // H)).double()[:, None].expand(B, H), rtol=1e-4)
    kv = kv4ref.cells(cache, D, *scales.values()).clone()
    kept, weights = native_gpu.evict_kv_cache(cache, tables, tokens, weights, small, keep,
                                              recent=recent)
    left = tokens.clamp(max=keep)
    now = kv4ref.cells(cache, D, *scales.values())
    for r in range(B):
        for h in range(H):
            t = kept[r, h, :int(left[r])]
            j = torch.arange(len(t), device=dev)
            assert torch.equal(now[:, small[r, j // bs], j % bs, h],
                               kv[:, tables[r, t // bs], t % bs, h])
            newest = int(tokens[r]) - torch.arange(min(recent, len(t)), 0, -1, device=dev)
            assert torch.equal(t[-len(newest):], newest)
    for _ in range(3):
        sums = weights.clone()
        query, after, starts, lse = step([1, 1, 1], small, left)
        weights = native_gpu.accumulate_attention_weights(
            query, cache, small, after, lse, weights, out=weights,
            max_tokens=min(weights.shape[2], narrow * bs),
            **({"k_scale": 0.05} if scales else {}))
        gain = (weights - sums).double().sum(-1)
        assert torch.allclose(gain, torch.full_like(gain, Hq // H), rtol=1e-4)
        left, place = after, place + 1


def test_refusals(cuda_device):
    w = Weights(cuda_device, tokens=(40, 33))
    e = Eviction(cuda_device)
    before = e.cache.clone()
    with pytest.raises(RuntimeError, match="float32 .requests, heads, places."):
        w.run(weights=w.weights.half())
    with pytest.raises(RuntimeError, match="float32 .requests, heads, places."):
        w.run(weights=w.weights[:1])
    with pytest.raises(RuntimeError, match="places must be contiguous"):
        w.run(weights=w.weights.transpose(1, 2).contiguous().transpose(1, 2))
    with pytest.raises(RuntimeError, match="out must have the weights' shape"):
        w.run(out=torch.zeros(2, 2, 5, device=cuda_device))
    with pytest.raises(RuntimeError, match="exceeds the weights' places"):
        w.run(max_tokens=48, weights=w.weights[..., :47])
    with pytest.raises(RuntimeError, match="exceeds the block tables"):
        w.run(max_tokens=49, weights=torch.zeros(2, 2, 80, device=cuda_device))
    with pytest.raises(RuntimeError, match="other elements of weights"):
        room = torch.zeros(2, 2, 101, device=cuda_device)
        w.run(weights=room[..., :100], out=room[..., 1:])
    with pytest.raises(RuntimeError, match="overlap itself"):
        w.run(out=torch.zeros(2, 1, w.weights.shape[2], device=cuda_device).expand(2, 2, -1))
    with pytest.raises(RuntimeError, match="lse must be float32"):
        w.lse = w.lse.double()
        w.run()
    w = Weights(cuda_device, tokens=(40, 33))
    with pytest.raises(RuntimeError, match="one query token"):
        w.query = torch.cat((w.query, w.query))
        w.run()
    with pytest.raises(RuntimeError, match="for float8_e4m3fn caches"):
        Weights(cuda_device).run(k_scale=2.0)
    with pytest.raises(RuntimeError, match="requires a gradient"):
        w = Weights(cuda_device)
        w.query.requires_grad_()
        w.run()

    with pytest.raises(RuntimeError, match="exceeds the new block tables"):
        e.keep = 33
        e.run()
    e.keep = -1
    with pytest.raises(RuntimeError, match="keep must not be negative"):
        e.run()
    e.keep = 20
    with pytest.raises(RuntimeError, match="must not be negative"):
        e.run(recent=-1)
    with pytest.raises(RuntimeError, match="exceeds the places of out_weights"):
        e.run(out_weights=torch.zeros(2, 2, 19, device=cuda_device))
    with pytest.raises(RuntimeError, match="out_weights must not overlap weights"):
        e.run(out_weights=e.weights)
    with pytest.raises(RuntimeError, match="a row for every request"):
        native_gpu.evict_kv_cache(e.cache, e.tables, e.tokens, e.weights, e.out_tables[:1], 20)
    with pytest.raises(RuntimeError, match="exceeds the weights' places"):
        e.run(max_tokens=64)
    with pytest.raises(RuntimeError, match="float16 or bfloat16"):
        native_gpu.evict_kv_cache(e.cache.float(), e.tables, e.tokens, e.weights, e.out_tables, 20,
                                  max_tokens=50)
    assert torch.equal(e.cache, before)


@pytest.mark.parametrize("tokens,queries", [
    ((70, 300, 0, 33), None), ((70, 300, 0, 33), (9, 40, 0, 2)), ((2000, 1500), (2000, 700)),
    ((5,) * 40, None)])
@pytest.mark.parametrize("spare", [1, 63, 20000])
@pytest.mark.parametrize("bound", ["most", "half", 0, None])
def test_weights_places_far_past_the_tokens(cuda_device, tokens, queries, spare, bound):
    """Sums for more tokens than there are, as a buffer that is kept for the longest context: the
    places past the bound are the sums before in a new buffer, and stay in the same one."""
    w = Weights(cuda_device, tokens=tokens, queries=queries, D=64, spare=spare, seed=spare)
    bound = {"most": w.most, "half": w.most // 2}.get(bound, bound)
    want = w.run(max_tokens=bound)
    cut = min(w.most if bound is None else bound, w.most)
    for start in (w.weights, torch.zeros_like(w.weights)):
        got = w.run(max_tokens=bound, weights=start)
        kv = kv4ref.cells(w.cache, w.D, w.k_scale)
        sums, added, largest = kv4ref.weigh(w.query, kv, w.tables, w.tokens, w.lse, start, w.starts)
        sums[..., cut:], added[..., cut:] = start[..., cut:].double(), 0.0
        tol = kv4ref.weigh_tolerance(w.D, largest, w.lse, added, sums)
        assert (got.double() - sums).abs().le(tol).all()
        assert torch.equal(got[..., cut:], start[..., cut:])
    B, H, S = w.weights.shape
    room = torch.full((H, B, S + 9), 5.0, device=cuda_device)  # a buffer of other strides
    out = room[..., 4:4 + S].transpose(0, 1)
    w.run(max_tokens=bound, out=out)
    assert torch.equal(out, want)
    assert (room[..., :4] == 5.0).all() and (room[..., 4 + S:] == 5.0).all()
    out.fill_(7.0)
    zero = w.run(max_tokens=min(bound, S) if bound is not None else w.most, weights=None, out=out)
    assert (zero[..., cut:] == 0).all()
    same = w.weights.clone()
    w.run(max_tokens=bound, weights=same, out=same)
    assert torch.equal(same, want)


@pytest.mark.parametrize("cache_dtype", [BF16, U8])
@pytest.mark.parametrize("requests,queries", [(64, 190), (20, 65), (300, 900)])
def test_weights_of_one_long_request_among_many(cuda_device, cache_dtype, requests, queries):
    """Requests of a row or two and one of many, whose sums lose no more than those of a prompt: its
    rows are added to each other first, and to what there was once."""
    at, group = requests // 2, 4
    counts, tokens = [1] * requests, [1 + 37 * i % 200 for i in range(requests)]
    counts[at], tokens[at], counts[-1], tokens[-2] = queries, queries + 70, 0, 0
    w = Weights(cuda_device, heads=2, group=group, D=64, tokens=tokens, queries=counts,
                cache_dtype=cache_dtype, seed=requests)
    w.check(w.run())
    same = w.weights.clone()
    assert torch.equal(w.run(weights=same, out=same), w.run())
    # 16 rows give 0.9, which is less than half a step of the sums before
    w.query.zero_()
    w.lse.fill_(math.log(16 / 0.9))
    w.weights.fill_(2.0 ** 24)
    added = w.check(w.run())
    assert added[at, 0, 0] > 14  # of which the sums have all but a step


def test_weights_of_parts_lose_nothing_between_them(cuda_device):
    """8192 rows are 32 parts; all but the first give 0.9 each, less than half a step (1) of what
    the first gives, and are not lost one by one."""
    w = Weights(cuda_device, heads=1, group=8, D=64, tokens=(2048,), queries=(1024,))
    w.query.zero_()
    w.lse.fill_(math.inf)
    w.lse[0, 0] = -math.log(1.5 * 2.0 ** 24)
    first = w.run(weights=None)[0, 0, :1024].double()  # tokens that all rows see
    assert ((first / 2.0 ** 24 - 1.5).abs() < 1e-4).all()
    w.lse[32:] = math.log(256 / 0.9)
    gain = w.run(weights=None)[0, 0, :1024].double() - first
    assert ((gain - 31 * 0.9).abs() <= 2.0).all()


@pytest.mark.parametrize("queries", [None, (9, 40), (1, 65)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_weights_of_infinite_and_nan_keys(cuda_device, queries, dtype):
    """What an odd key's token gets: infinity where a row's score is, nothing from scores of
    -infinity, NaN where a score is; and what other tokens get is the same."""
    w = Weights(cuda_device, tokens=(70, 300), queries=queries, dtype=dtype)
    want, t = w.run(), 250  # which all rows see
    clean, place = w.cache.clone(), (int(w.tables[1, t // w.bs]), t % w.bs)
    w.query[:, :4, 7] = w.query[:, :4, 7].abs() + 0.5  # of head 1 they stay of both signs
    base = w.run()
    for value in (math.inf, -math.inf, math.nan):
        w.cache.copy_(clean)
        w.cache[0, place[0], place[1], :, 7] = value
        got = w.run()
        w.check(got)
        others = torch.ones_like(got, dtype=torch.bool)
        others[1, :, t] = False
        assert torch.equal(got[others], base[others])
        if math.isnan(value):
            assert got[1, :, t].isnan().all()
        else:
            assert got[1, 0, t] == (math.inf if value > 0 else w.weights[1, 0, t])
    assert torch.equal(want[:, 1], base[:, 1])


@pytest.mark.parametrize("cache_dtype", [BF16, FP8, U8])
@pytest.mark.parametrize("D", [64, 80, 128, 256])
@pytest.mark.parametrize("group", [1, 4, 5])
def test_weights_of_uneven_drafts(cuda_device, cache_dtype, D, group):
    """16 rows and fewer on average, in requests of 16, of up to 32, and of more."""
    queries = (3, 5, 1, 7, 0, 4, 2, 8, 9, 1, 1, 1, 1, 1, 1, 1)
    w = Weights(cuda_device, heads=2, group=group, D=D, cache_dtype=cache_dtype, queries=queries,
                tokens=[q + 91 * i % 700 for i, q in enumerate(queries)], seed=D + group)
    w.check(w.run())
    same = w.weights.clone()
    assert torch.equal(w.run(weights=same, out=same), w.run())
