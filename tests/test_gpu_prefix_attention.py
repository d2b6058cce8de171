"""shared_prefix_attention on the GPU against plain 64-bit attention (tests/pagedref.py)."""
import math

import pytest
import torch

from origami_amd.lossless import native_gpu
from tests import pagedref

pytestmark = pytest.mark.gpu
BF16, F16, FP8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


class Batch:
    """A paged cache and a batch on it; every cell that the batch does not hold is NaN."""

    def __init__(self, dev, *, heads=2, group=4, D=128, bs=16, dtype=BF16, cache_dtype=None,
                 order="kv_first", prefix=100, own=(5, 33), queries=None, seed=0, spare=3,
                 peak=2.0):
        gen = torch.Generator().manual_seed(seed)
        self.heads, self.D, self.bs, self.dtype, self.prefix = heads, D, bs, dtype, prefix
        cache_dtype = cache_dtype or dtype
        width = max(-(-max(own, default=0) // bs), 1)
        shared = -(-prefix // bs)
        NB = shared + len(own) * width + spare
        ids = torch.randperm(NB, generator=gen)
        self.prefix_ids = ids[:shared].to(dev)
        self.tables = ids[shared:shared + len(own) * width].view(len(own), width).to(dev)
        kv = torch.randn(2, NB, bs, heads, D, generator=gen)
        self.k_scale, self.v_scale = (0.5, 0.25) if cache_dtype == FP8 else (1.0, 1.0)
        live = torch.zeros(NB, bs, dtype=torch.bool)
        for table, n in [(ids[:shared], prefix)] + [(t.cpu(), n) for t, n in zip(self.tables, own)]:
            for i in range(n):
                live[table[i // bs], i % bs] = True
        kv[:, ~live] = math.nan
        kv = kv if order == "kv_first" else kv.transpose(0, 1).contiguous()
        self.cache = kv.to(cache_dtype).to(dev)
        self.own = torch.tensor(own, dtype=torch.int64, device=dev)
        self.starts = None
        n = len(own)
        if queries is not None:
            self.starts = torch.tensor([0, *queries]).cumsum(0).to(dev)
            n = sum(queries)
        self.query = (peak * torch.randn(n, heads * group, D, generator=gen)).to(dtype).to(dev)

    def run(self, **kw):
        return native_gpu.shared_prefix_attention(
            self.query, self.cache, self.prefix_ids, self.prefix, self.tables, self.own,
            **{"query_starts": self.starts, "k_scale": self.k_scale, "v_scale": self.v_scale,
               "return_lse": True, **kw})

    def check(self, got, lse, rows=None, scale=None):
        ref, ref_lse, size, largest = pagedref.attend(
            self.query, self.cache, self.prefix_ids, self.prefix, self.tables, self.own,
            self.starts, scale, self.k_scale, self.v_scale)
        tokens = self.prefix + int(self.own.max()) if self.own.numel() else self.prefix
        rows = slice(None) if rows is None else rows
        tol = pagedref.attend_tolerance(self.dtype, self.D, tokens, size, largest, ref)
        assert torch.equal(got[rows].isnan(), ref[rows].isnan())
        off = (got.double() - ref).abs() - tol
        assert not (off[rows] > 0).any(), float(off[rows].nan_to_num(0).max())
        if lse is not None:
            same = lse.double() == ref_lse  # infinities
            off = (lse.double() - ref_lse).abs() - pagedref.lse_tolerance(
                self.D, tokens, largest, ref_lse)
            assert (same | (off <= 0) | ref_lse.isnan())[rows].all()


@pytest.mark.parametrize("dtype,cache_dtype", [(BF16, BF16), (F16, F16), (BF16, FP8), (F16, FP8)])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("order", ["kv_first", "blocks_first"])
def test_types_and_sizes(cuda_device, dtype, cache_dtype, D, order):
    b = Batch(cuda_device, D=D, dtype=dtype, cache_dtype=cache_dtype, order=order, prefix=150,
              own=(1, 40, 16, 77, 33))
    b.check(*b.run())


@pytest.mark.parametrize("heads,group", [(1, 1), (3, 1), (1, 7), (2, 16), (1, 17), (1, 48), (5, 8)])
@pytest.mark.parametrize("queries", [None, (2, 0, 5, 1)])
def test_head_groups(cuda_device, heads, group, queries):
    b = Batch(cuda_device, heads=heads, group=group, D=64, prefix=70, own=(9, 3, 50, 1),
              queries=queries, seed=heads * group)
    b.check(*b.run())


@pytest.mark.parametrize("D", [8, 16, 24, 40, 72, 80, 96, 120, 136, 192, 248])
@pytest.mark.parametrize("cache_dtype", [BF16, FP8])
def test_odd_head_sizes(cuda_device, D, cache_dtype):
    b = Batch(cuda_device, D=D, cache_dtype=cache_dtype, prefix=45, own=(3, 70), seed=D)
    b.check(*b.run())


@pytest.mark.parametrize("bs", [1, 2, 5, 8, 16, 24, 32, 64, 256])
@pytest.mark.parametrize("prefix", [0, 1, 31, 32, 33, 257])
def test_block_sizes(cuda_device, bs, prefix):
    b = Batch(cuda_device, bs=bs, prefix=prefix, own=(31, 1, 32, 65), D=64, seed=bs + prefix)
    b.check(*b.run())


@pytest.mark.parametrize("own", [(0,), (1,), (130,), (0, 0, 0), (0, 5, 0, 129), (511, 513, 512)])
@pytest.mark.parametrize("prefix", [0, 1, 700])
def test_lengths(cuda_device, own, prefix):
    b = Batch(cuda_device, prefix=prefix, own=own, D=64, seed=prefix + len(own))
    b.check(*b.run())


@pytest.mark.parametrize("prefix,own", [(5000, (1, 900)), (20011, (40,) * 20), (0, (9001, 17)),
                                        (2500, (2100,))])
@pytest.mark.parametrize("cache_dtype", [BF16, FP8])
def test_long(cuda_device, prefix, own, cache_dtype):
    b = Batch(cuda_device, prefix=prefix, own=own, cache_dtype=cache_dtype, seed=prefix)
    b.check(*b.run())


@pytest.mark.parametrize("queries,own,prefix", [
    ((1,), (1,), 0), ((5, 5, 5), (5, 90, 33), 300), ((3, 0, 7), (3, 4, 7), 50),
    ((64, 17), (64, 80), 129), ((130,), (130,), 0), ((200, 1, 77), (233, 9, 77), 400),
    ((129, 300), (400, 300), 64), ((70,) * 6, (75,) * 6, 1000)])
@pytest.mark.parametrize("heads,group", [(2, 1), (1, 5), (2, 4)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_several_queries(cuda_device, queries, own, prefix, heads, group, dtype):
    b = Batch(cuda_device, prefix=prefix, own=own, queries=queries, heads=heads, group=group,
              D=64 if group == 1 else 128, dtype=dtype, seed=sum(queries))
    b.check(*b.run())
    b.check(*b.run(max_query_tokens=max(queries), max_own_tokens=max(own)))
    b.check(*b.run(max_query_tokens=sum(queries) + 100))


def test_queries_beyond_the_own_tokens(cuda_device):
    """More query rows than own tokens: the first rows see the prefix alone, or nothing."""
    for prefix in (0, 40):
        b = Batch(cuda_device, prefix=prefix, own=(2, 0), queries=(6, 3), D=64)
        b.check(*b.run())


def test_masked_values_have_no_influence(cuda_device):
    """NaN and infinities in later own tokens reach the rows that see them and no others."""
    for value in (math.nan, math.inf, -math.inf):
        for half in (0, 1):
            b = Batch(cuda_device, prefix=20, own=(40, 37), queries=(30, 37), heads=2, group=2)
            table, bs = b.tables[0].tolist(), b.bs
            b.cache[half, table[25 // bs], 25 % bs, 1, 7] = value
            got, lse = b.run()
            # token 25 is that of query 15 of request 0; heads 2 and 3 read cache head 1
            sees = torch.zeros(67, 4, dtype=torch.bool, device=cuda_device)
            sees[15:30, 2:] = True
            clean = Batch(cuda_device, prefix=20, own=(40, 37), queries=(30, 37), heads=2, group=2)
            ref, ref_lse = clean.run()
            assert torch.equal(got[~sees], ref[~sees])
            assert torch.equal(lse[~sees], ref_lse[~sees])
            if half == 1:
                assert not got[sees][:, 7].isfinite().any()
                keep = [d for d in range(b.D) if d != 7]
                assert torch.equal(got[sees][:, keep], ref[sees][:, keep])
            elif math.isnan(value):
                assert got[sees].isnan().all()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("group", [1, 8, 40])
def test_odd_values_reach_the_rows_that_see_them(cuda_device, D, group):
    """Values of infinity and NaN anywhere in the tokens, in workgroups of every shape: the same
    channels are not finite as in the plain form, and all others are right."""
    for own, queries in (((40, 97), (30, 97)), ((300,), (257,)), ((64, 9), (1, 2))):
        b = Batch(cuda_device, prefix=75, own=own, queries=queries, heads=2, group=group, D=D,
                  seed=D + group)
        marks = [(b.prefix_ids, 3, 0, 5, math.nan), (b.prefix_ids, 74, 1, 6, math.inf),
                 (b.tables[0], 2, 0, 9, math.inf), (b.tables[0], own[0] - 3, 1, D - 1, -math.inf),
                 (b.tables[-1], own[-1] - 1, 0, 0, math.nan), (b.tables[-1], 0, 1, 1, -math.inf)]
        clean = b.cache.clone()
        for table, t, h, d, value in marks:
            b.cache[1, int(table[t // b.bs]), t % b.bs, h, d] = value
        got, lse = b.run()
        ref = pagedref.attend(b.query, b.cache, b.prefix_ids, b.prefix, b.tables, b.own,
                              b.starts)[0]
        fine = ref.isfinite()  # the plain form has no hidden tokens, so no 0 times infinity
        assert torch.equal(got.isfinite(), fine)
        b.cache = clean
        whole, whole_lse = b.run()
        assert torch.equal(got[fine], whole[fine]) and torch.equal(lse, whole_lse)


@pytest.mark.parametrize("peak", [0.0, 30.0])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_flat_and_steep_scores(cuda_device, peak, dtype):
    """Equal weights, and weights of one token: maxima that rise late in a long row."""
    b = Batch(cuda_device, prefix=3000, own=(700, 5), dtype=dtype, D=64, peak=peak, seed=3)
    b.check(*b.run())


@pytest.mark.parametrize("B,prefix,D", [(3, 1000, 128), (40, 600, 128), (70, 333, 64),
                                        (40, 600, 192)])
@pytest.mark.parametrize("queries", [1, 3, 11])
def test_batches_in_every_shape(cuda_device, B, prefix, D, queries):
    own = [(37 * i) % 150 + queries for i in range(B)]
    b = Batch(cuda_device, prefix=prefix, own=own, queries=[queries] * B, heads=1, group=5, D=D,
              seed=B + queries)
    b.check(*b.run())


def test_bounds_far_above_the_lengths(cuda_device):
    """Tables for much longer requests: ranges without a token are joined as nothing."""
    b = Batch(cuda_device, prefix=200, own=(3, 90, 41))
    plain = b.run()
    wide = torch.full((3, 4000), -1, dtype=torch.int64, device=cuda_device)
    wide[:, :b.tables.shape[1]] = b.tables
    b.tables = wide
    got = b.run()
    b.check(*got)
    assert (got[0].float() - plain[0].float()).abs().max() < 0.05


def test_blocks_outside_the_cache_are_not_seen(cuda_device):
    b = Batch(cuda_device, prefix=100, own=(50, 60, 3), D=64)
    NB = pagedref.halves(b.cache).shape[1]
    b.prefix_ids[2] = -1
    b.prefix_ids[6] = NB
    b.tables[0, 1] = 1 << 40
    b.tables[2, 0] = -(1 << 50)
    b.check(*b.run())
    b.prefix_ids.fill_(-1)
    b.tables.fill_(NB)
    got, lse = b.run()
    assert not got.any() and (lse == -math.inf).all()


def test_strided_inputs_and_output(cuda_device):
    """Queries inside a projection's rows, tables behind the prefix's columns, head-major output."""
    b = Batch(cuda_device, prefix=96, own=(50, 60, 3))
    rows = torch.full((3, 13, 128), math.nan, dtype=b.dtype, device=cuda_device)
    rows[:, 2:10] = b.query
    wide = torch.full((3, 9), -1, dtype=torch.int64, device=cuda_device)
    wide[:, 3:3 + b.tables.shape[1]] = b.tables
    plain, lse = b.run()
    out = torch.full((8, 3, 128), 7.0, dtype=b.dtype, device=cuda_device).transpose(0, 1)
    b.query, b.tables = rows[:, 2:10], wide[:, 3:3 + b.tables.shape[1]]
    got, again = b.run(out=out)
    assert got.data_ptr() == out.data_ptr()
    assert torch.equal(out, plain) and torch.equal(lse, again)
    odd = torch.zeros(3 * 8 * 129 + 1, dtype=b.dtype, device=cuda_device)[1:]
    odd = odd.as_strided((3, 8, 128), (8 * 129, 129, 1))
    odd.copy_(b.query)  # rows on two-byte boundaries
    b.query = odd
    out = torch.zeros(3 * 8 * 129 + 1, dtype=b.dtype, device=cuda_device)[1:]
    out = out.as_strided((3, 8, 128), (8 * 129, 129, 1))
    assert torch.equal(b.run(out=out)[0], plain)


def test_rows_of_no_request_stay(cuda_device):
    b = Batch(cuda_device, prefix=50, own=(9, 20), queries=(2, 3), D=64)
    b.query = torch.cat((b.query[:1], b.query, b.query[:4]))
    b.starts = b.starts + 1
    out = torch.full_like(b.query, 3.0)
    got, lse = b.run(out=out)
    rest = [0, 6, 7, 8, 9]
    assert (out[rest] == 3.0).all() and (lse[rest] == -math.inf).all()
    b.check(got, lse, rows=slice(1, 6))
    assert not b.run()[0][rest].any()


def test_scale(cuda_device):
    for scale in (0.0, 1.0, -0.3):
        b = Batch(cuda_device, prefix=50, own=(9, 20), D=64, peak=0.5)
        b.check(*b.run(scale=scale), scale=scale)


def test_far_blocks_of_a_large_cache(cuda_device):
    """Rows past 2^31 elements (and past 2^32 bytes) of the cache."""
    NB, bs, H, D = 40000, 16, 8, 256
    b = Batch(cuda_device, heads=H, D=D, bs=bs, prefix=40, own=(20, 33), group=1)
    kv = torch.empty(2, NB, bs, H, D, dtype=BF16, device=cuda_device)
    small = b.cache.shape[1]
    kv[:, NB - small:] = b.cache
    plain = b.run()
    b.cache, b.prefix_ids, b.tables = kv, b.prefix_ids + NB - small, b.tables + NB - small
    for x, y in zip(b.run(), plain):
        assert torch.equal(x, y)


def test_same_result_every_time_and_on_another_stream(cuda_device):
    b = Batch(cuda_device, prefix=3001, own=(900, 20, 400), queries=(4, 1, 9))
    plain, lse = b.run()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = [b.run() for _ in range(3)]
    torch.cuda.current_stream().wait_stream(stream)
    for x, y in got:
        assert torch.equal(x, plain) and torch.equal(y, lse)


def test_captured_steps_follow_the_lengths(cuda_device):
    """Two captured calls replayed in turn while lengths grow, with eager calls between."""
    bound = dict(max_own_tokens=208)
    batches = [Batch(cuda_device, prefix=300, own=(200, 200, 200), seed=s) for s in (1, 2)]
    graphs = []
    for b in batches:
        b.own.fill_(1)
        b.run(**bound)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            result = b.run(**bound)
        graphs.append((graph, result))
    for step in range(4):
        for b, (graph, result) in zip(batches, graphs):
            b.own.copy_(torch.tensor([3 + 40 * step, 200 - step, 64 * step]))
            graph.replay()
            eager = b.run(**bound)
            torch.cuda.synchronize()
            assert torch.equal(result[0], eager[0]) and torch.equal(result[1], eager[1])
            b.check(*result)


def test_parts_join_by_lse(cuda_device):
    """The results over the prefix alone and the own tokens alone, joined by their lse."""
    b = Batch(cuda_device, prefix=200, own=(30, 41), dtype=F16)
    whole, _ = b.run()
    none = torch.zeros_like(b.own)
    p, lp = native_gpu.shared_prefix_attention(b.query, b.cache, b.prefix_ids, 200, b.tables, none,
                                               return_lse=True)
    o, lo = native_gpu.shared_prefix_attention(b.query, b.cache, None, 0, b.tables, b.own,
                                               return_lse=True)
    w = torch.sigmoid(lp - lo)[..., None]
    joined = w * p.float() + (1 - w) * o.float()
    assert (joined - whole.float()).abs().max() < 4 * 2.0 ** -11 * 4  # four roundings of |v| < 4


def test_empty_calls(cuda_device):
    b = Batch(cuda_device, prefix=20, own=(5, 6), D=64)
    got, lse = native_gpu.shared_prefix_attention(
        b.query[:0], b.cache, b.prefix_ids, 20, b.tables[:0], b.own[:0], return_lse=True)
    assert got.shape == (0, 8, 64) and lse.shape == (0, 8)
    starts = torch.zeros(3, dtype=torch.int64, device=cuda_device)
    got, lse = native_gpu.shared_prefix_attention(
        b.query, b.cache, b.prefix_ids, 20, b.tables, b.own, query_starts=starts, return_lse=True)
    assert not got.any() and (lse == -math.inf).all()


def test_refusals(cuda_device):
    b = Batch(cuda_device, prefix=20, own=(5, 6), D=64)

    def refused(match, **kw):
        args = dict(query=b.query, kv_cache=b.cache, prefix_block_ids=b.prefix_ids,
                    prefix_tokens=20, block_tables=b.tables, own_tokens=b.own)
        args.update(kw)
        with pytest.raises(RuntimeError, match=match):
            native_gpu.shared_prefix_attention(**args)

    refused("same dtype|queries' dtype", query=b.query.half())
    refused("float16 or bfloat16", query=b.query.float())
    refused("head_dim differs", query=b.query[..., :32])
    refused("channels must be contiguous",
            query=b.query.transpose(1, 2).contiguous().transpose(1, 2))
    refused("multiple of the cache's heads", query=b.query[:, :3])
    refused("kv_cache device", query=b.query.cpu())
    refused("requires a gradient", query=b.query.clone().requires_grad_())
    refused("prefix tokens exceed", prefix_tokens=33)
    refused("prefix tokens exceed", prefix_block_ids=None)
    refused("must not be negative", prefix_tokens=-1)
    refused("must be a contiguous int64 vector", own_tokens=b.own.int())
    refused("must have 2 values", own_tokens=b.own[:1])
    refused("must have 3 values", query_starts=b.own)
    refused("int64 .requests, blocks.", block_tables=b.tables.int())
    refused("one query token", query=b.query[:1])
    refused("exceeds the block tables", max_own_tokens=1000)
    refused("scales are for float8", k_scale=0.5)
    refused("out must have", out=b.query[:1].clone())
    refused("rank 5", kv_cache=b.cache[0])
    refused("contiguous", kv_cache=b.cache[:, :, :, :1])


@pytest.mark.parametrize("own,queries,bound", [((20,), (5,), 10), ((20, 7), (5, 7), 10),
                                               ((300, 41, 3), (40, 1, 9), 200),
                                               ((600, 90), (200, 90), 450), ((30, 12), (3, 4), 0)])
@pytest.mark.parametrize("prefix", [0, 75, 900])
def test_lengths_above_the_bound(cuda_device, own, queries, bound, prefix):
    """A row's place follows from its request's whole length, and the bound only hides tokens: each
    row against a request of its own that has the tokens the row sees."""
    b = Batch(cuda_device, prefix=prefix, own=own, queries=queries, heads=2, group=3, D=64)
    got = b.run(max_own_tokens=bound)
    seen = [min(max(n - c + i + 1, 0), bound) for n, c in zip(own, queries) for i in range(c)]
    count = torch.tensor(queries, device=cuda_device)
    b.tables = torch.repeat_interleave(b.tables, count, 0)
    b.own, b.starts = torch.tensor(seen, device=cuda_device), None
    b.check(*got)


def test_lengths_above_the_block_tables(cuda_device):
    """The same where the bound is what the tables hold."""
    b = Batch(cuda_device, prefix=50, own=(64, 64), queries=(9, 5), D=64)
    b.own.copy_(torch.tensor([70, 66]))
    got = b.run()
    seen = [min(70 - 9 + i + 1, 64) for i in range(9)] + [min(66 - 5 + i + 1, 64) for i in range(5)]
    b.tables = torch.repeat_interleave(b.tables, torch.tensor([9, 5], device=cuda_device), 0)
    b.own, b.starts = torch.tensor(seen, device=cuda_device), None
    b.check(*got)


@pytest.mark.parametrize("far", [1 << 31, (1 << 40) + 7, (1 << 62)])
def test_lengths_past_32_bits(cuda_device, far):
    b = Batch(cuda_device, prefix=50, own=(64, 33), queries=(9, 5), D=64)
    b.own[0] = far
    got, _ = b.run()
    b.own[0] = 64 + 9
    want, _ = b.run()
    assert torch.equal(got, want)


@pytest.mark.parametrize("group", [1, 16, 17, 40, 200])
@pytest.mark.parametrize("own", [(20, 3), (2000,)])
def test_one_query_each_whatever_the_bound(cuda_device, group, own):
    """Without query_starts every request has one query, and a bound of none says nothing."""
    b = Batch(cuda_device, prefix=40, own=own, D=64, heads=1, group=group)
    out = torch.full_like(b.query, math.nan)
    b.check(*b.run(max_query_tokens=0, out=out))


@pytest.mark.parametrize("own", [(20,), (20, 3), (3000, 40)])  # one part, and several
@pytest.mark.parametrize("group", [2, 40])
@pytest.mark.parametrize("value", [math.inf, math.nan, 1.0])
def test_rows_of_scores_of_minus_infinity(cuda_device, own, group, value):
    """Tokens that are seen, with nothing but scores of -infinity: the row is zero, whatever
    the values are."""
    b = Batch(cuda_device, prefix=0, own=own, D=64, heads=1, group=group)
    b.cache[0, :, :, :, 0] = -math.inf
    b.cache[1, :, :, :, 3] = value
    b.query[:, ::2, 0] = 1.0
    b.query[:, 1::2, 0] = -1.0  # the others see scores of infinity: no defined weights
    got, lse = b.run()
    assert not got[:, ::2].any() and (lse[:, ::2] == -math.inf).all()
    assert got[:, 1::2].isnan().all()


# requests, their queries and rows of a KV head a query: workgroups of 16, 64, 128 and 256 rows
# for the batch and for a request, as far as a head size has them
SHAPES = {"16_16": (2, 1, 4), "64_16": (8, 1, 4), "64_64": (2, 5, 5), "128_16": (20, 1, 5),
          "128_64": (6, 5, 5), "128_128": (3, 20, 5), "one_128": (1, 21, 5), "256": (2, 31, 5)}


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("D", [40, 64, 72, 80, 96, 120, 128, 136, 192, 256])
@pytest.mark.parametrize("dtype,cache_dtype", [(BF16, FP8), (F16, FP8), (BF16, BF16), (F16, F16)])
def test_every_type_and_size_in_every_shape(cuda_device, shape, D, dtype, cache_dtype):
    requests, queries, group = SHAPES[shape]
    own = [queries + (53 * i) % 170 for i in range(requests)]
    counts = [queries - i % 2 * (queries // 3) for i in range(requests)]
    b = Batch(cuda_device, prefix=397, own=own, queries=counts if queries > 1 else None, heads=2,
              group=group, D=D, dtype=dtype, cache_dtype=cache_dtype, bs=(5, 24, 16)[D // 8 % 3],
              order=("kv_first", "blocks_first")[D // 8 % 2], seed=D)
    b.check(*b.run(max_query_tokens=queries))


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("D,bs", [(64, 16), (80, 24), (128, 5), (136, 24)])
def test_odd_values_of_an_e4m3_cache(cuda_device, shape, D, bs):
    """NaN among the values, in tiles that all rows see and in those that some see."""
    requests, queries, group = SHAPES[shape]
    own = [queries + (53 * i) % 170 for i in range(requests)]
    b = Batch(cuda_device, prefix=130, own=own, queries=[queries] * requests, heads=2, group=group,
              D=D, cache_dtype=FP8, bs=bs, seed=D)
    bound = dict(max_query_tokens=queries)
    whole, whole_lse = b.run(**bound)
    b.check(whole, whole_lse)
    marks = [(b.prefix_ids, 3, 0, 5), (b.prefix_ids, 129, 1, 6), (b.tables[0], own[0] - 1, 0, 9),
             (b.tables[-1], max(own[-1] - 3, 0), 1, D - 1), (b.tables[-1], 0, 1, 0)]
    cells = b.cache.view(torch.uint8)
    for table, t, h, d in marks:
        cells[1, int(table[t // bs]), t % bs, h, d] = 0x7f + 0x80 * (d % 2)
    got, lse = b.run(**bound)
    ref = pagedref.attend(b.query, b.cache, b.prefix_ids, b.prefix, b.tables, b.own, b.starts,
                          None, b.k_scale, b.v_scale)[0]
    fine = ref.isfinite()
    assert not fine.all() and torch.equal(got.isfinite(), fine)
    assert torch.equal(got[fine], whole[fine]) and torch.equal(lse, whole_lse)


@pytest.mark.parametrize("cache_dtype", [BF16, FP8])
def test_captured_ragged_queries_follow_starts_and_lengths(cuda_device, cache_dtype):
    """A captured call with query_starts, replayed with other rows for each request, rows of no
    request, and lengths past the bound; eager calls in between."""
    b = Batch(cuda_device, prefix=300, own=(200, 200, 200), queries=(4, 4, 4), D=64,
              cache_dtype=cache_dtype, seed=4)
    bound = dict(max_query_tokens=9, max_own_tokens=160)
    b.run(**bound)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, lse = b.run(**bound)
    for starts, own in (((0, 4, 8, 12), (200, 170, 31)), ((1, 1, 10, 11), (5, 163, 160)),
                        ((0, 9, 9, 9), (161, 0, 3)), ((2, 3, 5, 12), (1, 2, 168))):
        b.starts.copy_(torch.tensor(starts))
        b.own.copy_(torch.tensor(own))
        b.query.normal_()
        graph.replay()
        eager, eager_lse = b.run(**bound)
        torch.cuda.synchronize()
        assert torch.equal(got, eager) and torch.equal(lse, eager_lse)
        rows = torch.zeros(12, dtype=torch.bool)
        rows[starts[0]:starts[-1]] = True
        assert not got[~rows].any() and (lse[~rows] == -math.inf).all()
        # each row against a request of its own with the tokens it sees
        seen, request = [], []
        for r in range(3):
            n = starts[r + 1] - starts[r]
            seen += [min(max(own[r] - n + i + 1, 0), 160) for i in range(n)]
            request += [r] * n
        one = Batch.__new__(Batch)
        one.__dict__.update(b.__dict__)
        one.query, one.starts = b.query[starts[0]:starts[-1]], None
        one.tables, one.own = b.tables[request], torch.tensor(seen, device=cuda_device)
        one.check(got[starts[0]:starts[-1]], lse[starts[0]:starts[-1]])


def test_inference_mode(cuda_device):
    b = Batch(cuda_device, prefix=50, own=(9, 20), D=64)
    plain, lse = b.run()
    with torch.inference_mode():
        b.query = b.query.clone()
        got, again = b.run()
    assert torch.equal(got, plain) and torch.equal(again, lse)
    b.check(*b.run())  # an inference tensor outside of it
