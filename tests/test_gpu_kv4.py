"""Paged caches in 4 bits on the GPU: appending, reading and attention, against plain 64-bit forms
(tests/kv4ref.py, tests/pagedref.py)."""
import math

import pytest
import torch

from origami_amd.lossless import native_gpu
from tests import kv4ref, pagedref
from tests.test_gpu_append import Tokens
from tests.test_gpu_prefix_attention import Batch

pytestmark = pytest.mark.gpu
BF16, F16, FP8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


class Tokens4(Tokens):
    """Tokens for a cache in 4 bits, which holds any bytes at first."""

    def __init__(self, dev, *, D=128, seed=0, **kw):
        super().__init__(dev, D=D, seed=seed, **kw)
        gen = torch.Generator().manual_seed(seed + 1)
        shape = (*self.cache.shape[:4], native_gpu.kv4_row_bytes(D))
        self.cache = torch.randint(0, 256, shape, generator=gen, dtype=torch.uint8).to(dev)

    def check(self):
        before = self.cache.clone()
        query = self.run()
        kw = self.kw
        args = (kw.get("cos_sin"), kw.get("positions"), kw["interleaved"])
        ref = pagedref.rotate(self.query, *args, kw.get("query_norm"))
        tol = pagedref.rotate_tolerance(self.dtype, ref, self.query, kw.get("query_norm"), None)
        assert (query.double() - ref).abs().le(tol).all()
        place = (self.slots >= 0) & (self.slots < self.cache[..., 0, 0].numel() // 2)
        if "positions" in kw:
            place &= (kw["positions"] >= 0) & (kw["positions"] < kw["cos_sin"].shape[0])
        slots = self.slots[place]
        at = (slots // self.bs, slots % self.bs)
        got, old = kv4ref.halves(self.cache).clone(), kv4ref.halves(before).clone()
        # values are rounded from what they are: the same bytes, the filling too
        assert torch.equal(got[1][at], kv4ref.pack(self.value[place]))
        # keys after binary32 arithmetic: the nearest of a right scale, up to that arithmetic's error
        ref = pagedref.rotate(self.key, *args, kw.get("key_norm"))[place]
        most = ref.abs().amax(-1, keepdim=True)
        tol = (self.D / 2 + 8) * 2.0 ** -24 * 4 * most
        held = kv4ref.values(got[0][at], self.D)
        power = got[0][at][..., self.D // 2:][..., :math.ceil(self.D / 32)].double() - 127
        low, high = kv4ref.powers((ref.abs() - tol).clamp(min=0)), kv4ref.powers(ref.abs() + tol)
        assert ((power >= low) & (power <= high)).all()
        grid = torch.tensor(kv4ref.GRID, dtype=torch.float64, device=ref.device)
        scale = kv4ref.two_to(power.repeat_interleave(32, -1)[..., :self.D])
        nearest = (ref.abs()[..., None] - grid * scale[..., None]).abs().amin(-1)
        assert ((held - ref).abs() <= nearest + 2 * tol).all()
        for half in (0, 1):  # everything else stays
            old[half][at] = 0
            got[half][at] = 0
        assert torch.equal(got, old)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D,rot", [(8, 8), (24, 24), (40, 20), (64, 64), (80, 32), (96, 96),
                                   (128, 128), (136, 64), (192, 192), (256, 256)])
@pytest.mark.parametrize("norm", [False, True])
def test_append(cuda_device, dtype, D, rot, norm):
    for order in ("kv_first", "blocks_first"):
        for interleaved in (False, True):
            Tokens4(cuda_device, dtype=dtype, D=D, rot=rot, norm=norm, order=order,
                    interleaved=interleaved, seed=D).check()


@pytest.mark.parametrize("T", [0, 1, 2, 63, 257, 1031])
@pytest.mark.parametrize("Hq,H", [(1, 1), (7, 1), (8, 8), (28, 4), (0, 3)])
def test_append_tokens_and_heads(cuda_device, T, Hq, H):
    Tokens4(cuda_device, T=T, Hq=Hq, H=H, rot=64, norm=True, D=64, bs=5).check()


def test_append_padding(cuda_device):
    t = Tokens4(cuda_device, T=40, D=80, rot=80)
    t.slots[3:9] = -1
    t.slots[20] = t.cache[..., 0, 0].numel() // 2
    t.slots[21] = 1 << 40
    t.kw["positions"][30:32] = torch.tensor([-1, 50000], device=cuda_device)
    t.check()


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_append_ties_and_limits(cuda_device, dtype):
    """Every tie between two values, at every scale that is kept and past both ends; zeros of both
    signs; infinities and NaN."""
    dev, D = cuda_device, 64
    half_way = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0])
    near = torch.cat((half_way, half_way * (1 - 2.0 ** -7), half_way * (1 + 2.0 ** -7),
                      torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])))  # 32 numbers
    rows = [torch.cat((near, -near)) * 2.0 ** e for e in range(-30, 17)]
    rows += [torch.cat((near.clamp(max=6.875), near)) * 2.0 ** e for e in (-24, -1, 0, 12, 14)]
    odd = torch.zeros(8, D)
    odd[0, 5] = math.inf
    odd[1, 40] = -math.inf
    odd[2, 0] = math.nan
    odd[3, 63] = math.nan
    odd[3, 1] = -0.0
    odd[4] = -0.0
    odd[5, 3] = 2.0 ** -24
    odd[6, 31], odd[6, 32] = 65504.0, -65504.0
    odd[7, 2], odd[7, 3] = math.nan, math.inf
    x = torch.cat((torch.stack(rows), odd)).to(dtype).to(dev)
    n, bs = x.shape[0], 16
    cache = torch.full((2, -(-n // bs), bs, 1, native_gpu.kv4_row_bytes(D)), 7, dtype=torch.uint8,
                       device=dev)
    slots = torch.arange(n, device=dev)
    native_gpu.append_kv_cache(x[:, None], -x[:, None], cache, slots)
    flat = cache.flatten(1, 2)[:, :n, 0]
    for half, y in ((0, x), (1, -x)):
        want = kv4ref.pack(y)
        fine = ~y.isnan()
        got = kv4ref.values(flat[half], D)
        assert torch.equal(flat[half][:, D // 2:], want[:, D // 2:])
        assert torch.equal(got.isnan(), kv4ref.values(want, D).isnan())
        number = ~got.isnan()
        assert torch.equal(got[number], kv4ref.values(want, D)[number])
        assert torch.equal(torch.signbit(got)[number & fine], torch.signbit(y)[number & fine])


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D", [8, 40, 64, 80, 128, 200, 256])
def test_read_any_bytes(cuda_device, dtype, D):
    """Every value at every scale that the type holds, and NaN."""
    gen = torch.Generator().manual_seed(D)
    NB, bs, H, row = 7, 24, 3, native_gpu.kv4_row_bytes(D)
    rows = torch.randint(0, 256, (2, NB, bs, H, row), generator=gen, dtype=torch.uint8)
    low, high = (1, 252) if dtype == BF16 else (104, 140)
    n = math.ceil(D / 32)
    rows[..., D // 2:D // 2 + n] = torch.randint(low, high + 1, (2, NB, bs, H, n), generator=gen,
                                                 dtype=torch.uint8)
    rows[:, 1, 2, 1, D // 2] = 255
    rows[0, 0, 0, 0, D // 2], rows[0, 0, 1, 0, D // 2] = low, high
    for order in ("kv_first", "blocks_first"):
        cache = rows if order == "kv_first" else rows.transpose(0, 1).contiguous()
        cache = cache.to(cuda_device)
        slots = torch.randint(0, NB * bs, (133,), generator=gen)  # some twice
        slots[5], slots[6], slots[7], slots[8] = -1, NB * bs, 0, 1
        slots[9] = bs + 2
        key, value = native_gpu.read_kv_cache(cache, slots.to(cuda_device), dtype=dtype)
        kv = kv4ref.values(rows, D).flatten(1, 2)
        inside = (slots >= 0) & (slots < NB * bs)
        for half, got in ((0, key), (1, value)):
            want = torch.where(inside[:, None, None], kv[half][slots.clamp(0, NB * bs - 1)], 0.0)
            assert torch.equal(got.cpu().isnan(), want.isnan())
            assert torch.equal(got.cpu().double().nan_to_num(9.0), want.nan_to_num(9.0))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D", [8, 72, 128, 256])
@pytest.mark.parametrize("tokens", [0, 1, 500])
def test_read_other_caches(cuda_device, dtype, D, tokens):
    """Rows of 16 bits come as they are, NaN too; e4m3 times its scale, rounded once."""
    gen, NB, bs, H = torch.Generator().manual_seed(D), 40, 13, 2
    slots = torch.randint(-1, NB * bs, (tokens,), generator=gen).to(cuda_device)
    for cache_dtype in (dtype, FP8):
        cache = torch.randn(NB, 2, bs, H, D, generator=gen).to(cache_dtype).to(cuda_device)
        cache[1, 0, 1, 0, 3] = math.nan
        scales = dict(k_scale=0.3, v_scale=1.7) if cache_dtype == FP8 else {}
        room = torch.full((tokens, 2, H, D + 8), 5.0, dtype=dtype, device=cuda_device)
        results = [(None, None), (room[:, 0, :, :D], room[:, 1, :, :D])]
        if tokens:
            wide = torch.full((tokens, 2 * H, 2 * D + 1), 5.0, dtype=dtype, device=cuda_device)
            results.append((wide[:, 0::2, 1:D + 1], wide[:, 1::2, D + 1:]))  # rows off 16 bytes
        for key_out, value_out in results:
            key, value = native_gpu.read_kv_cache(cache, slots, dtype=dtype, key_out=key_out,
                                                  value_out=value_out, **scales)
            for half, got in ((0, key), (1, value)):
                flat = cache[:, half].flatten(0, 1)
                want = flat.view(torch.uint8 if cache_dtype == FP8 else torch.int16)
                want = want[slots.clamp(min=0)].view(cache_dtype)
                if cache_dtype == FP8:
                    want = (want.float() * scales["k_scale" if half == 0 else "v_scale"]).to(dtype)
                want = torch.where((slots >= 0)[:, None, None], want, torch.zeros_like(want))
                assert torch.equal(got.isnan(), want.isnan())
                same = got.contiguous().view(torch.int16) == want.contiguous().view(torch.int16)
                assert (same | want.isnan()).all()
        assert (room[..., D:] == 5.0).all()


def test_append_then_read(cuda_device):
    """What is read is what was appended, within half a step of 4 bits."""
    t = Tokens4(cuda_device, T=300, D=128, rot=128, norm=True)
    t.run()
    key, value = native_gpu.read_kv_cache(t.cache, t.slots, dtype=BF16)
    assert torch.equal(value.double(), kv4ref.values(kv4ref.pack(t.value), 128))
    ref = pagedref.rotate(t.key, t.kw["cos_sin"], t.kw["positions"], False, t.kw["key_norm"])
    step = kv4ref.two_to(kv4ref.powers(ref).repeat_interleave(32, -1))
    assert ((key.double() - ref).abs() <= (1 + 1e-5) * step).all()  # half of the largest step


class Batch4(Batch):
    """A batch on a cache in 4 bits; every cell that the batch does not hold is NaN."""

    def __init__(self, dev, *, D=128, **kw):
        super().__init__(dev, D=D, **kw)
        self.cache = kv4ref.pack(self.cache)

    def check(self, got, lse, rows=None, scale=None):
        held = self.cache
        self.cache = kv4ref.cells(held, self.D)  # float64, keys and values first
        try:
            super().check(got, lse, rows, scale)
        finally:
            self.cache = held


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("order", ["kv_first", "blocks_first"])
def test_attend_types_and_sizes(cuda_device, dtype, D, order):
    b = Batch4(cuda_device, D=D, dtype=dtype, order=order, prefix=150, own=(1, 40, 16, 77, 33))
    b.check(*b.run())


@pytest.mark.parametrize("heads,group", [(1, 1), (3, 1), (1, 7), (2, 16), (1, 17), (1, 48), (5, 8)])
@pytest.mark.parametrize("queries", [None, (2, 0, 5, 1)])
@pytest.mark.parametrize("prefix", [0, 70])
@pytest.mark.parametrize("D", [64, 128])
def test_attend_head_groups(cuda_device, heads, group, queries, prefix, D):
    b = Batch4(cuda_device, heads=heads, group=group, D=D, prefix=prefix, own=(9, 3, 50, 1),
               queries=queries, seed=heads * group)
    b.check(*b.run())


@pytest.mark.parametrize("D", [8, 16, 24, 40, 72, 80, 96, 120, 136, 160, 192, 248])
@pytest.mark.parametrize("prefix", [0, 45])
def test_attend_odd_head_sizes(cuda_device, D, prefix):
    b = Batch4(cuda_device, D=D, prefix=prefix, own=(3, 70), seed=D)
    b.check(*b.run())


@pytest.mark.parametrize("bs", [1, 2, 5, 8, 16, 24, 32, 64, 256])
@pytest.mark.parametrize("prefix", [0, 1, 33, 257])
def test_attend_block_sizes(cuda_device, bs, prefix):
    b = Batch4(cuda_device, bs=bs, prefix=prefix, own=(31, 1, 32, 65), D=128, seed=bs + prefix)
    b.check(*b.run())


@pytest.mark.parametrize("own", [(0,), (1,), (130,), (0, 0, 0), (0, 5, 0, 129), (511, 513, 512)])
@pytest.mark.parametrize("prefix", [0, 1, 700])
def test_attend_lengths(cuda_device, own, prefix):
    b = Batch4(cuda_device, prefix=prefix, own=own, D=128, seed=prefix + len(own))
    b.check(*b.run())


@pytest.mark.parametrize("prefix,own", [(5000, (1, 900)), (20011, (40,) * 20), (0, (9001, 17)),
                                        (2500, (2100,)), (0, (3001, 5, 700, 4096) * 5)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_attend_long(cuda_device, prefix, own, dtype):
    b = Batch4(cuda_device, prefix=prefix, own=own, dtype=dtype, seed=prefix)
    b.check(*b.run())
    b.check(*b.run(max_own_tokens=max(own)))


@pytest.mark.parametrize("queries,own,prefix", [
    ((1,), (1,), 0), ((5, 5, 5), (5, 90, 33), 300), ((3, 0, 7), (3, 4, 7), 50),
    ((64, 17), (64, 80), 129), ((130,), (130,), 0), ((200, 1, 77), (233, 9, 77), 400),
    ((129, 300), (400, 300), 64), ((70,) * 6, (75,) * 6, 1000), ((2, 4, 1), (900, 70, 1), 0)])
@pytest.mark.parametrize("heads,group", [(2, 1), (1, 5), (2, 4)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_attend_several_queries(cuda_device, queries, own, prefix, heads, group, dtype):
    b = Batch4(cuda_device, prefix=prefix, own=own, queries=queries, heads=heads, group=group,
               D=64 if group == 1 else 128, dtype=dtype, seed=sum(queries))
    b.check(*b.run())
    b.check(*b.run(max_query_tokens=max(queries), max_own_tokens=max(own)))


def test_attend_queries_beyond_the_own_tokens(cuda_device):
    for prefix in (0, 40):
        b = Batch4(cuda_device, prefix=prefix, own=(2, 0), queries=(6, 3), D=128)
        b.check(*b.run())


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("group", [1, 8, 40])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_attend_nan_reaches_the_rows_that_see_it(cuda_device, D, group, dtype):
    """NaN blocks of values and keys anywhere in the tokens, and values that float16 does not
    have, in workgroups of every shape."""
    for own, queries in (((40, 97), (30, 97)), ((300,), (257,)), ((64, 9), (1, 2)),
                         ((64, 9), None)):
        b = Batch4(cuda_device, prefix=75, own=own, queries=queries, heads=2, group=group, D=D,
                   seed=D + group, dtype=dtype)
        clean = b.cache.clone()
        whole, whole_lse = b.run()
        marks = [(b.prefix_ids, 3, 0, 0, 255), (b.prefix_ids, 74, 1, 1, 255),
                 (b.tables[0], own[0] - 3, 1, D // 32 - 1, 255), (b.tables[-1], own[-1] - 1, 0, 0, 255),
                 (b.tables[0], 2, 0, 1, 150)]
        for table, t, h, g, s in marks:
            b.cache[1, int(table[t // b.bs]), t % b.bs, h, D // 2 + g] = s
        got, lse = b.run()
        kv = kv4ref.cells(b.cache, D)
        kv = torch.where(kv.abs() > torch.finfo(dtype).max, torch.sign(kv) * math.inf, kv)
        ref = pagedref.attend(b.query, kv, b.prefix_ids, b.prefix, b.tables, b.own, b.starts)[0]
        fine = ref.isfinite()
        assert torch.equal(got.isfinite(), fine)
        plain = fine & (ref.abs() < 1000)  # the large values of bfloat16 are no NaN
        untouched = plain.clone()
        if dtype == BF16:
            untouched[..., 32:64] = False
        assert torch.equal(got[untouched], whole[untouched]) and torch.equal(lse, whole_lse)
        # a NaN key makes NaN of the rows that see it
        b.cache = clean
        t = own[-1] - 1
        b.cache[0, int(b.tables[-1][t // b.bs]), t % b.bs, 1, D // 2] = 255
        got, _ = b.run()
        sees = torch.zeros(got.shape[:2], dtype=torch.bool, device=cuda_device)
        sees[-1, group:] = True  # the newest query alone
        assert got[sees].isnan().all() and torch.equal(got[~sees], whole[~sees])


@pytest.mark.parametrize("peak", [0.0, 30.0])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("prefix", [0, 3000])
def test_attend_flat_and_steep_scores(cuda_device, peak, dtype, prefix):
    b = Batch4(cuda_device, prefix=prefix, own=(700, 5), dtype=dtype, peak=peak, seed=3)
    b.check(*b.run())


@pytest.mark.parametrize("B,prefix,D", [(3, 1000, 128), (40, 600, 128), (70, 333, 64),
                                        (40, 600, 192), (33, 0, 128), (33, 0, 64)])
@pytest.mark.parametrize("queries", [1, 3, 11])
def test_attend_batches_in_every_shape(cuda_device, B, prefix, D, queries):
    own = [(37 * i) % 150 + queries for i in range(B)]
    b = Batch4(cuda_device, prefix=prefix, own=own, queries=[queries] * B, heads=1, group=5, D=D,
               seed=B + queries)
    b.check(*b.run())
    if queries == 1:
        b.starts = None
        b.check(*b.run())


def test_attend_blocks_outside_the_cache(cuda_device):
    for prefix in (0, 100):
        b = Batch4(cuda_device, prefix=prefix, own=(70, 40, 33), D=128)
        b.tables[0, 1], b.tables[1, 0], b.tables[2] = -1, 1 << 40, -5
        b.check(*b.run())


def test_attend_strides(cuda_device):
    """Queries and outputs between other rows, and rows off 16 bytes."""
    b = Batch4(cuda_device, prefix=0, own=(70, 400), heads=2, group=3)
    n, D = b.query.shape[0], b.D
    for pad in (8, 1):
        room = torch.zeros(n, 9, D + pad, dtype=BF16, device=cuda_device)
        room[:, 2:8, :D] = b.query
        b.query = room[:, 2:8, :D]
        out = torch.full((n, 7, D + pad), 3.0, dtype=BF16, device=cuda_device)
        got, lse = b.run(out=out[:, :6, :D])
        b.check(got, lse)
        assert (out[:, 6] == 3.0).all() and (out[..., D:] == 3.0).all()


@pytest.mark.parametrize("prefix", [0, 200])
def test_attend_captured_as_lengths_grow(cuda_device, prefix):
    b = Batch4(cuda_device, prefix=prefix, own=(900, 1, 333, 40), D=128)
    grown = b.own.clone()
    b.own.fill_(1)
    b.run(return_lse=False)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = b.run(return_lse=False)
    for part in (0.0, 0.2, 0.5, 1.0, 0.7):
        b.own.copy_((grown * part).long().clamp(min=1))
        graph.replay()
        b.check(out, None)
        eager = b.run(return_lse=False)
        assert torch.equal(out, eager)


def test_attend_on_another_stream(cuda_device):
    b = Batch4(cuda_device, prefix=0, own=(900, 77), D=128)
    want, _ = b.run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, lse = b.run()
    side.synchronize()
    assert torch.equal(got, want)


# ---- attention over many tokens, whose requests are cut into shares by their lengths ----


def lengths_of(requests, most, seed):
    """Lengths with zeros, ones, and one far longer than the others."""
    gen = torch.Generator().manual_seed(seed)
    own = torch.randint(0, most // 8, (requests,), generator=gen)
    own[torch.rand(requests, generator=gen) < 0.2] = 0
    own[torch.rand(requests, generator=gen) < 0.1] = 1
    own[requests // 2] = most
    return tuple(own.tolist())


# on both sides of 64 and 256 requests, of one and of several heads a workgroup
@pytest.mark.parametrize("requests,heads,most", [
    (1, 8, 17000), (2, 8, 9000), (5, 3, 9000), (63, 1, 3000), (64, 8, 1500), (65, 2, 2050),
    (150, 5, 1031), (256, 1, 700), (257, 1, 700), (300, 4, 333)])
@pytest.mark.parametrize("D", [64, 128])
def test_attend_shares_of_any_lengths(cuda_device, requests, heads, most, D):
    b = Batch4(cuda_device, heads=heads, group=2, D=D, prefix=0,
               own=lengths_of(requests, most, requests), seed=requests)
    got, lse = b.run()
    b.check(got, lse)
    if requests * heads > 4:  # every run is the same, sum for sum
        again, again_lse = b.run()
        assert torch.equal(got, again) and torch.equal(lse, again_lse)


@pytest.mark.parametrize("own", [(0,) * 70, (1,) * 70, (0,) * 69 + (2500,), (2500,) + (0,) * 130])
def test_attend_shares_of_empty_requests(cuda_device, own):
    """The bound is of 2500 tokens for each, whatever they hold."""
    b = Batch4(cuda_device, heads=8, group=3, prefix=0, own=own, seed=len(own))
    if max(own) < 2500:
        b.tables = torch.cat([b.tables, b.tables[:, :1].expand(-1, 160)], 1).contiguous()
    got, lse = b.run()
    b.check(got, lse)
    empty = b.own == 0
    assert (got[empty] == 0).all() and (lse[empty] == -math.inf).all()


@pytest.mark.parametrize("D", [24, 80, 120, 200])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_attend_shares_of_odd_head_sizes(cuda_device, D, dtype):
    b = Batch4(cuda_device, heads=4, group=5, D=D, dtype=dtype, prefix=0, bs=24,
               own=(3000, 0, 77, 1999) * 5, seed=D)
    b.check(*b.run())


@pytest.mark.parametrize("queries", [(1, 0, 3, 2) * 20, (0,) * 79 + (1,), (2,) * 80])
def test_attend_shares_of_several_queries(cuda_device, queries):
    own = [n + q if n + q > 1 else q for n, q in zip(lengths_of(80, 1700, 7), queries)]
    b = Batch4(cuda_device, heads=2, group=4, prefix=0, own=own, queries=queries, seed=80)
    b.check(*b.run())


def test_attend_shares_of_a_prefix(cuda_device):
    """One request reads the prefix with its own tokens, in the same shares."""
    for own, queries in (((900,), (3,)), ((0,), None), ((5,), (5,))):
        b = Batch4(cuda_device, heads=8, group=4, prefix=17001, own=own, queries=queries, seed=9)
        b.check(*b.run())


@pytest.mark.parametrize("requests", [12, 90, 270])
def test_attend_shares_captured_as_lengths_grow(cuda_device, requests):
    """A bound far above the lengths, of which the graph knows nothing."""
    b = Batch4(cuda_device, heads=4, group=2, prefix=0, own=lengths_of(requests, 2600, 3), seed=3)
    grown = b.own.clone()
    b.own.fill_(1)
    b.run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = b.run()
    for part in (0.0, 0.05, 0.5, 1.0, 0.0):
        b.own.copy_((grown * part).long())
        graph.replay()
        b.check(out, lse)
        eager, eager_lse = b.run()
        assert torch.equal(out, eager) and torch.equal(lse, eager_lse)


@pytest.mark.parametrize("blocks", [1100, 4400, 9000])
def test_attend_shares_of_bounds_far_above_the_lengths(cuda_device, blocks):
    """Block tables of up to 144000 tokens for requests of up to 1700."""
    b = Batch4(cuda_device, heads=8, group=2, prefix=0, own=lengths_of(24, 1700, 11), seed=11)
    b.tables = torch.cat([b.tables, torch.full((24, blocks - b.tables.shape[1]), -1,
                                               device=cuda_device)], 1)
    b.check(*b.run())


def test_attend_shares_of_lengths_past_the_bound(cuda_device):
    """Lengths that the bound cuts off, up to the largest of their type, are no more than it."""
    b = Batch4(cuda_device, heads=8, group=2, prefix=0, own=(2000,) * 40, seed=5)
    whole, whole_lse = b.run(max_own_tokens=1600)
    b.own[:] = 1600
    want, want_lse = b.run(max_own_tokens=1600)
    assert torch.equal(whole, want) and torch.equal(whole_lse, want_lse)
    b.check(want, want_lse)
    b.own[3], b.own[4], b.own[5] = 1 << 62, -7, torch.iinfo(torch.int64).min
    got, lse = b.run(max_own_tokens=1600)
    assert (got[4:6] == 0).all() and (lse[4:6] == -math.inf).all()
    b.own[3], b.own[4], b.own[5] = 1600, 0, 0
    b.check(got, lse)


def test_attend_shares_nan_in_one_request(cuda_device):
    b = Batch4(cuda_device, heads=4, group=2, prefix=0, own=(1500, 2500, 0, 900) * 10, seed=6)
    whole, whole_lse = b.run()
    for r, t in ((1, 0), (1, 2499), (36, 1499), (39, 33)):
        b.cache[0, int(b.tables[r, t // b.bs]), t % b.bs, 2, b.D // 2] = 255
    got, lse = b.run()
    hit = torch.zeros(got.shape[:2], dtype=torch.bool, device=cuda_device)
    for r in (1, 36, 39):
        hit[r, 4:6] = True
    assert got[hit].isnan().all() and lse[hit].isnan().all()
    assert torch.equal(got[~hit], whole[~hit]) and torch.equal(lse[~hit], whole_lse[~hit])


def test_refusals(cuda_device):
    b = Batch4(cuda_device, prefix=0, own=(40, 3), D=128)
    whole = b.cache
    b.cache = whole[..., :64].contiguous()
    with pytest.raises(RuntimeError, match="rows of 68 bytes for 128 channels, not of 64"):
        b.run()
    b.cache = whole
    with pytest.raises(RuntimeError, match="for float8_e4m3fn caches"):
        b.run(k_scale=2.0)
    b.cache = whole[:, 1:]
    with pytest.raises(RuntimeError, match="must be contiguous"):
        b.run()
    t = Tokens4(cuda_device, D=64)
    before = t.cache.clone()
    t.cache = torch.zeros(2, 4, 16, 2, 64, dtype=torch.uint8, device=cuda_device)
    with pytest.raises(RuntimeError, match="rows of 36 bytes for 64 channels, not of 64"):
        t.run()
    slots = torch.zeros(3, dtype=torch.int64, device=cuda_device)
    read = native_gpu.read_kv_cache
    with pytest.raises(RuntimeError, match="no head_dim has rows of 72 bytes"):
        read(torch.zeros(2, 4, 16, 2, 72, dtype=torch.uint8, device=cuda_device), slots)
    with pytest.raises(RuntimeError, match="float16 or bfloat16"):
        read(before, slots, dtype=torch.float32)
    with pytest.raises(RuntimeError, match="keys' dtype or be float8_e4m3fn"):
        read(torch.zeros(2, 4, 16, 2, 64, dtype=F16, device=cuda_device), slots, dtype=BF16)
    with pytest.raises(RuntimeError, match="for float8_e4m3fn caches"):
        read(before, slots, v_scale=2.0)
    with pytest.raises(RuntimeError, match="contiguous int64 vector"):
        read(before, slots.int())
    with pytest.raises(RuntimeError, match="device"):
        read(before, slots.cpu())
    room = torch.zeros(3, 2, 64, dtype=BF16, device=cuda_device)
    with pytest.raises(RuntimeError, match="must not overlap"):
        read(before, slots, key_out=room, value_out=room)
    with pytest.raises(RuntimeError, match="must not overlap itself"):
        read(before, slots, key_out=room[:1].expand(3, 2, 64))
    with pytest.raises(RuntimeError, match="slots, heads"):
        read(before, slots, key_out=room[:2])
    memory = torch.zeros(1 << 16, dtype=torch.uint8, device=cuda_device)
    cache = memory[:2 * 4 * 16 * 2 * 36].view(2, 4, 16, 2, 36)
    with pytest.raises(RuntimeError, match="must not overlap kv_cache"):
        read(cache, slots, key_out=memory[512:512 + 768].view(BF16).view(3, 2, 64))


def test_attend_shares_memory_is_not_of_the_bound(cuda_device):
    """What a call takes beside its results follows from the batch, not from its block tables."""
    requests, heads, group = 128, 8, 8
    b = Batch4(cuda_device, heads=heads, group=group, prefix=0, own=lengths_of(requests, 900, 4))
    used = []
    for blocks in (b.tables.shape[1], 2048, 65536):
        b.tables = torch.cat([b.tables, torch.full((requests, blocks - b.tables.shape[1]), -1,
                                                   device=cuda_device)], 1)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        got, lse = b.run()
        used.append(torch.cuda.max_memory_allocated() - before)
        b.check(got, lse)
    results = got.nbytes + lse.nbytes
    # 2048 shares or two a request and head, with `group` rows each; lists of 8 bytes a row
    most = (2048 + 2 * requests * heads) * group * 130 * 4 + 8 * lse.numel() + 4096
    assert max(used) <= results + most


@pytest.mark.parametrize("filled", [0xff, 0x7f, 0x00, 0x80])
def test_attend_shares_leave_other_rows(cuda_device, filled):
    """Rows before the first request and behind the last are left as they were; a request with more
    queries than its bound harms no other, whatever the workspace held before."""
    queries = (2, 1, 5, 0, 2, 1) * 9
    own = [n + q for n, q in zip(lengths_of(54, 2300, 8), queries)]
    b = Batch4(cuda_device, heads=4, group=4, prefix=0, own=own, queries=queries, seed=2)
    b.query = torch.cat([b.query[:3], b.query, b.query[:4]])
    b.starts = b.starts + 3
    n = b.query.shape[0]
    out = torch.full_like(b.query, 3.0)
    # the memory that the call's workspace gets: its own size first, then filled
    b.run(out=out, max_query_tokens=2)
    workspaces = [torch.full((1 << k,), filled, dtype=torch.uint8, device=cuda_device)
                  for k in range(21, 28)]
    del workspaces
    out.fill_(3.0)
    got, lse = b.run(out=out, max_query_tokens=2)
    assert (got[:3] == 3.0).all() and (got[n - 4:] == 3.0).all()
    request = torch.repeat_interleave(torch.arange(54), torch.tensor(queries))
    fine = torch.cat([torch.zeros(3, dtype=torch.bool), torch.tensor(queries)[request] <= 2,
                      torch.zeros(4, dtype=torch.bool)]).to(cuda_device)
    b.check(got, lse, rows=fine)


@pytest.mark.parametrize("requests,bound", [(60, 4096), (256, 40960), (257, 40960), (400, 131072)])
def test_attend_many_requests_with_a_bound_far_above(cuda_device, requests, bound):
    """On both sides of where shares end; the longest request far beyond the others."""
    b = Batch4(cuda_device, heads=1, group=3, D=64, prefix=0, seed=requests,
               own=lengths_of(requests, 1100, requests))
    want, want_lse = b.run()
    b.check(want, want_lse)
    b.tables = torch.cat([b.tables, torch.full((requests, bound // b.bs - b.tables.shape[1]), -1,
                                               device=cuda_device)], 1)
    b.check(*b.run())


@pytest.mark.parametrize("requests", [24, 200, 270])
def test_attend_beside_other_lengths(cuda_device, requests):
    """One request's length changes: the others' results are as near as before, but in shares (up to
    256 requests) their sums may be made of other parts.  In equal ranges, and over other types of
    caches, they are the same bits."""
    own = [1 + n for n in lengths_of(requests, 2500 if requests < 100 else 700, 12)]
    for make in (Batch4, Batch):
        b = make(cuda_device, heads=4 if requests < 100 else 1, group=2, D=64, prefix=0, own=own,
                 seed=4)
        most, first = max(own), requests // 2
        whole, whole_lse = b.run(max_own_tokens=most)
        b.check(whole, whole_lse)
        b.own[first] = 3  # the longest
        got, lse = b.run(max_own_tokens=most)
        b.check(got, lse)
        again, again_lse = b.run(max_own_tokens=most)
        assert torch.equal(got, again) and torch.equal(lse, again_lse)
        others = torch.arange(requests, device=cuda_device) != first
        if make is Batch or requests > 256:
            assert torch.equal(got[others], whole[others])
            assert torch.equal(lse[others], whole_lse[others])


@pytest.mark.parametrize("D", [16, 32, 48, 64, 80, 96, 112, 128])
def test_read_refuses_8_bit_caches_seen_as_bytes(cuda_device, D):
    """A view of an e4m3 cache, as the layout calls take it, is not taken for 4 bits, though some
    head size has rows of as many bytes."""
    gen = torch.Generator().manual_seed(D)
    cache = torch.randn(2, 4, 16, 3, D, generator=gen).to(FP8).to(cuda_device)
    slots = torch.arange(33, device=cuda_device)
    read = native_gpu.read_kv_cache
    with pytest.raises(RuntimeError, match="head_dim must be given"):
        read(cache.view(torch.uint8), slots)
    with pytest.raises(RuntimeError, match=f"bytes for {D} channels, not of {D}"):
        read(cache.view(torch.uint8), slots, head_dim=D)
    room = torch.empty(33, 3, D, dtype=BF16, device=cuda_device)
    with pytest.raises(RuntimeError, match=f"bytes for {D} channels, not of {D}"):
        read(cache.view(torch.uint8), slots, value_out=room)
    with pytest.raises(RuntimeError, match="head_dim differs from the kv_cache's"):
        read(cache, slots, head_dim=D + 8)
    key, value = read(cache, slots, head_dim=D)
    for half, got in ((0, key), (1, value)):
        assert torch.equal(got.float(), cache[half].flatten(0, 1)[:33].float())


@pytest.mark.parametrize("D", [24, 56, 88, 120, 144, 176, 208, 240])
def test_read_of_rows_of_whole_16_bytes(cuda_device, D):
    """4-bit rows of as many bytes as common head sizes have in 8 bits, where it is said."""
    gen = torch.Generator().manual_seed(D)
    kv = torch.randn(2, 4, 16, 3, D, generator=gen)
    cache = kv4ref.pack(kv).to(cuda_device)
    assert cache.shape[-1] % 16 == 0
    slots = torch.arange(33, device=cuda_device)
    want = kv4ref.values(cache, D).flatten(1, 2)[:, :33]
    room = torch.empty(33, 3, D, dtype=F16, device=cuda_device)
    for kw in (dict(head_dim=D), dict(key_out=room), dict(value_out=room)):
        key, value = native_gpu.read_kv_cache(cache, slots, dtype=F16, **kw)
        assert torch.equal(key.double(), want[0]) and torch.equal(value.double(), want[1])
    for other in (D + 8, D - 8):
        with pytest.raises(RuntimeError, match=f"bytes for {other} channels"):
            native_gpu.read_kv_cache(cache, slots, head_dim=other)
    with pytest.raises(RuntimeError, match="multiple of 8"):
        native_gpu.read_kv_cache(cache, slots, head_dim=D + 1)


@pytest.mark.parametrize("heads,bound", [(1, 40000), (1, 1 << 20), (3, 1 << 20), (8, 1 << 22)])
def test_attend_one_request_in_all_shares(cuda_device, heads, bound):
    """A request beside empty ones is cut into as many parts as a row can have, whatever the bound
    allows."""
    own = (0,) * 5 + (40000,) + (1,) * 3
    b = Batch4(cuda_device, heads=heads, group=2, D=8, prefix=0, own=own, seed=heads)
    want, want_lse = b.run()
    b.check(want, want_lse)
    width = -(-bound // b.bs) - b.tables.shape[1]
    b.tables = torch.cat([b.tables, torch.full((len(own), width), -1, device=cuda_device)], 1)
    b.check(*b.run())
