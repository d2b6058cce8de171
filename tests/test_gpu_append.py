"""append_kv_cache on the GPU against its plain 64-bit form (tests/pagedref.py)."""
import math

import pytest
import torch

from origami_amd.lossless import native_gpu
from tests import pagedref

pytestmark = pytest.mark.gpu
BF16, F16, FP8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def table_of(positions, rot, dev):
    angle = (torch.arange(positions, dtype=torch.float64)[:, None]
             * 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot))
    return torch.cat((angle.cos(), angle.sin()), 1).float().to(dev)


class Tokens:
    def __init__(self, dev, *, T=19, Hq=4, H=2, D=128, bs=16, dtype=BF16, cache_dtype=None,
                 order="kv_first", rot=None, interleaved=False, norm=False, norm_dtype=None,
                 seed=0, positions=50000):
        gen = torch.Generator().manual_seed(seed)
        self.dtype, self.D, self.bs = dtype, D, bs
        cache_dtype = cache_dtype or dtype
        NB = -(-T // bs) + 3
        shape = (2, NB, bs, H, D) if order == "kv_first" else (NB, 2, bs, H, D)
        self.cache = torch.randn(*shape, generator=gen).to(cache_dtype).to(dev)
        self.rows = torch.randn(T, Hq + 2 * H, D, generator=gen).to(dtype).to(dev)
        self.query, self.key, self.value = (self.rows[:, :Hq], self.rows[:, Hq:Hq + H],
                                            self.rows[:, Hq + H:])
        self.slots = torch.randperm(NB * bs, generator=gen)[:T].to(dev)
        self.kw = dict(interleaved=interleaved)
        if rot:
            self.kw.update(cos_sin=table_of(positions, rot, dev),
                           positions=torch.randint(0, positions, (T,), generator=gen).to(dev))
        if norm:
            w = [(1 + 0.3 * torch.randn(D, generator=gen)).to(norm_dtype or dtype).to(dev)
                 for _ in range(2)]
            self.kw.update(query_norm=w[0], key_norm=w[1])
        self.k_scale, self.v_scale = (0.07, 0.3) if cache_dtype == FP8 else (1.0, 1.0)

    def run(self, **kw):
        return native_gpu.append_kv_cache(
            self.key, self.value, self.cache, self.slots,
            **{"query": self.query, "k_scale": self.k_scale, "v_scale": self.v_scale, **self.kw,
               **kw})

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
        ct = self.cache.dtype
        got, old = pagedref.cells(self.cache), pagedref.cells(before)
        at = (slots // self.bs, slots % self.bs)
        ref = pagedref.rotate(self.key, *args, kw.get("key_norm"))[place]
        tol = pagedref.rotate_tolerance(ct, ref / self.k_scale, self.key[place] / self.k_scale,
                                        None, None)
        if kw.get("key_norm") is not None:
            most = ref.abs().amax(-1, keepdim=True) / self.k_scale * 2
            tol = tol + (self.D / 2 + 8) * 2.0 ** -24 * 2 * most
        ref = (ref / self.k_scale).clamp(-448, 448) if ct == FP8 else ref
        assert (got[0][at] - ref).abs().le(tol).all()
        ref = self.value[place].double() / self.v_scale
        if ct == FP8:
            ref = ref.clamp(-448, 448)
            tol = pagedref.HALF_STEP[FP8] * (1 + 2.0 ** -20) * ref.abs() + pagedref.TINY[FP8]
            assert (got[1][at] - ref).abs().le(tol).all()
        else:
            assert torch.equal(got[1][at], ref)
        for half in (0, 1):  # everything else stays
            old[half][at] = 0
            got[half][at] = 0
        assert torch.equal(got, old)
        return query


@pytest.mark.parametrize("dtype,cache_dtype", [(BF16, BF16), (F16, F16), (BF16, FP8), (F16, FP8)])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
def test_types_and_sizes(cuda_device, dtype, cache_dtype, D, norm, interleaved):
    for order in ("kv_first", "blocks_first"):
        Tokens(cuda_device, dtype=dtype, cache_dtype=cache_dtype, D=D, norm=norm, rot=D,
               interleaved=interleaved, order=order).check()


@pytest.mark.parametrize("D,rot", [(8, 8), (8, 2), (24, 16), (40, 20), (80, 32), (80, 20), (96, 96),
                                   (128, 64), (128, 6), (136, 136), (192, 64), (248, 248),
                                   (256, 2)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm_dtype", [None, BF16, torch.float32])
def test_rotary_sizes(cuda_device, D, rot, interleaved, norm_dtype):
    for cache_dtype in (BF16, FP8):
        Tokens(cuda_device, D=D, rot=rot, interleaved=interleaved, norm=norm_dtype is not None,
               norm_dtype=norm_dtype, cache_dtype=cache_dtype, seed=D + rot).check()


@pytest.mark.parametrize("T", [0, 1, 2, 63, 257, 1031])
@pytest.mark.parametrize("Hq,H", [(1, 1), (7, 1), (8, 8), (28, 4), (0, 3)])
def test_tokens_and_heads(cuda_device, T, Hq, H):
    t = Tokens(cuda_device, T=T, Hq=Hq, H=H, rot=64, norm=True, D=64, bs=5)
    t.check()


@pytest.mark.parametrize("exponent", [-66, -52, -48, -47, 0, 50])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_norm_without_eps_of_small_and_large_rows(cuda_device, exponent, D):
    """Mean squares of 2^-132 to 2^100.  In binary32 the least lose at most D 2^-150 of
    D 2^-132 or so, 2^-19 of their root; sums and products lose (D / 2 + 8) 2^-24.  A row of
    zeros has no direction: 0 / 0."""
    t = Tokens(cuda_device, D=D, Hq=5, H=3, norm=True)
    t.rows.mul_(2.0 ** exponent)
    t.rows[3, :8] = 0
    query = t.run(eps=0.0)
    key = pagedref.cells(t.cache)[0][t.slots // t.bs, t.slots % t.bs]
    for got, x, w in ((query, t.query, t.kw["query_norm"]), (key, t.key, t.kw["key_norm"])):
        x = x.double()
        ref = x / x.square().mean(-1, keepdim=True).sqrt() * w.double()
        assert ref[3].isnan().all() and got[3].isnan().all()
        got, ref = got.double()[torch.arange(len(x)) != 3], ref[torch.arange(len(x)) != 3]
        assert (got - ref).abs().le(2.0 ** -8 * (1 + 2.0 ** -6) * ref.abs()).all()


def test_plain_append_is_exact(cuda_device):
    """Without a norm or a rotation rows are copied bit by bit, NaN and subnormals included."""
    for dtype in (BF16, F16):
        t = Tokens(cuda_device, dtype=dtype, T=512, D=128)
        t.rows.view(torch.int16).copy_(torch.randint(-2 ** 15, 2 ** 15, t.rows.shape))
        query = t.run()
        at = (t.slots // t.bs, t.slots % t.bs)
        bits = t.cache.view(torch.int16)
        assert torch.equal(bits[0][at], t.key.contiguous().view(torch.int16))
        assert torch.equal(bits[1][at], t.value.contiguous().view(torch.int16))
        assert torch.equal(query.view(torch.int16), t.query.contiguous().view(torch.int16))
        assert native_gpu.append_kv_cache(t.key, t.value, t.cache, t.slots) is None


def test_fp8_values(cuda_device):
    """Ties go to even, what is too large to 448, and NaN stays NaN."""
    t = Tokens(cuda_device, T=1, Hq=0, H=1, D=16, cache_dtype=FP8)
    x = torch.tensor([448., 464., 1e6, -1e6, math.inf, -math.inf, math.nan, 17., 19., 2 ** -10,
                      3 * 2 ** -10, 2 ** -9, -0.0, 0.0, 1.0625, 1.1875])
    want = torch.tensor([448., 448., 448., -448., 448., -448., math.nan, 16., 20., 0., 2 ** -8,
                         2 ** -9, -0.0, 0.0, 1.0, 1.25])
    rows = x.to(BF16).view(1, 1, 16).to(cuda_device)
    native_gpu.append_kv_cache(rows, rows, t.cache, t.slots)
    for half in (0, 1):
        got = pagedref.cells(t.cache)[half].view(-1, 16)[t.slots[0]].cpu().float()
        assert torch.equal(got.nan_to_num(7), want.nan_to_num(7))
        assert torch.equal(got.signbit()[12:14], want.signbit()[12:14])


def test_slots_and_positions_outside(cuda_device):
    """Padding and positions past the table: nothing written, queries of the latter zero."""
    t = Tokens(cuda_device, T=40, rot=32, D=64, positions=100, norm=True)
    n = t.cache.shape[1] * t.bs
    t.slots[3], t.slots[7], t.slots[8], t.slots[20] = -1, n, 1 << 40, -(1 << 50)
    t.kw["positions"][5], t.kw["positions"][6] = -1, 100
    t.kw["positions"][7], t.kw["positions"][9] = 1 << 40, -(1 << 60)
    query = t.check()
    assert not query[[5, 6, 7, 9]].any() and query[[3, 8, 20]].abs().sum() > 0


def test_strides_and_in_place(cuda_device):
    """Rows inside wider ones, head-major rows, rows off 16 bytes; queries rotated in place."""
    for norm in (False, True):
        for rot in (128, 20):
            t = Tokens(cuda_device, T=33, rot=rot, norm=norm)
            plain_query, plain = t.run(), t.cache.clone()
            t.cache.zero_()
            t.key = t.key.transpose(0, 1).contiguous().transpose(0, 1)
            odd = torch.zeros(33 * 2 * 129 + 1, dtype=BF16, device=cuda_device)[1:]
            odd = odd.as_strided((33, 2, 128), (2 * 129, 129, 1))
            odd.copy_(t.value)
            t.value = odd
            t.cache.copy_(plain)
            got = t.run(query_out=t.query)
            assert got.data_ptr() == t.query.data_ptr()
            assert torch.equal(t.query, plain_query) and torch.equal(t.cache, plain)


def test_far_slots_of_a_large_cache(cuda_device):
    NB, bs, H, D = 40000, 16, 8, 256
    t = Tokens(cuda_device, H=H, D=D, bs=bs, rot=D)
    plain_query, small = t.run(), t.cache.shape[1]
    cache = torch.zeros(2, NB, bs, H, D, dtype=BF16, device=cuda_device)
    at = (t.slots // bs, t.slots % bs)
    want = t.cache[0][at], t.cache[1][at]
    t.slots += (NB - small) * bs
    t.cache = cache
    assert torch.equal(t.run(), plain_query)
    at = (t.slots // bs, t.slots % bs)
    assert torch.equal(cache[0][at], want[0]) and torch.equal(cache[1][at], want[1])


def test_captured_and_on_another_stream(cuda_device):
    t = Tokens(cuda_device, T=8, rot=128, norm=True)
    t.run()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = t.run()
    for step in range(4):
        t.rows.normal_()
        t.slots.copy_((t.slots + 5) % (t.cache.shape[1] * t.bs))
        t.kw["positions"].add_(1)
        t.cache.zero_()
        graph.replay()
        torch.cuda.synchronize()
        query, cache = out.clone(), t.cache.clone()
        t.cache.zero_()
        with torch.cuda.stream(stream):
            again = t.run()
        torch.cuda.synchronize()
        assert torch.equal(query, again) and torch.equal(cache, t.cache)


def test_refusals(cuda_device):
    t = Tokens(cuda_device, rot=32, norm=True)

    def refused(match, **kw):
        args = dict(key=t.key, value=t.value, kv_cache=t.cache, slots=t.slots, query=t.query,
                    **t.kw)
        args.update(kw)
        with pytest.raises(RuntimeError, match=match):
            native_gpu.append_kv_cache(**args)

    refused("float16 or bfloat16", key=t.key.float(), value=t.value.float())
    refused("keys' dtype or be float8", kv_cache=t.cache.half())
    refused("same dtype", value=t.value.half())
    refused("heads differ", key=t.key[:, :1])
    refused("same tokens", value=t.value[:3])
    refused("same tokens", query=t.query[:3])
    refused("head_dim differs", query=t.query[..., :64])
    refused("channels must be contiguous", key=t.key.transpose(1, 2).contiguous().transpose(1, 2))
    refused("must have 19 values", slots=t.slots[:3])
    refused("int64 vector", slots=t.slots.int())
    refused("kv_cache device", slots=t.slots.cpu())
    refused("both positions and cos_sin", positions=None)
    refused("float32", cos_sin=t.kw["cos_sin"].double())
    refused("even rotary size", cos_sin=t.kw["cos_sin"][:, :5].contiguous())
    refused("even rotary size", cos_sin=torch.zeros(4, 130, device=cuda_device))
    refused("head_dim values", key_norm=t.kw["key_norm"][:7])
    refused("same dtype", key_norm=t.kw["key_norm"].float())
    refused("must have the keys' dtype or be float32", key_norm=t.kw["key_norm"].half(),
            query_norm=None)
    refused("needs a query", query=None)
    refused("scales are for float8", k_scale=2.0)
    refused("eps must not be negative", eps=-1.0)
    refused("requires a gradient", key=t.key.clone().requires_grad_())
    refused("query's shape", query_out=t.query[:, :1].clone())
    refused("rank 5", kv_cache=t.cache[0])
    before = t.cache.clone()
    assert torch.equal(before, t.cache)


def test_refuses_results_over_inputs(cuda_device):
    t = Tokens(cuda_device, T=8, Hq=2, H=2, D=64, rot=64)
    both = torch.zeros(9, 2, 64, dtype=BF16, device=cuda_device)
    before = t.cache.clone()
    t.query = both[:8]
    with pytest.raises(RuntimeError, match="overlap|single memory location"):
        t.run(query_out=both[1:])
    t.key = both[1:]
    with pytest.raises(RuntimeError, match="overlap|single memory location"):
        t.run(query_out=t.query)
    t.key = t.value
    cells = t.cache.view(-1)[:8 * 2 * 64].view(8, 2, 64)
    with pytest.raises(RuntimeError, match="overlap|single memory location"):
        t.run(query_out=cells)
    assert torch.equal(t.cache, before) and not both.any()
    assert t.run(query_out=t.query) is not None
