"""A prompt's prefix restored into the paged cache, then a batch that goes on from it: drafted
prompts first, single tokens after, each step appended and attended to."""
import pytest
import torch

from origami_amd.layout import kv_symbol_layout
from origami_amd.lossless import native_gpu
from tests import pagedref
from tests.test_gpu_append import table_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,cache_dtype", [(torch.bfloat16, torch.bfloat16),
                                               (torch.float16, torch.float8_e4m3fn)])
@pytest.mark.parametrize("order", ["kv_first", "blocks_first"])
@pytest.mark.parametrize("captured", [False, True])
def test_restore_append_attend(cuda_device, dtype, cache_dtype, order, captured):
    dev, gen = cuda_device, torch.Generator().manual_seed(7)
    B, Hq, H, D, bs, prefix, width = 3, 8, 2, 64, 16, 100, 6
    shared = -(-prefix // bs)
    NB = shared + B * width + 4

    def cache_of(values):
        return values if order == "kv_first" else values.transpose(0, 1).contiguous()

    # the prefix as it was saved: rotated keys of 100 tokens in another cache
    saved = cache_of(torch.randn(2, NB, bs, H, D, generator=gen).to(cache_dtype)).to(dev)
    saved_ids = torch.randperm(NB, generator=gen)[:shared].to(dev)
    C = D * saved.element_size()
    layout = kv_symbol_layout(prefix, H, C, 8, [[0, H, 0, C, 0, 2 * prefix]])
    stream = native_gpu.pack_from_kv_cache(saved, saved_ids, prefix, layout)

    cache = cache_of(torch.zeros(2, NB, bs, H, D).to(cache_dtype)).to(dev)
    ids = torch.randperm(NB, generator=gen).to(dev)
    prefix_ids, tables = ids[:shared], ids[shared:shared + B * width].view(B, width)
    native_gpu.unpack_to_kv_cache(stream, layout, prefix, cache, prefix_ids)

    table = table_of(1000, D, dev)
    norms = [(1 + 0.2 * torch.randn(D, generator=gen)).to(dtype).to(dev) for _ in range(2)]
    scales = dict(k_scale=0.05, v_scale=0.04) if cache_dtype == torch.float8_e4m3fn else {}
    own = torch.zeros(B, dtype=torch.int64, device=dev)

    def layer(rows, positions, slots, starts):
        query = native_gpu.append_kv_cache(
            rows[:, Hq:Hq + H], rows[:, Hq + H:], cache, slots, query=rows[:, :Hq],
            positions=positions, cos_sin=table, query_norm=norms[0], key_norm=norms[1], **scales)
        return query, native_gpu.shared_prefix_attention(
            query, cache, prefix_ids, prefix, tables, own, query_starts=starts,
            max_query_tokens=None if starts is None else 9, **scales)

    def step(counts, run):
        """Appends counts[r] tokens of each request and checks what they attend to."""
        n, r = sum(counts), torch.repeat_interleave(torch.arange(B), torch.tensor(counts)).to(dev)
        i = torch.cat([torch.arange(c) for c in counts]).to(dev)
        at = own[r] + i
        own.add_(torch.tensor(counts, device=dev))
        rows = torch.randn(n, Hq + 2 * H, D, generator=gen).to(dtype).to(dev)
        slots = tables[r, at // bs] * bs + at % bs
        starts = None
        if counts != [1] * B:
            starts = torch.tensor([0, *counts]).cumsum(0).to(dev)
        query, got = run(rows, prefix + at, slots, starts)
        # the query against the plain form; what the cache holds is checked by the append's tests
        ref = pagedref.rotate(rows[:, :Hq], table, prefix + at, False, norms[0])
        tol = pagedref.rotate_tolerance(dtype, ref, rows[:, :Hq], norms[0], None)
        assert (query.double() - ref).abs().le(tol).all()
        key = pagedref.rotate(rows[:, Hq:Hq + H], table, prefix + at, False, norms[1])
        held = pagedref.cells(cache)[0][slots // bs, slots % bs] * scales.get("k_scale", 1.0)
        assert ((held - key).abs() <= 2 * pagedref.HALF_STEP[cache_dtype] * key.abs() + 0.01).all()
        ref, _, size, largest = pagedref.attend(query, cache, prefix_ids, prefix, tables, own,
                                                starts, **scales)
        tol = pagedref.attend_tolerance(dtype, D, prefix + int(own.max()), size, largest, ref)
        assert (got.double() - ref).abs().le(tol).all()

    # the restored prefix is the saved one
    t = torch.arange(prefix, device=dev)
    was, now = pagedref.cells(saved), pagedref.cells(cache)
    assert torch.equal(was[:, saved_ids[t // bs], t % bs], now[:, prefix_ids[t // bs], t % bs])

    step([5, 9, 1], layer)
    step([1, 1, 1], layer)
    if not captured:
        for counts in ([1, 1, 1], [2, 0, 3], [1, 1, 1]):
            step(counts, layer)
        return
    inputs = (torch.zeros(B, Hq + 2 * H, D, dtype=dtype, device=dev),
              torch.zeros(B, dtype=torch.int64, device=dev),
              torch.full((B,), -1, dtype=torch.int64, device=dev))
    layer(*inputs, None)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outputs = layer(*inputs, None)

    def replay(rows, positions, slots, starts):
        for x, y in zip(inputs, (rows, positions, slots)):
            x.copy_(y)
        graph.replay()
        return outputs

    for _ in range(5):
        step([1, 1, 1], replay)
    step([3, 2, 2], layer)
    step([1, 1, 1], replay)
