"""Refusals of the C entry points of the operators on the paged cache; no GPU is needed, since
they are checked before anything is launched."""
import random

import pytest
import torch

from origami_amd import _ext, _native

BF16, FP8, F32 = _native.DTYPE_BFLOAT16, _native.DTYPE_FLOAT8_E4M3FN, _native.DTYPE_FLOAT32


def _append(**kw):
    a = dict(key=16, value=16, query=16, query_out=16, dtype=BF16, strides=[8] * 8, tokens=4,
             query_heads=4, kv_cache=16, cache_dtype=BF16, layout=0, num_blocks=4, block_size=16,
             heads=2, head_dim=64, slots=16, positions=16, cos_sin=16, table_rows=10,
             rotary_dim=64, interleaved=0, query_norm=None, key_norm=None, norm_dtype=BF16,
             eps=1e-6, k_scale=1.0, v_scale=1.0, stream=None)
    a.update(kw)
    strides = _native.i64_array(a["strides"])
    a["strides"] = strides.ctypes.data
    return _native.call("origami_append_kv_cache", *a.values())


@pytest.mark.parametrize("change,message", [
    (dict(dtype=F32), "must be float16 or bfloat16"),
    (dict(cache_dtype=F32), "keys' dtype or be float8_e4m3fn"),
    (dict(tokens=-1), "must not be negative"),
    (dict(heads=0), "must not be negative"),
    (dict(head_dim=60), "multiple of 8"),
    (dict(head_dim=264), "at most 256"),
    (dict(block_size=0), "block size must be positive"),
    (dict(layout=7), "kv_cache must be"),
    (dict(num_blocks=1 << 40), "too many token slots"),
    (dict(query_out=None), "need an output"),
    (dict(rotary_dim=7), "even rotary size"),
    (dict(rotary_dim=66), "even rotary size"),
    (dict(positions=None), "needs positions"),
    (dict(table_rows=0), "needs positions"),
    (dict(key_norm=16, norm_dtype=_native.DTYPE_FLOAT16), "norm weights"),
    (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps"),
    (dict(cache_dtype=FP8, k_scale=0.0), "scales must be positive"),
    (dict(cache_dtype=FP8, v_scale=float("nan")), "scales must be positive"),
    (dict(v_scale=2.0), "for float8_e4m3fn"),
    (dict(kv_cache=24), "16-byte aligned"),
    (dict(tokens=1 << 25), "too many rows"),
    (dict(query_heads=1 << 16), "too many rows"),
    (dict(strides=[8, 8, 8, 8, -8, 8, 8, 8]), "must not be negative"),
    (dict(key=None), "must not be null"),
    (dict(slots=None), "must not be null"),
    (dict(kv_cache=None), "must not be null"),
])
def test_append_refuses(change, message):
    with pytest.raises(_native.OrigamiNativeError, match=message) as e:
        _append(**change)
    assert e.value.code == _native.ORIGAMI_ERR_INVALID


def _attend(**kw):
    a = dict(query=16, dtype=BF16, strides=[8] * 4, tokens=3, query_heads=4, kv_cache=16,
             cache_dtype=BF16, layout=0, num_blocks=4, block_size=16, heads=2, head_dim=64,
             prefix_ids=16, prefix_blocks=2, prefix=32, tables=16, table_stride=2, table_blocks=2,
             own=16, requests=3, starts=None, max_query=1, max_own=32, scale=1.0, k_scale=1.0,
             v_scale=1.0, out=16, lse=None, workspace=16, workspace_bytes=1 << 30, stream=None)
    a.update(kw)
    strides = _native.i64_array(a["strides"])
    a["strides"] = strides.ctypes.data
    return _native.call("origami_shared_prefix_attention", *a.values())


@pytest.mark.parametrize("change,message", [
    (dict(dtype=F32), "queries must be float16 or bfloat16"),
    (dict(cache_dtype=F32), "queries' dtype or be float8_e4m3fn"),
    (dict(query_heads=3), "multiple of the cache's heads"),
    (dict(heads=0), "multiple of the cache's heads"),
    (dict(head_dim=4), "multiple of 8"),
    (dict(head_dim=512), "at most 256"),
    (dict(tokens=-1), "must not be negative"),
    (dict(prefix=-1), "must not be negative"),
    (dict(prefix=1 << 30), "too many tokens"),
    (dict(tokens=1 << 22, starts=16), "too many query rows"),
    (dict(num_blocks=1 << 28), "too many token slots"),
    (dict(block_size=0), "block size must be positive"),
    (dict(layout=3), "kv_cache must be"),
    (dict(prefix=33), "exceed the prefix blocks"),
    (dict(max_own=33), "exceeds the block tables"),
    (dict(tokens=4), "one query token"),
    (dict(k_scale=-1.0), "scales must be positive"),
    (dict(v_scale=0.5), "for float8_e4m3fn"),
    (dict(kv_cache=17), "16-byte aligned"),
    (dict(workspace_bytes=8), "workspace is too small"),
    (dict(workspace=None), "workspace is too small"),
    (dict(strides=[8, -8, 8, 8]), "must not be negative"),
    (dict(table_stride=-2), "must not be negative"),
    (dict(out=None), "must not be null"),
    (dict(own=None), "must not be null"),
    (dict(tables=None), "must not be null"),
    (dict(prefix_ids=None), "must not be null"),
    (dict(kv_cache=None), "must not be null"),
])
def test_attention_refuses(change, message):
    with pytest.raises(_native.OrigamiNativeError, match=message) as e:
        _attend(**change)
    assert e.value.code == _native.ORIGAMI_ERR_INVALID


def test_workspace_sizes():
    size = _native.lib().origami_shared_prefix_attention_workspace
    assert size(3, 4, 2, 64, 32, 3, 1, 32, BF16) > 0
    assert size(0, 4, 2, 64, 32, 3, 0, 32, BF16) == 0
    assert size(3, 3, 2, 64, 32, 3, 1, 32, BF16) == -1
    assert size(1, 4, 2, 64, 0, 1, 1, 16, FP8) == 0  # one part: the rows are written at once


INF, NAN, BIG = float("inf"), float("nan"), 1 << 62


@pytest.mark.parametrize("change,message", [
    (dict(heads=BIG), "too many rows"),
    (dict(heads=BIG + (1 << 15)), "too many rows"),
    (dict(query_heads=BIG, heads=BIG), "too many rows"),
    (dict(num_blocks=0, block_size=1 << 40), "too many token slots"),
])
def test_append_refuses_sizes_past_its_integers(change, message):
    with pytest.raises(_native.OrigamiNativeError, match=message) as e:
        _append(**change)
    assert e.value.code == _native.ORIGAMI_ERR_INVALID


@pytest.mark.parametrize("change,message", [
    # a block size that 32 bits do not hold would give block numbers past the tables
    (dict(num_blocks=0, block_size=1 << 40, prefix_blocks=1, table_blocks=1),
     "too many token slots"),
    (dict(num_blocks=0, block_size=(1 << 32) + 1, prefix_blocks=1, table_blocks=1),
     "too many token slots"),
    (dict(prefix=BIG, max_own=BIG, prefix_blocks=BIG, table_blocks=BIG), "too many tokens"),
    (dict(prefix=0, max_own=BIG + BIG - 1, table_blocks=BIG), "too many tokens"),
    (dict(starts=16, requests=1 << 40), "too many requests"),
    (dict(starts=16, requests=BIG), "too many requests"),
    (dict(starts=16, requests=BIG, tokens=0), "too many requests"),
    (dict(query_heads=BIG, heads=BIG, tokens=0), "too many query rows"),
])
def test_attention_refuses_sizes_past_its_integers(change, message):
    with pytest.raises(_native.OrigamiNativeError, match=message) as e:
        _attend(**change)
    assert e.value.code == _native.ORIGAMI_ERR_INVALID


def test_workspace_refuses_sizes_past_its_integers():
    size = _native.lib().origami_shared_prefix_attention_workspace
    assert size(3, 4, 2, 64, BIG, 3, 1, BIG, BF16) == -1
    assert size(3, 4, 2, 64, 32, BIG, 1, 32, BF16) == -1
    assert size(3, 4, 2, 64, 32, 1 << 23, 1, 32, BF16) == -1


@pytest.mark.parametrize("change,message", [
    (dict(eps=INF), "eps must not be negative or infinite"),
    (dict(eps=1e39), "eps must not be negative or infinite"),
    (dict(cache_dtype=FP8, k_scale=INF), "scales must be positive"),
    (dict(cache_dtype=FP8, v_scale=1e39), "scales must be positive"),
    (dict(cache_dtype=FP8, k_scale=1e-60), "scales must be positive"),
])
def test_append_refuses_numbers_that_binary32_does_not_hold(change, message):
    with pytest.raises(_native.OrigamiNativeError, match=message) as e:
        _append(**change)
    assert e.value.code == _native.ORIGAMI_ERR_INVALID


@pytest.mark.parametrize("change,message", [
    (dict(scale=NAN), "scale must be finite"),
    (dict(scale=-INF), "scale must be finite"),
    (dict(scale=3e38), "scale must be finite"),  # times log2 e
    (dict(cache_dtype=FP8, scale=1e30, k_scale=1e10), "scale must be finite"),
    (dict(cache_dtype=FP8, k_scale=INF), "scales must be positive"),
    (dict(cache_dtype=FP8, v_scale=1e39), "scales must be positive"),
    (dict(cache_dtype=FP8, v_scale=1e-60), "scales must be positive"),
])
def test_attention_refuses_numbers_that_binary32_does_not_hold(change, message):
    with pytest.raises(_native.OrigamiNativeError, match=message) as e:
        _attend(**change)
    assert e.value.code == _native.ORIGAMI_ERR_INVALID


def _bytes(t):
    at = torch.zeros((), dtype=torch.int64)
    for n, step in zip(t.shape, t.stride()):
        at = at[..., None] + torch.arange(n) * step
    at = (t.data_ptr() + at.reshape(-1) * t.element_size())[:, None]
    return (at + torch.arange(t.element_size())).reshape(-1)


def _view(rng, memory, dtype):
    """A view of `memory` with any strides, inside it."""
    typed = memory.view(dtype)
    shape = [rng.choice([0, 1, 1, 2, 3, 5, 7]) if rng.random() < 0.1 else rng.randint(1, 6)
             for _ in range(rng.randint(1, 3))]
    while True:
        strides = [rng.choice([0, 1, 1, 2, 3, 8, 9, 16, 24, 25, 48, 50]) for _ in shape]
        room = typed.numel() - sum(max(n - 1, 0) * s for n, s in zip(shape, strides))
        if room > 0:
            return typed.as_strided(shape, strides, rng.randrange(room))


def test_overlap_of_strided_tensors():
    """Which tensors share bytes, against sets of their bytes."""
    ext, rng, found = _ext.ext(), random.Random(0), [0, 0, 0]
    memory = torch.zeros(2048, dtype=torch.uint8)
    types = [torch.uint8, torch.bfloat16, torch.float32, torch.int64]
    for _ in range(4000):
        a, b = (_view(rng, memory, rng.choice(types)) for _ in range(2))
        x, y = _bytes(a), _bytes(b)
        both = len(set(x.tolist()) & set(y.tolist())) > 0
        assert ext._tensors_overlap(a, b) == both == ext._tensors_overlap(b, a), (a.shape, b.shape)
        assert ext._tensor_overlaps_itself(a) == (len(set(x.tolist())) < x.numel())
        found[0] += both
        found[1] += not both and bool(x.numel() and y.numel() and x.min() <= y.max()
                                      and y.min() <= x.max())
        found[2] += len(set(x.tolist())) < x.numel()
    assert min(found) > 100  # overlaps, views in each other's gaps, and overlaps with oneself


def test_overlap_of_a_projections_parts():
    """The views of a large projection, whose parts lie between each other's rows."""
    ext = _ext.ext()
    rows = torch.empty(100_000, 48, 8, dtype=torch.bfloat16)
    query, key, value = rows[:, :32], rows[:, 32:40], rows[:, 40:]
    for a, b in ((query, key), (key, value), (query, value), (rows[::2], rows[1::2]),
                 (rows[:, :, :4], rows[:, :, 4:]), (rows[:50_000], rows[50_000:])):
        assert not ext._tensors_overlap(a, b) and not ext._tensors_overlap(b, a)
    for a, b in ((query, rows[:, 31:35]), (rows[:-1, :32], rows[1:, :32]), (query, query[777:778]),
                 (rows.transpose(0, 1)[:32], query), (key, rows.view(-1)[32 * 8:32 * 8 + 1])):
        assert ext._tensors_overlap(a, b) and ext._tensors_overlap(b, a)
    assert not ext._tensor_overlaps_itself(query)
    assert ext._tensor_overlaps_itself(rows[:, :1].expand(-1, 2, -1))
    assert ext._tensor_overlaps_itself(rows.view(-1).as_strided((5, 2, 8), (16, 7, 1)))
