"""Refusals of the C entry points of caches in 4 bits and of eviction, and the plain forms of
their tests; no GPU is needed."""
import math

import pytest
import torch

from origami_amd import _native
from origami_amd.lossless import native_gpu
from tests import kv4ref
from tests.test_paged_ops import _append, _attend

BF16, F16, F32, FP8, FP4 = (_native.DTYPE_BFLOAT16, _native.DTYPE_FLOAT16, _native.DTYPE_FLOAT32,
                            _native.DTYPE_FLOAT8_E4M3FN, _native.DTYPE_FLOAT4_E2M1)
BIG, NAN = 1 << 62, float("nan")


def refused(call, change, message):
    with pytest.raises(_native.OrigamiNativeError, match=message) as e:
        call(**change)
    assert e.value.code == _native.ORIGAMI_ERR_INVALID


@pytest.mark.parametrize("D", range(8, 257, 8))
def test_row_bytes(D):
    assert native_gpu.kv4_row_bytes(D) == kv4ref.row_bytes(D)
    assert kv4ref.row_bytes(D) % 4 == 0


@pytest.mark.parametrize("D", [-8, 0, 4, 12, 264, BIG])
def test_row_bytes_refuses(D):
    with pytest.raises(ValueError, match="multiple of 8"):
        native_gpu.kv4_row_bytes(D)


def test_pack_of_the_plain_form():
    """The plain form's own rounding, against every pair of neighbours."""
    x = torch.zeros(1, 32, dtype=torch.float64)
    x[0, :9] = torch.tensor([6.0, 0.25, 0.26, 0.75, 2.5, -3.5, 5.0, -0.0, 7.0])
    rows = kv4ref.pack(x)
    assert rows.shape == (1, 20) and rows[0, 16] == 127 and (rows[0, 17:] == 0).all()
    assert kv4ref.values(rows, 32)[0, :9].tolist() == [6, 0, 0.5, 1, 2, -4, 4, 0, 6]
    x[0, 8] = 7.1
    assert kv4ref.pack(x)[0, 16] == 128
    x[0, 8] = math.inf
    assert kv4ref.values(kv4ref.pack(x), 32)[0, 8] == 49152
    x[0, 3] = NAN
    assert kv4ref.values(kv4ref.pack(x), 32).isnan().all()
    gen = torch.Generator().manual_seed(0)
    y = torch.randn(50, 40, generator=gen, dtype=torch.float64)
    held = kv4ref.values(kv4ref.pack(y), 40)
    step = 2.0 ** kv4ref.powers(y).repeat_interleave(32, -1)[..., :40]
    assert ((held - y).abs() <= step).all()


def test_kept_places_of_the_plain_form():
    w = torch.tensor([[[3.0, 1.0, 3.0, NAN, 0.0, 9.0, 9.0]]])
    assert kv4ref.kept_places(w, [6], 3, 1) == [[[0, 3, 5]]]
    assert kv4ref.kept_places(w, [6], 4, 1) == [[[0, 2, 3, 5]]]
    assert kv4ref.kept_places(w, [3], 4, 1) == [[[0, 1, 2]]]
    assert kv4ref.kept_places(w, [7], 2, 5) == [[[5, 6]]]


@pytest.mark.parametrize("change,message", [
    (dict(k_scale=0.5), "for float8_e4m3fn"), (dict(v_scale=2.0), "for float8_e4m3fn"),
    (dict(kv_cache=20), "16-byte aligned"), (dict(head_dim=60), "multiple of 8")])
def test_append_and_attention_in_4_bits_refuse(change, message):
    refused(_append, dict(change, cache_dtype=FP4), message)
    refused(_attend, dict(change, cache_dtype=FP4), message)


def _read(**kw):
    a = dict(kv_cache=16, cache_dtype=FP4, layout=0, num_blocks=4, block_size=16, heads=2,
             head_dim=64, slots=16, tokens=3, k_scale=1.0, v_scale=1.0, key=16, value=16,
             dtype=BF16, strides=[8] * 4, stream=None)
    a.update(kw)
    strides = _native.i64_array(a["strides"])
    a["strides"] = strides.ctypes.data
    return _native.call("origami_read_kv_cache", *a.values())


@pytest.mark.parametrize("change,message", [
    (dict(dtype=F32), "must be float16 or bfloat16"), (dict(dtype=FP4), "must be float16"),
    (dict(cache_dtype=F32), "keys' dtype or be float8_e4m3fn or in 4 bits"),
    (dict(cache_dtype=F16), "keys' dtype or be float8_e4m3fn or in 4 bits"),
    (dict(tokens=-1), "must not be negative"), (dict(heads=0), "must not be negative"),
    (dict(head_dim=12), "multiple of 8"), (dict(head_dim=264), "at most 256"),
    (dict(block_size=0), "block size must be positive"), (dict(layout=2), "kv_cache must be"),
    (dict(num_blocks=1 << 40), "too many token slots"),
    (dict(num_blocks=0, block_size=1 << 40), "too many token slots"),
    (dict(k_scale=2.0), "for float8_e4m3fn"), (dict(cache_dtype=FP8, v_scale=NAN), "must be positive"),
    (dict(kv_cache=8), "16-byte aligned"), (dict(tokens=1 << 27), "too many rows"),
    (dict(heads=BIG), "too many rows"), (dict(strides=[8, -8, 8, 8]), "must not be negative"),
    (dict(key=None), "must not be null"), (dict(value=None), "must not be null"),
    (dict(slots=None), "must not be null"), (dict(kv_cache=None), "must not be null")])
def test_read_refuses(change, message):
    refused(_read, change, message)


def test_nothing_to_read():
    assert _read(tokens=0, key=None, value=None, slots=None) == 0


def _weigh(**kw):
    a = dict(query=16, dtype=BF16, strides=[8, 8], tokens=3, query_heads=4, lse=16, kv_cache=16,
             cache_dtype=FP4, layout=0, num_blocks=4, block_size=16, heads=2, head_dim=64,
             tables=16, table_stride=2, table_blocks=2, lengths=16, requests=3, starts=None,
             max_tokens=32, scale=1.0, k_scale=1.0, weights=16, out=16, places=40,
             weight_strides=[8] * 4, workspace=16, workspace_bytes=1 << 40, stream=None)
    a.update(kw)
    strides, more = (_native.i64_array(a[n]) for n in ("strides", "weight_strides"))
    a["strides"], a["weight_strides"] = strides.ctypes.data, more.ctypes.data
    return _native.call("origami_accumulate_attention_weights", *a.values())


@pytest.mark.parametrize("change,message", [
    (dict(dtype=F32), "queries must be float16 or bfloat16"),
    (dict(cache_dtype=F16), "queries' dtype or be float8_e4m3fn or in 4 bits"),
    (dict(heads=0), "heads must be positive"), (dict(query_heads=3), "multiple of the cache's"),
    (dict(head_dim=4), "multiple of 8"), (dict(block_size=0), "block size must be positive"),
    (dict(layout=9), "kv_cache must be"), (dict(num_blocks=1 << 28), "too many token slots"),
    (dict(tokens=-1), "must not be negative"), (dict(places=-1), "must not be negative"),
    (dict(places=BIG), "too many tokens"), (dict(tokens=1 << 22, starts=16), "too many query rows"),
    (dict(requests=BIG, starts=16), "too many requests"),
    (dict(heads=1 << 22, query_heads=1 << 22), "too many heads"),
    (dict(max_tokens=41), "exceeds the weights' places"),
    (dict(max_tokens=33), "exceeds the block tables"), (dict(tokens=4), "one query token"),
    (dict(k_scale=0.5), "for float8_e4m3fn"), (dict(cache_dtype=FP8, k_scale=0.0), "be positive"),
    (dict(scale=NAN), "scale must be finite"), (dict(scale=1e39), "scale must be finite"),
    (dict(kv_cache=24), "16-byte aligned"), (dict(strides=[-8, 8]), "row strides"),
    (dict(weight_strides=[8, 8, 8, -1]), "weight strides"),
    (dict(table_stride=-1), "table stride"), (dict(query=None), "must not be null"),
    (dict(lse=None), "must not be null"), (dict(out=None), "must not be null"),
    (dict(lengths=None), "must not be null"), (dict(tables=None), "must not be null"),
    (dict(kv_cache=None), "must not be null"),
    (dict(places=1 << 30, requests=1 << 10, starts=16, tokens=1 << 20),
     "too many tokens for one call")])
def test_weights_refuse(change, message):
    refused(_weigh, change, message)


@pytest.mark.parametrize("change", [dict(workspace_bytes=8), dict(workspace=None),
                                    dict(workspace=8)])
def test_weights_refuse_workspaces(change):
    prompt = dict(tokens=4096, requests=1, starts=16, places=4096)
    refused(_weigh, dict(prompt, **change), "workspace of the weights is too small")


@pytest.mark.parametrize("places", [4096, 131072, 1 << 30])
def test_weights_are_split_by_the_bound(places):
    """Two prompts of 4096 tokens take parts of their rows (and room for their sums), however wide
    the buffer of the sums is."""
    prompts = dict(tokens=8000, requests=2, starts=16, heads=4, query_heads=28, table_blocks=256,
                   max_tokens=4096, places=places)
    refused(_weigh, dict(prompts, workspace_bytes=8), "workspace of the weights is too small")


def test_weights_workspace_is_enough_for_every_bound():
    size = _native.lib().origami_accumulate_attention_weights_workspace
    for requests, heads in ((1, 1), (1, 8), (2, 4), (60, 8), (300, 8)):
        sizes = [size(1 << 18, 4 * heads, heads, requests, n)
                 for n in (1, 255, 256, 257, 1000, 4096, 20000, 131072, 1 << 30)]
        assert sizes == sorted(sizes) and sizes[-1] <= 2 * 2048 * 256 * 4
        assert sizes[0] >= 0 and (sizes[0] > 0) == (requests * heads < 2048)


def test_weights_workspace_sizes():
    size = _native.lib().origami_accumulate_attention_weights_workspace
    assert size(4096, 8, 2, 1, 4096) > 0 and size(4096, 8, 2, 1, 4096) % (2 * 4096 * 4) == 0
    assert size(64, 32, 8, 64, 32768) == 0  # single tokens: one part
    assert size(64, 8, 2, 0, 100) == 0
    for sizes in ((-1, 4, 2, 1, 8), (1, 3, 2, 1, 8), (1, 4, 0, 1, 8), (1, 4, 2, BIG, 8),
                  (BIG, 4, 2, 1, 8), (1, 4, 2, 1, BIG)):
        assert size(*sizes) == -1


def test_nothing_to_weigh():
    assert _weigh(requests=0, tokens=0, query=None, out=None, lengths=None) == 0
    assert _weigh(places=0, max_tokens=0, out=None) == 0


def _evict(**kw):
    a = dict(kv_cache=16, cache_dtype=FP4, layout=0, num_blocks=4, block_size=16, heads=2,
             head_dim=64, tables=16, table_stride=2, table_blocks=2, lengths=16, requests=3,
             max_tokens=32, weights=16, places=40, out_tables=16, out_stride=1, out_blocks=1,
             keep=10, recent=3, kept=16, out_weights=16, out_places=40, weight_strides=[8] * 4,
             stream=None)
    a.update(kw)
    strides = _native.i64_array(a["weight_strides"])
    a["weight_strides"] = strides.ctypes.data
    return _native.call("origami_evict_kv_cache", *a.values())


@pytest.mark.parametrize("change,message", [
    (dict(cache_dtype=F32), "kv_cache must be float16, bfloat16"),
    (dict(heads=0), "heads must be positive"), (dict(head_dim=20), "multiple of 8"),
    (dict(head_dim=BIG), "at most 256"), (dict(block_size=-1), "block size must be positive"),
    (dict(layout=-1), "kv_cache must be"), (dict(num_blocks=1 << 28), "too many token slots"),
    (dict(requests=-1), "must not be negative"), (dict(keep=-1), "must not be negative"),
    (dict(recent=-1), "must not be negative"), (dict(out_places=-5), "must not be negative"),
    (dict(max_tokens=BIG, places=BIG), "too many tokens"),
    (dict(keep=BIG, out_places=BIG), "too many tokens"),
    (dict(requests=BIG), "too many requests"), (dict(heads=BIG), "too many heads"),
    (dict(heads=1 << 22), "too many heads"), (dict(heads=1 << 21, requests=2), "too many requests"),
    (dict(max_tokens=41), "exceeds the weights' places"),
    (dict(max_tokens=33), "exceeds the block tables"),
    (dict(out_places=9), "places of out_weights"), (dict(keep=17), "new block tables"),
    (dict(weight_strides=[-1, 8, 8, 8]), "weight strides"),
    (dict(out_stride=-1), "table strides"), (dict(kv_cache=4), "16-byte aligned"),
    (dict(lengths=None), "must not be null"), (dict(weights=None), "must not be null"),
    (dict(kept=None), "must not be null"), (dict(out_weights=None), "must not be null"),
    (dict(tables=None), "must not be null"), (dict(out_tables=None), "must not be null"),
    (dict(kv_cache=None), "must not be null"),
    (dict(keep=1 << 28, max_tokens=1 << 28, places=1 << 28, out_places=1 << 28, block_size=1 << 26,
          out_blocks=4, table_blocks=4, requests=1 << 10), "too many tokens for one call")])
def test_evict_refuses(change, message):
    refused(_evict, change, message)


def test_nothing_to_evict():
    assert _evict(requests=0, lengths=None, kept=None, out_weights=None) == 0


@pytest.mark.parametrize("heads,query_heads", [(8, 64), (8, 32), (1, 16), (4, 28)])
@pytest.mark.parametrize("requests", [1, 16, 128, 256, 257, 512, 2000])
def test_attention_workspace_is_not_of_the_bound(heads, query_heads, requests):
    """Decode steps over a cache in 4 bits, however far the bound is above what the requests hold.
    There are shares for 2048 waves or two for each request and head, each with a request's rows of
    D + 2 numbers, and 8 bytes a row; of equal ranges, past 256 requests, 256 MiB or what 2048 waves
    take."""
    size, D = _native.lib().origami_shared_prefix_attention_workspace, 128
    row = (D + 2) * 4
    for bound in (1, 4096, 32768, 131072, 1 << 20, 1 << 22):
        got = size(requests, query_heads, heads, D, 0, requests, 1, bound, FP4)
        waves = (2048 + 2 * requests * heads) * (query_heads // heads) * row
        most = waves + requests * query_heads * 8 if requests <= 256 else max(256 << 20, waves)
        assert 0 <= got <= most, (bound, got, most)
