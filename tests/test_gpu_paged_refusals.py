"""What the operators on the paged cache refuse beyond sizes and types: tensors that a launch on
addresses would not be right for, and results over inputs."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

from origami_amd import _ext
from origami_amd.lossless import native_gpu
from tests.test_gpu_append import Tokens
from tests.test_gpu_prefix_attention import Batch

pytestmark = pytest.mark.gpu


class Append:
    """append_kv_cache as a function of one of its inputs."""

    def __init__(self, dev, name, tokens=None):
        self.tokens, self.name = tokens or Tokens(dev, T=5, D=64, rot=64, norm=True), name
        self.before = self.tokens.cache.clone()

    @property
    def input(self):
        t = self.tokens
        return t.kw[self.name] if self.name in t.kw else getattr(t, self.name)

    def __call__(self, x):
        t = self.tokens
        kept = self.input
        try:
            if self.name in t.kw:
                t.kw[self.name] = x
            else:
                setattr(t, self.name, x)
            return t.run()
        finally:
            if self.name in t.kw:
                t.kw[self.name] = kept
            else:
                setattr(t, self.name, kept)

    def untouched(self):
        return torch.equal(self.tokens.cache, self.before)


class Attend:
    def __init__(self, dev, name):
        self.batch, self.name = Batch(dev, prefix=20, own=(5, 6), queries=(2, 3), D=64), name

    @property
    def input(self):
        return getattr(self.batch, self.name)

    def __call__(self, x):
        kept = self.input
        try:
            setattr(self.batch, self.name, x)
            return self.batch.run()[0]
        finally:
            setattr(self.batch, self.name, kept)

    def untouched(self):
        return True


FLOATING = [(Append, n) for n in ("key", "value", "query", "cache", "cos_sin", "query_norm",
                                  "key_norm")] + [(Attend, "query"), (Attend, "cache")]
WHOLE = [(Append, n) for n in ("slots", "positions")] + [
    (Attend, n) for n in ("prefix_ids", "tables", "own", "starts")]


@pytest.mark.parametrize("op,name", FLOATING)
def test_tangents_and_gradients(cuda_device, op, name):
    call = op(cuda_device, name)
    x = call.input
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(RuntimeError, match="requires a gradient"):
            call(dual)
        with forward_ad._set_fwd_grad_enabled(False):
            call(dual)
    call = op(cuda_device, name)
    with pytest.raises(RuntimeError, match="requires a gradient"):
        call(call.input.clone().requires_grad_())
    with torch.no_grad():
        call(call.input.clone().requires_grad_())


@pytest.mark.parametrize("op,name", FLOATING + WHOLE)
def test_transformed_and_traced_tensors(cuda_device, op, name):
    call = op(cuda_device, name)
    x = call.input
    for run in (lambda: torch.func.vmap(call)(x[None]),
                lambda: torch.jit.trace(call.__call__, (x,), check_trace=False),
                lambda: make_fx(call)(x)):
        with pytest.raises(RuntimeError, match="plain tensor|traced"):
            run()
    with FakeTensorMode(allow_non_fake_inputs=True) as mode:
        with pytest.raises(RuntimeError, match="plain tensor|traced"):
            call(mode.from_tensor(x))
    if name not in ("slots", "positions", "prefix_ids", "tables", "own", "starts"):
        with pytest.raises(RuntimeError, match="plain tensor"):
            call(torch._neg_view(x))
    assert call.untouched()


@pytest.mark.parametrize("op,name", [(Append, "key"), (Attend, "query")])
def test_jvp(cuda_device, op, name):
    call = op(cuda_device, name)
    with pytest.raises(RuntimeError, match="plain tensor|requires a gradient"):
        torch.func.jvp(call, (call.input,), (torch.ones_like(call.input),))
    assert call.untouched()


# -- results over inputs.  A refused call launches nothing, so these race on nothing. --------


def _inside(t, shape, dtype):
    """The first bytes of `t` as another tensor."""
    return t.view(torch.uint8).view(-1)[:1 << 14].view(dtype)[:shape.numel()].view(shape)


@pytest.mark.parametrize("name", ["key", "value", "query", "slots", "positions", "cos_sin",
                                  "query_norm", "key_norm"])
def test_append_refuses_inputs_in_the_cache(cuda_device, name):
    """Tokens moved to other slots, say: one workgroup would read what another has written."""
    t = Tokens(cuda_device, T=5, D=64, rot=64, norm=True, positions=20)
    call = Append(cuda_device, name, t)
    inside = _inside(t.cache, call.input.shape, call.input.dtype)
    inside.copy_(call.input)
    before = t.cache.view(torch.int16).clone()  # as numbers, some of the bytes are NaN
    with pytest.raises(RuntimeError, match=f"kv_cache must not overlap {name}"):
        call(inside)
    assert torch.equal(t.cache.view(torch.int16), before)


def test_append_refuses_strided_queries_over_each_other(cuda_device):
    """Views of one projection: parts beside each other are apart, shifted heads are not."""
    t = Tokens(cuda_device, T=6, Hq=4, H=2, D=64, rot=64)
    rows = t.rows.clone()
    plain, cache = t.run(), t.cache.clone()
    t.query = t.rows[:, :4]
    for out in (t.rows[:, 1:5], t.rows[:, 2:6], t.rows[:, 4:8],
                t.rows.as_strided((6, 4, 64), (512, 63, 1)),
                t.rows[:1, :4].expand(6, 4, 64)):
        with pytest.raises(RuntimeError, match="must not overlap"):
            t.run(query_out=out)
    assert torch.equal(t.rows, rows)
    wide = torch.zeros(6, 12, 64, dtype=t.dtype, device=cuda_device)
    wide[:, :8] = rows
    t.query, t.key, t.value = wide[:, :4], wide[:, 4:6], wide[:, 6:8]
    t.run(query_out=wide[:, 8:])
    assert torch.equal(wide[:, 8:], plain) and torch.equal(t.cache, cache)
    t.run(query_out=wide[:, :4])
    assert torch.equal(wide[:, :4], plain) and torch.equal(t.cache, cache)


@pytest.mark.parametrize("name", ["positions", "cos_sin", "query_norm", "key_norm", "slots"])
def test_append_refuses_queries_over_other_inputs(cuda_device, name):
    t = Tokens(cuda_device, T=5, D=64, rot=64, norm=True, positions=20)
    call = Append(cuda_device, name, t)
    memory = torch.zeros(1 << 14, dtype=torch.uint8, device=cuda_device)
    shared = _inside(memory, call.input.shape, call.input.dtype)
    shared.copy_(call.input)
    if name in t.kw:
        t.kw[name] = shared
    else:
        t.slots = shared
    out, before = _inside(memory, t.query.shape, t.query.dtype), t.cache.clone()
    with pytest.raises(RuntimeError, match=f"query_out must not overlap {name}"):
        t.run(query_out=out)
    assert torch.equal(t.cache, before)


@pytest.mark.parametrize("name", ["query", "cache", "tables", "own", "starts", "prefix_ids"])
def test_attention_refuses_an_output_over_inputs(cuda_device, name):
    b = Batch(cuda_device, prefix=20, own=(5, 6), queries=(2, 3), D=64)
    memory = torch.zeros(1 << 20, dtype=torch.uint8, device=cuda_device)
    x = getattr(b, name)
    shared = memory[:x.numel() * x.element_size()].view(x.dtype).view(x.shape)
    shared.copy_(x)
    setattr(b, name, shared)
    before = shared.clone()
    out = _inside(memory, b.query.shape, b.query.dtype)
    argument = {"cache": "kv_cache", "tables": "block_tables", "own": "own_tokens",
                "starts": "query_starts", "prefix_ids": "prefix_block_ids"}.get(name, name)
    with pytest.raises(RuntimeError, match=f"out must not overlap {argument}"):
        b.run(out=out)
    lse = _inside(memory, b.query.shape[:2], torch.float32)
    plain = torch.empty_like(b.query)

    def direct(out, lse):
        return _ext.ext().shared_prefix_attention(
            b.query, b.cache, b.prefix_ids, b.prefix, b.tables, b.own, b.starts, None, None, None,
            1.0, 1.0, out, lse)

    with pytest.raises(RuntimeError, match=f"lse must not overlap {argument}"):
        direct(plain, lse)
    with pytest.raises(RuntimeError, match="out must not overlap lse"):
        both = torch.zeros(b.query.numel(), dtype=b.dtype, device=cuda_device)
        direct(both.view(b.query.shape), both.view(torch.float32)[:lse.numel()].view(lse.shape))
    assert torch.equal(shared.view(torch.uint8), before.view(torch.uint8))
    direct(plain, torch.zeros(lse.shape, device=cuda_device))


def test_attention_refuses_strided_outputs_over_each_other(cuda_device):
    b = Batch(cuda_device, prefix=20, own=(5, 6), D=64)
    plain = b.run()[0]
    rows = torch.zeros(2, 20, 64, dtype=b.dtype, device=cuda_device)
    rows[:, :8] = b.query
    b.query = rows[:, :8]
    for out in (rows[:, :8], rows[:, 7:15], rows[:, :1].expand(2, 8, 64),
                rows.as_strided((2, 8, 64), (1280, 48, 1), 512)):
        with pytest.raises(RuntimeError, match="out must not overlap"):
            b.run(out=out)
    assert torch.equal(b.run(out=rows[:, 12:])[0], plain)
    assert torch.equal(rows[:, 12:], plain)


def test_refused_appends_leave_the_cache_and_the_output(cuda_device):
    t = Tokens(cuda_device, rot=32, norm=True)
    out = torch.full_like(t.query, 3.0)
    t.cache.fill_(5.0)
    w, table = t.kw["key_norm"], t.kw["cos_sin"]
    for change in (dict(key=t.key[:, :1]), dict(value=t.value[:3]), dict(query=t.query[:3]),
                   dict(slots=t.slots[:3]), dict(slots=t.slots.int()), dict(positions=None),
                   dict(cos_sin=table.double()), dict(cos_sin=table[:, :5].contiguous()),
                   dict(cos_sin=table[:0]), dict(key_norm=w[:7]), dict(key_norm=w.float()),
                   dict(key_norm=w.half(), query_norm=None), dict(k_scale=2.0), dict(eps=-1.0),
                   dict(eps=float("nan")), dict(key=t.key.clone().requires_grad_()),
                   dict(query_out=out[:, :1]), dict(query_out=out.float()),
                   dict(kv_cache=t.cache.half()), dict(query=None)):
        args = dict(key=t.key, value=t.value, kv_cache=t.cache, slots=t.slots, query=t.query,
                    query_out=out, **t.kw)
        args.update(change)
        with pytest.raises(RuntimeError):
            native_gpu.append_kv_cache(**args)
    assert (t.cache == 5.0).all() and (out == 3.0).all()
    t.run(query_out=out)
    assert (t.cache != 5.0).any() and (out != 3.0).any()
