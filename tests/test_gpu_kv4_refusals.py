"""What reading, adding up weights and evicting refuse beyond sizes and types, as the other operators
on the paged cache do; and a cache in 4 bits saved and restored."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

from origami_amd.layout import kv_symbol_layout
from origami_amd.lossless import native_gpu
from tests import kv4ref
from tests.test_gpu_evict import Eviction, Weights, make_cache
from tests.test_gpu_kv4 import Batch4, Tokens4

pytestmark = pytest.mark.gpu


class Call:
    """An operator as a function of one of its inputs, an attribute of `held`."""

    def __init__(self, held, name, run):
        self.held, self.name, self.run = held, name, run
        self.before = held.cache.clone()

    @property
    def input(self):
        return getattr(self.held, self.name)

    def __call__(self, x):
        kept = self.input
        try:
            setattr(self.held, self.name, x)
            return self.run()
        finally:
            setattr(self.held, self.name, kept)

    def untouched(self):
        return torch.equal(self.held.cache.view(torch.uint8), self.before.view(torch.uint8))


def read(dev, name):
    held = Weights(dev, tokens=(30, 20), cache_dtype=torch.bfloat16)
    held.slots = torch.arange(40, device=dev)
    return Call(held, name, lambda: native_gpu.read_kv_cache(held.cache, held.slots)[0])


def weigh(dev, name):
    held = Weights(dev, tokens=(30, 20), queries=(3, 2))
    return Call(held, name, held.run)


def evict(dev, name):
    held = Eviction(dev)
    return Call(held, name, lambda: held.run()[1])


def append4(dev, name):
    held = Tokens4(dev, D=64, T=9)
    return Call(held, name, held.run)


def attend4(dev, name):
    held = Batch4(dev, D=64, prefix=0, own=(20, 30))
    return Call(held, name, lambda: held.run()[0])


FLOATING = [(read, "cache"), (weigh, "query"), (weigh, "cache"), (weigh, "lse"),
            (weigh, "weights"), (evict, "cache"), (evict, "weights"), (append4, "key"),
            (attend4, "query")]
WHOLE = [(read, "slots"), (weigh, "tables"), (weigh, "tokens"), (weigh, "starts"),
         (evict, "tables"), (evict, "tokens"), (evict, "out_tables"), (append4, "cache"),
         (attend4, "cache"), (attend4, "tables")]


@pytest.mark.parametrize("op,name", FLOATING)
def test_tangents_and_gradients(cuda_device, op, name):
    call = op(cuda_device, name)
    x = call.input
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="requires a gradient"):
            call(forward_ad.make_dual(x, torch.ones_like(x)))
    with pytest.raises(RuntimeError, match="requires a gradient"):
        call(x.clone().requires_grad_())
    assert call.untouched()
    with torch.no_grad():
        call(x.clone().requires_grad_())


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
    assert call.untouched()


@pytest.mark.parametrize("op,name", FLOATING + WHOLE)
def test_inputs_on_the_host(cuda_device, op, name):
    call = op(cuda_device, name)
    with pytest.raises(RuntimeError, match="device|CUDA"):
        call(call.input.cpu())
    assert call.untouched()


@pytest.mark.parametrize("op,name", [w for w in WHOLE if w[1] not in ("cache",)])
def test_other_integers(cuda_device, op, name):
    call = op(cuda_device, name)
    with pytest.raises(RuntimeError, match="int64"):
        call(call.input.int())
    assert call.untouched()


def test_inference_mode(cuda_device):
    with torch.inference_mode():
        for op, name in FLOATING:
            call = op(cuda_device, name)
            call(call.input)


@pytest.mark.parametrize("order", ["kv_first", "blocks_first"])
@pytest.mark.parametrize("D,heads,prefix", [(128, 2, 100), (64, 3, 37), (80, 1, 64)])
def test_save_and_restore_a_cache_in_4_bits(cuda_device, order, D, heads, prefix):
    """A cache in 4 bits is a cache of bytes to the layout calls: what is packed from its blocks and
    restored elsewhere reads and attends the same."""
    dev, gen, bs, NB = cuda_device, torch.Generator().manual_seed(D), 16, 20
    saved = make_cache(gen, torch.uint8, NB, bs, heads, D, order, dev)
    shared = -(-prefix // bs)
    ids = torch.randperm(NB, generator=gen).to(dev)
    C = native_gpu.kv4_row_bytes(D)
    layout = kv_symbol_layout(prefix, heads, C, 8, [[0, heads, 0, C, 0, 2 * prefix]])
    stream = native_gpu.pack_from_kv_cache(saved, ids[:shared], prefix, layout)
    cache = torch.zeros_like(saved)
    new = ids[shared:2 * shared]
    native_gpu.unpack_to_kv_cache(stream, layout, prefix, cache, new)
    t = torch.arange(prefix, device=dev)
    was = native_gpu.read_kv_cache(saved, ids[t // bs] * bs + t % bs)
    now = native_gpu.read_kv_cache(cache, new[t // bs] * bs + t % bs)
    assert all(torch.equal(a, b) for a, b in zip(was, now))
    assert torch.equal(was[0].double(), kv4ref.cells(saved, D)[0][ids[t // bs], t % bs])
    query = torch.randn(1, 4 * heads, D, generator=gen).to(torch.bfloat16).to(dev)
    tokens = torch.tensor([prefix], device=dev)
    out = [native_gpu.shared_prefix_attention(query, c, None, 0, i[None], tokens)
           for c, i in ((saved, ids[:shared]), (cache, new))]
    assert torch.equal(*out)
