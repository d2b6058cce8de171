"""What the operators on the paged cache refuse beyond sizes and types: tensors that a launch on
addresses would not be right for, and results over inputs."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

from tests.test_gpu_append import Tokens
from tests.test_gpu_prefix_attention import Batch

pytestmark = pytest.mark.gpu


class Append:
    """append_kv_cache as a function of one of its inputs."""

    def __init__(self, dev, name):
        self.tokens, self.name = Tokens(dev, T=5, D=64, rot=64, norm=True), name
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
