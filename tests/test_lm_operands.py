"""What the language-model operators' kernels cannot see of an operand: a tangent,
a tracer and another tensor inside are refused, in front of every look at the
device, so that this can be tested without one; a negation is resolved."""
import pytest
import torch
import torch.autograd.forward_ad as fw
from torch._subclasses import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

from dear_pytorch_amd.ops.fused_ln import layer_norm
from dear_pytorch_amd.ops.token_loss import token_logprobs, topk_distill_loss


def operands(dev, seed=0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(3, 8, generator=gen)
    ids = torch.tensor([[1, 2], [3, 4], [0, 7]])
    lp = torch.log_softmax(torch.randn(3, 8, generator=gen), -1).gather(1, ids)
    w = torch.randn(8, generator=gen)
    return {k: t.to(dev) for k, t in
            dict(x=x, w=w, b=w - 1, r=x.flip(0), ids=ids, lp=lp).items()}


# the public entry points, and the operands of each that are numbers
CALLS = {
    "layer_norm": (lambda o: layer_norm(o["x"], o["w"], o["b"], 1e-5,
                                        residual=o["r"]),
                   ("x", "w", "b", "r")),
    "token_logprobs": (lambda o: token_logprobs(o["x"], o["ids"][:, 0],
                                                top=2).logprob, ("x",)),
    "topk_distill_loss": (lambda o: topk_distill_loss(o["x"], o["ids"],
                                                      o["lp"], tail=True),
                          ("x", "lp")),
}


# the same calls of the extension, which refuses before it asks for the device
def native(name):
    k = pytest.importorskip("dear_pytorch_amd._kernels")
    return {
        "layer_norm": lambda o: k.layer_norm(o["x"], o["w"], o["b"], 1e-5,
                                             o["r"]),
        "token_logprobs": lambda o: k.token_logprobs(
            o["x"], o["ids"][:, 0].contiguous(), 2, 1.0, -1),
        "topk_distill_loss": lambda o: k.topk_distill_loss(
            o["x"], o["ids"], o["lp"], 1.0, True),
    }[name]


EACH = [(n, k) for n, (_, keys) in CALLS.items() for k in keys]


def tangents(call, name, key, dev):
    for grad in (False, True):
        o = operands(dev)
        if grad:
            o["x"].requires_grad_(True)
        for mode in (torch.enable_grad, torch.no_grad):
            with mode(), fw.dual_level():
                dual = dict(o)
                dual[key] = fw.make_dual(o[key], torch.ones_like(o[key]))
                with pytest.raises(NotImplementedError, match=name):
                    call(dual)


@pytest.mark.parametrize("name,key", EACH)
def test_tangents_are_refused(name, key):
    tangents(native(name), name, key, "cpu")


def test_cpu_paths_have_tangents():
    for name, (call, keys) in CALLS.items():
        o = operands("cpu")
        with fw.dual_level():
            o["x"] = fw.make_dual(o["x"], torch.ones_like(o["x"]) * 0.3)
            assert fw.unpack_dual(call(o)).tangent is not None, name


def traces(call, name, dev):
    o = operands(dev)
    for grad in (False, True):
        x = o["x"].clone().requires_grad_(grad)
        with pytest.raises(NotImplementedError, match=name):
            torch.jit.trace(lambda x: call({**o, "x": x}), (x,))
        with pytest.raises(NotImplementedError, match=name):
            make_fx(lambda x: call({**o, "x": x}))(x)
    assert not torch.jit.is_tracing()


@pytest.mark.parametrize("name", CALLS)
def test_tracing_is_refused(name):
    traces(native(name), name, "cpu")


@pytest.mark.parametrize("name", CALLS)
def test_cpu_paths_can_be_traced(name):
    o, call = operands("cpu"), CALLS[name][0]
    run = lambda x: call({**o, "x": x})
    for traced in (torch.jit.trace(run, (o["x"],), check_trace=False),
                   make_fx(run)(o["x"])):
        x = operands("cpu", seed=1)["x"]
        assert torch.equal(traced(x), run(x))


class Wrapper(torch.Tensor):
    """A tensor around another one, as distributed tensors are."""

    @staticmethod
    def __new__(cls, t):
        return torch.Tensor._make_wrapper_subclass(
            cls, t.shape, dtype=t.dtype, device=t.device)

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise AssertionError(func)


EVERY = [(n, k) for n, keys in (
    ("layer_norm", ("x", "w", "b", "r")), ("token_logprobs", ("x", "tokens")),
    ("topk_distill_loss", ("x", "ids", "lp"))) for k in keys]


@pytest.mark.parametrize("name,key", EVERY)
def test_operands_without_memory_are_refused(name, key):
    k = pytest.importorskip("dear_pytorch_amd._kernels")
    call = native(name)
    if key == "tokens":
        call = lambda o: k.token_logprobs(o["x"], o["tokens"], 2, 1.0, -1)
    with FakeTensorMode():
        fake = operands("cpu")
        fake["tokens"] = torch.zeros(3, dtype=torch.long)
    for grad in (False, True):
        o = operands("cpu")
        o["tokens"] = o["ids"][:, 0].contiguous()
        if key != "x":
            o["x"].requires_grad_(grad)
        for bad in (Wrapper(o[key]), fake[key],
                    torch._efficientzerotensor(o[key].shape,
                                               dtype=o[key].dtype)):
            with pytest.raises(TypeError, match=name):
                call({**o, key: bad})


@pytest.mark.gpu
@pytest.mark.parametrize("name", CALLS)
def test_gpu_tracing_is_refused(name):
    traces(CALLS[name][0], name, "cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("name,key", EACH)
def test_gpu_tangents_are_refused(name, key):
    tangents(CALLS[name][0], name, key, "cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("name", CALLS)
def test_gpu_tangents_of_upstream_gradients_are_refused(name):
    o = operands("cuda")
    o["x"].requires_grad_(True)
    y = CALLS[name][0](o)
    with fw.dual_level():
        up = fw.make_dual(torch.ones_like(y), torch.ones_like(y))
        with pytest.raises(NotImplementedError, match=name):
            torch.autograd.grad(y, o["x"], up)


@pytest.mark.gpu
@pytest.mark.parametrize("name,key", EACH)
def test_gpu_operands_that_are_negated_when_read(name, key):
    """The same numbers as their copies, upstream gradients as well."""
    def both(o, change):
        o["x"] = o["x"].detach().requires_grad_(True)
        y = call({**o, key: change(o[key])})
        with torch.no_grad():
            again = call({**o, key: change(o[key])})
        up = change(torch.full_like(y, 0.75))
        return y.detach(), again, torch.autograd.grad(y, o["x"], up)[0]

    def negated(t):
        t = torch._neg_view(-t)
        assert t.is_neg() and t.is_contiguous()
        return t

    call, o = CALLS[name][0], operands("cuda")
    want, got = both(o, lambda t: t), both(o, negated)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
