"""Second derivatives that the regularised operators do not have are refused
whichever way they are asked for: a gradient taken with create_graph may be used
as a value, but no derivative of it is left out of a sum.
"""
import pytest
import torch

from terra_amd import autograd
from terra_amd.kernels import Norm

pytestmark = pytest.mark.gpu


def _rand(shape, seed, dev):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dev).requires_grad_()


def _gelu(v, dev):
    return autograd.gelu_dropout(v["h"] * v["w"], 0.3, torch.tensor([5], device=dev))


def _tail(v, dev):
    y, z = autograd.residual_norm(v["h"] * v["w"], v["x"], Norm(v["w"]), v["g"], Norm(v["w"]), p=0.3,
                                  seed=torch.tensor([5], device=dev))
    return y + z


@pytest.mark.parametrize("f", [_gelu, _tail])
def test_gradient_penalty_is_refused(dev, f):
    v = {n: _rand(s, i, dev) for i, (n, s) in enumerate(dict(h=(8, 64), x=(8, 64), w=(64,), g=(64,)).items())}
    used = [t for n, t in v.items() if n in ("h", "w") or f is _tail]
    out = f(v, dev)
    plain = torch.autograd.grad(out.square().sum(), used, retain_graph=True)
    grads = torch.autograd.grad(out.square().sum(), used, create_graph=True)
    for a, b in zip(grads, plain):
        assert torch.equal(a, b)
    penalty = sum(g.square().sum() for g in grads)
    for t in used:  # the loss beside it reaches t another way
        with pytest.raises((RuntimeError, NotImplementedError), match="twice"):
            torch.autograd.grad(penalty + t.square().sum(), t, retain_graph=True)
    with pytest.raises((RuntimeError, NotImplementedError), match="twice"):
        (penalty + out.square().sum()).backward()


@pytest.mark.parametrize("f", [_gelu, _tail])
def test_through_the_output_gradient_is_refused(dev, f):
    """The gradient is linear in the output's; that derivative is not there either."""
    v = {n: _rand(s, i, dev) for i, (n, s) in enumerate(dict(h=(8, 64), x=(8, 64), w=(64,), g=(64,)).items())}
    d = torch.ones(8, 64, device=dev, requires_grad=True)
    g, = torch.autograd.grad(f(v, dev), v["h"], d, create_graph=True)
    with pytest.raises((RuntimeError, NotImplementedError), match="twice"):
        torch.autograd.grad(g.sum() + d.sum(), d)
