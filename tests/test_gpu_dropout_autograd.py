"""Derivatives of autograd.dropout and autograd.gelu_dropout beside the first
backward: forward mode, and second derivatives.

Both maps act element by element, so a tangent is multiplied by what a gradient
is: equal bit for bit to the backward kernel's result on it.
"""
import pytest
import torch
from torch.autograd import forward_ad

from terra_amd import autograd, kernels

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _rand(shape, dt, seed, dev):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dt).to(dev)


def _seed(dev, value=0x1234567890ABCDE):
    return torch.tensor([value], dtype=torch.int64, device=dev)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("needs_grad", [False, True])
@pytest.mark.parametrize("p", [0.0, 0.3])
def test_tangents(dev, dt, needs_grad, p):
    x, t = _rand((37, 100), dt, 1, dev).requires_grad_(needs_grad), _rand((37, 100), dt, 2, dev)
    seed = _seed(dev) if p else None
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, t)
        y = forward_ad.unpack_dual(autograd.dropout(dual, p, seed, 4))
        assert torch.equal(y.primal, kernels.dropout(x, p, seed, 4))
        assert torch.equal(y.tangent, kernels.dropout(t, p, seed, 4))
        a = forward_ad.unpack_dual(autograd.gelu_dropout(dual, p, seed, 4))
        assert torch.equal(a.primal, kernels.gelu_dropout(x.detach(), p, seed, 4))
        assert torch.equal(a.tangent, kernels.gelu_dropout_backward(t, x.detach(), p, seed, 4))
        with torch.no_grad():
            assert torch.equal(forward_ad.unpack_dual(autograd.dropout(dual, p, seed, 4)).tangent, y.tangent)
        # one without a tangent stays without
        assert forward_ad.unpack_dual(autograd.dropout(x, p, seed, 4)).tangent is None


def test_tangent_of_strided_rows(dev):
    """A tangent comes in its primal's strides, or as an expanded one."""
    x, t = _rand((20, 192), torch.float32, 3, dev)[:, 64:128], _rand((20, 64), torch.float32, 4, dev)
    with forward_ad.dual_level():
        y = forward_ad.unpack_dual(autograd.dropout(forward_ad.make_dual(x, t), 0.25, _seed(dev)))
        assert torch.equal(y.tangent, kernels.dropout(t, 0.25, _seed(dev)))
        one = torch.ones((), device=dev).expand(20, 64)
        y = forward_ad.unpack_dual(autograd.dropout(forward_ad.make_dual(x.contiguous(), one), 0.25, _seed(dev)))
        assert torch.equal(y.tangent, kernels.dropout(torch.ones(20, 64, device=dev), 0.25, _seed(dev)))


def test_tangents_of_no_rows(dev):
    x = torch.empty(0, 8, device=dev)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, x.clone())
        for f in (autograd.dropout, autograd.gelu_dropout):
            assert forward_ad.unpack_dual(f(dual, 0.3, _seed(dev))).tangent.shape == (0, 8)


@pytest.mark.parametrize("dt", TYPES)
def test_dropout_twice_differentiated(dev, dt):
    """Of sum(w y^2) with y = d x (d the mask times the scale): the gradient is 2 w d^2 x, its derivative along v
    2 w d^2 v.  Products of values rounded to the type one after the other: six roundings of half an eps."""
    x, v, w = (_rand((37, 100), dt, i, dev) for i in (6, 7, 8))
    x.requires_grad_()
    d = kernels.dropout(torch.ones(37, 100, device=dev), 0.3, _seed(dev), 4).double()
    y = autograd.dropout(x, 0.3, _seed(dev), 4)
    g, = torch.autograd.grad((w * y * y).sum(), x, create_graph=True)
    want = 2 * w.double() * d * d
    tol = 3 * torch.finfo(dt).eps + 4 * torch.finfo(torch.float32).eps
    near = lambda a, b: bool(((a.detach().double() - b).abs() <= tol * b.abs() + 1e-6).all())  # noqa: E731
    assert near(g, want * x.detach().double())
    h, = torch.autograd.grad((g * v).sum(), x)
    assert near(h, want * v.double())


def test_out_of_a_saved_tensor(dev):
    """A tensor that a graph has saved and a call then writes into is refused by the backward, as after torch's own
    in-place operations."""
    calls = {
        "dropout": lambda t: kernels.dropout(t, 0.3, _seed(dev), out=t),
        "gelu_dropout": lambda t: kernels.gelu_dropout(t, 0.3, _seed(dev), out=t),
        "gelu_dropout_backward": lambda t: kernels.gelu_dropout_backward(t, t.clone(), 0.3, _seed(dev), out=t),
    }
    for name, call in calls.items():
        for shape in ((16, 64), (0, 64)):
            x = _rand(shape, torch.float32, 5, dev).requires_grad_()
            v = torch.exp(x)  # saves its result
            before = v._version
            call(v.detach())
            assert v._version == before + 1, name
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                v.sum().backward()
        with pytest.raises(ValueError, match="out must be"):  # a refused call leaves the count
            kernels.dropout(v.detach(), 0.3, _seed(dev), out=v.detach().half())
        assert v._version == before + 1
    with torch.inference_mode():
        t = torch.ones(8, 8, device=dev)
        assert kernels.dropout(t, 0.3, _seed(dev), out=t) is t
    assert kernels.dropout(t, 0.3, _seed(dev), out=t) is t
