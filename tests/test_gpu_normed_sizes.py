"""Norms of the halves that the kernels do not take are torch's: they ran as modules before there were kernels for them."""
import pytest
import torch

from terra_amd import kernels, workloads
from terra_amd.attention import normed
from terra_amd.kernels import Norm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", [torch.nn.LayerNorm, torch.nn.RMSNorm])
@pytest.mark.parametrize("C,rows,eps", [((1 << 24) + 8, 1, 1e-5), (64, 5, -1e-3), (0, 4, 1e-5)])
def test_what_the_kernels_do_not_take(dev, kind, C, rows, eps):
    module = kind(C, eps=eps, device=dev)
    x = (workloads.activations((rows, C), 3, torch.float32) if C else torch.zeros(rows, 0)).to(dev).requires_grad_()
    with pytest.raises(ValueError):
        kernels.layer_norm(x.detach(), Norm.of(module))
    y = normed(module, x)
    assert y.grad_fn.name() != "LayerNormBackward"
    assert torch.equal(y, module(x))
    y.sum().backward()
    assert x.grad.shape == x.shape


@pytest.mark.parametrize("C,rows,eps", [(64, 0, 1e-5), (64, 5, 0.0), (1, 7, 1e-5)])
def test_what_they_take(dev, C, rows, eps):
    module = torch.nn.LayerNorm(C, eps=eps, device=dev)
    x = torch.randn(rows, C, device=dev, generator=torch.Generator(dev).manual_seed(1)).requires_grad_()
    y = normed(module, x)
    assert y.grad_fn.name() == "LayerNormBackward"
    # Two norms in fp32, each within a few roundings of values of at most sqrt(C).
    assert y.shape == x.shape and bool(((y - module(x)).abs() <= 16 * 2.0 ** -24 * max(C, 1) ** 0.5).all())
