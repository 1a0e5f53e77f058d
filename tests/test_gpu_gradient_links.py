"""Gradients handed from one node's backward to another's: a pass over a
retained graph that reaches the second node alone takes nothing of an earlier
pass.  Each gradient is compared with the same one taken first, bit for bit but
for the parameter gradients that are summed with atomics (not looked at here).
"""
import pytest
import torch

from terra_amd import autograd, kernels
from terra_amd.mlp import SequentialMlp
from terra_amd.transformer import SequentialSwinTransformer

pytestmark = pytest.mark.gpu


def _rand(shape, seed, dev):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dev)


def test_branch_gradient_after_one_of_the_gate(dev):
    """An auxiliary loss on the branch of a half, after a pass for the layer scale alone."""
    torch.manual_seed(3)
    attn = SequentialSwinTransformer(1, 16, 16, 96, window_size=8, num_heads=3, layer_scale=0.3, residual_scale=0.9).to(dev)
    kept = []
    attn.attn.register_forward_hook(lambda m, i, o: kept.append(o))
    x = _rand((1, 256, 96), 1, dev).requires_grad_()
    y, h = attn(x), kept[0]
    grad = lambda out, to: torch.autograd.grad(out.square().sum(), to, retain_graph=True)[0]  # noqa: E731
    aux, main = grad(h, x), grad(y, x)
    for alone in (attn.layer_scale1, attn.attn.proj.weight):
        grad(y, alone)
        assert torch.equal(grad(h, x), aux)
        assert torch.equal(grad(y, x), main)
    both, = torch.autograd.grad(y.square().sum() + h.square().sum(), x)
    assert (both - aux - main).norm() <= 1e-5 * both.norm()


@pytest.mark.parametrize("tail", [False, True])
def test_residual_links(dev, tail):
    """partition_ln with the ends that hand it the residual's gradient."""
    C = 96
    geom = kernels.WindowGeometry(1, 16, 16, C, 8, 4, 4)
    x, w = _rand((1, 16, 16, C), 2, dev).requires_grad_(), _rand((C,), 3, dev).requires_grad_()
    link = autograd.ResidualLink()
    windows = autograd.partition_ln(x, geom, w, None, 1e-5, link=link)
    h = windows * 2
    y = autograd.residual_norm(h, x, geom=geom, link=link) if tail else autograd.reverse(h, geom, residual=x, link=link)
    grad = lambda out, to: torch.autograd.grad(out.square().sum(), to, retain_graph=True)[0]  # noqa: E731
    aux, main = grad(h, x), grad(y, x)
    grad(y, h)
    assert torch.equal(grad(h, x), aux)
    assert torch.equal(grad(y, x), main)


def test_column_sums(dev):
    x, w, b = _rand((64, 96), 4, dev), _rand((128, 96), 5, dev).requires_grad_(), _rand((128,), 6, dev).requires_grad_()
    link = autograd.ColumnSumLink()
    h = autograd.linear(x, w, b, bias_sums=link)
    a = autograd.gelu_dropout(h, 0.3, torch.tensor([5], device=dev), bias_sums=link)
    grad = lambda out, to: torch.autograd.grad(out.square().sum(), to, retain_graph=True)[0]  # noqa: E731
    aux, main = grad(h, b), grad(a, b)
    grad(a, h)
    assert torch.equal(grad(h, b), aux)
    assert torch.equal(grad(a, b), main)


@pytest.mark.parametrize("reentrant", [False, True])
def test_links_in_a_checkpointed_half(dev, reentrant):
    """The passes of a reentrant checkpoint are passes of their own."""
    from torch.utils.checkpoint import checkpoint

    torch.manual_seed(3)
    opts = dict(layer_scale=0.3, residual_scale=0.9, dropout=0.2)
    halves = [SequentialSwinTransformer(1, 16, 16, 96, window_size=8, num_heads=3, **opts),
              SequentialMlp(96, 384, hidden_dropout=0.2, **opts)]
    x = _rand((1, 256, 96), 7, dev)
    for half in halves:
        half.to(dev).train()
        grads = []
        for f in (half, lambda t: checkpoint(half, t, use_reentrant=reentrant)):
            torch.manual_seed(8)
            v = x.clone().requires_grad_()
            f(v).square().sum().backward()
            grads.append(v.grad)
        assert torch.equal(*grads)


def test_links_with_the_engine_in_the_callers_thread(dev):
    torch.manual_seed(3)
    opts = dict(layer_scale=0.3, residual_scale=0.9, dropout=0.2)
    for half in (SequentialSwinTransformer(1, 16, 16, 96, window_size=8, num_heads=3, **opts),
                 SequentialMlp(96, 384, hidden_dropout=0.2, **opts)):
        half.to(dev).train()
        grads = []
        for threads in (True, False):
            torch.manual_seed(8)
            x = _rand((1, 256, 96), 7, dev).requires_grad_()
            y = half(x)
            with torch.autograd.set_multithreading_enabled(threads):
                grads.append(torch.autograd.grad(y.square().sum(), x)[0])
        assert torch.equal(*grads)
