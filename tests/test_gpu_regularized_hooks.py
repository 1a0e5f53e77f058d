"""Modules of the regularised halves that something watches or that are of
another class are called, not passed by: what their hooks see and change counts.

Tolerance: as in test_gpu_regularized_block.py, 2e-5 of the norm between two
fp32 paths of one forward, 1e-4 for gradients.
"""
import pytest
import torch

from terra_amd.mlp import SequentialMlp
from terra_amd.transformer import SequentialSwinTransformer

pytestmark = pytest.mark.gpu

OPTIONS = dict(post_norm=True, layer_scale=0.3, residual_scale=0.9, dropout=0.2)


def _halves(dev, **kw):
    torch.manual_seed(3)
    opts = {**OPTIONS, **kw}
    attn = SequentialSwinTransformer(1, 14, 14, 96, window_size=7, num_heads=3, init_seed_base=5, **opts)
    opts.pop("norm_layer", None)
    mlp = SequentialMlp(96, 384, init_seed_base=6, hidden_dropout=0.25, **opts)
    g = torch.Generator().manual_seed(7)
    with torch.no_grad():
        for b in (attn, mlp):
            for n, p in b.named_parameters():
                if "norm" in n:
                    p.add_(0.2 * torch.randn(p.shape, generator=g))
    return attn.to(dev).train(), mlp.to(dev).train()


def _input(dev):
    return torch.randn(2, 196, 96, generator=torch.Generator().manual_seed(8)).to(dev)


def _step(f, x):
    """f's output and input gradient with fixed masks."""
    x = x.detach().requires_grad_()
    torch.manual_seed(4)
    y = f(x)
    dy = torch.randn(y.shape, generator=torch.Generator().manual_seed(9)).to(y.device)
    return y.detach(), torch.autograd.grad(y, x, dy)[0]


def _close(got, want):
    for a, b, tol in zip(got, want, (2e-5, 1e-4)):
        assert (a - b).norm() <= tol * b.norm()


@pytest.mark.parametrize("name", ["fc1", "act", "fc2"])
def test_backward_hooks_of_layers(dev, name):
    _, mlp = _halves(dev)
    x = _input(dev)
    want = _step(mlp, x)
    layer, seen = getattr(mlp, name), []
    for register in (layer.register_full_backward_hook, layer.register_full_backward_pre_hook):
        handle = register(lambda *a: seen.append(len(a)))
        _close(_step(mlp, x), want)
        handle.remove()
    assert seen == [3, 2]
    # one that changes the gradient
    handle = layer.register_full_backward_hook(lambda m, gi, go: (2 * gi[0],))
    y, dx = _step(mlp, x)
    handle.remove()
    assert (dx - want[1]).norm() > 1e-2 * want[1].norm()


def test_global_backward_hooks(dev):
    _, mlp = _halves(dev)
    seen = []
    handle = torch.nn.modules.module.register_module_full_backward_hook(lambda m, gi, go: seen.append(m))
    try:
        _step(mlp, _input(dev))
    finally:
        handle.remove()
    assert {mlp.fc1, mlp.act, mlp.fc2} <= set(seen)
