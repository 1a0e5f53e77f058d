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


def _watched(half):
    """The half's call, and its norms by name."""
    attn, mlp = half
    names = {"norm1": attn.norm1, "post_norm1": attn.post_norm1, "norm2": mlp.norm2, "post_norm2": mlp.post_norm2}
    return lambda x: mlp(attn(x)), names


@pytest.mark.parametrize("name", ["norm1", "post_norm1", "norm2", "post_norm2"])
def test_hooks_of_norms(dev, name):
    f, norms = _watched(_halves(dev))
    x, norm, seen = _input(dev), norms[name], []
    want = _step(f, x)
    for register in (norm.register_forward_hook, norm.register_forward_pre_hook, norm.register_full_backward_hook,
                     norm.register_full_backward_pre_hook):
        handle = register(lambda *a: seen.append(len(a)))
        _close(_step(f, x), want)
        handle.remove()
    assert seen == [3, 2, 3, 2]
    handle = norm.register_forward_hook(lambda m, i, o: 2 * o)
    got = _step(f, x)
    handle.remove()
    with torch.no_grad():  # the same as a norm of twice the size
        norm.weight.mul_(2)
        norm.bias.mul_(2)
    assert (got[0] - want[0]).norm() > 1e-2 * want[0].norm()
    _close(got, _step(f, x))


@pytest.mark.parametrize("watched", [False, True])
def test_hooks_of_the_next_norm(dev, watched):
    attn, mlp = _halves(dev)
    x, seen = _input(dev), []
    with torch.no_grad():
        torch.manual_seed(4)
        y, z = attn(x, next_norm=mlp.norm2)
        if watched:
            mlp.norm2.register_forward_hook(lambda m, i, o: seen.append(o.shape))
        torch.manual_seed(4)
        y2, z2 = attn(x, next_norm=mlp.norm2)
    assert torch.equal(y, y2) and len(seen) == watched
    assert (z - z2).norm() <= 2e-5 * z.norm() and z2.dtype == z.dtype and z2.shape == z.shape


@pytest.mark.parametrize("autocast", [False, True])
def test_hooks_keep_the_types(dev, autocast):
    """Under autocast torch's LayerNorm gives fp32: the stream and the handed-over norm keep the launch's types."""
    attn, mlp = _halves(dev)
    x = _input(dev)

    def run():
        with torch.no_grad(), torch.amp.autocast("cuda", dtype=torch.bfloat16, enabled=autocast):
            y, z = attn(x, next_norm=mlp.norm2)
            return [t.dtype for t in (y, z, mlp(y, normed=z), mlp(y))]

    want = run()
    for norm in (attn.post_norm1, mlp.norm2, mlp.post_norm2):
        norm.register_forward_hook(lambda *a: None)
    assert run() == want


class Centred(torch.nn.Module):
    """A norm of another class: takes the mean off, and counts its calls."""

    def __init__(self, channels):
        super().__init__()
        self.weight, self.calls = torch.nn.Parameter(torch.ones(channels)), 0

    def forward(self, v):
        self.calls += 1
        return (v - v.mean(-1, keepdim=True)) * self.weight


def test_norms_of_another_class(dev):
    """Against the half composed of torch operations around the same branch."""
    attn, mlp = _halves(dev, norm_layer=Centred, dropout=0.0)
    mlp.norm2, mlp.post_norm2, mlp.hidden_dropout = Centred(96).to(dev), Centred(96).to(dev), 0.0
    off = SequentialSwinTransformer(1, 14, 14, 96, window_size=7, num_heads=3, norm_layer=Centred).to(dev)
    off.load_state_dict({k: v for k, v in attn.state_dict().items() if "post_norm" not in k and "scale" not in k})

    def ref(x):
        branch = off(x) - x
        y = 0.9 * x + 0.3 * attn.post_norm1(branch)
        h = mlp.fc2(torch.nn.functional.gelu(mlp.fc1(mlp.norm2(y))))
        return 0.9 * y + 0.3 * mlp.post_norm2(h)

    x = _input(dev)
    want = _step(ref, x)
    for norm in (attn.norm1, attn.post_norm1, mlp.norm2, mlp.post_norm2):
        norm.calls = 0
    _close(_step(lambda x: mlp(attn(x)), x), want)
    assert [n.calls for n in (attn.norm1, attn.post_norm1, mlp.norm2, mlp.post_norm2)] == [1] * 4
    y, z = attn(x, next_norm=mlp.norm2)
    assert (mlp(y, normed=z) - want[0]).norm() <= 2e-5 * want[0].norm()


def test_norms_over_other_dimensions_are_refused(dev):
    """A norm without an affine map over fewer channels has no parameter whose size would show it."""
    attn, mlp = _halves(dev)
    x = _input(dev)
    attn.post_norm1 = torch.nn.LayerNorm(48, elementwise_affine=False).to(dev)
    mlp.post_norm2 = torch.nn.LayerNorm((196, 48), elementwise_affine=False).to(dev)
    for half in (attn, mlp):
        with pytest.raises(RuntimeError, match="normalized_shape"):
            half(x)
    mlp.post_norm2 = torch.nn.LayerNorm((196, 96)).to(dev)  # over the tokens too: called, and right
    with torch.no_grad():
        torch.manual_seed(4)
        y = mlp(x)
        assert y.shape == x.shape
