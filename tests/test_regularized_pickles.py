"""Halves pickled before the regularisation options were there."""
import io

import pytest
import torch

from terra_amd.mlp import SequentialMlp
from terra_amd.transformer import SequentialSwinTransformer

OPTIONS = ("post_norm1", "post_norm2", "layer_scale1", "layer_scale2", "residual_scale", "hidden_dropout", "dropout")


def _half(kind, **kw):
    if kind == "mlp":
        return SequentialMlp(96, 384, init_seed_base=6, **kw)
    return SequentialSwinTransformer(1, 14, 14, 96, window_size=7, num_heads=3, init_seed_base=5, **kw)


def _through_a_pickle(module):
    f = io.BytesIO()
    torch.save(module, f)
    f.seek(0)
    return torch.load(f, weights_only=False)  # of a file that this test wrote


def _older(kind):
    """A half as an earlier version would have pickled it."""
    module = _half(kind)
    for name in OPTIONS:
        module.__dict__.pop(name, None)
    return _through_a_pickle(module)


@pytest.mark.parametrize("kind", ["attention", "mlp"])
def test_options_are_off(kind):
    old, new = _older(kind), _half(kind)
    names = [n for n in OPTIONS if hasattr(new, n)]
    assert len(names) == (4 if kind == "attention" else 5)
    assert all(getattr(old, n) == getattr(new, n) for n in names)
    assert old.state_dict().keys() == new.state_dict().keys()


@pytest.mark.parametrize("kind", ["attention", "mlp"])
def test_options_come_back(kind):
    kw = dict(post_norm=True, layer_scale=0.3, residual_scale=0.9, dropout=0.1)
    want = _half(kind, **kw)
    got = _through_a_pickle(want)
    i = 1 if kind == "attention" else 2
    assert type(getattr(got, f"post_norm{i}")) is torch.nn.LayerNorm
    assert torch.equal(getattr(got, f"layer_scale{i}"), getattr(want, f"layer_scale{i}"))
    assert (got.residual_scale, got.dropout) == (0.9, 0.1)
    assert got.state_dict().keys() == want.state_dict().keys()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["attention", "mlp"])
def test_forward_of_an_older_half(dev, kind):
    x = torch.randn(1, 196, 96, generator=torch.Generator().manual_seed(1)).to(dev)
    old, new = _older(kind).to(dev).train(), _half(kind).to(dev).train()
    for a, b in zip(old.parameters(), new.parameters()):
        assert torch.equal(a, b)
    with torch.no_grad():
        assert torch.equal(old(x), new(x))
