"""The attention half with rotary positions and a regularised tail, and with an RMS norm of its own, against 64 bits,
forward and gradients.

fp32: normwise within 1e-5 of the oracle, as the halves without rotary positions."""
import pytest
import torch

from helpers import gain_block, rel_norm
from oracle import regularize as rg
from oracle import swin_oracle as so
from oracle import training as tr
from terra_amd import workloads
from terra_amd.transformer import SequentialSwinTransformer

pytestmark = pytest.mark.gpu

F32 = torch.float32


def _filled(blk):
    """Norms and gates that show in the output."""
    with torch.no_grad():
        for i, (name, p) in enumerate(blk.named_parameters()):
            if "post_norm" in name or "layer_scale" in name:
                p.copy_(0.7 + 0.3 * workloads.activations(p.shape, 70 + i, F32))
    return blk


@pytest.mark.parametrize("post_norm,layer_scale,residual_scale", [(True, 0.5, 0.75), (True, None, 1.0), (False, 0.5, 1.5)])
def test_tail(dev, post_norm, layer_scale, residual_scale):
    H = W = 16
    kw = dict(window_size=8, num_heads=6, rotary=True, post_norm=post_norm, layer_scale=layer_scale, residual_scale=residual_scale,
              init_seed_base=11)
    blk = _filled(gain_block(SequentialSwinTransformer(1, H, W, 192, **kw)))
    nxt = torch.nn.LayerNorm(192)
    with torch.no_grad():
        nxt.weight.copy_(1.0 + 0.2 * workloads.activations((192,), 90, F32))
    x = workloads.activations((2, H * W, 192), 7, F32)
    dy, dz = (workloads.activations((2, H * W, 192), i, F32) for i in (8, 9))

    ps = {k: p.detach().double().requires_grad_() for k, p in blk.named_parameters()}
    pn = [p.detach().double().requires_grad_() for p in (nxt.weight, nxt.bias)]
    xr, rot = x.double().requires_grad_(), blk.attn.rotary
    block = {k: v for k, v in ps.items() if "post_norm" not in k and "layer_scale" not in k}
    h = tr.swin_block_rotary(xr, H, W, 8, blk.shift_size, 6, block, rot.rates, rot.dim) - xr  # a norm of each token: order is all the same to it
    post = (ps["post_norm1.weight"], ps["post_norm1.bias"], blk.post_norm1.eps, False) if post_norm else None
    y, z = rg.residual_norm(h, xr, post, ps.get("layer_scale1"), (*pn, nxt.eps, False), None, residual_scale)
    z = z.view(y.shape)
    ref = torch.autograd.grad([y, z], [xr, *ps.values(), *pn], [dy.double(), dz.double()])

    blk, nxt = blk.to(dev), nxt.to(dev)
    xd = x.to(dev).requires_grad_()
    yd, zd = blk(xd, next_norm=nxt)
    assert rel_norm(yd.detach(), y.detach()) <= 1e-5 and rel_norm(zd.detach(), z.detach()) <= 1e-5
    got = torch.autograd.grad([yd, zd], [xd, *blk.parameters(), *nxt.parameters()], [dy.to(dev), dz.to(dev)])
    for name, a, b in zip(["x", *ps, "next.weight", "next.bias"], got, ref):
        assert rel_norm(a, b) <= 1e-5, name


def test_gradients_of_a_half_with_an_rms_norm(dev):
    """Against the same half in 64 bits, its norm an RMS norm over the rows."""
    H = W = 14
    blk = SequentialSwinTransformer(0, H, W, 96, window_size=7, num_heads=3, norm_layer=torch.nn.RMSNorm, rotary=True, init_seed_base=5)
    with torch.no_grad():
        for lin in (blk.attn.q_linear, blk.attn.k_linear, blk.attn.v_linear, blk.attn.proj):
            lin.weight.mul_(6.0)
        blk.norm1.weight.copy_(1.0 + 0.2 * workloads.activations((96,), 90, F32))
    x, dy = (workloads.activations((2, H * W, 96), i, F32) for i in (7, 8))
    ps = {k: p.detach().double().requires_grad_() for k, p in blk.named_parameters()}
    xr, rot = x.double().requires_grad_(), blk.attn.rotary
    n = tr.layer_norm(xr, ps["norm1.weight"], None, torch.finfo(F32).eps if blk.norm1.eps is None else blk.norm1.eps, True)[0]
    win = so.partition_frame(n.view(2, H, W, 96), 7, 0, 0)
    at = torch.arange(49)
    positions = torch.stack((at // 7, at % 7), -1)
    lin = lambda t, name: t @ ps[f"attn.{name}.weight"].T + ps[f"attn.{name}.bias"]  # noqa: E731
    turned = lambda t: tr.rotary(t.unflatten(-1, (3, 32)), positions, rot.rates, 32, 2).flatten(-2)  # noqa: E731
    o = so.window_attention_core(turned(lin(win, "q_linear")), turned(lin(win, "k_linear")), lin(win, "v_linear"), 3, 32 ** -0.5,
                                 ps["attn.relative_position_bias_table"], (7, 7), None, compute_dtype=torch.float64)
    y = so.reverse_frame(lin(o, "proj"), 2, H, W, 7, 0, 0, residual=xr).view(2, H * W, 96)
    ref = torch.autograd.grad(y, [xr, *ps.values()], dy.double())
    blk = blk.to(dev)
    xd = x.to(dev).requires_grad_()
    yd = blk(xd)
    assert rel_norm(yd.detach(), y.detach()) <= 1e-5
    for name, a, b in zip(["x", *ps], torch.autograd.grad(yd, [xd, *blk.parameters()], dy.to(dev)), ref):
        assert rel_norm(a, b) <= 1e-5, name
