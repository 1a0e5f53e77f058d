"""Rotary positions (terra_swin_rotary) against the 64-bit oracle.

Tolerances, with u = 2^-24: the turn reduced to fp32 is off by at most 2^-26 of a turn, an
angle by 1.6 u; sine and cosine add 2 u, the amplitude and the two products and
their sum 5 more: 9 u a (|u| + |v|), and half a step of the type.
"""
import pytest
import torch

from oracle import training as tr
from terra_amd import autograd, kernels
from terra_amd.kernels import Rotary

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _rand(shape, dt, seed=1):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dt)


def check(y, x, rot, positions, inverse=False):
    x, d = x.detach().cpu(), rot.dim
    rate = rot.rates
    ref = tr.rotary(x, positions.cpu(), rate, d, rot.axes, rot.interleaved, rot.amplitude, inverse)
    a = x.double().abs()
    pair = torch.zeros_like(a)
    first, second = (slice(0, d, 2), slice(1, d, 2)) if rot.interleaved else (slice(0, d // 2), slice(d // 2, d))
    pair[..., first] = pair[..., second] = a[..., first] + a[..., second]
    dt = y.dtype
    tol = 9 * U * abs(rot.amplitude) * pair + torch.finfo(dt).eps / 2 * ref.abs() + torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
    y = y.double().cpu()
    assert y.shape == ref.shape
    assert bool(((y - ref).abs() <= tol).all()), ((y - ref).abs() / tol).max()
    assert torch.equal(y[..., d:], x[..., d:].double())


@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("heads,head_dim,dim", [(1, 2, 2), (3, 8, 8), (2, 10, 6), (5, 16, 4), (1, 33, 12), (4, 64, 64), (6, 80, 40),
                                                (2, 96, 44), (16, 128, 128), (2, 257, 250), (3, 1200, 1100)])
def test_against_oracle(dev, dt, interleaved, heads, head_dim, dim):
    x, positions = _rand((3, 7, heads, head_dim), dt), torch.tensor([0, 1, 2, 5, 100, 4097, 1048576])
    rot = Rotary(dim, interleaved=interleaved)
    y = kernels.rotary(x.to(dev), rot, positions.to(dev))
    assert y.is_contiguous() and y.dtype == dt
    check(y, x, rot, positions)
    check(kernels.rotary(x.to(dev), rot, positions.to(dev), inverse=True), x, rot, positions, inverse=True)


@pytest.mark.parametrize("kw", [dict(scaling="linear", factor=4.0), dict(scaling="ntk", factor=8.0),
                                dict(scaling="yarn", factor=16.0, original_length=4096), dict(base=5e5, amplitude=0.5)])
def test_scaled(dev, kw):
    x, positions, rot = _rand((50, 4, 64), BF16), torch.arange(50) * 2999, Rotary(64, **kw)
    check(kernels.rotary(x.to(dev), rot, positions.to(dev)), x, rot, positions)


@pytest.mark.parametrize("dt", [torch.int32, torch.int64])
def test_positions(dev, dt):
    """Of both types: negative, the largest, of each sequence's own."""
    x, rot = _rand((2, 4, 3, 16), F32), Rotary(16)
    low, high = (-(1 << 31), (1 << 31) - 1) if dt == torch.int32 else (-(1 << 40), 1 << 40)
    positions = torch.tensor([[0, -1, low, high], [7, 7, 12345678, 3]], dtype=dt)
    check(kernels.rotary(x.to(dev), rot, positions.to(dev)), x, rot, positions)
    one = torch.tensor(17, dtype=dt)  # one for all tokens
    check(kernels.rotary(x.to(dev), rot, one.to(dev)), x, rot, one.expand(2, 4))


@pytest.mark.parametrize("window", [(7, 7), (8, 8), (5, 3)])
def test_two_axes(dev, window):
    n = window[0] * window[1]
    at = torch.arange(n)
    positions = torch.stack((at // window[1], at % window[1]), -1)
    x = _rand((6, n, 4, 32), BF16)
    for dim in (32, 20):
        rot = Rotary(dim, axes=2)
        check(kernels.rotary(x.to(dev), rot, positions.to(dev)), x, rot, positions)


def _views(big):
    """Heads that are not packed: [tokens.., heads, head_dim] views of big [3, 5, 8, 32]."""
    return {
        "query and key heads": big[:, :, :5],
        "every other head": big[:, :, ::2],
        "part of a head": big[..., 4:21],
        "heads before tokens": big.view(3, 8, 5, 32).transpose(1, 2),
        "some tokens": big[:, 1:4],
        "one token": big[1:2, 2:3, 3:5],
        "one head": big[:, :, 3:4],
    }


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("kind", list(_views(torch.zeros(3, 5, 8, 32))))
def test_strides(dev, kind, dt):
    big = _rand((3, 5, 8, 32), dt)
    x, xd = _views(big)[kind], _views(big.to(dev).clone())[kind]
    positions = torch.arange(x.shape[0] * x.shape[1]).view(x.shape[:2]) * 3 + 1
    for dim in (16, 10):
        for interleaved in (False, True):
            rot = Rotary(dim, interleaved=interleaved)
            check(kernels.rotary(xd, rot, positions.to(dev)), x, rot, positions)


@pytest.mark.parametrize("kind", list(_views(torch.zeros(3, 5, 8, 32))))
def test_in_place(dev, kind):
    big = _rand((3, 5, 8, 32), BF16)
    whole = big.to(dev)
    x, xd = _views(big)[kind], _views(whole)[kind]
    positions = torch.arange(x.shape[1]) + 5
    rot = Rotary(12)
    before = xd._version
    assert kernels.rotary(xd, rot, positions.to(dev), out=xd) is xd
    assert xd._version > before
    check(xd, x, rot, positions)
    _views(whole)[kind].copy_(x.to(dev))  # what stands beside it is left
    assert torch.equal(whole.cpu(), big)


def test_into_another_layout(dev):
    x, rot, positions = _rand((3, 5, 8, 32), F16), Rotary(32), torch.arange(5)
    for out in (torch.zeros(3, 8, 5, 32, dtype=F16, device=dev).transpose(1, 2), torch.zeros(3, 5, 9, 40, dtype=F16, device=dev)[:, :, 1:, 4:36],
                torch.zeros(3, 6, 8, 32, dtype=F16, device=dev)[:, 1:]):
        check(kernels.rotary(x.to(dev), rot, positions.to(dev), out=out), x, rot, positions)
    src = x.to(dev).transpose(1, 2).contiguous().transpose(1, 2)  # rows of two strides into rows of one
    check(kernels.rotary(src, rot, positions.to(dev), out=torch.zeros(3, 5, 8, 32, dtype=F16, device=dev)), x, rot, positions)


@pytest.mark.parametrize("shape", [(0, 4, 8), (3, 0, 4, 8), (3, 5, 0, 8)])
def test_empty(dev, shape):
    x = torch.zeros(shape, device=dev)
    positions = torch.zeros(shape[-3], dtype=torch.int64, device=dev)
    assert kernels.rotary(x, Rotary(8), positions).shape == x.shape


def test_infinities_and_nan_stay_in_their_pairs(dev):
    x = _rand((4, 2, 16), F32)
    x[1, 0, 3], x[2, 1, 15] = float("inf"), float("nan")
    y = kernels.rotary(x.to(dev), Rotary(16), torch.arange(4, device=dev)).cpu()
    bad = (~y.isfinite()).nonzero().tolist()
    assert bad == [[1, 0, 3], [1, 0, 11], [2, 1, 7], [2, 1, 15]]


def test_tokens_past_32_bits_of_elements(dev):
    tokens, heads, head_dim = 1 << 20, 16, 136  # 2.3e9 elements, 4.6 GB
    x = torch.zeros(tokens, heads, head_dim, dtype=BF16, device=dev)
    x[-3:] = _rand((3, heads, head_dim), BF16).to(dev)
    positions, rot = torch.arange(tokens, device=dev), Rotary(136)
    kernels.rotary(x, rot, positions, out=x)
    check(x[-3:].clone(), _rand((3, heads, head_dim), BF16), rot, positions[-3:])


class TestAutograd:
    def test_gradient_is_the_turn_back(self, dev):
        x, rot, positions = _rand((2, 9, 4, 64), BF16).to(dev).requires_grad_(), Rotary(32, interleaved=True), torch.arange(9, device=dev)
        dy = _rand((2, 9, 4, 64), BF16, 2).to(dev)
        y = autograd.rotary(x, rot, positions)
        check(y, x, rot, positions)
        y.backward(dy)
        check(x.grad, dy, rot, positions, inverse=True)

    def test_derivatives_of_every_order_and_mode(self, dev):
        x, rot, positions = _rand((5, 2, 8), F32).to(dev), Rotary(8), torch.arange(5, device=dev)
        from torch.autograd import forward_ad

        with forward_ad.dual_level():
            t = _rand((5, 2, 8), F32, 2).to(dev)
            out = forward_ad.unpack_dual(autograd.rotary(forward_ad.make_dual(x, t), rot, positions))
            check(out.tangent, t, rot, positions)
        x.requires_grad_()
        y = autograd.rotary(x, rot, positions)
        g, = torch.autograd.grad((y ** 3).sum(), x, create_graph=True)
        h, = torch.autograd.grad(g.square().sum(), x)
        ref = x.detach().cpu().double().requires_grad_()
        yr = tr.rotary(ref, positions.cpu(), rot.rates, 8)
        gr, = torch.autograd.grad((yr ** 3).sum(), ref, create_graph=True)
        hr, = torch.autograd.grad(gr.square().sum(), ref)
        # Four turns, each off by 9 u of at most sqrt 2 times its pair's length, in an expression of the fourth degree,
        # whose other products add 8 roundings: (4 x 9 x 4 + 8) (sqrt 2)^4 u of the largest value's scale.
        scale = 24 * x.detach().abs().max().item() ** 3 * x.detach().abs().max().item() ** 2
        assert (h.cpu().double() - hr).abs().max() <= 608 * U * scale

    def test_first_used_in_inference_mode(self, dev):
        rot, positions = Rotary(16), torch.arange(4, device=dev)
        with torch.inference_mode():
            kernels.rotary(torch.zeros(4, 2, 16, device=dev), rot, positions)
        x, dy = _rand((4, 2, 16), F32).to(dev).requires_grad_(), _rand((4, 2, 16), F32, 2).to(dev)
        autograd.rotary(x, rot, positions).backward(dy)
        check(x.grad, dy, rot, positions, inverse=True)

    def test_checkpointed(self, dev):
        from torch.utils.checkpoint import checkpoint

        rot, positions = Rotary(16), torch.arange(4, device=dev)
        x, dy = _rand((4, 2, 16), F32).to(dev).requires_grad_(), _rand((4, 2, 16), F32, 2).to(dev)
        checkpoint(lambda t: autograd.rotary(t, rot, positions), x, use_reentrant=False).backward(dy)
        check(x.grad, dy, rot, positions, inverse=True)

    def test_heads_of_a_packed_row(self, dev):
        qkv = _rand((6, 9, 16), BF16).to(dev).requires_grad_()
        rot, positions, dy = Rotary(16), torch.arange(6, device=dev), _rand((6, 6, 16), BF16, 2).to(dev)
        autograd.rotary(qkv[:, :6], rot, positions).backward(dy)
        check(qkv.grad[:, :6], dy, rot, positions, inverse=True)
        assert not qkv.grad[:, 6:].any()

    def test_heads_of_other_strides_are_copied(self, dev):
        x = _rand((4, 16, 3), F32).to(dev).transpose(1, 2)
        rot, positions = Rotary(16), torch.arange(4, device=dev)
        with pytest.raises(ValueError, match="unit stride"):
            kernels.rotary(x, rot, positions)
        check(autograd.rotary(x, rot, positions), x, rot, positions)


def test_captured(dev):
    x, rot, positions = _rand((33, 4, 64), BF16).to(dev), Rotary(64), torch.arange(33, device=dev)
    kernels.rotary(x, rot, positions)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = kernels.rotary(x, rot, positions)
    for seed in range(4):
        x.copy_(_rand((33, 4, 64), BF16, seed))
        positions.add_(1000)
        graph.replay()
        eager = kernels.rotary(x, rot, positions)
        torch.cuda.synchronize()
        assert torch.equal(y, eager)


def test_refusals(dev):
    x, p = torch.zeros(2, 4, 3, 16, device=dev), torch.arange(4, device=dev)
    r = Rotary(16)
    for bad, error, text in (
        (lambda: kernels.rotary(x.double(), r, p), TypeError, "not supported"),
        (lambda: kernels.rotary(x[0, 0, 0], r, p), ValueError, "heads, head_dim"),
        (lambda: kernels.rotary(x[..., :8], r, p), ValueError, "rotated elements"),
        (lambda: kernels.rotary(x, r, p[:3]), ValueError, "positions of the tokens"),
        (lambda: kernels.rotary(x, r, p.view(4, 1)), ValueError, "positions of the tokens"),
        (lambda: kernels.rotary(x, r, p.float()), ValueError, "int32 or int64"),
        (lambda: kernels.rotary(x, r, torch.arange(8, device=dev)[::2]), ValueError, "contiguous"),
        (lambda: kernels.rotary(x, r, p.cpu()), RuntimeError, "ROCm devices only"),
        (lambda: kernels.rotary(x, Rotary(16, axes=2), p), ValueError, "2 values for each token"),
        (lambda: kernels.rotary(x, r, p, out=x[:1]), ValueError, "out must be"),
        (lambda: kernels.rotary(x, r, p, out=x.half()), ValueError, "out must be"),
        (lambda: kernels.rotary(x[:, 1:3], r, p[:2], out=x[:, :2]), ValueError, "overlap"),
        (lambda: kernels.rotary(x, r, p, out=x[:1].expand(2, 4, 3, 16)), ValueError, "share a place"),
    ):
        with pytest.raises(error, match=text):
            bad()
