"""The 64-bit oracle of the training step's operators against torch and closed forms (CPU)."""
import math

import pytest
import torch
import torch.nn.functional as F

from oracle import regularize as rg
from oracle import training as tr


def _rand(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)


@pytest.mark.parametrize("rms", [False, True])
def test_norms_against_torch(rms):
    x, w, b, dy = _rand(3, 5, 17), _rand(17, seed=1), _rand(17, seed=2), _rand(3, 5, 17, seed=3)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = F.rms_norm(x, (17,), w, 1e-3) + b if rms else F.layer_norm(x, (17,), w, b, 1e-3)
    torch.testing.assert_close(tr.layer_norm(x, w, b, 1e-3, rms)[0], y)
    grads = torch.autograd.grad(y, leaves, dy)
    for got, ref in zip(tr.layer_norm_backward(dy, x, w, 1e-3, rms), grads):
        torch.testing.assert_close(got, ref)


def test_rotary_is_a_turn():
    x, rate = _rand(2, 7, 3, 10), tr.rates(8)[0]
    positions = torch.arange(7) * 3
    for interleaved in (False, True):
        y = tr.rotary(x, positions, rate, 8, interleaved=interleaved)
        assert torch.equal(y[..., 8:], x[..., 8:])
        torch.testing.assert_close(y[..., :8].norm(dim=-1), x[..., :8].norm(dim=-1))
        torch.testing.assert_close(tr.rotary(y, positions, rate, 8, interleaved=interleaved, inverse=True), x)
        # Products of two turned vectors depend on the difference of their positions alone.
        a, b = _rand(1, 1, 8, seed=4), _rand(1, 1, 8, seed=5)
        at = lambda v, p: tr.rotary(v, torch.tensor([p]), rate, 8, interleaved=interleaved)  # noqa: E731
        torch.testing.assert_close((at(a, 9) * at(b, 4)).sum(), (at(a, 105) * at(b, 100)).sum())
    pair = tr.rotary(torch.tensor([[[1.0, 0.0]]]), torch.tensor([1]), tr.rates(2)[0], 2)
    torch.testing.assert_close(pair, torch.tensor([[[math.cos(1.0), math.sin(1.0)]]], dtype=torch.float64))


def test_rates():
    f = tr.rates(16)[0]
    torch.testing.assert_close(f, 10000.0 ** (-torch.arange(8, dtype=torch.float64) / 8))
    torch.testing.assert_close(tr.rates(16, scaling="linear", factor=4.0)[0], f / 4)
    g = tr.rates(16, scaling="ntk", factor=4.0)[0]
    assert g[0] == f[0] and abs(g[-1] / f[-1] * 4 - 1) < 1e-12  # the slowest by the factor, the fastest not at all
    h, amplitude = tr.rates(16, scaling="yarn", factor=4.0, original_length=4096)
    assert h[0] == f[0] and abs(h[-1] / f[-1] * 4 - 1) < 1e-12 and amplitude == 0.1 * math.log(4.0) + 1
    assert tr.rates(16, axes=2)[0].numel() == 4


@pytest.mark.parametrize("maximize", [False, True])
def test_adamw_against_torch(maximize):
    p, grads = torch.nn.Parameter(_rand(50)), [_rand(50, seed=s) for s in range(1, 6)]
    opt = torch.optim.AdamW([p], lr=1e-2, betas=(0.8, 0.95), eps=1e-6, weight_decay=0.1, maximize=maximize)
    q, m, v = p.detach().clone(), torch.zeros(50).double(), torch.zeros(50).double()
    for step, g in enumerate(grads, 1):
        p.grad = g
        opt.step()
        m, v = tr.moments(-g if maximize else g, m, v, 0.8, 0.95)
        q, _ = tr.updated(q, m, v, step, 1e-2, 0.8, 0.95, 1e-6, 0.1)
        torch.testing.assert_close(q, p.detach())


def test_e4m3():
    values = tr.e4m3_values()
    codes = torch.arange(127, dtype=torch.uint8)
    assert torch.equal(codes.view(torch.float8_e4m3fn).double(), values)
    x = torch.cat((_rand(20000) * 100, _rand(20000, seed=1) * 0.01, values, -values, (values[1:] + values[:-1]) / 2))
    x = x.clamp(-448, 448).float().double()  # torch rounds from float32
    code, _ = tr.nearest_code(x)
    assert torch.equal(code, x.float().to(torch.float8_e4m3fn).view(torch.uint8))


def test_root_codes_have_the_mean():
    values = tr.e4m3_values()
    all_draws = torch.arange(65536)
    for w in (1.2345, 300.0 ** 2, 0.003 ** 2, 2.0 ** -9 * 1.7, 447.0 ** 2):
        codes, _ = tr.root_code(torch.full((65536,), w, dtype=torch.float64), all_draws)
        mean = values[codes.long()].square().mean().item()
        assert abs(mean - w) <= w * 1e-4, w
    assert tr.root_code(torch.tensor([0.0, 1e-30]).double(), torch.tensor([65535, 0]))[0].tolist() == [0, 1]
    assert tr.root_code(torch.tensor([448.0 ** 2 * 1.0001]).double(), torch.tensor([0]))[0].tolist() == [126]


def test_draws_are_those_of_dropout():
    """With the counter's third word 0 they are the dropout mask's, whose oracle is another one."""
    seed = 0x1234567890ABCDE
    d = tr.draws(seed, 77, tensor=5, step=0, stream=3)
    for p in (0.1, 0.5, 0.9):
        keep = rg.keep_mask(seed, 6, 77, p, 3)[5]
        assert torch.equal(d >= round(p * 65536), keep)


def test_positions_of_a_module_built_without_memory():
    from terra_amd.attention import WindowAttention

    real = WindowAttention(32, (3, 5), 2, rotary=True)
    with torch.device("meta"):
        m = WindowAttention(32, (3, 5), 2, rotary=True)
    m = m.to_empty(device="cpu")
    m.token_positions.fill_(77)
    m.load_state_dict(real.state_dict())
    assert torch.equal(m.token_positions, real.token_positions)
    assert torch.equal(m.rotary.rates, real.rotary.rates)
