"""The oracle of the regularised training operators: its generator against the
published known answers, its masks' statistics, its norms against torch."""
import numpy as np
import pytest
import torch

from oracle import regularize as rg
from oracle import swin_oracle as so
from terra_amd.kernels import WindowGeometry


@pytest.mark.parametrize("counter,key,want", [
    ((0, 0, 0, 0), (0, 0), (0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8)),
    ((0xffffffff,) * 4, (0xffffffff,) * 2, (0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd)),
    ((0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344), (0xa4093822, 0x299f31d0),
     (0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1)),
])
def test_philox_known_answers(counter, key, want):
    assert tuple(int(v) for v in rg.philox4x32_10(counter, key)) == want


@pytest.mark.parametrize("p", [0.05, 0.3, 0.5])
def test_mask_rate_and_independence(p):
    # n draws of a Bernoulli(p): the rate is off by more than 5 sqrt(p (1 - p) / n) once in 1.7 million.
    rows, C = 512, 1000
    keep = rg.keep_mask(1234567890123, rows, C, p, 7)
    sigma = (p * (1 - p) / keep.numel()) ** 0.5
    assert abs((~keep).double().mean().item() - p) < 5 * sigma + 2.0 ** -17
    other = rg.keep_mask(1234567890123, rows, C, p, 8)
    both = ((~keep) & (~other)).double().mean().item()
    assert abs(both - p * p) < 5 * (p * p * (1 - p * p) / keep.numel()) ** 0.5 + 2.0 ** -16
    # neighbouring columns and rows are as independent as streams
    for a, b in ((keep[:, 1:], keep[:, :-1]), (keep[1:], keep[:-1])):
        both = ((~a) & (~b)).double().mean().item()
        assert abs(both - p * p) < 5 * (p * p * (1 - p * p) / a.numel()) ** 0.5 + 2.0 ** -16


def test_mask_of_a_row_depends_on_the_row_alone():
    full = rg.keep_mask(99, 40, 50, 0.4)
    assert torch.equal(rg.keep_mask(99, 1, 50, 0.4, first_row=17), full[17:18])
    assert torch.equal(rg.keep_mask(99, 40, 30, 0.4), full[:, :30])


def test_scale_makes_the_mean_exact_and_p_one_drops_all():
    for p in (0.0, 0.1, 1 / 3, 0.999):
        t = rg.threshold(p)
        assert abs(rg.keep_scale(p) * (65536 - t) / 65536 - 1) < 1e-15
    assert rg.keep_scale(1.0) == 0.0 and not rg.keep_mask(5, 4, 16, 1.0).any()
    assert rg.keep_mask(5, 4, 16, 0.0).all()


def test_norms_are_torchs():
    x = torch.randn(5, 24, dtype=torch.float64, generator=torch.Generator().manual_seed(1))
    w, b = torch.randn(24, dtype=torch.float64), torch.randn(24, dtype=torch.float64)
    assert torch.allclose(rg.norm(x, w, b, 1e-5, False), torch.nn.functional.layer_norm(x, (24,), w, b, 1e-5), atol=1e-13)
    assert torch.allclose(rg.norm(x, w, None, 1e-6, True), torch.nn.functional.rms_norm(x, (24,), w, 1e-6), atol=1e-13)
    assert torch.allclose(rg.gelu(x), torch.nn.functional.gelu(x), atol=1e-14)


@pytest.mark.parametrize("B,H,W,ws,s", [(1, 14, 21, 7, 3), (2, 16, 24, 8, 4), (1, 8, 8, 8, 0)])
def test_window_sources_are_reverse_and_roll(B, H, W, ws, s):
    geom = WindowGeometry(B, H, W, 1, ws, s, s)
    rows = torch.arange(geom.num_windows * ws * ws).view(-1, ws, ws, 1)
    grid = so.reverse_unroll(rows, ws, H, W, s)
    assert torch.equal(rg.window_sources(geom), grid.reshape(-1))


def test_gradients_of_the_oracle_by_differences():
    g = torch.Generator().manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64).requires_grad_()  # noqa: E731
    h, x, gate, pw, pb, nw, nb = r(2, 3, 9), r(2, 3, 9), r(2, 9), r(9), r(9), r(9), r(9)

    def f(h, x, gate, pw, pb, nw, nb):
        return rg.residual_norm(h, x, (pw, pb, 1e-3, False), gate, (nw, nb, 1e-3, True), None, 0.7, 0.3, 11, 2)

    assert torch.autograd.gradcheck(f, (h, x, gate, pw, pb, nw, nb))
    assert np.isfinite(f(h, x, gate, pw, pb, nw, nb)[0].sum().item())
