"""WindowAttention.core on projected q, k, v of a module with rotary positions.

core turns the heads by the kernel that attend uses and calls the same attention, so the two differ by roundings
alone: fp32 within 1e-5 of the largest value, bf16 within 2e-2, as in the block's other tests."""
import pytest
import torch

from helpers import rel_maxabs
from terra_amd import workloads
from terra_amd.attention import WindowAttention
from terra_amd.kernels import Rotary, ShiftMask

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def _attn(dev, dtype, rot, bias=True, C=96, heads=3, window=(7, 7)):
    attn = WindowAttention(C, window, heads, rotary=rot, use_relative_position_bias=bias, init_seed_base=5)
    with torch.no_grad():
        for p in attn.parameters():
            p.mul_(6.0)
    return attn.to(dev).to(dtype)


@pytest.mark.parametrize("rot", [True, Rotary(16, axes=2, interleaved=True, amplitude=1.25)])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("packed", [True, False])
def test_core_is_attends(dev, rot, dtype, packed):
    attn = _attn(dev, dtype, rot)
    tol = 1e-5 if dtype == F32 else 2e-2
    x = workloads.activations((8, 49, 96), 3, dtype).to(dev)
    mask = ShiftMask(14, 14, 3, 3, 0, 2, 2)
    with torch.no_grad():
        parts = attn.qkv(x).chunk(3, -1)
        q, k, v = parts if packed else (t.contiguous() for t in parts)
        ref, got = attn.attend(x, mask), attn.core(q, k, v, mask)
        assert rel_maxabs(got, ref) <= tol
        attn.rotary = None
        assert rel_maxabs(attn.core(q, k, v, mask), ref) > 0.05  # without positions it is another attention


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_gradients_of_the_core(dev, dtype):
    attn = _attn(dev, dtype, True, bias=False)
    tol = 1e-5 if dtype == F32 else 2e-2
    x = workloads.activations((4, 49, 96), 3, dtype).to(dev).requires_grad_()
    dy = workloads.activations((4, 49, 96), 4, dtype).to(dev)
    grads = []
    for call in (attn.attend, lambda t: attn.core(*attn.qkv(t).chunk(3, -1))):
        grads.append(torch.autograd.grad(call(x), [x, attn.q_linear.weight, attn.k_linear.weight, attn.v_linear.weight], dy))
    for a, b in zip(*grads):
        assert rel_maxabs(b, a) <= tol


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_windows_in_padded_rows(dev, dtype):
    """49 tokens in 64 rows: those of the window are the same, whatever stands in the others."""
    attn = _attn(dev, dtype, True)
    x = workloads.activations((4, 49, 96), 3, dtype).to(dev)
    with torch.no_grad():
        parts = attn.qkv(x).chunk(3, -1)
        padded = [torch.cat((t, torch.full((4, 15, 96), 3.0, dtype=dtype, device=dev)), 1) for t in parts]
        got = attn.core(*padded, n_real=49)[:, :49]
        assert rel_maxabs(got, attn.attend(x)) <= (1e-5 if dtype == F32 else 2e-2)
        with pytest.raises(ValueError, match="positions of the tokens"):
            attn.core(*padded)


def test_only_one_derivative_of_the_core(dev):
    """As attend's: a second one would leave terms out without a word."""
    attn = _attn(dev, F32, True)
    x = workloads.activations((4, 49, 96), 3, F32).to(dev).requires_grad_()
    g, = torch.autograd.grad(attn.core(*attn.qkv(x).chunk(3, -1)).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()
