"""The positions of WindowAttention(rotary=...) on the device: moved there with the module, so that a first call of it
may be captured, and kept from a first call in inference mode for a later one with gradients."""
import pytest
import torch

from terra_amd import workloads
from terra_amd.attention import WindowAttention
from terra_amd.kernels import Rotary

pytestmark = pytest.mark.gpu


def test_moved_with_the_module(dev):
    rot = Rotary(32, axes=2)
    warm, attn = (WindowAttention(96, (7, 7), 3, rotary=rot, init_seed_base=5).to(dev) for _ in range(2))
    assert attn._positions.device == torch.device("cuda", torch.cuda.current_device())
    x = workloads.activations((4, 49, 96), 3, torch.float32).to(dev)
    with torch.no_grad():
        ref = warm(x)  # sends the rates, which the two share, and prepares the library
        attn.qkv(x)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = attn(x)
        for _ in range(3):
            y.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, ref)
            x.mul_(-0.5)
            ref = warm(x)


def test_built_without_memory(dev):
    real = WindowAttention(96, (7, 7), 3, rotary=True, init_seed_base=5).to(dev)
    x = workloads.activations((4, 49, 96), 3, torch.float32).to(dev)
    with torch.inference_mode():
        y = real(x)
    for assign in (True, False):
        with torch.device("meta"):
            m = WindowAttention(96, (7, 7), 3, rotary=True)
        if not assign:
            m = m.to_empty(device=dev)
        m.load_state_dict(real.state_dict(), assign=assign)
        with torch.inference_mode():
            assert torch.equal(m(x), y)
        t = x.clone().requires_grad_()
        m(t).sum().backward()  # of positions that were made in inference mode
        assert t.grad.isfinite().all()
