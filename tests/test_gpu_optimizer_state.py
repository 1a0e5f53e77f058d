"""State dicts between terra_amd.optimizer.AdamW and torch's, groups and draws, on the device.

Tolerances, with u = 2^-24, as in the other tests of the optimizer: n steps of fp32 parameters against 64 bits are off by 3 u of the
parameter and 40 u of what a step takes off, at most 10 lr a step: n (3 u max|p| + 400 u lr)."""
import copy

import pytest
import torch

from terra_amd import kernels, workloads
from terra_amd.optimizer import AdamW

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
SHAPES = [(70, 90), (90,), (5000,), (1,)]
OPTS = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-6, weight_decay=0.1)


def _params(dev, dtype=torch.float32):
    return [torch.nn.Parameter(workloads.activations(s, 10 + i, torch.float32).to(dtype).to(dev)) for i, s in enumerate(SHAPES)]


def _set_grads(params, step):
    for i, p in enumerate(params):
        p.grad = (workloads.activations(tuple(p.shape), 100 * step + i, torch.float32) * 0.3).to(p.dtype).to(p.device)


def _steps(opt, steps):
    params = [p for g in opt.param_groups for p in g["params"]]
    for step in steps:
        _set_grads(params, step)
        opt.step()


def _near(params, ref, n, lr=OPTS["lr"]):
    for p, r in zip(params, ref):
        e = (p.detach().double().cpu() - r.detach()).abs().max().item()
        assert e <= n * (3 * U * r.detach().abs().max().item() + 400 * U * lr), e


def test_moments_of_torchs_step_on_in_8_bits(dev):
    """What was loaded is what the next step takes: its first moment is beta1 times the codes' value and the gradient's part.
    The sum in 64 bits of two terms rounded to 32, 2 u of their magnitudes, and half a step of e4m3 at most, 2^-4 of
    the value or half of the least step, 2^-10 of the scale."""
    theirs = torch.optim.AdamW(_params(dev), **OPTS)
    _steps(theirs, (1, 2))
    params = [torch.nn.Parameter(p.detach().clone()) for p in theirs.param_groups[0]["params"]]
    ours = AdamW(params, bits=8, min_8bit_size=100, seed=3)
    ours.load_state_dict(copy.deepcopy(theirs.state_dict()))
    read = {}
    for p in params:
        s = ours.state[p]
        assert ("scales" in s) == (p.numel() >= 100) and s["step"] == 2
        if "scales" in s:
            read[p] = [t.double() for t in kernels.Moments(s["exp_avg"], s["exp_avg_sq"], s["scales"]).values()]
    _steps(ours, (3,))
    for p, (m, v) in read.items():
        s = ours.state[p]
        got = kernels.Moments(s["exp_avg"], s["exp_avg_sq"], s["scales"]).values()[0].double()
        terms = 0.9 * m, 0.1 * p.grad.double()
        least = 2.0 ** -10 * s["scales"][0].double().repeat_interleave(256)[:p.numel()].view(p.shape)
        tol = 2 * U * (terms[0].abs() + terms[1].abs()) + torch.maximum(2.0 ** -4 * (terms[0] + terms[1]).abs() * (1 + 4 * U), least)
        assert bool(((got - terms[0] - terms[1]).abs() <= tol * (1 + 8 * U)).all())
        assert p.isfinite().all()
    with_codes = ours.state_dict()
    again = AdamW([torch.nn.Parameter(p.detach().clone()) for p in params], bits=8)
    again.load_state_dict(copy.deepcopy(with_codes))
    _steps(ours, (4,))
    _steps(again, (4,))
    assert all(torch.equal(p, q) for p, q in zip(params, again.param_groups[0]["params"]))


@pytest.mark.parametrize("kw", [dict(capturable=True), dict(skip_nonfinite=True), dict()])
@pytest.mark.parametrize("form", [dict(foreach=False), dict(foreach=True), dict(capturable=True), dict(fused=True)])
def test_counts_step_on_in_torchs(dev, kw, form):
    """From counts in device memory to each form of torch's step and back, against 64 bits all the way."""
    params = _params(dev)
    ref = [torch.nn.Parameter(p.detach().double().cpu()) for p in params]
    ref_opt = torch.optim.AdamW(ref, **OPTS)
    ours = AdamW(params, **OPTS, **kw)
    _steps(ours, (1, 2))
    back = torch.optim.AdamW(params, **form)
    made = copy.deepcopy(ours.state_dict())
    made["param_groups"][0].update(form)  # torch takes its options from the state dict
    back.load_state_dict(made)
    _steps(back, (3, 4))
    _steps(ref_opt, (1, 2, 3, 4))
    assert [int(back.state[p]["step"]) for p in params] == [4] * len(params)
    assert [int(ours.state[p]["step"]) for p in params] == [2] * len(params)
    _near(params, ref, 4)
    ours.load_state_dict(copy.deepcopy(back.state_dict()))
    _steps(ours, (5,))
    _steps(ref_opt, (5,))
    _near(params, ref, 5)


def _codes(opt, p):
    return opt.state[p]["exp_avg_sq"].view(torch.uint8)


@pytest.mark.parametrize("capturable", [True, False])
def test_draws_of_tensors_that_step_apart(dev, capturable):
    """Two parameters of one group with the same gradients and as many steps, which each left out another step: their
    codes are drawn apart."""
    params = [torch.nn.Parameter(torch.zeros(5000, device=dev)) for _ in range(3)]
    opt = AdamW(params, bits=8, min_8bit_size=100, seed=5, capturable=capturable)
    for left in (0, 1, None, None):
        for i, p in enumerate(params):
            p.grad = None if i == left else torch.linspace(0.01, 1.0, 5000, device=dev)
        opt.step()
    assert [int(opt.state[p]["step"]) for p in params] == [3, 3, 4]
    a, b, c = (_codes(opt, p) for p in params)
    assert not torch.equal(a, b) and not torch.equal(a, c) and not torch.equal(b, c)


def test_draws_do_not_go_by_what_else_steps(dev):
    """The same parameter at the same place of its group: alone, or with others that step, or that have no gradient."""
    def run(with_gradient):
        params = [torch.nn.Parameter(torch.zeros(n, device=dev)) for n in (300, 5000)]
        opt = AdamW(params, bits=8, min_8bit_size=100, seed=5)
        for _ in range(3):
            params[1].grad = torch.linspace(0.01, 1.0, 5000, device=dev)
            params[0].grad = torch.ones(300, device=dev) if with_gradient else None
            opt.step()
        return _codes(opt, params[1])

    assert torch.equal(run(True), run(False))


def test_places(dev):
    """A call's places are the tensors' numbers; without, their places in the list."""
    def run(order, **kw):
        params = [torch.zeros(1000, device=dev) for _ in range(3)]
        moments = [kernels.moments(p, 8) for p in params]
        grads = [torch.linspace(0.01, 1.0 + i, 1000, device=dev) for i in range(3)]
        pick = lambda ts: [ts[i] for i in order]  # noqa: E731
        kernels.adamw_step(pick(params), pick(grads), pick(moments), 1, seed=torch.tensor([9], device=dev), **kw)
        return [m.exp_avg_sq.view(torch.uint8) for m in moments]

    ref = run((0, 1, 2))
    for got in (run((0, 1, 2), places=(0, 1, 2)), run((2, 0, 1), places=[2, 0, 1])):
        assert all(torch.equal(a, b) for a, b in zip(got, ref))
    assert all(not torch.equal(a, b) for a, b in zip(run((0, 1, 2), places=(5, (1 << 32) - 1, 7)), ref))
    for bad in ((), (0, 1), (0, 1, 2, 3), (0, 1, -1), (0, 1, 1 << 32)):
        with pytest.raises(ValueError, match="places"):
            run((0, 1, 2), places=bad)
