"""State dicts, groups and seeds of terra_amd.optimizer.AdamW (on the CPU: no step of it runs)."""
import copy
import io

import pytest
import torch

from terra_amd import kernels
from terra_amd.optimizer import AdamW

SIZES = [(70, 90), (90,), (5000,), (1,)]
OPTS = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-6, weight_decay=0.1)


def _params(dtype=torch.float32):
    return [torch.nn.Parameter(torch.randn(s, generator=torch.Generator().manual_seed(i)).to(dtype)) for i, s in enumerate(SIZES)]


def _set_grads(params, step):
    for i, p in enumerate(params):
        p.grad = torch.randn(p.shape, generator=torch.Generator().manual_seed(100 * step + i)).to(p.dtype)


def _theirs(steps=2, cls=torch.optim.AdamW, **kw):
    """An optimizer of torch's after some steps."""
    opt = cls(_params(), **{**OPTS, **kw})
    for step in range(1, steps + 1):
        _set_grads(opt.param_groups[0]["params"], step)
        opt.step()
    return opt


def _snapshot(opt):
    return copy.deepcopy([{k: v for k, v in g.items() if k != "params"} for g in opt.param_groups]), \
        {i: dict(opt.state[p]) for i, p in enumerate(p for g in opt.param_groups for p in g["params"]) if p in opt.state}


# ---- steps that are not this optimizer's ------------------------------------------


@pytest.mark.parametrize("cls,kw,text", [(torch.optim.AdamW, dict(amsgrad=True), "amsgrad"),
                                         (torch.optim.Adam, dict(), "decoupled_weight_decay"),
                                         (torch.optim.AdamW, dict(differentiable=True), "differentiable")])
def test_state_of_another_update_is_refused(cls, kw, text):
    theirs = _theirs(steps=0 if "differentiable" in kw else 2, cls=cls, **kw)
    ours = AdamW(_params(), lr=0.5)
    ours.load_state_dict(_theirs(3).state_dict())
    before = _snapshot(ours)
    with pytest.raises(ValueError, match=text):
        ours.load_state_dict(theirs.state_dict())
    after = _snapshot(ours)
    assert after[0] == before[0]  # nothing has been taken of it
    assert all(after[1][i][k] is before[1][i][k] for i in before[1] for k in before[1][i])


def test_one_refused_group_of_many():
    params = _params()
    theirs = torch.optim.AdamW([dict(params=params[:2]), dict(params=params[2:], amsgrad=True)])
    with pytest.raises(ValueError, match="amsgrad"):
        AdamW([dict(params=params[:2]), dict(params=params[2:])]).load_state_dict(theirs.state_dict())


def test_refused_as_a_group_too():
    for kw in (dict(amsgrad=True), dict(differentiable=True), dict(decoupled_weight_decay=False)):  # of the default decay
        with pytest.raises(ValueError, match=next(iter(kw))):
            AdamW([dict(params=_params(), **kw)])
    opt = AdamW(_params()[:2])
    with pytest.raises(ValueError, match="amsgrad"):
        opt.add_param_group(dict(params=_params()[2:], amsgrad=True))
    assert len(opt.param_groups) == 1


def test_what_the_options_do_not_change_loads():
    """torch's other forms of the same step, and Adam's without a decay."""
    for theirs in (_theirs(foreach=True), _theirs(foreach=False), _theirs(cls=torch.optim.Adam, weight_decay=0.0),
                   _theirs(maximize=True)):
        ours = AdamW(_params())
        ours.load_state_dict(copy.deepcopy(theirs.state_dict()))
        group = ours.param_groups[0]
        assert group["lr"] == OPTS["lr"] and group["betas"] == OPTS["betas"] and group["decoupled_weight_decay"]
        assert group["maximize"] == theirs.param_groups[0]["maximize"]
        for p, q in zip(theirs.param_groups[0]["params"], group["params"]):
            assert ours.state[q]["step"] == 2 and torch.equal(ours.state[q]["exp_avg"], theirs.state[p]["exp_avg"])


# ---- hooks -----------------------------------------------------------------------


@pytest.mark.parametrize("steps", [(1,), (1, 2)])
def test_state_dicts_that_hooks_make(steps):
    """What load_state_dict's hooks give is what is loaded, moments in their own types."""
    theirs = _theirs()
    saved = {"optimizer": copy.deepcopy(theirs.state_dict())}
    ours = AdamW(_params(torch.bfloat16))
    ours.register_load_state_dict_pre_hook(lambda _, d: d["optimizer"])
    if 2 in steps:  # and one that changes it in place, a copy of the first level
        def double(_, d):
            d["state"] = {i: {**s, "exp_avg": 2 * s["exp_avg"]} for i, s in d["state"].items()}
        ours.register_load_state_dict_pre_hook(double)
    for _ in range(2):  # the hooks are those of before each time
        ours.load_state_dict(copy.deepcopy(saved))  # the second hook writes into it
        for p, q in zip(theirs.param_groups[0]["params"], ours.param_groups[0]["params"]):
            a, b = theirs.state[p], ours.state[q]
            assert b["exp_avg"].dtype == b["exp_avg_sq"].dtype == torch.float32 and b["step"] == 2
            assert torch.equal(b["exp_avg"], steps[-1] * a["exp_avg"]) and torch.equal(b["exp_avg_sq"], a["exp_avg_sq"])


# ---- options that torch's groups do not have -----------------------------------------


def _groups(params, **first):
    return [dict(params=params[:2], **first), dict(params=params[2:])]


def test_options_of_ones_own_groups_stay():
    """What a state dict does not say of a group is the group's own, not the optimizer's."""
    theirs = torch.optim.AdamW(_groups(_params(), lr=0.3))
    ours = AdamW(_groups(_params(), bits=8, min_8bit_size=100, seed=9), lr=1.0)
    ours.load_state_dict(theirs.state_dict())
    a, b = ours.param_groups
    assert (a["bits"], a["min_8bit_size"], a["seed"], a["lr"]) == (8, 100, 9, 0.3)
    assert (b["bits"], b["min_8bit_size"], b["lr"]) == (32, 4096, 1e-3)
    ours.load_state_dict(AdamW(_groups(_params(), bits=8, min_8bit_size=7, seed=11)).state_dict())
    assert (ours.param_groups[0]["min_8bit_size"], ours.param_groups[0]["seed"]) == (7, 11)  # said, so taken
