"""State dicts, groups and seeds of terra_amd.optimizer.AdamW (on the CPU: no step of it runs)."""
import copy
import io

import pytest
import torch

from oracle import training as tr
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


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_moments_of_torchs_in_8_bits(dtype):
    """A group of 8 bits has what it loads in 8 bits.  With u = 2^-24, a scale is off by a rounding and a quotient by another:
    the nearest code is that of a value within 3 u of the quotient (the root: one more rounding), half a step of e4m3 at most, 2^-4 of
    the value or half of its least step, from it."""
    theirs = torch.optim.AdamW(_params(), **OPTS)
    theirs.param_groups[0]["params"][0].data = theirs.param_groups[0]["params"][0].data.t().contiguous().t()
    for step in (1, 2):
        _set_grads(theirs.param_groups[0]["params"], step)
        theirs.param_groups[0]["params"][2].grad[256:600] *= 10.0 ** torch.linspace(-9, 3, 344)
        theirs.param_groups[0]["params"][2].grad[768:1024] = 0.0
        theirs.step()
    params = _params(dtype)
    params[0].data = params[0].data.t().contiguous().t()
    ours = AdamW(params, bits=8, min_8bit_size=100, seed=1)
    ours.load_state_dict(copy.deepcopy(theirs.state_dict()))
    for p, q in zip(theirs.param_groups[0]["params"], params):
        a, b = theirs.state[p], ours.state[q]
        assert b["step"] == 2 and ("scales" in b) == (q.numel() >= 100)
        if "scales" not in b:
            assert torch.equal(b["exp_avg"], a["exp_avg"]) and torch.equal(b["exp_avg_sq"], a["exp_avg_sq"])
            continue
        held = kernels.Moments(b["exp_avg"], b["exp_avg_sq"], b["scales"])
        assert all(t.dtype == torch.float8_e4m3fn and t.shape == q.shape and t.stride() == q.stride() for t in held[:2])
        for i, values in enumerate((a["exp_avg"].double(), a["exp_avg_sq"].double().sqrt())):
            lain = torch.empty_like(q, dtype=torch.float64).copy_(values).as_strided((q.numel(),), (1,))
            codes = held[i].as_strided((q.numel(),), (1,))
            block = torch.arange(q.numel()) // 256
            top = torch.zeros(held.scales.shape[1], dtype=torch.float64).scatter_reduce_(0, block, lain.abs(), "amax")
            scales = held.scales[i].double()
            assert bool(((scales - top / 448).abs() <= 2 * 2.0 ** -24 * top / 448).all())
            per = scales[block]
            e = (codes.double() * per - lain).abs()
            low = 2.0 ** -10 * (1 if i == 0 else 2)  # a root below the least code is held as that
            assert bool((e <= torch.maximum((2.0 ** -4 + 8 * 2.0 ** -24) * lain.abs(), low * per)).all())
            assert i == 0 or torch.equal(lain > 0, codes.float() > 0)


def test_nearest_codes_of_moments():
    """Against the oracle's codes, away from the borders of two; infinities and NaN make a block NaN, as in a step."""
    from terra_amd.optimizer import _in_8_bits

    gen = torch.Generator().manual_seed(3)
    m = torch.randn(1000, generator=gen) * 10.0 ** (torch.rand(1000, generator=gen) * 6 - 6)
    v = torch.rand(1000, generator=gen) * 10.0 ** (torch.rand(1000, generator=gen) * 12 - 12)
    m[600], v[900] = float("nan"), float("inf")
    held = _in_8_bits(torch.zeros(1000), m, v)
    block = torch.arange(1000) // 256
    a, b = held.values()
    assert a.isnan().nonzero().view(-1).tolist() == list(range(512, 768)) and b.isnan().nonzero().view(-1).tolist() == list(range(768, 1000))
    ok = block != 2
    code, near = tr.nearest_code((m.double() / held.scales[0].double()[block])[ok])
    same = code == held.exp_avg.view(torch.uint8)[ok]
    assert bool((same | (near < 8 * 2.0 ** -24) | ((code % 128 == 0) & (held.exp_avg.view(torch.uint8)[ok] % 128 == 0))).all())
    empty = _in_8_bits(torch.zeros(3, 0), torch.zeros(3, 0), torch.zeros(3, 0))
    assert empty.scales.shape == (2, 0) and empty.exp_avg.shape == (3, 0)


def _in_8_bits(params):
    """An optimizer with 8-bit moments after two steps of torch's."""
    opt = AdamW(params, bits=8, min_8bit_size=100, seed=1)
    opt.load_state_dict(_theirs().state_dict())
    return opt


def test_moments_in_8_bits_of_another_layout_are_refused_as_a_whole():
    """Their scales go by blocks of memory.  What was there stays, all of it."""
    theirs, params = _in_8_bits(_params()), _params()
    params[0].data = params[0].data.t().contiguous().t()
    ours = AdamW(params, lr=0.5)
    ours.load_state_dict(_theirs(3).state_dict())
    before = _snapshot(ours)
    with pytest.raises(ValueError, match="lay otherwise in memory"):
        ours.load_state_dict(theirs.state_dict())
    after = _snapshot(ours)
    assert after[0] == before[0]
    assert all(after[1][i][k] is before[1][i][k] for i in before[1] for k in before[1][i])
    with pytest.raises(ValueError, match="match the size"):
        AdamW(_params()[:3]).load_state_dict(theirs.state_dict())
    with pytest.raises(ValueError, match="number of parameter groups"):
        AdamW(_groups(_params())).load_state_dict(theirs.state_dict())


# ---- counts in device memory ---------------------------------------------------------


@pytest.mark.parametrize("kw", [dict(capturable=True), dict(skip_nonfinite=True), dict()])
@pytest.mark.parametrize("foreach", [False, True])
@pytest.mark.parametrize("saved", [True, False])
def test_counts_that_load_into_torchs(kw, foreach, saved):
    """Each parameter's count is its own in torch's optimizer, and steps there leave this one's."""
    theirs, ours = _theirs(), AdamW(_params(), **kw)
    ours.load_state_dict(copy.deepcopy(theirs.state_dict()))
    made = ours.state_dict()
    assert all(type(s["step"]) is int for s in made["state"].values())
    if saved:
        f = io.BytesIO()
        torch.save(made, f)
        f.seek(0)
        made = torch.load(f, weights_only=True)
    back = torch.optim.AdamW([torch.nn.Parameter(p.detach().clone()) for p in theirs.param_groups[0]["params"]], foreach=foreach)
    back.load_state_dict(made)
    back.param_groups[0]["foreach"] = foreach
    for step in (3, 4):
        for opt in (theirs, back):
            _set_grads(opt.param_groups[0]["params"], step)
            opt.step()
    for p, q in zip(theirs.param_groups[0]["params"], back.param_groups[0]["params"]):
        assert int(back.state[q]["step"]) == int(theirs.state[p]["step"]) == 4
        assert torch.allclose(p, q, rtol=1e-6, atol=1e-7)
    assert all(int(ours.state[p]["step"]) == 2 for p in ours.param_groups[0]["params"])


def test_parameters_share_their_counter_again():
    theirs = _theirs()
    ours, other = (AdamW(_params(), capturable=True) for _ in range(2))
    ours.load_state_dict(theirs.state_dict())
    other.load_state_dict(ours.state_dict())
    for opt in (ours, other):
        counts = [opt.state[p]["step"] for p in opt.param_groups[0]["params"]]
        assert all(c is counts[0] for c in counts) and counts[0].dtype == torch.int64 and int(counts[0]) == 2
    assert other.state[other.param_groups[0]["params"][0]]["step"] is not ours.state[ours.param_groups[0]["params"][0]]["step"]


def test_hooks_see_the_counts_that_are_saved():
    ours, seen = AdamW(_params(), capturable=True), []
    ours.load_state_dict(_theirs().state_dict())
    ours.register_state_dict_post_hook(lambda _, d: seen.append([s["step"] for s in d["state"].values()]) or {"optimizer": d})
    for _ in range(2):
        made = ours.state_dict()
        assert list(made) == ["optimizer"] and [s["step"] for s in made["optimizer"]["state"].values()] == [2] * 4
    assert seen == [[2] * 4] * 2 and all(type(n) is int for n in seen[0])


# ---- seeds -------------------------------------------------------------------------


def _drawn(n):
    """The n seeds that torch's generator would give after seed 5."""
    with torch.random.fork_rng(devices=[]):
        torch.manual_seed(5)
        return [int(torch.randint(0, 1 << 62, (1,)).item()) for _ in range(n)]


def test_seeds_of_groups():
    """A group of 8 bits has a seed of torch's generator wherever it said so; nothing is drawn without one."""
    first, _ = _drawn(2)
    with torch.random.fork_rng(devices=[]):
        torch.manual_seed(5)
        before = torch.get_rng_state()
        AdamW(_params())
        AdamW(_params(), bits=8, seed=3)
        AdamW([dict(params=_params(), bits=8, seed=0)])
        assert torch.equal(torch.get_rng_state(), before)
        assert AdamW(_params(), bits=8).param_groups[0]["seed"] == first
        torch.manual_seed(5)
        opt = AdamW(_groups(_params(), bits=8))  # the group says 8 bits, the optimizer 32
        assert opt.param_groups[0]["seed"] == first
        opt.add_param_group(dict(params=_params(), bits=8))
        opt.add_param_group(dict(params=_params(), bits=8, seed=0))
        assert [g["seed"] for g in opt.param_groups[2:]] == [first, 0]
    assert AdamW(_groups(_params(), bits=8), seed=12).param_groups[0]["seed"] == 12
    assert [g["seed"] for g in AdamW(_groups(_params(), bits=8, seed=4), bits=8, seed=12).param_groups] == [4, 12]


def test_a_group_whose_bits_are_set_later_has_a_seed():
    first, = _drawn(1)
    opt = AdamW(_params())
    opt.param_groups[0]["bits"] = 8
    with torch.random.fork_rng(devices=[]):
        torch.manual_seed(5)
        assert opt._seed(opt.param_groups[0], torch.device("cpu")).tolist() == [first]
    assert opt._seed(opt.param_groups[0], torch.device("cpu")).tolist() == [first] == [opt.param_groups[0]["seed"]]
    assert opt.state_dict()["param_groups"][0]["seed"] == first


def test_seeds_go_with_state_dicts():
    opt = AdamW(_groups(_params(), bits=8))
    other = AdamW(_groups(_params(), bits=8))
    other.load_state_dict(opt.state_dict())
    assert other.param_groups[0]["seed"] == opt.param_groups[0]["seed"]
    eight = AdamW(_params(), bits=8, seed=3)
    eight.load_state_dict(AdamW(_params()).state_dict())  # of 32 bits: it names no seed
    assert (eight.param_groups[0]["bits"], eight.param_groups[0]["seed"]) == (32, 3)
