"""terra_amd.optimizer.AdamW, and a training step of a block with rotary
positions, wide norms, clipping and the step together.

Tolerances, with u = 2^-24: n steps of fp32 parameters against 64 bits are off by 3 u of the parameter and
40 u of what a step takes off, which is at most 10 lr (m / sqrt(v) <= 1 / (1 - beta1)), a step:
n (3 u max|p| + 400 u lr)."""
import copy
import io
import pickle

import pytest
import torch

from helpers import gain_block
from oracle import training as tr
from terra_amd import autograd, kernels, workloads
from terra_amd.kernels import Norm
from terra_amd.mlp import SequentialMlp
from terra_amd.optimizer import AdamW
from terra_amd.transformer import SequentialSwinTransformer

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
SHAPES = [(70, 90), (90,), (3, 5, 7), (1,), (5000,)]
OPTS = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-6, weight_decay=0.1)


def _params(dev, dtype=torch.float32):
    return [torch.nn.Parameter(workloads.activations(s, 10 + i, torch.float32).to(dtype).to(dev)) for i, s in enumerate(SHAPES)]


def _grad(p, i, step):
    return (workloads.activations(tuple(p.shape), 100 * step + i, torch.float32) * 0.3).to(p.dtype).to(p.device)


def _set_grads(params, step, only=None):
    for i, p in enumerate(params):
        p.grad = _grad(p, i, step) if only is None or i in only else None


def _reference(params, **kw):
    """The same parameters in 64 bits on the CPU under torch's AdamW."""
    ref = [torch.nn.Parameter(p.detach().double().cpu()) for p in params]
    return ref, torch.optim.AdamW(ref, **{**OPTS, **kw})


def _near(params, ref, n, lr=OPTS["lr"]):
    for p, r in zip(params, ref):
        e = (p.detach().double().cpu() - r.detach()).abs().max().item()
        assert e <= n * (3 * U * r.detach().abs().max().item() + 400 * U * lr), e


@pytest.mark.parametrize("kw", [{}, dict(capturable=True), dict(maximize=True)])
def test_steps(dev, kw):
    params = _params(dev)
    ref, ref_opt = _reference(params, maximize=kw.get("maximize", False))
    opt = AdamW(params, **OPTS, **kw)
    for step in range(1, 6):
        _set_grads(params, step)
        _set_grads(ref, step)
        opt.step()
        ref_opt.step()
    _near(params, ref, 5)


@pytest.mark.parametrize("max_norm", [0.5, 1e4])
def test_clipped(dev, max_norm):
    params = _params(dev)
    ref, ref_opt = _reference(params)
    opt = AdamW(params, **OPTS, max_grad_norm=max_norm)
    for step in range(1, 4):
        _set_grads(params, step)
        _set_grads(ref, step)
        before = [p.grad.clone() for p in params]
        opt.step()
        n = torch.nn.utils.clip_grad_norm_(ref, max_norm)
        ref_opt.step()
        assert opt.grad_norm.item() == pytest.approx(n.item(), rel=1e-6)
        assert all(torch.equal(p.grad, b) for p, b in zip(params, before))
    _near(params, ref, 3)


@pytest.mark.parametrize("capturable", [False, True])
def test_parameters_without_gradients(dev, capturable):
    """A parameter that takes part in some steps alone counts those."""
    params = _params(dev)
    ref, ref_opt = _reference(params)
    opt = AdamW(params, **OPTS, capturable=capturable)
    for step, only in enumerate([(0, 1, 2), (0, 2, 3), (1, 2, 3, 4), (0, 1, 2, 3, 4), (4,)], 1):
        _set_grads(params, step, only)
        _set_grads(ref, step, only)
        opt.step()
        ref_opt.step()
    _near(params, ref, 5)
    assert [int(opt.state[p]["step"]) for p in params] == [int(ref_opt.state[p]["step"]) for p in ref]
    opt.zero_grad()
    opt.step()  # of nothing


def test_groups_rates_and_closures(dev):
    params = _params(dev)
    ref = [torch.nn.Parameter(p.detach().double().cpu()) for p in params]
    groups = lambda ps: [dict(params=ps[:2], lr=3e-2, weight_decay=0.0), dict(params=ps[2:], betas=(0.5, 0.9))]  # noqa: E731
    opt, ref_opt = AdamW(groups(params), **OPTS), torch.optim.AdamW(groups(ref), **OPTS)
    sched, ref_sched = (torch.optim.lr_scheduler.ExponentialLR(o, 0.5) for o in (opt, ref_opt))
    for step in range(1, 5):
        _set_grads(params, step)
        _set_grads(ref, step)
        assert opt.step(lambda: 17) == 17
        ref_opt.step()
        sched.step()
        ref_sched.step()
    _near(params, ref, 4, 3e-2)


@pytest.mark.parametrize("bits", [32, 8])
def test_a_step_that_is_not_finite_is_left_out(dev, bits):
    params, twin = _params(dev), _params(dev)
    kw = dict(bits=bits, min_8bit_size=100, max_grad_norm=1.0, skip_nonfinite=True, seed=5)
    opt, other = AdamW(params, **OPTS, **kw), AdamW(twin, **OPTS, **kw)
    for step in range(1, 5):
        _set_grads(params, step)
        if step == 3:
            params[4].grad[7] = float("inf")
        else:
            _set_grads(twin, step)
            other.step()
        opt.step()
    assert all(torch.equal(p, q) for p, q in zip(params, twin))
    assert int(opt.state[params[0]]["step"]) == 3


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_8_bits(dev, dtype):
    """Large parameters have moments in 8 bits, the others in 32; 20 steps end near those of 32 bits: what a step takes
    off differs by a fraction of itself (codes of an eighth, rounded to nearest or at random), so on the whole by much less than all of it."""
    params, twin = _params(dev, dtype), _params(dev, dtype)
    start = [p.detach().clone() for p in params]
    opt, other = AdamW(params, **OPTS, bits=8, min_8bit_size=4000, seed=1), AdamW(twin, **OPTS)
    for step in range(1, 21):
        _set_grads(params, step)
        _set_grads(twin, step)
        opt.step()
        other.step()
    for i, (p, q, s) in enumerate(zip(params, twin, start)):
        state = opt.state[p]
        assert ("scales" in state) == (p.numel() >= 4000)
        assert state["exp_avg"].dtype == (torch.float8_e4m3fn if p.numel() >= 4000 else torch.float32)
        if "scales" not in state:
            assert torch.equal(p, q)
        elif dtype == torch.float32:
            moved = (q - s).norm().item()
            assert moved > 0 and (p - q).norm().item() <= 0.5 * moved


def _round_trip(state):
    f = io.BytesIO()
    torch.save(state, f)
    f.seek(0)
    return torch.load(f, weights_only=True)


@pytest.mark.parametrize("bits,dtype,capturable", [(32, torch.float32, False), (32, torch.bfloat16, True), (8, torch.float32, False),
                                                   (8, torch.bfloat16, True)])
def test_state_dicts(dev, bits, dtype, capturable):
    params = _params(dev, dtype)
    kw = dict(bits=bits, min_8bit_size=100, seed=3, capturable=capturable)
    opt = AdamW(params, **OPTS, **kw)
    for step in (1, 2):
        _set_grads(params, step)
        opt.step()
    saved = _round_trip(opt.state_dict())
    twin = [torch.nn.Parameter(p.detach().clone()) for p in params]
    other = AdamW(twin, lr=1.0, bits=bits, capturable=capturable)
    other.load_state_dict(saved)
    for p, q in zip(params, twin):
        a, b = opt.state[p], other.state[q]
        assert a.keys() == b.keys() and int(a["step"]) == int(b["step"]) == 2
        for k in ("exp_avg", "exp_avg_sq", "scales"):
            if k in a:
                assert a[k].dtype == b[k].dtype and a[k].data_ptr() != b[k].data_ptr()
                assert torch.equal(a[k].view(torch.uint8), b[k].view(torch.uint8))
    for step in (3, 4):
        _set_grads(params, step)
        _set_grads(twin, step)
        opt.step()
        other.step()
    assert all(torch.equal(p, q) for p, q in zip(params, twin))


def test_state_dicts_of_torchs_adamw(dev):
    params = _params(dev)
    ref, ref_opt = _reference(params)
    theirs = torch.optim.AdamW([torch.nn.Parameter(p.detach().clone()) for p in params], **OPTS)
    for step in (1, 2):
        _set_grads(theirs.param_groups[0]["params"], step)
        _set_grads(ref, step)
        theirs.step()
        ref_opt.step()
    ours = AdamW(theirs.param_groups[0]["params"])
    ours.load_state_dict(copy.deepcopy(theirs.state_dict()))
    _set_grads(ours.param_groups[0]["params"], 3)
    _set_grads(ref, 3)
    ours.step()
    ref_opt.step()
    _near(ours.param_groups[0]["params"], ref, 3)
    back = torch.optim.AdamW(ours.param_groups[0]["params"])
    back.load_state_dict(copy.deepcopy(ours.state_dict()))
    _set_grads(back.param_groups[0]["params"], 4)
    _set_grads(ref, 4)
    back.step()
    ref_opt.step()
    _near(back.param_groups[0]["params"], ref, 4)


@pytest.mark.parametrize("bits", [32, 8])
def test_saved_whole(dev, bits):
    """(pickle alone takes no tensors in 8 bits; torch.save and deepcopy do.)"""
    params = _params(dev)
    opt = AdamW(params, **OPTS, max_grad_norm=1.0, bits=bits, min_8bit_size=100)
    _set_grads(params, 1)
    opt.step()
    if bits == 32:
        other = pickle.loads(pickle.dumps(opt))
    else:
        f = io.BytesIO()
        torch.save(opt, f)
        f.seek(0)
        other = torch.load(f, weights_only=False)  # of a file that this test wrote
    assert other.max_grad_norm == 1.0
    _set_grads(other.param_groups[0]["params"], 2)
    _set_grads(params, 2)
    opt.step()
    other.step()
    assert all(torch.equal(p, q) for p, q in zip(params, other.param_groups[0]["params"]))


def test_captured(dev):
    params, twin = _params(dev), _params(dev)
    kw = dict(capturable=True, max_grad_norm=1.0, skip_nonfinite=True, bits=8, min_8bit_size=100, seed=7)
    lr, lr2 = torch.tensor(1e-2, device=dev), torch.tensor(1e-2, device=dev)
    opt, other = AdamW(params, **{**OPTS, "lr": lr}, **kw), AdamW(twin, **{**OPTS, "lr": lr2}, **kw)
    for o, ps in ((opt, params), (other, twin)):
        _set_grads(ps, 1)
        o.step()
    grads = [p.grad for p in params]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for step in range(2, 6):
        for i, (p, g) in enumerate(zip(params, grads)):
            g.copy_(_grad(p, i, step))
        _set_grads(twin, step)
        lr.mul_(0.5)
        lr2.mul_(0.5)
        graph.replay()
        other.step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(params, twin)), step


def test_refusals(dev):
    params = _params(dev)
    for kw in (dict(bits=16), dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(eps=-1.0), dict(weight_decay=-0.1), dict(max_grad_norm=0.0)):
        with pytest.raises(ValueError):
            AdamW(params, **kw)
    emb = torch.nn.Embedding(4, 8, sparse=True, device=dev)
    emb(torch.tensor([1], device=dev)).sum().backward()
    with pytest.raises(TypeError, match="not dense"):
        AdamW(emb.parameters()).step()


class _Stack(torch.nn.Module):
    """Two half-blocks with rotary positions, four neighbours merged and normed, a head."""

    def __init__(self, C=288, heads=9, H=14, W=14):
        super().__init__()
        self.attn = gain_block(SequentialSwinTransformer(1, H, W, C, window_size=7, num_heads=heads, rotary=True, init_seed_base=21))
        self.mlp = SequentialMlp(C, 2 * C, init_seed_base=31)
        self.norm = torch.nn.LayerNorm(4 * C)  # 1152: wider than the gather's norm
        self.head = torch.nn.Linear(4 * C, 24)
        self.size = H, W
        with torch.no_grad():
            self.head.weight.copy_(workloads.activations((24, 4 * C), 77, torch.float32) * 0.05)
            self.norm.weight.add_(workloads.activations((4 * C,), 78, torch.float32) * 0.2)

    @staticmethod
    def merged(x, H, W):
        B, _, C = x.shape
        return x.view(B, H // 2, 2, W // 2, 2, C).permute(0, 1, 3, 2, 4, 5).reshape(B, -1, 4 * C)

    def forward(self, x):
        y = self.merged(self.mlp(self.attn(x)), *self.size)
        return self.head(autograd.layer_norm(y, Norm.of(self.norm)))

    def oracle(self, x, params):
        part = lambda name: {k[len(name) + 1:]: v for k, v in params.items() if k.startswith(name + ".")}  # noqa: E731
        a, rot = self.attn, self.attn.attn.rotary
        y = tr.swin_block_rotary(x, *self.size, 7, a.shift_size, a.attn.num_heads, part("attn"), rot.rates, rot.dim)
        y = self.merged(tr.mlp(y, part("mlp")), *self.size)
        n, h = part("norm"), part("head")
        return tr.layer_norm(y, n["weight"], n["bias"])[0] @ h["weight"].double().T + h["bias"].double()


def test_a_training_run(dev):
    """Forward, backward, clipping and three steps against 64 bits.  With gradients clipped to norm 1 and within 1e-5 of their
    largest, and eps = 1e-2, what a step takes off is within lr 2e-5 / eps = 2e-3 lr of the reference's; the parameters after
    that move the next gradients by a similar part: 1e-2 lr a step."""
    model = _Stack()
    x, target = workloads.activations((2, 196, 288), 7, torch.float32), workloads.activations((2, 49, 24), 8, torch.float32)
    opts = dict(lr=1e-3, betas=(0.9, 0.99), eps=1e-2, weight_decay=0.05)
    ref = {k: torch.nn.Parameter(p.detach().double()) for k, p in model.named_parameters()}
    ref_opt = torch.optim.AdamW(ref.values(), **opts)
    model = model.to(dev)
    opt = AdamW(model.parameters(), **opts, max_grad_norm=1.0)
    start = {k: p.detach().clone() for k, p in model.named_parameters()}
    for step in range(1, 4):
        loss = (model(x.to(dev)) - target.to(dev)).square().sum()
        opt.zero_grad()
        loss.backward()
        loss_ref = (model.oracle(x.double(), ref) - target.double()).square().sum()
        ref_opt.zero_grad()
        loss_ref.backward()
        assert loss.item() == pytest.approx(loss_ref.item(), rel=1e-4)
        if step == 1:
            for k, p in model.named_parameters():
                g = ref[k].grad
                assert (p.grad.double().cpu() - g).abs().max() <= 1e-5 * g.abs().max(), k
        torch.nn.utils.clip_grad_norm_(ref.values(), 1.0)
        opt.step()
        ref_opt.step()
    for k, p in model.named_parameters():
        assert (p.detach().double().cpu() - ref[k].detach()).abs().max().item() <= 3 * 1e-2 * opts["lr"], k
    assert any((p - start[k]).abs().max().item() > 1e-4 for k, p in model.named_parameters())


def test_a_training_run_in_bf16_with_8_bits(dev):
    """Under autocast, moments in 8 bits: it runs, everything stays finite, every parameter moves."""
    model = _Stack().to(dev)
    x, target = workloads.activations((2, 196, 288), 7, torch.float32).to(dev), workloads.activations((2, 49, 24), 8, torch.float32).to(dev)
    opt = AdamW(model.parameters(), lr=1e-3, bits=8, max_grad_norm=1.0, skip_nonfinite=True)
    start = {k: p.detach().clone() for k, p in model.named_parameters()}
    for _ in range(3):
        with torch.autocast("cuda", torch.bfloat16):
            loss = (model(x).float() - target).square().mean()
        opt.zero_grad()
        loss.backward()
        opt.step()
    assert opt.grad_norm.isfinite() and all(p.isfinite().all() for p in model.parameters())
    assert all(not torch.equal(p, start[k]) for k, p in model.named_parameters())


def test_packed_weights_follow_the_step(dev):
    """The halves keep packed copies of their weights until a parameter's version changes: a step changes it."""
    m = SequentialMlp(128, 512, init_seed_base=3).to(dev).to(torch.bfloat16)
    x = workloads.activations((64, 128), 7, torch.bfloat16).to(dev)
    with torch.no_grad():
        before = m(x)
    for p in m.parameters():
        p.grad = torch.ones_like(p)
    AdamW(m.parameters(), lr=0.1).step()
    with torch.no_grad():
        after = m(x)
        fresh = SequentialMlp(128, 512).to(dev).to(torch.bfloat16)
        fresh.load_state_dict(m.state_dict())
        assert torch.equal(after, fresh(x)) and not torch.equal(after, before)


def test_packed_weights_follow_replays(dev):
    """A replayed step changes no version: the halves are told."""
    m = SequentialMlp(128, 512, init_seed_base=3).to(dev).to(torch.bfloat16)
    x = workloads.activations((64, 128), 7, torch.bfloat16).to(dev)
    for p in m.parameters():
        p.grad = torch.ones_like(p)
    opt = AdamW(m.parameters(), lr=0.1, capturable=True)
    opt.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for _ in range(3):
        with torch.no_grad():
            m(x)
        graph.replay()
        opt.replayed()
        with torch.no_grad():
            fresh = SequentialMlp(128, 512).to(dev).to(torch.bfloat16)
            fresh.load_state_dict(m.state_dict())
            assert torch.equal(m(x), fresh(x))


def test_groups_of_different_bits(dev):
    a, b = (torch.nn.Parameter(torch.ones(5000, device=dev)) for _ in range(2))
    opt = AdamW([dict(params=[a], bits=8), dict(params=[b])], lr=0.1)
    a.grad = b.grad = torch.full_like(a, 0.5)
    opt.step()
    assert opt.state[a]["exp_avg"].dtype == torch.float8_e4m3fn and opt.state[b]["exp_avg"].dtype == torch.float32
    # The first step comes before the first rounding of a moment: some ten roundings of 0.1 and one of 0.9 apart on each side.
    assert (a - b).abs().max().item() <= 2 * (10 * 0.1 + 1) * 2.0 ** -24
    c = torch.nn.Parameter(torch.ones(8, device=dev))
    c.grad = torch.ones_like(c)
    with pytest.raises(ValueError, match="32 bits or in 8"):
        AdamW([dict(params=[c], bits=16)]).step()


def test_options_set_between_steps(dev):
    """The count moves to the device and back; the steps are those of an optimizer that counts on the host."""
    a, b = ([torch.nn.Parameter(torch.linspace(-1, 1, n, device=dev)) for n in (33, 700)] for _ in range(2))
    one, two = AdamW(a, lr=0.1), AdamW(b, lr=0.1)
    for step in range(6):
        one.capturable, one.skip_nonfinite = step in (2, 3), step == 3
        for ps, opt in ((a, one), (b, two)):
            for k, p in enumerate(ps):
                p.grad = torch.full_like(p, 0.3 * (k + 1) - 0.1 * step)
            opt.step()
    assert all(torch.equal(p, q) for p, q in zip(a, b)) and one.state[a[0]]["step"] == two.state[b[0]]["step"] == 6
