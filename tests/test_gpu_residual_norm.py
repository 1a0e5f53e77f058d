"""The end of a half-block (terra_swin_residual_norm and its backward) against
the 64-bit oracle, whose gradients come from torch autograd over float64.

Tolerances, with e = eps of fp32 and K = 64 e.  All arithmetic is fp32 on exact
inputs, and every result is rounded once to its type (half an eps of it).  A
row's sums run over at most 16 values a lane and then a tree, so a mean is off
by at most 24 e of the row's largest magnitude, the reciprocal root by as much
relatively, and each further product by e / 2: K covers them.  A norm divides by
the row's spread, so an error of its input grows by r max|v| (A below) where the
mean is large beside the spread.  Per row, with the maxima over its channels:
  y   K (|alpha x| + |gate| s (|n|))
  z   K |w| (r2 Y)(1 + A2) with Y the scale of y and A2 = r2 Y
  dY  K (|dy| + r2 G (2 + Zh)(1 + A2)), G = max |dz w2|, Zh = max |yhat|
  dx  alpha times it;  dn  s |gate| times it
  dh  K r1 U (2 + Nh)(1 + A1), U = dn's scale times max|w1|
and the parameters' gradients K times the sum over rows of the scales of their
terms.
"""
import itertools
import threading

import pytest
import torch

from oracle import regularize as rg
from terra_amd import autograd, kernels
from terra_amd.kernels import Norm, WindowGeometry

pytestmark = pytest.mark.gpu

E32 = torch.finfo(torch.float32).eps
K = 64 * E32
SEED = 0x7EDCBA9876543210
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [(F32, F32), (BF16, BF16), (F16, F16), (BF16, F32), (F16, F32)]
NAMES = ("dpost_weight", "dpost_bias", "dgate", "dnext_weight", "dnext_bias")


def _half(dt):
    return torch.finfo(dt).eps / 2 if dt != F32 else 0.0


def _tiny(dt):
    return torch.finfo(dt).smallest_normal * torch.finfo(dt).eps


class Case:
    """Inputs on the CPU, made from a seed; the kernels' calls; the oracle's results and tolerances."""

    def __init__(self, grid, dts=(F32, F32), post="layer", nxt="layer", gate="channel", alpha=1.0, p=0.0, geom=None, seed=0,
                 eps=1e-5, affine=True, stream=3):
        g = torch.Generator().manual_seed(1000 + seed)
        r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
        C = grid[-1]
        self.C, self.grid, self.geom, self.alpha, self.p, self.stream = C, tuple(grid), geom, alpha, p, stream
        hd, xd = self.dts = dts
        hs = grid if geom is None else (geom.num_windows, geom.window ** 2, C)
        self.h = (r(*hs) * 0.8 + 0.1).to(hd)
        self.x = (r(*grid) * 2 + 0.3).to(xd)
        self.dy, self.dz = r(*grid).to(xd), (r(*grid).to(hd) if nxt else None)
        self.kinds = tuple(None if k is None else (eps, k == "rms") for k in (post, nxt))
        self.pw, self.pb, self.nw, self.nb = (
            (1 + 0.2 * r(C) if i % 2 == 0 else 0.1 * r(C)) if affine and k else None for i, k in enumerate((post, post, nxt, nxt)))
        self.gate = {None: None, "channel": 0.3 + 0.2 * r(C), "sample": 0.5 * r(grid[0], C)}[gate]

    def tensors(self):
        return {k: v for k in ("h", "x", "dy", "dz", "pw", "pb", "gate", "nw", "nb") if (v := getattr(self, k)) is not None}

    def args(self, dev):
        t = {k: v.to(dev) for k, v in self.tensors().items()}
        post, nxt = (None if k is None else Norm(t.get(w), t.get(b), *k)
                     for k, w, b in zip(self.kinds, ("pw", "nw"), ("pb", "nb")))
        kw = dict(post_norm=post, gate=t.get("gate"), next_norm=nxt, geom=self.geom, residual_scale=self.alpha, p=self.p,
                  seed=torch.tensor([SEED], device=dev) if self.p else None, stream=self.stream)
        return t, kw

    def run(self, dev):
        t, kw = self.args(dev)
        out = kernels.residual_norm(t["h"], t["x"], **kw)
        y, z = out if kw["next_norm"] is not None else (out, None)
        g = kernels.residual_norm_backward(t["h"], t["x"], t["dy"], t.get("dz"), **kw)
        return y, z, g

    def oracle(self):
        v = {k: t.double().requires_grad_() for k, t in self.tensors().items() if k not in ("dy", "dz")}
        post, nxt = (None if k is None else (v.get(w), v.get(b), *k)
                     for k, w, b in zip(self.kinds, ("pw", "nw"), ("pb", "nb")))
        y, z = rg.residual_norm(v["h"], v["x"], post, v.get("gate"), nxt, self.geom, self.alpha, self.p, SEED, self.stream)
        outs = [y] if z is None else [y, z]
        gs = torch.autograd.grad(outs, list(v.values()), [self.dy.double()] + ([] if z is None else [self.dz.double()]))
        return y.detach(), None if z is None else z.detach(), dict(zip(v, gs))

    def check(self, dev, got=None):
        """The kernels' results (of ``got``: those of an equal call) against the oracle's."""
        y, z, g = self.run(dev) if got is None else got
        assert y.shape == self.grid and y.dtype == self.dts[1]
        yr, zr, gr = self.oracle()
        C, R = self.C, self.x.numel() // self.C
        rows = lambda t: t.double().reshape(-1, C)  # noqa: E731
        top = lambda t: t.abs().amax(-1, keepdim=True)  # noqa: E731
        one = torch.ones(1, dtype=torch.float64)
        s = rg.keep_scale(self.p)
        h = rows(self.h)
        if self.geom is not None:
            src = rg.window_sources(self.geom)
            have = (src >= 0)[:, None]
            h = h[src.clamp(min=0)] * have
        w = lambda t: top(t.double()[None]) if t is not None else one  # noqa: E731
        bias = lambda t: t.double().abs().max() if t is not None else 0.0  # noqa: E731
        gate = one if self.gate is None else (
            top(self.gate.double()[None]) if self.gate.dim() == 1
            else top(self.gate.double()).repeat_interleave(R // self.gate.shape[0], 0))

        def stats(v, kind):
            d = v if kind[1] else v - v.mean(-1, keepdim=True)
            r = 1 / torch.sqrt((d * d).mean(-1, keepdim=True) + kind[0])
            return d * r, r

        n, A1, Nh, r1 = top(h), 0.0, 1.0, one
        if self.kinds[0] is not None:
            hat, r1 = stats(h, self.kinds[0])
            A1, Nh = r1 * top(h), top(hat)
            n = w(self.pw) * Nh * (1 + A1) + bias(self.pb)
        Y = top(rows(self.x) * self.alpha) + gate * s * n

        def near(got, ref, tol, dt, what):
            got, ref = got.detach().double().cpu().reshape(ref.shape), ref
            bad = ((got - ref).abs() - (_half(dt) * ref.abs() + tol + _tiny(dt))).max().item()
            assert bad <= 0, (what, bad, (got - ref).abs().max().item())

        near(rows(y.cpu()), rows(yr), K * Y, self.dts[1], "y")
        dY = top(rows(self.dy))
        if zr is not None:
            assert z.shape == self.grid and z.dtype == self.dts[0]
            yhat, r2 = stats(rows(yr), self.kinds[1])
            A2, Zh = r2 * Y, top(yhat)
            near(rows(z.cpu()), rows(zr), K * (w(self.nw) * A2 * (1 + A2) + bias(self.nb)), self.dts[0], "z")
            dz = top(rows(self.dz))
            dY = dY + r2 * dz * w(self.nw) * (2 + Zh) * (1 + A2)
            self._sum(near, g.dnext_weight, gr.get("nw"), dz * (Zh + A2 * (1 + A2)), "dnext_weight")
            self._sum(near, g.dnext_bias, gr.get("nb"), dz, "dnext_bias")
        near(rows(g.dx.cpu()), rows(gr["x"]), K * abs(self.alpha) * dY, self.dts[1], "dx")
        if self.gate is not None:
            terms = dY * s * n
            terms = terms.view(self.gate.shape[0], -1).sum(1, keepdim=True) if self.gate.dim() == 2 else terms.sum()
            near(g.dgate, gr["gate"], K * terms, F32, "dgate")
        dn = s * gate * dY
        self._sum(near, g.dpost_weight, gr.get("pw"), dn * (Nh + A1 * (1 + A1)), "dpost_weight")
        self._sum(near, g.dpost_bias, gr.get("pb"), dn, "dpost_bias")
        tol = K * dn if self.kinds[0] is None else K * r1 * dn * w(self.pw) * (2 + Nh) * (1 + A1)
        if self.geom is not None:
            full = torch.zeros(self.h.numel() // C, 1, dtype=torch.float64)
            full[src[have[:, 0]]] = tol.expand(R, 1)[have[:, 0]]
            tol = full
        near(rows(g.dh.cpu()), rows(gr["h"]), tol, self.dts[0], "dh")
        return y, z, g

    @staticmethod
    def _sum(near, got, ref, terms, what):
        if ref is None:
            assert got is None
        else:
            near(got, ref, K * terms.sum(), F32, what)


WIDTHS = [1, 7, 8, 33, 96, 128, 192, 250, 256, 385, 512, 515, 1000, 1024, 1030, 2048, 2050, 4096, 4097, 8192]


@pytest.mark.parametrize("C", WIDTHS)
@pytest.mark.parametrize("dts", TYPES, ids=lambda d: "-".join(str(t)[6:] for t in d))
def test_widths_and_types(dev, C, dts):
    Case((5, C), dts, p=0.2, seed=C).check(dev)
    Case((2, 19, C), dts, post="rms", nxt="rms", gate="sample", alpha=0.75, seed=C + 1).check(dev)


@pytest.mark.parametrize("post,nxt,gate,p", itertools.product([None, "layer", "rms"], [None, "layer", "rms"],
                                                            [None, "channel", "sample"], [0.0, 0.3]))
def test_every_combination(dev, post, nxt, gate, p):
    Case((3, 23, 72), (BF16, F32), post, nxt, gate, 1.0, p, seed=5).check(dev)
    Case((3, 23, 70), (BF16, BF16), post, nxt, gate, -0.5, p, seed=6).check(dev)


@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 63, 65, 1000, 4099, 20000])
@pytest.mark.parametrize("C", [24, 192, 1024])
def test_rows(dev, rows, C):
    if rows * C > 1 << 22:
        rows = (1 << 22) // C + 3
    Case((rows, C), (BF16, BF16), p=0.1, seed=rows).check(dev)


@pytest.mark.parametrize("B,R", [(1, 1), (7, 1), (40, 1), (3, 700), (64, 33), (2000, 2), (1500, 3)])
def test_sample_gates(dev, B, R):
    """More samples than workgroups, one row a sample, several slabs a sample."""
    Case((B, R, 48), (F16, F16), gate="sample", p=0.1, seed=B).check(dev)


def test_without_affine_parameters(dev):
    for post, nxt in itertools.product(("layer", "rms"), repeat=2):
        Case((9, 100), (F32, F32), post, nxt, affine=False).check(dev)


GEOMS = [
    WindowGeometry(1, 14, 21, 96, 7, 3, 3),
    WindowGeometry(2, 16, 24, 192, 8, 4, 4),
    WindowGeometry(2, 10, 13, 64, 7, 3, 2, (1, 3, 2, 6)),
    WindowGeometry(1, 40, 16, 72, 8, 4, 4, (0, 8, 0, 0), 1, 4, (1, 7)),
    WindowGeometry(3, 9, 6, 33, 3),
]


@pytest.mark.parametrize("geom", GEOMS)
@pytest.mark.parametrize("post,nxt,gate,p", [("layer", "layer", "channel", 0.2), (None, "rms", "sample", 0.0),
                                             ("rms", None, None, 0.3)])
def test_window_order(dev, geom, post, nxt, gate, p):
    grid = (geom.batch, geom.height, geom.width, geom.channels)
    for dts in ((BF16, F32), (F32, F32)):
        y, z, g = Case(grid, dts, post, nxt, gate, 0.9, p, geom).check(dev)
    c = Case(grid, (BF16, BF16), None, None, None, geom=geom)  # with nothing on, the residual scatter itself
    y, _, _ = c.run(dev)
    assert torch.equal(y, kernels.swin_reverse(c.h.to(dev), geom, residual=c.x.to(dev)))


def test_bitwise_the_same_each_time(dev):
    c = Case((3, 1111, 200), (BF16, F32), gate="sample", p=0.2)
    y, z, g = c.run(dev)
    for _ in range(3):
        y2, z2, g2 = c.run(dev)
        assert torch.equal(y, y2) and torch.equal(z, z2)
        assert all(torch.equal(a, b) for a, b in zip(g, g2))


@pytest.mark.parametrize("dts", TYPES)
@pytest.mark.parametrize("C", [96, 100])
@pytest.mark.parametrize("extra", [8, 9])
def test_strides_and_alignment(dev, C, extra, dts):
    """Column blocks of wider rows, on the 16-byte grid (C = 96, 8 more) and off
    it: each against the oracle, and those of one kind the same bit for bit."""
    c = Case((37, C), dts, p=0.1, seed=8)
    packed = c.check(dev)
    t, kw = c.args(dev)
    first = {C % 8 == 0: packed}
    for lo in (0, 8, 5):
        h, x = (torch.zeros(37, 2 * C + extra, dtype=d, device=dev)[:, lo:lo + C].copy_(t[n]) for n, d in zip("hx", dts))
        got = (*kernels.residual_norm(h, x, **kw), kernels.residual_norm_backward(h, x, t["dy"], t["dz"], **kw))
        c.check(dev, got)
        same = first.setdefault(all(v.stride(0) * v.element_size() % 16 == 0 and v.data_ptr() % 16 == 0 for v in (h, x))
                                and C % 8 == 0, got)
        assert torch.equal(got[0], same[0]) and torch.equal(got[1], same[1])
        assert all(torch.equal(a, b) for a, b in zip(got[2], same[2]))


@pytest.mark.parametrize("gate", [None, "channel", "sample"])
def test_gradients_that_are_not_there(dev, gate):
    """dy or dz of zero, both, and parameters whose gradients are not asked for."""
    c = Case((2, 33, 64), (F32, F32), gate=gate, p=0.2, seed=9)
    t, kw = c.args(dev)
    zero = torch.zeros_like(t["dy"])
    for dy, dz in ((None, t["dz"]), (t["dy"], None), (None, None)):
        got = kernels.residual_norm_backward(t["h"], t["x"], dy, dz, **kw)
        want = kernels.residual_norm_backward(t["h"], t["x"], zero if dy is None else dy, zero if dz is None else dz, **kw)
        for a, b in zip(got, want):
            assert (a is None) == (b is None) and (a is None or torch.allclose(a, b, rtol=1e-5, atol=1e-6))
    full = kernels.residual_norm_backward(t["h"], t["x"], t["dy"], t["dz"], **kw)
    for i in range(5):
        needs = [j == i for j in range(5)]
        part = kernels.residual_norm_backward(t["h"], t["x"], t["dy"], t["dz"], needs=needs, **kw)
        assert torch.equal(part.dh, full.dh) and torch.equal(part.dx, full.dx)
        for j, (a, b) in enumerate(zip(part[2:], full[2:])):
            assert (a is None) == (j != i or b is None) and (a is None or torch.equal(a, b))


def test_no_rows(dev):
    c = Case((2, 3, 16), (BF16, F32), gate="sample")
    t, kw = c.args(dev)
    h, x = t["h"][:, :0], t["x"][:, :0]
    y, z = kernels.residual_norm(h, x, **kw)
    assert y.shape == z.shape == (2, 0, 16)
    g = kernels.residual_norm_backward(h, x, t["dy"][:, :0].contiguous(), t["dz"][:, :0].contiguous(), **kw)
    assert all(bool((q == 0).all()) for q in g[2:]) and g.dgate.shape == (2, 16)


@pytest.mark.parametrize("p", [1.0, 2.0 ** -18])
def test_everything_and_nothing_dropped(dev, p):
    Case((11, 80), (BF16, BF16), p=p, seed=10).check(dev)


def test_non_finite_rows_stay_in_their_rows(dev):
    """A row with NaN or infinity, one of a type's lowest values, one of zeros."""
    c = Case((8, 64), (BF16, BF16), p=0.3, seed=11)
    clean = c.run(dev)
    t, kw = c.args(dev)
    h = t["h"].clone()
    h[2, 5], h[4, 6], h[6] = float("nan"), float("-inf"), torch.finfo(BF16).min
    h[7] = 0
    y, z = kernels.residual_norm(h, t["x"], **kw)
    g = kernels.residual_norm_backward(h, t["x"], t["dy"], t["dz"], **kw)
    for row in (0, 1, 3, 5):
        for a, b in ((y, clean[0]), (z, clean[1]), (g.dh, clean[2].dh), (g.dx, clean[2].dx)):
            assert torch.equal(a[row], b[row])
    assert bool(torch.isnan(z[2]).all()) and bool(torch.isfinite(y[7]).all())
    # what is dropped is 0 whatever the norm gave
    keep = rg.keep_mask(SEED, 8, 64, 0.3, c.stream).to(dev)
    assert torch.equal(y[2][~keep[2]], t["x"][2][~keep[2]])


def test_dropped_branch_without_norm(dev):
    """NaN and infinities of the branch in dropped places leave no trace."""
    c = Case((16, 40), (F32, F32), None, "layer", None, p=0.5, seed=12)
    t, kw = c.args(dev)
    keep = rg.keep_mask(SEED, 16, 40, 0.5, c.stream).to(dev)
    clean = kernels.residual_norm(t["h"], t["x"], **kw)
    for bad in (float("nan"), float("inf"), torch.finfo(F32).min):
        h = torch.where(keep, t["h"], torch.full_like(t["h"], bad))
        out = kernels.residual_norm(h, t["x"], **kw)
        assert torch.equal(out[0], clean[0]) and torch.equal(out[1], clean[1])


def test_autograd_matches_the_kernels_and_differences(dev):
    c = Case((2, 12, 9, 40), (F32, F32), gate="sample", p=0.25, seed=13)
    t, kw = c.args(dev)
    names = ("h", "x", "pw", "pb", "gate", "nw", "nb")
    v = {n: t[n].requires_grad_() for n in names}
    kw.update(post_norm=Norm(v["pw"], v["pb"], *c.kinds[0]), next_norm=Norm(v["nw"], v["nb"], *c.kinds[1]), gate=v["gate"])
    y, z = autograd.residual_norm(v["h"], v["x"], **kw)
    grads = torch.autograd.grad((y, z), list(v.values()), (t["dy"], t["dz"]))
    g = kernels.residual_norm_backward(v["h"].detach(), v["x"].detach(), t["dy"], t["dz"], **kw)
    for a, b in zip(grads, (g.dh, g.dx, g.dpost_weight, g.dpost_bias, g.dgate, g.dnext_weight, g.dnext_bias)):
        assert torch.equal(a, b)
    # central differences of the 64-bit forward along a random direction of each input
    step = 1e-6

    def loss(**moved):
        u = {n: moved.get(n, getattr(c, n).double()) for n in names}
        yy, zz = rg.residual_norm(u["h"], u["x"], (u["pw"], u["pb"], *c.kinds[0]), u["gate"], (u["nw"], u["nb"], *c.kinds[1]),
                                  None, c.alpha, c.p, SEED, c.stream)
        return ((yy * c.dy.double()).sum() + (zz * c.dz.double()).sum()).item()

    gen = torch.Generator().manual_seed(14)
    for n, got in zip(names, grads):
        base = getattr(c, n).double()
        d = torch.randn(base.shape, generator=gen, dtype=torch.float64)
        slope = (loss(**{n: base + step * d}) - loss(**{n: base - step * d})) / (2 * step)
        got = (got.double().cpu() * d)
        # 1e-6 steps: 1e-12 curvature, 1e-16 / 1e-6 cancellation; the kernel's fp32 sums
        assert abs(got.sum().item() - slope) <= 1e-5 * got.abs().sum().item(), n


def test_autograd_forms(dev):
    """A branch's gradient alone, y unused, 16-bit parameters, a promoted stream, no second derivative."""
    c = Case((4, 6, 32), (BF16, BF16), gate="sample", seed=15)
    t, kw = c.args(dev)
    h = t["h"].clone().requires_grad_()
    y, z = autograd.residual_norm(h, t["x"], **kw)
    dh, = torch.autograd.grad(z, h, t["dz"])
    assert torch.equal(dh, kernels.residual_norm_backward(t["h"], t["x"], None, t["dz"], needs=(False,) * 5, **kw).dh)
    gate = t["gate"].bfloat16().requires_grad_()
    y, z = autograd.residual_norm(t["h"], t["x"], **{**kw, "gate": gate})
    dgate, = torch.autograd.grad((y, z), gate, (t["dy"], t["dz"].expand_as(z)))
    want = kernels.residual_norm_backward(t["h"], t["x"], t["dy"], t["dz"], **{**kw, "gate": gate.detach()}).dgate
    assert dgate.dtype == BF16 and torch.equal(dgate, want.bfloat16())
    y, z = autograd.residual_norm(t["h"].float(), t["x"], **kw)
    assert y.dtype == z.dtype == F32
    h = t["h"].clone().requires_grad_()
    y, z = autograd.residual_norm(h, t["x"], **kw)
    dh, = torch.autograd.grad((y * y).sum() + z.float().sum(), h, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable|twice"):
        dh.float().sum().backward()


def test_the_node_keeps_torchs_rules(dev):
    """A graph that is kept gives its gradients again, one that is freed or whose saved tensors changed refuses;
    the engine may run in the caller's thread; only the gradients asked for are taken."""
    c = Case((3, 17, 96), (BF16, F32), gate="sample", p=0.2, seed=34)
    t, kw = c.args(dev)
    want = kernels.residual_norm_backward(t["h"], t["x"], t["dy"], t["dz"], **kw)
    leaves = {k: t[k].clone().requires_grad_() for k in ("h", "x", "pw", "pb", "gate", "nw", "nb")}
    given = dict(kw, post_norm=Norm(leaves["pw"], leaves["pb"], 1e-5), gate=leaves["gate"],
                 next_norm=Norm(leaves["nw"], leaves["nb"], 1e-5))
    call = lambda: autograd.residual_norm(leaves["h"], leaves["x"], **given)  # noqa: E731
    outs = call()
    with torch.autograd.set_multithreading_enabled(False):
        first = torch.autograd.grad(outs, list(leaves.values()), (t["dy"], t["dz"]), retain_graph=True)
    again = torch.autograd.grad(outs, list(leaves.values()), (t["dy"], t["dz"]))
    order = (want.dh, want.dx, want.dpost_weight, want.dpost_bias, want.dgate, want.dnext_weight, want.dnext_bias)
    for a, b, ref in zip(first, again, order):
        assert torch.equal(a, ref) and torch.equal(b, ref)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(outs, leaves["h"], (t["dy"], t["dz"]))
    for name in ("h", "pw"):
        outs = call()
        with torch.no_grad():
            leaves[name].mul_(1)
        with pytest.raises(RuntimeError, match="inplace|in-place"):
            torch.autograd.grad(outs, leaves["x"], (t["dy"], t["dz"]))
    dnb, = torch.autograd.grad(call(), leaves["nb"], (t["dy"], t["dz"]))
    assert torch.equal(dnb, want.dnext_bias)
    import torch.autograd.forward_ad as fwad

    with fwad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        autograd.residual_norm(fwad.make_dual(t["h"], t["h"]), t["x"], **kw)
    leaves["h"].requires_grad_(False)
    y, z = autograd.residual_norm(leaves["h"], t["x"], **kw)
    assert not y.requires_grad and not z.requires_grad
    with torch.no_grad():
        assert not call()[0].requires_grad


def test_saved_tensors_that_come_back_packed(dev):
    """save_on_cpu keeps a copy of a column block, and gives it back packed."""
    c = Case((9, 64), (BF16, F32), p=0.1, seed=16)
    t, kw = c.args(dev)
    wide = torch.zeros(9, 200, dtype=BF16, device=dev)
    wide[:, 8:72] = t["h"]
    grads = []
    for hooks in (False, True):
        h, x = wide.clone().requires_grad_(), t["x"].clone().requires_grad_()
        with torch.autograd.graph.save_on_cpu() if hooks else torch.enable_grad():
            y, z = autograd.residual_norm(h[:, 8:72], x, **kw)
        grads.append(torch.autograd.grad((y, z), (h, x), (t["dy"], t["dz"])))
    for a, b in zip(*grads):
        assert torch.equal(a, b)


@pytest.mark.parametrize("C,rows", [(1024, (1 << 21) + 37), (8, (1 << 28) + 5)])
def test_offsets_past_32_bits(dev, C, rows):
    """Tensors of over 2^32 bytes, and more row groups than one launch has workgroups: the last
    rows are those of a call of their own."""
    h = torch.empty(rows, C, dtype=BF16, device=dev).normal_(generator=torch.Generator(dev).manual_seed(1))
    x = h.roll(1, 0)
    ln = Norm(1 + 0.1 * torch.randn(C, device=dev), 0.1 * torch.randn(C, device=dev))
    kw = dict(post_norm=ln, gate=torch.rand(C, device=dev), next_norm=ln)
    y, z = kernels.residual_norm(h, x, **kw)
    for at in (slice(rows - 9, rows), slice(rows // 2, rows // 2 + 9)):
        a, b = kernels.residual_norm(h[at].contiguous(), x[at].contiguous(), **kw)
        assert torch.equal(y[at], a) and torch.equal(z[at], b)
    del y
    g = kernels.residual_norm_backward(h, x, z, x, **kw)
    for at in (slice(rows - 9, rows), slice(rows // 2, rows // 2 + 9)):
        part = kernels.residual_norm_backward(*(t[at].contiguous() for t in (h, x, z, x)), **kw)
        assert torch.equal(g.dh[at], part.dh) and torch.equal(g.dx[at], part.dx)
    total = x.sum(0, dtype=torch.float64)
    # each of the at most 2^19 terms a lane adds in a row, and the rest in fp64, by magnitude
    assert bool(((g.dnext_bias.double() - total).abs() <= 2 ** 18 * E32 * x.abs().sum(0, dtype=torch.float64)).all())
    del h, x, z, g
    torch.cuda.empty_cache()


def test_infinite_gate_of_dropped_elements(dev):
    """A dropped element's branch and its gradient are 0 whatever the gate is."""
    c = Case((16, 40), (F32, F32), None, "layer", "channel", p=0.5, seed=17)
    t, kw = c.args(dev)
    keep = rg.keep_mask(SEED, 16, 40, 0.5, c.stream).to(dev)
    for bad in (float("inf"), float("nan")):
        kw["gate"] = torch.where(torch.arange(40, device=dev) == 3, bad, t["gate"])
        y = kernels.residual_norm(t["h"], t["x"], **kw)[0]
        dh = kernels.residual_norm_backward(t["h"], t["x"], t["dy"], None, **kw).dh
        assert torch.equal(y[~keep], t["x"][~keep]) and bool((dh[~keep] == 0).all())


def test_refusals(dev):
    c = Case((4, 6, 32), (BF16, BF16), gate="sample")
    t, kw = c.args(dev)
    h, x = t["h"], t["x"]
    bad = [
        (ValueError, "x's shape", dict(), h[:2], x),
        (ValueError, "channels", dict(), h[..., :16], x),
        (TypeError, "float32", dict(), h, x.half()),
        (TypeError, "float32", dict(), h.float(), x),
        (ValueError, "gate", dict(gate=torch.ones(3, 32, device=dev)), h, x),
        (ValueError, "gate", dict(gate=torch.ones(31, device=dev)), h, x),
        (ValueError, "weight", dict(post_norm=Norm(torch.ones(31, device=dev))), h, x),
        (ValueError, "needs a seed", dict(p=0.1, seed=None), h, x),
        (ValueError, "grid", dict(geom=WindowGeometry(1, 4, 8, 32, 4)), h, x),
        (ValueError, "unit channel stride", dict(), h.transpose(0, 1), x.transpose(0, 1)),
    ]
    for err, text, change, hh, xx in bad:
        with pytest.raises(err, match=text):
            kernels.residual_norm(hh, xx, **{**kw, **change})
    with pytest.raises(ValueError, match="8192"):
        kernels.residual_norm(torch.zeros(1, 8200, device=dev), torch.zeros(1, 8200, device=dev))
    with pytest.raises(ValueError, match="dz"):
        kernels.residual_norm_backward(h, x, t["dy"], t["dz"].float(), **kw)
    with pytest.raises(ValueError, match="without a next_norm"):
        kernels.residual_norm_backward(h, x, t["dy"], t["dz"], **{**kw, "next_norm": None})


def test_a_call_like_an_earlier_one(dev):
    """Calls of the same shapes and options check what they are given anew, and take numbers of any kind."""
    c = Case((2, 16, 24, 40), (BF16, F32), p=0.25, alpha=0.5, seed=30, geom=WindowGeometry(2, 16, 24, 40, 8, 4, 4))
    t, kw = c.args(dev)
    want = kernels.residual_norm(t["h"], t["x"], **kw)
    listed = WindowGeometry(2, 16, 24, 40, 8, 4, 4, [0, 0, 0, 0])
    for change in (dict(geom=listed), dict(residual_scale=torch.tensor(0.5), p=torch.tensor(0.25)), dict()):
        got = kernels.residual_norm(t["h"], t["x"], **{**kw, **change})
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    for seed in (None, torch.zeros(2, dtype=torch.int64, device=dev), torch.zeros(1, dtype=torch.int64)):
        with pytest.raises(ValueError, match="seed"):
            kernels.residual_norm(t["h"], t["x"], **{**kw, "seed": seed})
    with pytest.raises(ValueError, match="gate"):
        kernels.residual_norm(t["h"], t["x"], **{**kw, "gate": kw["gate"][:1]})
    changed = kernels.residual_norm(t["h"], t["x"], **{**kw, "residual_scale": torch.tensor(2.0)})
    assert not torch.equal(changed[0], want[0])


def test_one_tensor_twice(dev):
    """h and x may be one tensor, whose gradient is the sum of both."""
    g = torch.Generator(dev).manual_seed(31)
    v = torch.randn(50, 96, device=dev, generator=g, requires_grad=True)
    w = torch.randn(96, device=dev, generator=g, requires_grad=True)
    y = autograd.residual_norm(v, v, Norm(w), w)
    dy = torch.randn(50, 96, device=dev, generator=g)
    dv, dw = torch.autograd.grad(y, (v, w), dy)
    part = kernels.residual_norm_backward(v.detach(), v.detach(), dy, None, Norm(w.detach()), w.detach())
    assert torch.equal(dv, part.dh + part.dx) and torch.equal(dw, part.dpost_weight + part.dgate)


def test_calls_of_two_threads(dev):
    cs = [Case((3, 130, 96), (BF16, F32), gate="sample", p=0.2, seed=s) for s in (32, 33)]
    want, bad = [c.run(dev) for c in cs], []

    def calls(c, ref):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                y, z, g = c.run(dev)
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, b) for a, b in zip((y, z, *g), (ref[0], ref[1], *ref[2]))):
                    bad.append(c)

    torch.cuda.synchronize()
    threads = [threading.Thread(target=calls, args=a) for a in zip(cs, want)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not bad


def test_other_streams_and_graphs(dev):
    """Two graphs replayed in turn, with new inputs and seeds, eager calls between the replays."""
    cs = [Case((3, 130, 96), (BF16, F32), gate="sample", p=0.2, seed=s) for s in (20, 21)]
    want = [c.run(dev) for c in cs]
    t, kw = cs[0].args(dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y, z = kernels.residual_norm(t["h"], t["x"], **kw)
        g = kernels.residual_norm_backward(t["h"], t["x"], t["dy"], t["dz"], **kw)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, want[0][0]) and all(torch.equal(a, b) for a, b in zip(g, want[0][2]))
    graphs, outs = [], []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            y, z = kernels.residual_norm(t["h"], t["x"], **kw)
            g = kernels.residual_norm_backward(t["h"], t["x"], t["dy"], t["dz"], **kw)
        graphs.append(gr)
        outs.append((y, z, *g))
    for i in (1, 0, 1, 1):
        for name, v in cs[i].tensors().items():
            t[name].copy_(v)
        for gr, out in zip(graphs, outs):
            gr.replay()
            torch.cuda.synchronize()
            ref = (want[i][0], want[i][1], *want[i][2])
            assert all(torch.equal(a, b) for a, b in zip(out, ref))
            assert torch.equal(kernels.residual_norm(t["h"], t["x"], **kw)[0], want[i][0])
