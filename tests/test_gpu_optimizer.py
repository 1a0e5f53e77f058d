"""The gradient norm and the AdamW step (terra_swin_gradient_norm,
terra_swin_adamw) against the 64-bit oracle.

Tolerances, with u = 2^-24.  The norm is summed in 64 bits: one rounding, 2 u.
Moments in 32 bits: g times the factor, the two products and their sum, and the
betas as fp32 numbers, 4 u of the terms' magnitudes, 6 u for the second moment's square.  The
parameter: 3 u of itself (its factor's rounding, the product, the difference), of what is taken off 12 u (root, quotient,
rate, and half of the second moment's 6 u) and the first moment's error in it, and half a step of its type.
In 8 bits the moments are computed in 64 and then rounded to 32: the first one's scale is off by that and a
division, 2 u; the root by half the rounding of its square and an ulp (2 u), with the division 4 u.  Codes are
the oracle's except where the oracle's value is within a rounding to 32 bits (2 u) of the border of two
codes; or within 40 u of its draw's threshold: the root over its scale is off by 4 u, its square by 8 u of high^2, which is
at most 4.8 times high^2 - low^2 (low / high <= 8 / 9).
"""
import pytest
import torch

from oracle import training as tr
from terra_amd import kernels
from terra_amd.kernels import Moments

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
PAIRS = [(F32, F32), (F32, BF16), (F32, F16), (BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)]
OPTS = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-6, weight_decay=0.1)
SIZES = [(1,), (7,), (3, 5), (255,), (256,), (257,), (64, 64), (1000,), (33, 129), (8192,), (8193,), (3, 0), (), (20011,)]


def _rand(shape, dt, seed, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dt)


def _seed(dev, value=0x1234567890ABCDE):
    return torch.tensor([value], dtype=torch.int64, device=dev)


# ---- the norm ----------------------------------------------------------------------


def check_norm(r, grads, max_norm):
    n, f = tr.gradient_norm([g.cpu() for g in grads], max_norm)
    assert abs(r.norm.item() - n) <= 2 * U * n and abs(r.factor.item() - f) <= 2 * U * f
    assert r.nonfinite.item() == 0 and all(t.shape == () and t.dtype == F32 for t in r)


@pytest.mark.parametrize("max_norm", [None, 1.0, 1e6])
def test_norm(dev, max_norm):
    grads = [_rand(s, dt, i, 10.0 ** (i % 5 - 3)).to(dev) for i, s in enumerate(SIZES) for dt in (F32, BF16, F16)]
    check_norm(kernels.gradient_norm(grads, max_norm), grads, max_norm)
    for i in range(0, len(grads), 5):
        if grads[i].numel() > 0:
            check_norm(kernels.gradient_norm([grads[i]], max_norm), [grads[i]], max_norm)


def test_norm_of_many_and_large(dev):
    many = [_rand((17 + i % 50,), F32, i).to(dev) for i in range(300)]
    check_norm(kernels.gradient_norm(many, 1.0), many, 1.0)
    large = [_rand((1000, 1001), BF16, 1).to(dev), _rand((1 << 20,), F32, 2).to(dev)[3:]]
    a, b = (kernels.gradient_norm(large, 1.0) for _ in range(2))
    check_norm(a, large, 1.0)
    assert torch.equal(a.norm, b.norm)


def test_norm_of_values_whose_squares_overflow(dev):
    for scale in (1e25, 1e-30):
        g = [_rand((3000,), F32, 1, scale).to(dev)]
        check_norm(kernels.gradient_norm(g, 1.0), g, 1.0)


def test_norm_of_nothing_and_of_what_is_not_finite(dev):
    r = kernels.gradient_norm([torch.zeros(0, device=dev)], 1.0)
    assert (r.norm.item(), r.factor.item(), r.nonfinite.item()) == (0.0, 1.0, 0.0)
    r = kernels.gradient_norm([torch.zeros(9, device=dev)], 1e-3)
    assert r.norm.item() == 0.0 and r.factor.item() == 1.0
    for bad in (float("inf"), float("nan")):
        r = kernels.gradient_norm([torch.ones(5, device=dev), torch.tensor([1.0, bad], device=dev)], 1.0)
        assert r.nonfinite.item() == 1.0 and not r.norm.isfinite()
        assert r.factor.item() == 0.0 if bad == float("inf") else r.factor.isnan()


def test_norm_of_other_strides(dev):
    g = [_rand((30, 40), F32, 1).to(dev).t(), _rand((30, 40), F32, 2).to(dev)[:, ::3], torch.ones(1, device=dev).expand(77)]
    check_norm(kernels.gradient_norm(g, 1.0), g, 1.0)


# ---- the step, moments in 32 bits ----------------------------------------------------


def check_step(after, before, g, step, factor=1.0, sign=1.0, opts=OPTS):
    """after, before: (param, exp_avg, exp_avg_sq) on the CPU."""
    b1, b2 = opts["betas"]
    p, m0, v0 = (t.double() for t in before)
    g = sign * g.double() * factor
    m, v = tr.moments(g, m0, v0, b1, b2)
    q, d = tr.updated(p, m, v, step, opts["lr"], b1, b2, opts["eps"], opts["weight_decay"])
    em = 4 * U * ((b1 * m0).abs() + ((1 - b1) * g).abs())
    ev = 6 * U * v
    off = d.abs() / m.abs().clamp_min(1e-300) * em
    dt = after[0].dtype
    ep = 3 * U * p.abs() + 12 * U * d.abs() + off + torch.finfo(dt).eps / 2 * q.abs() + torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
    for name, got, ref, tol in (("param", after[0], q, ep), ("exp_avg", after[1], m, em + 1e-44), ("exp_avg_sq", after[2], v, ev + 1e-44)):
        e = (got.double() - ref).abs()
        assert bool((e <= tol).all()), (name, (e / tol).max())


def _state(shape, pt, i, dev, old=True):
    p = _rand(shape, pt, 3 * i)
    m = _rand(shape, F32, 3 * i + 1, 0.1) if old else torch.zeros(shape)
    v = _rand(shape, F32, 3 * i + 2, 0.1).square() if old else torch.zeros(shape)
    return p, m, v


@pytest.mark.parametrize("pt,gt", PAIRS)
@pytest.mark.parametrize("step", [1, 1000])
def test_step(dev, pt, gt, step):
    before = [_state(s, pt, i, dev, step > 1) for i, s in enumerate(SIZES)]
    grads = [_rand(s, gt, 100 + i, 0.3) for i, s in enumerate(SIZES)]
    now = [[t.to(dev) for t in b] for b in before]
    kernels.adamw_step([t[0] for t in now], [g.to(dev) for g in grads], [Moments(t[1], t[2]) for t in now], step, **OPTS)
    for after, b, g in zip(now, before, grads):
        check_step([t.cpu() for t in after], b, g, step)


def test_step_of_many_mixed_tensors(dev):
    """More than a launch lists, of all pairs of types, in 32 and 8 bits, in one call."""
    n = 200
    before = [_state((11 + i,), PAIRS[i % 7][0], i, dev) for i in range(n)]
    grads = [_rand((11 + i,), PAIRS[i % 7][1], 900 + i, 0.3) for i in range(n)]
    now = [[t.to(dev) for t in b] for b in before]
    moments = [Moments(t[1], t[2]) if i % 3 else kernels.moments(t[0], 8) for i, t in enumerate(now)]
    kernels.adamw_step([t[0] for t in now], [g.to(dev) for g in grads], moments, 7, **OPTS, seed=_seed(dev))
    for i, (after, b, g) in enumerate(zip(now, before, grads)):
        if i % 3:
            check_step([t.cpu() for t in after], b, g, 7)
        else:
            assert moments[i].scales.min() > 0


@pytest.mark.parametrize("offset", [1, 2, 3])
def test_step_off_any_alignment(dev, offset):
    for pt, gt in PAIRS:
        for n in (5, 1000, 9001):
            p, m, v = _state((n,), pt, 5, dev)
            g = _rand((n,), gt, 9)
            shifted = []
            for t in (p, m, v, g):
                buf = torch.full((n + 8,), 3.0, dtype=t.dtype, device=dev)
                buf[offset:offset + n] = t.to(dev)
                shifted.append(buf)
            a = [t[offset:offset + n] for t in shifted]
            kernels.adamw_step([a[0]], [a[3]], [Moments(a[1], a[2])], 3, **OPTS)
            check_step([t.cpu() for t in a[:3]], (p, m, v), g, 3)
            for buf in shifted:  # what stands beside it is left
                assert bool((buf[:offset] == 3).all()) and bool((buf[offset + n:] == 3).all())


def test_step_options(dev):
    p, m, v = _state((3000,), F32, 1, dev)
    g = _rand((3000,), F32, 9)
    for kw, factor, sign in ((dict(grad_factor=torch.tensor(0.25, device=dev)), 0.25, 1.0), (dict(maximize=True), 1.0, -1.0),
                             (dict(found_inf=torch.tensor(0.0, device=dev)), 1.0, 1.0)):
        now = [t.to(dev) for t in (p, m, v)]
        kernels.adamw_step([now[0]], [g.to(dev)], [Moments(*now[1:])], 5, **OPTS, **kw)
        check_step([t.cpu() for t in now], (p, m, v), g, 5, factor, sign)
    for opts in (dict(lr=0.0, betas=(0.0, 0.0), eps=1e-8, weight_decay=0.0), dict(lr=1.0, betas=(0.5, 0.9999), eps=1.0, weight_decay=0.0)):
        now = [t.to(dev) for t in (p, m, v)]
        kernels.adamw_step([now[0]], [g.to(dev)], [Moments(*now[1:])], 2, **opts)
        check_step([t.cpu() for t in now], (p, m, v), g, 2, opts=opts)


@pytest.mark.parametrize("bits", [32, 8])
def test_a_step_left_out(dev, bits):
    p, g = _rand((777,), F32, 1).to(dev), _rand((777,), F32, 2).to(dev)
    m = kernels.moments(p, bits)
    kernels.adamw_step([p], [g], [m], 1, **OPTS, seed=_seed(dev))
    kept = [t.clone() for t in (p, *m) if t is not None]
    g[3] = float("nan")
    n = kernels.gradient_norm([g], 1.0)
    kernels.adamw_step([p], [g], [m], 2, **OPTS, grad_factor=n.factor, found_inf=n.nonfinite, seed=_seed(dev))
    for a, b in zip(kept, (t for t in (p, *m) if t is not None)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_step_and_rate_in_device_memory(dev):
    p, m, v = _state((500,), F32, 1, dev)
    g = _rand((500,), F32, 9)
    now = [t.to(dev) for t in (p, m, v)]
    opts = dict(OPTS, lr=torch.tensor(3e-3, device=dev))
    kernels.adamw_step([now[0]], [g.to(dev)], [Moments(*now[1:])], torch.tensor([12], device=dev), **opts)
    check_step([t.cpu() for t in now], (p, m, v), g, 12, opts=dict(OPTS, lr=torch.tensor(3e-3).item()))


def test_dense_tensors_of_other_strides(dev):
    p, m, v = (t.t() for t in _state((40, 30), F32, 1, dev))
    g = _rand((30, 40), F32, 9)  # packed: of other strides than the parameter
    now = [t.t().to(dev).t() for t in (p, m, v)]
    assert now[0].stride() == (1, 30)
    kernels.adamw_step([now[0]], [g.to(dev)], [Moments(*now[1:])], 3, **OPTS)
    check_step([t.cpu() for t in now], (p, m, v), g, 3)


def test_infinities_and_nan_stay_in_their_elements(dev):
    p, g = _rand((600,), F32, 1).to(dev), _rand((600,), F32, 2).to(dev)
    g[5], g[300] = float("inf"), float("nan")
    m = kernels.moments(p)
    kernels.adamw_step([p], [g], [m], 1, **OPTS)
    assert (~p.isfinite()).nonzero().view(-1).tolist() == [5, 300]
    q, h = _rand((600,), F32, 1).to(dev), g.clone()
    m = kernels.moments(q, 8)
    kernels.adamw_step([q], [h], [m], 1, **OPTS, seed=_seed(dev))
    assert (~q.isfinite()).nonzero().view(-1).tolist() == [5, 300]
    kernels.adamw_step([q], [torch.ones_like(q)], [m], 2, **OPTS, seed=_seed(dev))
    assert not q[:512].isfinite().any() and q[512:].isfinite().all()  # their blocks are NaN from then on


def test_changed_tensors_are_counted(dev):
    p = torch.nn.Parameter(torch.ones(9, device=dev))
    m = kernels.moments(p)
    versions = [t._version for t in (p, *m[:2])]
    y = p * p
    kernels.adamw_step([p], [torch.ones(9, device=dev)], [m], 1)
    assert all(t._version > v for t, v in zip((p, *m[:2]), versions))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


# ---- moments in 8 bits ---------------------------------------------------------------


def _codes(t):
    return t.cpu().view(torch.uint8).reshape(-1)


def check_step_8bit(p_after, m_after, before, m_before, g, step, seed, index, factor=1.0, opts=OPTS, stream=0):
    """One tensor; before, g on the CPU; m_before, m_after Moments on the CPU."""
    b1, b2 = opts["betas"]
    values = tr.e4m3_values()
    n = before.numel()
    block = torch.arange(n) // 256
    signed = lambda c: torch.where(c >= 128, -1.0, 1.0).double() * values[(c % 128).long()]  # noqa: E731
    m0 = signed(_codes(m_before.exp_avg)) * m_before.scales[0].double()[block]
    v0 = (signed(_codes(m_before.exp_avg_sq)) * m_before.scales[1].double()[block]).square()
    g, p = g.double().reshape(-1) * factor, before.double().reshape(-1)
    m, v = tr.moments(g, m0, v0, b1, b2)
    q, d = tr.updated(p, m, v, step, opts["lr"], b1, b2, opts["eps"], opts["weight_decay"])
    dt = before.dtype
    tol = 3 * U * p.abs() + 12 * U * d.abs() + torch.finfo(dt).eps / 2 * q.abs() + torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
    assert bool(((p_after.double().reshape(-1) - q).abs() <= tol).all())
    blocks = -(-n // 256)
    top = torch.zeros(2, blocks, dtype=torch.float64).scatter_reduce_(1, block.expand(2, n), torch.stack((m.abs(), v)), "amax")
    top[1] = top[1].sqrt()
    scales = m_after.scales.double()
    assert bool(((scales - top / 448).abs() <= torch.tensor([[2.0], [4.0]]).double() * U * top / 448 + 1e-44).all())
    inv = torch.where(scales > 0, 1 / scales, torch.zeros_like(scales))
    code, near = tr.nearest_code((m * inv[0][block]).clamp(-448, 448))
    same = code == _codes(m_after.exp_avg)
    zero = (code % 128 == 0) & (_codes(m_after.exp_avg) % 128 == 0)  # of either sign
    assert bool((same | zero | (near < 2 * U)).all())
    code, near = tr.root_code(v * inv[1][block].square(), tr.draws(seed, n, index, step, stream))
    same = code == _codes(m_after.exp_avg_sq)
    assert bool((same | (near < 40 * U)).all())
    assert int((~same).sum()) <= n // 1000


def _cpu(m):
    return Moments(*(t.cpu() for t in m))


@pytest.mark.parametrize("pt,gt", PAIRS)
def test_steps_in_8_bits(dev, pt, gt):
    seed = 0x0FEDCBA987654321
    params = [_rand(s, pt, i) for i, s in enumerate(SIZES)]
    now = [p.to(dev) for p in params]
    moments = [kernels.moments(p, 8) for p in now]
    for step in (1, 2, 3):
        grads = [_rand(s, gt, 50 * step + i, 0.3 * 10.0 ** (i % 4 - 2)) for i, s in enumerate(SIZES)]
        before = [(p.cpu(), _cpu(Moments(*(t.clone() for t in m)))) for p, m in zip(now, moments)]
        kernels.adamw_step(now, [g.to(dev) for g in grads], moments, step, **OPTS, seed=_seed(dev, seed), stream=4)
        for i, (p, m, g, (b, mb)) in enumerate(zip(now, moments, grads, before)):
            if p.numel() > 0:
                check_step_8bit(p.cpu(), _cpu(m), b, mb, g, step, seed, i, stream=4)


def test_8_bits_off_any_alignment(dev):
    for offset in (1, 2, 5):
        for n in (300, 9003):
            p, g = _rand((n,), F32, 1), _rand((n,), F32, 2)
            pb, gb = torch.zeros(n + 8, device=dev), torch.zeros(n + 8, device=dev)
            cb = [torch.zeros(n + 16, dtype=torch.uint8, device=dev) for _ in range(2)]
            pb[offset:offset + n], gb[offset:offset + n] = p.to(dev), g.to(dev)
            m = Moments(*(c[offset:offset + n].view(torch.float8_e4m3fn) for c in cb), torch.zeros(2, -(-n // 256), device=dev))
            before = _cpu(Moments(*(t.clone() for t in m)))
            kernels.adamw_step([pb[offset:offset + n]], [gb[offset:offset + n]], [m], 1, **OPTS, seed=_seed(dev, 77))
            check_step_8bit(pb[offset:offset + n].cpu(), _cpu(m), p, before, g, 1, 77, 0)
            for c in cb:
                assert not c[:offset].any() and not c[offset + n:].any()


def test_8_bits_of_tiny_and_wide_values(dev):
    """Blocks of very small gradients, of a wide range, and of zeros; the second moment is never lost."""
    g = torch.cat((torch.full((256,), 1e-30), 10.0 ** (torch.arange(256) / 16 - 12), torch.zeros(256), torch.full((256,), 3e4)))
    p = torch.zeros(1024)
    now = p.to(dev)
    m = kernels.moments(now, 8)
    for step in (1, 2):
        before, b = _cpu(Moments(*(t.clone() for t in m))), now.cpu()
        kernels.adamw_step([now], [g.to(dev)], [m], step, **OPTS, seed=_seed(dev, 5))
        check_step_8bit(now.cpu(), _cpu(m), b, before, g, step, 5, 0)
    codes = _codes(m.exp_avg_sq)
    assert bool((codes[:512] > 0).all()) and not codes[512:768].any()
    assert now.isfinite().all()


def test_second_moment_in_8_bits_follows_the_gradients(dev):
    """The mean of v over many elements with the same gradients is that of 32 bits: 200 steps of beta2 = 0.99 on
    gradients that grow tenfold.  An element's v varies by about a third of itself at each
    end (a code's step is a quarter of v); the mean of 65536 of them by 0.0013, and is tested to 0.02."""
    n = 1 << 16
    p = torch.zeros(n, device=dev)
    m8, m32 = kernels.moments(p, 8), kernels.moments(p)
    q = p.clone()
    gen = torch.Generator(device=dev).manual_seed(0)
    for step in range(1, 201):
        g = torch.full((n,), 0.1 if step <= 100 else 1.0, device=dev)
        g[::256] = 8.0  # one large element in each block, so that the others have codes of their own
        g *= torch.where(torch.rand(n, generator=gen, device=dev) < 0.5, 1.0, -1.0)
        kernels.adamw_step([p, q], [g, g], [m8, m32], step, **OPTS, seed=_seed(dev, 99))
    v8, v32 = m8.values()[1], m32.values()[1]
    others = torch.arange(n, device=dev) % 256 != 0
    assert abs(v8[others].mean().item() / v32[others].mean().item() - 1) < 0.02


# ---- both ------------------------------------------------------------------------------


def test_past_32_bits_of_elements(dev):
    n = (1 << 31) + 5000  # 4.3 GB of bf16, 8.6 of each moment
    p = torch.zeros(n, dtype=BF16, device=dev)
    g = torch.zeros(n, dtype=BF16, device=dev)
    tail = slice(n - 3000, n)
    p[tail], g[tail] = _rand((3000,), BF16, 1).to(dev), _rand((3000,), BF16, 2).to(dev)
    r = kernels.gradient_norm([g], 1.0)
    check_norm(r, [g[tail]], 1.0)
    m = kernels.moments(p)
    before = p[tail].cpu()
    kernels.adamw_step([p], [g], [m], 1, **OPTS)
    check_step([t[tail].cpu() for t in (p, *m[:2])], (before, torch.zeros(3000), torch.zeros(3000)), g[tail].cpu(), 1)
    assert not p[:n - 3000].any() and not m.exp_avg[:n - 3000].any()


@pytest.mark.parametrize("bits", [32, 8])
def test_captured(dev, bits):
    """Norm and step in a graph, with the count, the rate and the seed in device memory."""
    sizes = [(300,), (64, 65), (9000,)]

    def fresh():
        ps = [_rand(s, F32, i).to(dev) for i, s in enumerate(sizes)]
        return ps, [kernels.moments(p, bits) for p in ps]

    grads = [torch.zeros(s, device=dev) for s in sizes]
    count, lr, seed = torch.zeros(1, dtype=torch.int64, device=dev), torch.tensor(1e-2, device=dev), _seed(dev, 3)
    (ps, ms), (qs, ns) = fresh(), fresh()

    def work(params, moments):
        n = kernels.gradient_norm(grads, 1.0)
        kernels.adamw_step(params, grads, moments, count, lr=lr, grad_factor=n.factor, found_inf=n.nonfinite, seed=seed)
        return n.norm

    warm, warm_m = fresh()
    count.fill_(1)
    work(warm, warm_m)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = work(ps, ms)
    for step in range(1, 5):
        for i, g in enumerate(grads):
            g.copy_(_rand(g.shape, F32, 100 * step + i))
        count.fill_(step)
        lr.fill_(1e-2 / step)
        seed.add_(1)
        graph.replay()
        eager = work(qs, ns)
        torch.cuda.synchronize()
        assert torch.equal(norm, eager)
        for a, b in zip(ps + [t for m in ms for t in m if t is not None], qs + [t for m in ns for t in m if t is not None]):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_on_another_stream(dev):
    p, g = _rand((5000,), F32, 1).to(dev), _rand((5000,), F32, 2).to(dev)
    q, m, n = p.clone(), kernels.moments(p), kernels.moments(p)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        kernels.adamw_step([p], [g], [m], 1, grad_factor=kernels.gradient_norm([g], 1.0).factor)
    s.synchronize()
    kernels.adamw_step([q], [g], [n], 1, grad_factor=kernels.gradient_norm([g], 1.0).factor)
    assert torch.equal(p, q)


def test_refusals(dev):
    p, g = torch.zeros(8, device=dev), torch.zeros(8, device=dev)
    m, m8 = kernels.moments(p), kernels.moments(p, 8)
    one = torch.ones(1, device=dev)
    step = lambda *a, **kw: kernels.adamw_step(*a, **kw)  # noqa: E731
    for bad, error, text in (
        (lambda: kernels.gradient_norm([g.double()]), TypeError, "not supported"),
        (lambda: kernels.gradient_norm([g.to_sparse()]), TypeError, "not dense"),
        (lambda: kernels.gradient_norm([g, torch.zeros(8)]), RuntimeError, "ROCm devices only"),
        (lambda: step([p], [], [m], 1), ValueError, "as many"),
        (lambda: step([p], [g[:7]], [m], 1), ValueError, "shape"),
        (lambda: step([p], [g.double()], [m], 1), TypeError, "not supported"),
        (lambda: step([p], [g.to_sparse()], [m], 1), TypeError, "not dense"),
        (lambda: step([p.bfloat16()], [g.half()], [m], 1), ValueError, "of one dtype"),
        (lambda: step([p], [g], [Moments(m[0].half(), m[1])], 1), ValueError, "moments of parameter 0"),
        (lambda: step([p], [g], [Moments(m[0][:4], m[1])], 1), ValueError, "moments of parameter 0"),
        (lambda: step([p], [g], [Moments(m[0], m[1], m8[2])], 1, seed=_seed(dev)), ValueError, "moments of parameter 0"),
        (lambda: step([p], [g], [Moments(m8[0], m8[1], torch.zeros(2, 2, device=dev))], 1, seed=_seed(dev)), ValueError, "scales"),
        (lambda: step([p], [g], [m8], 1), ValueError, "need a seed"),
        (lambda: step([p, p], [g, g], [m, kernels.moments(p)], 1), ValueError, "overlap"),
        (lambda: step([p], [p], [m], 1), ValueError, "overlap"),
        (lambda: step([p], [g], [Moments(m[0], m[0])], 1), ValueError, "overlap"),
        (lambda: step([p[:6], p[4:]], [g[:6], g[4:]], [kernels.moments(p[:6]), kernels.moments(p[4:])], 1), ValueError, "overlap"),
        (lambda: step([torch.zeros(4, 4, device=dev)[:, ::2]], [torch.zeros(4, 2, device=dev)],
                      [kernels.moments(torch.zeros(4, 2, device=dev))], 1), ValueError, "side by side"),
        (lambda: step([p], [g], [m], 0), ValueError, "step counts from 1"),
        (lambda: step([p], [g], [m], 1, betas=(1.0, 0.9)), ValueError, "betas"),
        (lambda: step([p], [g], [m], 1, lr=-1.0), ValueError, "lr"),
        (lambda: step([p], [g], [m], one), ValueError, "step must be one"),
        (lambda: step([p], [g], [m], 1, lr=one.double()), ValueError, "lr must be one"),
        (lambda: step([p], [g], [m], 1, grad_factor=torch.ones(2, device=dev)), ValueError, "grad_factor must be one"),
        (lambda: step([p], [g], [m], 1, found_inf=torch.ones(1)), ValueError, "found_inf must be one"),
        (lambda: step([p], [g], [m8], 1, seed=one), ValueError, "seed must be one"),
    ):
        with pytest.raises(error, match=text):
            bad()
    assert not p.any() and not m.exp_avg.any()
