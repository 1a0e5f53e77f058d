"""Norms over rows (terra_swin_layer_norm and its backward) against the 64-bit
oracle.

Tolerances, with u = 2^-24.  Sums over a row of C values are taken by lanes of
at most C / 8 + 8 values one after the other (far fewer in fact) and a tree of at most 16
steps, so with n = C / 8 + 24 a mean is off by n u of the mean of the magnitudes, and the reciprocal root
by (n + 4) u of itself; the normalised value by
    e = r n u mean|x| + (n + 6) u |xh|.
y adds four roundings of its terms, dx those of g and of its two means, and
both half a step of their type.  Sums over rows are at most R terms one after
the other: R u of the sum of the magnitudes, plus the error of xh in each term, plus half a step.
"""
import pytest
import torch

from oracle import training as tr
from terra_amd import autograd, kernels
from terra_amd.kernels import Norm

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [(F32, F32), (F32, BF16), (F32, F16), (BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)]


def _half(dt):
    return torch.finfo(dt).eps / 2


def _tiny(dt):
    return torch.finfo(dt).smallest_normal * torch.finfo(dt).eps


def _rand(shape, dt, seed, scale=1.0, mean=0.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale + mean).to(dt)


def _x(shape, dt, seed=1):
    x = _rand(shape, torch.float32, seed, 2.0, 0.4)
    x[..., ::7] *= 6.0
    return x.to(dt)


def _norm(C, dt=F32, rms=False, weight=True, bias=True, eps=1e-5, dev="cpu"):
    return Norm(_rand((C,), dt, 11, 0.3, 1.0).to(dev) if weight else None, _rand((C,), dt, 12, 0.2).to(dev) if bias else None,
                eps, rms)


def _errors(x, norm):
    """(xh, r, the bound of xh's error) of the oracle."""
    C = x.shape[-1]
    _, xh, _, r = tr.layer_norm(x, eps=norm.eps, rms=norm.rms)
    n = C / 8 + 24
    return xh, r, (0.0 if norm.rms else r * n * U * x.double().abs().mean(-1, keepdim=True)) + (n + 6) * U * xh.abs()


def _cpu(norm):
    return Norm(*(None if t is None else t.detach().cpu() for t in (norm.weight, norm.bias)), norm.eps, norm.rms)


def check_forward(y, x, norm):
    norm, x = _cpu(norm), x.detach().cpu()
    ref, xh, _, _ = tr.layer_norm(x, norm.weight, norm.bias, norm.eps, norm.rms)
    _, _, e = _errors(x, norm)
    w = torch.ones(()).double() if norm.weight is None else norm.weight.double().abs()
    b = torch.zeros(()).double() if norm.bias is None else norm.bias.double().abs()
    tol = _half(y.dtype) * ref.abs() + w * e + 4 * U * (xh.abs() * w + b) + _tiny(y.dtype)
    assert y.shape == x.shape and y.is_contiguous()
    assert bool(((y.double().cpu() - ref).abs() <= tol).all()), ((y.double().cpu() - ref).abs() / tol).max()


def check_backward(grads, dy, x, norm):
    norm, x, dy = _cpu(norm), x.detach().cpu(), dy.cpu().double()
    C, R = x.shape[-1], max(x.numel() // x.shape[-1], 1)
    xh, r, e = _errors(x, norm)
    w = torch.ones(()).double() if norm.weight is None else norm.weight.double()
    g, n = (dy * w).abs(), C / 8 + 24
    mean = lambda t: t.mean(-1, keepdim=True)  # noqa: E731
    s1 = mean(dy * w * xh).abs()
    dx, dw, db = tr.layer_norm_backward(dy, x, norm.weight, norm.eps, norm.rms)
    tol = r * (6 * U * g + (n + 4) * U * mean(g) + xh.abs() * ((n + 6) * U * mean(g * xh.abs()) + mean(g * e)) + e * s1) \
        + (n + 8) * U * dx.abs() + 4 * U * r * xh.abs() * s1
    over_rows = lambda t: t.reshape(-1, C).sum(0)  # noqa: E731
    bounds = [tol, R * U * over_rows((dy * xh).abs()) + over_rows(dy.abs() * e), R * U * over_rows(dy.abs())]
    for got, ref, bound in zip(grads, (dx, dw, db), bounds):
        if got is None:
            continue
        assert got.shape == ref.shape
        bound = bound + (_half(got.dtype) + 2 * U) * ref.abs() + _tiny(got.dtype)
        assert bool(((got.double().cpu() - ref).abs() <= bound).all()), ((got.double().cpu() - ref).abs() / bound).max()


SHAPES = [(1, 1), (1, 8), (3, 7), (2, 5, 16), (9, 33), (5, 64), (67, 96), (130, 100), (33, 192), (7, 386), (21, 768),
          (17, 1024), (5, 1030), (6, 2048), (4, 4096), (3, 4098), (2, 8192), (3, 8200), (2, 8201), (2, 20000), (1, 40001),
          (2, 16), (70, 24), (5, 32), (1, 385), (200, 385), (77, 1001), (9, 1101), (5, 1601), (40, 2049), (9, 5001),
          (3, 12000), (2, 16384), (3, 16383), (2, 16385)]


@pytest.mark.parametrize("rms", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("xt,yt", TYPES)
def test_against_oracle(dev, xt, yt, shape, rms):
    C = shape[-1]
    x, norm, dy = _x(shape, xt).to(dev), _norm(C, rms=rms, dev=dev), _rand(shape, yt, 3).to(dev)
    y, st = kernels.layer_norm(x, norm, yt, statistics=True)
    assert y.dtype == yt
    check_forward(y, x, norm)
    assert torch.equal(kernels.layer_norm(x, norm, yt), y)
    grads = kernels.layer_norm_backward(dy, x, norm, st)
    assert grads.dx.dtype == xt and grads.dweight.dtype == grads.dbias.dtype == F32
    check_backward(grads, dy, x, norm)


@pytest.mark.parametrize("C", [16, 24, 99, 100, 130, 385, 768, 1001, 9000, 9001])
@pytest.mark.parametrize("rows", [40, 3001])
def test_sums_over_many_rows(dev, rows, C):
    """Rows of many workgroups; the sums are the same in a second call."""
    rows = rows if C < 1000 else rows // 10
    x, norm, dy = _x((rows, C), BF16).to(dev), _norm(C, BF16, dev=dev), _rand((rows, C), BF16, 3, mean=0.2).to(dev)
    _, st = kernels.layer_norm(x, norm, statistics=True)
    a, b = (kernels.layer_norm_backward(dy, x, norm, st) for _ in range(2))
    assert a.dweight.dtype == BF16
    check_backward(a, dy, x, norm)
    assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("pt", [F32, BF16, F16])
@pytest.mark.parametrize("weight,bias", [(True, True), (True, False), (False, True), (False, False)])
def test_parameters(dev, pt, weight, bias):
    shape = (19, 72)
    x, norm, dy = _x(shape, F16).to(dev), _norm(72, pt, False, weight, bias, dev=dev), _rand(shape, F16, 3).to(dev)
    y, st = kernels.layer_norm(x, norm, statistics=True)
    check_forward(y, x, norm)
    grads = kernels.layer_norm_backward(dy, x, norm, st)
    assert (grads.dweight is not None) == weight and (grads.dbias is not None) == bias
    check_backward(grads, dy, x, norm)
    for needs in ((True, False, False), (False, True, False), (False, False, True), (False, False, False)):
        some = kernels.layer_norm_backward(dy, x, norm, st, needs)
        for a, b, need in zip(some, grads, needs):
            assert (a is None) if not need or b is None else torch.equal(a, b)


def test_parameters_of_two_types(dev):
    x, dy = _x((6, 40), BF16).to(dev), _rand((6, 40), BF16, 3).to(dev)
    norm = Norm(_rand((40,), BF16, 1).to(dev), _rand((40,), F32, 2).to(dev))
    y, st = kernels.layer_norm(x, norm, statistics=True)
    check_forward(y, x, norm)
    grads = kernels.layer_norm_backward(dy, x, norm, st)
    assert grads.dweight.dtype == BF16 and grads.dbias.dtype == F32
    check_backward(grads, dy, x, norm)


def _strided(kind, dt):
    """Rows that are not packed: (x, its values)."""
    big = _x((7, 9, 6, 32), dt)
    return {
        "heads": big[:, :, 2:5],                        # of a packed row: rows of two strides
        "columns": big.view(7, 9, 192)[..., 32:96],     # a column block of wider rows
        "odd columns": big.view(7, 9, 192)[..., 5:82],  # the same off any alignment
        "every other": big[:, ::2, 0],
        "transposed": big[:, :, 1].transpose(0, 1),
        "broadcast": big[:1, :1, 0].expand(7, 9, 32),
        "one row": big[3, 4, 5],
    }[kind]


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("kind", ["heads", "columns", "odd columns", "every other", "transposed", "broadcast", "one row"])
def test_rows_of_other_strides(dev, kind, dt):
    x = _strided(kind, dt)
    xd = torch.empty(0, dtype=dt, device=dev).set_(_device_storage(x, dev), x.storage_offset(), x.shape, x.stride())
    C = x.shape[-1]
    norm, dy = _norm(C, dev=dev), _rand(x.shape, dt, 3).to(dev)
    y, st = kernels.layer_norm(xd, norm, statistics=True)
    check_forward(y, x, norm)
    check_backward(kernels.layer_norm_backward(dy, xd, norm, st), dy, x, norm)


def _device_storage(x, dev):
    whole = torch.empty(0, dtype=x.dtype).set_(x.untyped_storage(), 0, (x.untyped_storage().nbytes() // x.element_size(),), (1,))
    return whole.to(dev).untyped_storage()


@pytest.mark.parametrize("offset", [0, 1, 3, 8])
@pytest.mark.parametrize("rows,C", [(11, 64), (11, 63), (1, 17), (5, 1001), (3, 2051), (2, 9001)])
def test_addresses_off_any_alignment(dev, offset, rows, C):
    buf = _x((rows * C + 8,), BF16).to(dev)
    x = buf[offset:offset + rows * C].view(rows, C)
    norm = _norm(C, dev=dev)
    out = torch.full((rows * C + 16,), 7.0, dtype=BF16, device=dev)
    y = out[offset:offset + rows * C].view(rows, C)
    assert kernels.layer_norm(x, norm, out=y).data_ptr() == y.data_ptr()
    check_forward(y, x, norm)
    assert bool((out[:offset] == 7).all()) and bool((out[offset + rows * C:] == 7).all())  # what stands beside it is left
    _, st = kernels.layer_norm(x, norm, statistics=True)
    dy = torch.zeros_like(out)
    dy[offset:offset + rows * C] = _rand((rows * C,), BF16, 3).to(dev)
    dy = dy[offset:offset + rows * C].view(rows, C)
    check_backward(kernels.layer_norm_backward(dy, x, norm, st), dy, x, norm)


@pytest.mark.parametrize("shape", [(0, 8), (4, 0, 8), (0, 9000)])
def test_no_rows(dev, shape):
    norm = _norm(shape[-1], dev=dev)
    x = torch.zeros(shape, device=dev)
    y, st = kernels.layer_norm(x, norm, statistics=True)
    assert y.shape == x.shape and tuple(st.shape) == (0, 2)
    grads = kernels.layer_norm_backward(x, x, norm, st)
    assert grads.dx.shape == x.shape and not grads.dweight.any() and not grads.dbias.any()


def test_infinities_and_nan_stay_in_their_rows(dev):
    for C in (40, 768, 9000):
        x, norm, dy = _x((6, C), BF16).to(dev), _norm(C, dev=dev), _rand((6, C), BF16, 3).to(dev)
        clean = kernels.layer_norm(x, norm)
        x[1, 3], x[4, C - 1] = float("inf"), float("nan")
        y, st = kernels.layer_norm(x, norm, statistics=True)
        keep = torch.tensor([0, 2, 3, 5], device=dev)
        assert torch.equal(y[keep], clean[keep])
        assert y[4].isnan().all() and y[1, 3].isnan()
        dx = kernels.layer_norm_backward(dy, x, norm, st).dx
        assert dx[keep].isfinite().all() and dx[4].isnan().all()


def test_constant_rows_and_far_means(dev):
    """A row of one value has no spread but eps; a mean far from 0 costs what its magnitude does."""
    x = torch.full((3, 192), 1000.0)
    x[1] += torch.randn(192, generator=torch.Generator().manual_seed(0))
    norm = _norm(192, dev=dev)
    y = kernels.layer_norm(x.to(dev), norm)
    check_forward(y, x, norm)


def test_rows_past_32_bits_of_elements(dev):
    rows, C = 2_200_000, 1000  # 2.2e9 elements, 4.4 GB
    x = torch.empty(rows, C, dtype=BF16, device=dev)
    x[:4], x[-4:] = _x((4, C), BF16).to(dev), _x((4, C), BF16, 2).to(dev)
    x[4:-4] = 0
    norm = _norm(C, dev=dev)
    y, st = kernels.layer_norm(x, norm, statistics=True)
    check_forward(y[-4:].clone(), x[-4:], norm)
    check_forward(y[:4].clone(), x[:4], norm)
    dy = y.zero_()
    dy[-4:] = _rand((4, C), BF16, 3).to(dev)
    g = kernels.layer_norm_backward(dy, x, norm, st)
    check_backward((g.dx[-4:], g.dweight, g.dbias), dy[-4:].clone(), x[-4:], norm)


def test_odd_rows_past_32_bits_of_elements(dev):
    rows, C = 2_200_001, 999
    x = torch.empty(rows, C, dtype=BF16, device=dev)
    x[:4], x[-4:] = _x((4, C), BF16).to(dev), _x((4, C), BF16, 2).to(dev)
    x[4:-4] = 0
    norm = _norm(C, dev=dev)
    y, st = kernels.layer_norm(x, norm, statistics=True)
    check_forward(y[-4:].clone(), x[-4:], norm)
    check_forward(y[:4].clone(), x[:4], norm)
    dy = y.zero_()
    dy[-4:] = _rand((4, C), BF16, 3).to(dev)
    g = kernels.layer_norm_backward(dy, x, norm, st)
    check_backward((g.dx[-4:], g.dweight, g.dbias), dy[-4:].clone(), x[-4:], norm)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("C", [33, 65, 99, 385, 1030, 2049, 5001, 9001])
def test_nan_of_neighbours_that_share_a_chunk(dev, C, dt):
    """Every other row is NaN: the rows between them are as they are by themselves, bit by bit."""
    x, norm, dy = _x((40, C), dt).to(dev), _norm(C, dev=dev), _rand((40, C), dt, 3).to(dev)
    y, st = kernels.layer_norm(x, norm, statistics=True)
    dx = kernels.layer_norm_backward(dy, x, norm, st).dx
    x[1::2], dy[::2] = float("nan"), float("nan")
    z, _ = kernels.layer_norm(x, norm, statistics=True)
    assert torch.equal(z[::2], y[::2]) and bool(z[1::2].isnan().all())
    x = _x((40, C), dt).to(dev)
    again = kernels.layer_norm_backward(dy, x, norm, st).dx
    assert torch.equal(again[1::2], dx[1::2]) and bool(again[::2].isnan().all())


class TestAutograd:
    def test_gradients(self, dev):
        x = _x((5, 7, 96), F32).to(dev).requires_grad_()
        norm = Norm(*(t.requires_grad_() for t in (_norm(96, dev=dev).weight, _norm(96, dev=dev).bias)))
        y = autograd.layer_norm(x, norm)
        dy = _rand((5, 7, 96), F32, 3).to(dev)
        grads = torch.autograd.grad(y, (x, norm.weight, norm.bias), dy)
        check_backward(grads, dy, x, norm)

    def test_gradients_against_differences(self, dev):
        """Along a direction d, in fp32: the quotient of differences h = 2^-6 apart has the curvature's error, of order h^2
        (1e-3 of what moves), and that of fp32 sums of 2000 terms divided by h (2000 u / h = 8e-3 of their mean magnitude)."""
        for rms in (False, True):
            x, d = _rand((20, 100), F32, 1).to(dev), _rand((20, 100), F32, 2).to(dev)
            norm, dy, h = _norm(100, rms=rms, dev=dev), _rand((20, 100), F32, 3).to(dev), 2.0 ** -6
            f = lambda t: (kernels.layer_norm(t, norm).double() * dy.double()).sum().item()  # noqa: E731
            _, st = kernels.layer_norm(x, norm, statistics=True)
            along = (kernels.layer_norm_backward(dy, x, norm, st).dx.double() * d.double()).sum().item()
            scale = (kernels.layer_norm(x, norm).abs() * dy.abs()).sum().item()
            assert abs((f(x + h * d) - f(x - h * d)) / (2 * h) - along) <= 1e-3 * scale

    @pytest.mark.parametrize("needs", [(True, False, False), (False, True, False), (False, False, True), (False, True, True)])
    def test_only_what_is_asked(self, dev, needs):
        x, norm, dy = _x((9, 64), BF16).to(dev), _norm(64, dev=dev), _rand((9, 64), BF16, 3).to(dev)
        leaves = (x, norm.weight, norm.bias)
        for t, need in zip(leaves, needs):
            t.requires_grad_(need)
        autograd.layer_norm(x, norm).backward(dy)
        check_backward([t.grad for t in leaves], dy, x, norm)
        assert [t.grad is not None for t in leaves] == list(needs)

    def test_a_gradient_of_other_strides(self, dev):
        x = _x((6, 64), F32).to(dev).requires_grad_()
        autograd.layer_norm(x, Norm()).sum().backward()  # an expanded gradient
        check_backward((x.grad,), torch.ones(6, 64), x, Norm())

    def test_heads_of_a_packed_row(self, dev):
        qkv = _x((5, 4, 9, 32), BF16).to(dev).requires_grad_()
        dy = _rand((5, 4, 6, 32), BF16, 3).to(dev)
        autograd.layer_norm(qkv[:, :, :6], Norm(rms=True)).backward(dy)
        check_backward((qkv.grad[:, :, :6],), dy, qkv[:, :, :6], Norm(rms=True))
        assert not qkv.grad[:, :, 6:].any()

    def test_rows_of_many_strides_are_copied(self, dev):
        big = _x((4, 6, 5, 16), F32).to(dev)
        x = big[:, :4, :3]
        with pytest.raises(ValueError, match="at most two strides"):
            kernels.layer_norm(x, Norm())
        check_forward(autograd.layer_norm(x, Norm()), x, Norm())
        t = big.transpose(2, 3)
        with pytest.raises(ValueError, match="unit channel stride"):
            kernels.layer_norm(t, Norm())
        check_forward(autograd.layer_norm(t, Norm()), t, Norm())

    @pytest.mark.parametrize("rms", [False, True])
    def test_second_derivatives(self, dev, rms):
        """Of a pass in fp32 operations of torch: each of the some ten operations between the leaves and the second
        derivative is off by C / 8 + 24 roundings of its largest terms."""
        x, norm = _rand((4, 32), F32, 1).to(dev).requires_grad_(), _norm(32, rms=rms, dev=dev)
        norm = Norm(norm.weight.requires_grad_(), norm.bias.requires_grad_(), norm.eps, rms)
        leaves = (x, norm.weight, norm.bias)
        y = autograd.layer_norm(x, norm)
        g = torch.autograd.grad(y.pow(3).sum(), leaves, create_graph=True)
        h = torch.autograd.grad(sum(t.square().sum() for t in g), leaves)
        ref = [t.detach().cpu().double().requires_grad_() for t in leaves]
        yr = tr.layer_norm(ref[0], ref[1], ref[2], norm.eps, rms)[0]
        gr = torch.autograd.grad(yr.pow(3).sum(), ref, create_graph=True)
        hr = torch.autograd.grad(sum(t.square().sum() for t in gr), ref)
        for a, b in zip(g, gr):
            check = (a.detach().cpu().double() - b.detach()).abs().max()
            assert check <= 10 * 28 * U * max(t.abs().max() for t in gr).detach()
        for a, b in zip(h, hr):
            assert (a.cpu().double() - b).abs().max() <= 20 * 28 * U * max(t.abs().max() for t in hr)

    def test_forward_mode_is_refused(self, dev):
        x = _x((4, 32), F32).to(dev)
        with torch.autograd.forward_ad.dual_level():
            d = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                autograd.layer_norm(d, Norm())

    def test_a_changed_input_is_noticed(self, dev):
        x = _x((4, 32), F32).to(dev).requires_grad_()
        h = x * 1.0
        y = autograd.layer_norm(h, Norm())
        h.add_(1.0)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()
        a = torch.ones(4, 32, device=dev, requires_grad=True)
        b = a * 1.0
        z = b * b
        kernels.layer_norm(x.detach(), Norm(), out=b.detach())
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            z.sum().backward()

    def test_saved_tensors_packed_by_a_hook(self, dev):
        big = _x((6, 3, 64), F32).to(dev).requires_grad_()
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.to(dev)):
            y = autograd.layer_norm(big[:, 1], Norm())
        dy = _rand((6, 64), F32, 3).to(dev)
        y.backward(dy)
        check_backward((big.grad[:, 1],), dy, big[:, 1], Norm())

    def test_an_exception_of_a_hook_passes(self, dev):
        def full(t):
            raise KeyError("full")

        x = _x((6, 64), F32).to(dev).requires_grad_()
        with torch.autograd.graph.saved_tensors_hooks(full, lambda t: t):
            with pytest.raises(KeyError, match="full"):
                autograd.layer_norm(x, Norm())

    @pytest.mark.parametrize("reentrant", [False, True])
    def test_checkpointed(self, dev, reentrant):
        from torch.utils.checkpoint import checkpoint

        x, norm, dy = _x((6, 64), F32).to(dev).requires_grad_(), _norm(64, dev=dev), _rand((6, 64), F32, 3).to(dev)
        checkpoint(lambda t: autograd.layer_norm(t, norm), x, use_reentrant=reentrant).backward(dy)
        check_backward((x.grad,), dy, x, norm)

    def test_twice_over_a_retained_graph(self, dev):
        x = _x((4, 64), F32).to(dev).requires_grad_()
        y = autograd.layer_norm(x, Norm())
        a, = torch.autograd.grad(y, x, torch.ones_like(y), retain_graph=True)
        b, = torch.autograd.grad(y, x, torch.ones_like(y))
        assert torch.equal(a, b)

    def test_inference_mode(self, dev):
        with torch.inference_mode():
            x = _x((4, 64), BF16).to(dev)
            check_forward(autograd.layer_norm(x, Norm()).clone(), x, Norm())


def test_on_another_stream(dev):
    x, norm = _x((300, 768), BF16).to(dev), _norm(768, dev=dev)
    ref = kernels.layer_norm(x, norm)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        y = kernels.layer_norm(x, norm)
    s.synchronize()
    assert torch.equal(y, ref)


@pytest.mark.parametrize("C", [96, 1024, 9000])
def test_captured(dev, C):
    x, norm, dy = _x((40, C), BF16).to(dev), _norm(C, dev=dev), _rand((40, C), BF16, 3).to(dev)

    def work():
        y, st = kernels.layer_norm(x, norm, statistics=True)
        return y, *kernels.layer_norm_backward(dy, x, norm, st)

    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        work()
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    for seed in range(4):
        x.copy_(_x((40, C), BF16, seed))
        graph.replay()
        eager = work()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager))


def test_refusals(dev):
    x = torch.zeros(4, 32, device=dev)
    for bad, error, text in (
        (lambda: kernels.layer_norm(x, Norm(torch.zeros(31, device=dev))), ValueError, "32 channels"),
        (lambda: kernels.layer_norm(x, Norm(torch.zeros(32))), RuntimeError, "ROCm devices only"),
        (lambda: kernels.layer_norm(x, Norm(torch.zeros(32, device=dev, dtype=torch.float64))), TypeError, "not supported"),
        (lambda: kernels.layer_norm(x.double(), Norm()), TypeError, "not supported"),
        (lambda: kernels.layer_norm(x.half(), Norm(), BF16), TypeError, "out_dtype"),
        (lambda: kernels.layer_norm(x, Norm(), torch.float64), TypeError, "out_dtype"),
        (lambda: kernels.layer_norm(x[0, 0], Norm()), ValueError, "C >= 1"),
        (lambda: kernels.layer_norm(x[:, :0], Norm()), ValueError, "C >= 1"),
        (lambda: kernels.layer_norm(x, Norm(eps=-1.0)), ValueError, "eps"),
        (lambda: kernels.layer_norm(x, Norm(), out=x), ValueError, "overlap"),
        (lambda: kernels.layer_norm(x, Norm(), out=torch.zeros(4, 31, device=dev)), ValueError, "out must be"),
        (lambda: kernels.layer_norm_backward(x[:3], x, Norm(), torch.zeros(4, 2, device=dev)), ValueError, "dy must be"),
        (lambda: kernels.layer_norm_backward(x, x, Norm(), torch.zeros(3, 2, device=dev)), ValueError, "statistics"),
    ):
        with pytest.raises(error, match=text):
            bad()
