"""Dropout and GELU + dropout kernels (terra_swin_dropout,
terra_swin_gelu_dropout and its backward) against the 64-bit oracle.

Tolerances.  A kept element of dropout is one fp32 product rounded once more to
the type: |y - ref| <= (eps_t / 2 + 2 eps_32) |ref| (the product's and the
scale's own rounding), plus half the type's smallest subnormal.  GELU and its
slope go through erfc and exp of fp32 (a few ulp each, taken as 16 eps_32 of
the terms): |a - ref| <= eps_t / 2 |ref| + 16 eps_32 |h|, |dh - ref| <=
eps_t / 2 |ref| + 16 eps_32 |da| (1 + |h|) s.  Column sums of n rows add the
terms' errors and at most n eps_32 / 8 of the sum of their magnitudes (rows are
dealt to at least eight adders): (16 + n / 8) eps_32 sum |terms|.  Masks are
equal element for element.
"""
import pytest
import torch

from oracle import regularize as rg
from terra_amd import autograd, kernels

pytestmark = pytest.mark.gpu

E32 = torch.finfo(torch.float32).eps
TYPES = [torch.float32, torch.bfloat16, torch.float16]
SEED = 0x1234567890ABCDE


def _half(dt):
    return torch.finfo(dt).eps / 2 if dt != torch.float32 else 0.0


def _tiny(dt):
    return torch.finfo(dt).smallest_normal * torch.finfo(dt).eps


def _rand(shape, dt, seed, scale=1.5):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dt)


def _seed(dev, value=SEED):
    return torch.tensor([value], dtype=torch.int64, device=dev)


def _check_dropout(y, x, p, seed, stream):
    ref = rg.dropout(x.double(), p, seed, stream)
    y = y.double().cpu()
    tol = (_half(x.dtype) + 2 * E32) * ref.abs() + _tiny(x.dtype)
    assert bool(((y - ref).abs() <= tol).all())
    keep = rg.keep_mask(seed, x.numel() // x.shape[-1], x.shape[-1], p, stream).view(x.shape)
    assert bool((y[~keep] == 0).all())


SHAPES = [(1, 1), (1, 7), (1, 8), (3, 9), (2, 1, 16), (5, 96), (67, 100), (1030, 24), (33, 1001), (9, 2048), (5, 2050),
          (3, 5, 4104), (20011,)]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_dropout_against_oracle(dev, dt, shape):
    x = _rand(shape, dt, 1)
    y = kernels.dropout(x.to(dev), 0.3, _seed(dev), stream=5)
    assert y.shape == x.shape and y.dtype == dt
    _check_dropout(y, x, 0.3, SEED, 5)


@pytest.mark.parametrize("p", [0.0, 2.0 ** -18, 0.5, 0.9999, 1.0])
def test_dropout_probabilities_and_seeds(dev, p):
    x = _rand((64, 72), torch.bfloat16, 2)
    for seed in (0, -1, -(1 << 63), (1 << 63) - 1):
        _check_dropout(kernels.dropout(x.to(dev), p, _seed(dev, seed), 0xFFFFFFFF), x, p, seed, 0xFFFFFFFF)
    if p == 0.0:
        assert torch.equal(kernels.dropout(x.to(dev), 0.0, None).cpu(), x)


@pytest.mark.parametrize("dt", TYPES)
def test_dropout_of_infinities_and_nan(dev, dt):
    x = _rand((32, 40), dt, 3)
    x[::3, ::7] = float("nan")
    x[1::3, ::5] = float("inf")
    x[2::3, ::5] = torch.finfo(dt).min
    y = kernels.dropout(x.to(dev), 0.5, _seed(dev)).cpu()
    keep = rg.keep_mask(SEED, 32, 40, 0.5)
    assert bool((y[~keep] == 0).all())
    want = (x.float() * rg.keep_scale(0.5)).to(dt)
    assert torch.equal(torch.nan_to_num(y[keep], 7.0), torch.nan_to_num(want[keep], 7.0))


@pytest.mark.parametrize("dt", TYPES)
def test_dropout_strides_and_alignment(dev, dt):
    x = _rand((50, 3 * 64), dt, 4)
    for lo, hi in ((0, 64), (64, 128), (3, 67), (5, 6)):  # column blocks, some off the 16-byte grid
        _check_dropout(kernels.dropout(x.to(dev)[:, lo:hi], 0.25, _seed(dev)), x[:, lo:hi].contiguous(), 0.25, SEED, 0)
    flat = _rand((50 * 64 + 1,), dt, 5)
    _check_dropout(kernels.dropout(flat.to(dev)[1:].view(50, 64), 0.25, _seed(dev)), flat[1:].view(50, 64), 0.25, SEED, 0)


def test_dropout_in_place_and_out(dev):
    x = _rand((300, 96), torch.bfloat16, 6)
    want = kernels.dropout(x.to(dev), 0.4, _seed(dev))
    y = x.to(dev)
    assert kernels.dropout(y, 0.4, _seed(dev), out=y) is y and torch.equal(y, want)
    with pytest.raises(ValueError, match="overlap"):
        kernels.dropout(y.view(-1)[96:].view(-1, 96), 0.4, _seed(dev), out=y.view(-1)[:-96].view(-1, 96))


def test_dropout_large_rows_and_offsets(dev):
    """Rows whose bytes end past 2^32: the last ones against the oracle."""
    rows, C = (1 << 32) // (2 * 2048) + 5, 2048
    x = torch.ones(rows, C, dtype=torch.bfloat16, device=dev)
    y = kernels.dropout(x, 0.5, _seed(dev), 1)
    for first in (0, (1 << 31) // (2 * C) - 1, rows - 6):
        keep = rg.keep_mask(SEED, 6, C, 0.5, 1, first_row=first)
        assert torch.equal(y[first:first + 6].cpu() != 0, keep)
    del x, y
    torch.cuda.empty_cache()


def test_one_long_row(dev):
    """A flat tensor of 2^25 + 3 elements: one row of many strips of columns."""
    n = (1 << 25) + 3
    y = kernels.dropout(torch.ones(n, dtype=torch.float16, device=dev), 0.5, _seed(dev), 1)
    assert torch.equal(y.cpu() != 0, rg.keep_mask(SEED, 1, n, 0.5, 1)[0])
    h, da = torch.ones(n, device=dev), torch.ones(n, device=dev)
    dh, sums = kernels.gelu_dropout_backward(da, h, 0.5, _seed(dev), 1, column_sums=True)
    assert torch.equal(dh, sums) and torch.equal(dh != 0, y != 0)


def test_dropout_empty(dev):
    for shape in ((0, 8), (3, 0), (0,)):
        assert kernels.dropout(torch.empty(shape, device=dev), 0.5, _seed(dev)).shape == shape
    dh, db = kernels.gelu_dropout_backward(torch.empty(0, 8, device=dev), torch.empty(0, 8, device=dev), 0.5, _seed(dev),
                                           column_sums=True)
    assert dh.shape == (0, 8) and torch.equal(db.cpu(), torch.zeros(8))


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("shape", [(1, 1), (1, 8), (3, 9), (67, 100), (2, 515, 24), (33, 1001), (9, 2048), (5, 2050),
                                   (1, 4104), (20011, 16)])
@pytest.mark.parametrize("p", [0.0, 0.3])
def test_gelu_dropout_against_oracle(dev, dt, shape, p):
    h, da = _rand(shape, dt, 7, 2.0), _rand(shape, dt, 8)
    h.view(-1)[:1] = -20.0
    ref_h = h.double().requires_grad_()
    ref = rg.dropout(rg.gelu(ref_h), p, SEED, 2)
    ref_dh, = torch.autograd.grad(ref, ref_h, da.double())
    ref, s = ref.detach(), rg.keep_scale(p)
    a = kernels.gelu_dropout(h.to(dev), p, _seed(dev), 2).double().cpu()
    hd, dad = h.double().abs(), da.double().abs()
    assert bool(((a - ref).abs() <= _half(dt) * ref.abs() + 16 * E32 * hd * s + _tiny(dt)).all())
    dh, db = kernels.gelu_dropout_backward(da.to(dev), h.to(dev), p, _seed(dev), 2, column_sums=True)
    terms = dad * (1 + hd) * s
    assert bool(((dh.double().cpu() - ref_dh).abs() <= _half(dt) * ref_dh.abs() + 16 * E32 * terms + _tiny(dt)).all())
    rows = h.numel() // shape[-1]
    tol = (16 + rows / 8) * E32 * terms.view(rows, -1).sum(0)
    assert bool(((db.double().cpu() - ref_dh.view(rows, -1).sum(0)).abs() <= tol).all())
    assert torch.equal(kernels.gelu_dropout_backward(da.to(dev), h.to(dev), p, _seed(dev), 2), dh)
    keep = rg.keep_mask(SEED, rows, shape[-1], p, 2).view(shape)
    assert bool((a[~keep] == 0).all()) and bool((dh.cpu()[~keep] == 0).all())


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_gelu_dropout_of_every_value(dev, dt):
    """All 2^16 values of a 16-bit type, without and with dropout: NaN and the
    infinities as the formulas give them (GELU(-inf) = -inf * 0 is NaN)."""
    h = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(dt).view(256, 256)
    one = torch.ones_like(h)
    a = kernels.gelu_dropout(h.to(dev), 0.0, None).cpu()
    dh = kernels.gelu_dropout_backward(one.to(dev), h.to(dev), 0.0, None).cpu()
    hd = h.double()
    ref = rg.gelu(hd)
    slope = 0.5 * torch.erfc(-hd / 2 ** 0.5) + hd * torch.exp(-0.5 * hd * hd) / (2 * torch.pi) ** 0.5
    fine = torch.isfinite(hd)
    for got, want, tol in ((a, ref, 16 * E32 * hd.abs()), (dh, slope, 16 * E32 * (1 + hd.abs().clamp(max=20)))):
        got = got.double()
        assert bool(((got - want).abs() <= _half(dt) * want.abs() + tol + _tiny(dt))[fine].all())
    assert bool(torch.isnan(a[torch.isnan(hd)]).all()) and bool(torch.isnan(dh[torch.isnan(hd)]).all())
    assert a[hd == float("inf")].item() == float("inf") and bool(torch.isnan(a[hd == -float("inf")]).all())
    keep = rg.keep_mask(SEED, 256, 256, 0.5)
    a = kernels.gelu_dropout(h.to(dev), 0.5, _seed(dev)).cpu()
    assert bool((a[~keep] == 0).all())


def test_gelu_dropout_backward_in_place_and_repeatable(dev):
    h, da = _rand((4099, 136), torch.bfloat16, 9).to(dev), _rand((4099, 136), torch.bfloat16, 10).to(dev)
    want, db = kernels.gelu_dropout_backward(da, h, 0.2, _seed(dev), column_sums=True)
    for _ in range(3):  # the same order of additions each time
        dh, db2 = kernels.gelu_dropout_backward(da, h, 0.2, _seed(dev), column_sums=True)
        assert torch.equal(dh, want) and torch.equal(db, db2)
    buf = da.clone()
    dh, db2 = kernels.gelu_dropout_backward(buf, h, 0.2, _seed(dev), column_sums=True, out=buf)
    assert dh is buf and torch.equal(dh, want) and torch.equal(db, db2)


def test_seed_draws(dev):
    torch.manual_seed(5)
    a, b = kernels.dropout_seed(dev), kernels.dropout_seed(dev)
    torch.manual_seed(5)
    assert torch.equal(a, kernels.dropout_seed(dev)) and not torch.equal(a, b)
    x = torch.ones(64, 64, device=dev, requires_grad=True)
    torch.manual_seed(6)
    y = autograd.dropout(x, 0.5)
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    assert torch.equal(dx, y.detach())  # the backward's mask is the forward's
    torch.manual_seed(6)
    assert torch.equal(autograd.dropout(x, 0.5), y) and not torch.equal(autograd.dropout(x, 0.5), y)


def test_autograd_functions(dev):
    h = _rand((40, 72), torch.bfloat16, 11).to(dev).requires_grad_()
    da = _rand((40, 72), torch.bfloat16, 12).to(dev)
    link = autograd.ColumnSumLink()
    a = autograd.gelu_dropout(h, 0.3, _seed(dev), 4, bias_sums=link)
    dh, = torch.autograd.grad(a, h, da)
    want, sums = kernels.gelu_dropout_backward(da, h.detach(), 0.3, _seed(dev), 4, column_sums=True)
    assert torch.equal(dh, want) and torch.equal(link.sums, sums)
    # an expanded gradient, as a sum's backward gives it
    y = autograd.dropout(h, 0.3, _seed(dev))
    dh, = torch.autograd.grad(y.sum(), h)
    assert torch.equal(dh, kernels.dropout(torch.ones_like(h), 0.3, _seed(dev)))
    # the mask's seed must not change between forward and backward
    s = _seed(dev)
    y = autograd.dropout(h, 0.3, s)
    s.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y.sum(), h)


def test_dropout_on_another_stream_and_in_graphs(dev):
    x = _rand((513, 96), torch.bfloat16, 13).to(dev)
    seeds = [_seed(dev, v) for v in (1, 2, 3)]
    want = [kernels.dropout(x, 0.3, s) for s in seeds]
    da = torch.ones_like(x)
    want_b = [kernels.gelu_dropout_backward(da, x, 0.3, s, column_sums=True) for s in seeds]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = kernels.dropout(x, 0.3, seeds[0])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, want[0])
    state = seeds[0].clone()
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    outs = []
    for g in graphs:
        with torch.cuda.graph(g):
            outs.append((kernels.dropout(x, 0.3, state), *kernels.gelu_dropout_backward(da, x, 0.3, state, column_sums=True)))
    for i in (1, 2, 0, 1):  # a replay takes the seed that is there; eager work in between
        state.copy_(seeds[i])
        for g, (y, dh, db) in zip(graphs, outs):
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, want[i]) and torch.equal(dh, want_b[i][0]) and torch.equal(db, want_b[i][1])
            assert torch.equal(kernels.dropout(x, 0.3, seeds[i]), want[i])


def test_drawn_seeds_in_a_graph_differ_from_replay_to_replay(dev):
    x = torch.ones(64, 512, device=dev)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = kernels.dropout(x, 0.5, kernels.dropout_seed(dev))
    got = []
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        got.append(y.clone())
    assert not torch.equal(got[0], got[1]) and not torch.equal(got[1], got[2])


def test_columns_to_the_limit(dev):
    """A row of more columns than one grid of the column sums' launch has workgroups for (2^25 at a time, 2^26 and a few
    here), sums of no rows, and a row of the most columns there may be."""
    n = (1 << 26) + 5
    da, h = torch.randn(1, n, device=dev, generator=torch.Generator(dev).manual_seed(1)), torch.ones(1, n, device=dev)
    dh, sums = kernels.gelu_dropout_backward(da, h, 0.0, None, column_sums=True)
    assert torch.equal(dh[0], sums)  # one row: its own sum
    slope = 0.5 * (1 + torch.erf(torch.tensor(0.5, dtype=torch.float64).sqrt())) + torch.exp(
        torch.tensor(-0.5, dtype=torch.float64)) / (2 * torch.pi) ** 0.5
    assert bool(((sums.double() - da[0].double() * slope).abs() <= 16 * E32 * 2 * da[0].double().abs()).all())
    del da, h, dh, sums
    empty = torch.empty(0, n, device=dev)
    sums = kernels.gelu_dropout_backward(empty, empty, 0.0, None, column_sums=True)[1]
    assert not bool(sums.any())
    del sums, empty
    n = (1 << 27) - 1
    y = kernels.dropout(torch.ones(1, n, dtype=torch.bfloat16, device=dev), 0.5, _seed(dev), 1)
    first = (n // 8) - 100  # the last chunks' draws
    words = rg.philox4x32_10((torch.arange(first, n // 8 + 1).numpy().astype("uint64"), 0, 0, 1),
                             (SEED & 0xFFFFFFFF, SEED >> 32))
    draws = torch.stack([torch.from_numpy((w >> (16 * k) & 0xFFFF).astype("int64")) for w in map(lambda w: w.astype("int64"), words)
                         for k in (0, 1)], -1).view(-1)
    assert torch.equal(y[0, 8 * first:].cpu() != 0, (draws >= rg.threshold(0.5))[:n - 8 * first])
    del y
    torch.cuda.empty_cache()


def _every_value(rows):
    """[rows, 256] bf16 rows that go through all 2^16 values again and again: 0, values below 2^-12 and from 16 on,
    infinities and NaN among them."""
    at = torch.arange(256 * rows, dtype=torch.int32) * 40503  # odd: neighbouring lanes see values far apart
    return (at & 0xFFFF).to(torch.int16).view(torch.bfloat16).view(rows, 256)


@pytest.mark.parametrize("rows,p", [(1 << 14, 0.0), (1 << 14, 0.3), ((1 << 14) + 19, 0.3)])
def test_gelu_dropout_of_many_bf16_values(dev, rows, p):
    """From 2^22 aligned bf16 elements on the factors come from a table: against the oracle, and against the calls of
    fewer rows, which compute them (two roundings to the type from values 32 eps_32 apart: one step of the type)."""
    h = _every_value(rows)
    seed = _seed(dev) if p else None
    a = kernels.gelu_dropout(h.to(dev), p, seed, 2).cpu()
    hd, s = h.double(), rg.keep_scale(p)
    ref = rg.dropout(rg.gelu(hd), p, SEED, 2)
    fine = torch.isfinite(hd)
    tol = _half(torch.bfloat16) * ref.abs() + 16 * E32 * hd.abs() * s + _tiny(torch.bfloat16)
    top = torch.finfo(torch.bfloat16).max
    near = ((a.double() - ref).abs() <= tol) | ((ref.abs() > top * (1 - _half(torch.bfloat16))) & torch.isinf(a))
    assert bool(near[fine].all())
    keep = rg.keep_mask(SEED, rows, 256, p, 2)
    assert bool((a[~keep] == 0).all())
    assert bool(torch.isnan(a[keep & torch.isnan(hd)]).all())
    assert bool((a[keep & (hd == float("inf"))] == float("inf")).all())
    assert bool(torch.isnan(a[keep & (hd == -float("inf"))]).all())
    few = kernels.gelu_dropout(h[:4099].to(dev), p, seed, 2).cpu()
    big = a[:4099]
    assert torch.equal(torch.isnan(few), torch.isnan(big)) and torch.equal(torch.isinf(few), torch.isinf(big))
    both = torch.isfinite(few)
    step = torch.finfo(torch.bfloat16).eps * torch.maximum(few.abs(), big.abs()).float() + 2 * _tiny(torch.bfloat16)
    wide = 32 * E32 * hd[:4099].abs().nan_to_num() * s  # a dropped NaN is 0 in both
    assert bool(((few.float() - big.float()).abs() <= step + wide)[both].all())
    dst = h.to(dev)
    assert torch.equal(kernels.gelu_dropout(dst, p, seed, 2, out=dst).view(torch.int16).cpu(), a.view(torch.int16))


def test_gelu_tail_in_fp32(dev):
    """The negative tail keeps its relative precision but for the exponent's: exp(-h^2 / 2) is taken from a product
    rounded twice (half an eps of h^2 / 2 each) with a constant rounded once (another half), 0.75 eps h^2 in all; the
    polynomial, its seven steps, the reciprocal and exp2 (one ulp each) and the last products add 8 eps.  The
    slope at h <= -2 takes both terms' errors, at most (1 + h^2) / (h^2 - 1) <= 5 / 3 of it."""
    h = torch.linspace(-12.5, -0.001, 200_003)
    a = kernels.gelu_dropout(h.to(dev).view(1, -1), 0.0, None)[0].double().cpu()
    hd = h.double()
    ref = rg.gelu(hd)
    tol = E32 * (8 + 0.75 * hd * hd)
    assert bool(((a - ref).abs() <= tol * ref.abs()).all())
    far = h <= -2
    h, hd, tol = h[far], hd[far], tol[far] * 5 / 3
    dh = kernels.gelu_dropout_backward(torch.ones(1, len(h), device=dev), h.to(dev).view(1, -1), 0.0, None)[0].double().cpu()
    slope = 0.5 * torch.erfc(-hd / 2 ** 0.5) + hd * torch.exp(-0.5 * hd * hd) / (2 * torch.pi) ** 0.5
    assert bool(((dh - slope).abs() <= tol * slope.abs()).all())
