"""Argument checks of the training step's operators (on the CPU, no kernel
runs): the C entry points and the tensor-level wrappers."""
import ctypes

import pytest
import torch

import terra_amd._lib as L
from terra_amd import autograd, kernels
from terra_amd.kernels import Norm, Rotary

A = 1 << 24


def at(i, off=0):
    return ctypes.c_void_p(A * (i + 1) * 64 + off)


def test_descriptors_mirror_the_header():
    assert ctypes.sizeof(L.LayerNormDesc) == 4 * 8 + 6 * 4
    assert ctypes.sizeof(L.RotaryDesc) == 9 * 8 + 9 * 4 + 4
    assert ctypes.sizeof(L.TensorList) == 24
    assert ctypes.sizeof(L.AdamWTensor) == 6 * 8 + 3 * 4 + 4
    assert ctypes.sizeof(L.AdamWDesc) == 11 * 8 + 2 * 4


def _set(d, vals, kw):
    for k, v in {**vals, **kw}.items():
        setattr(d, k, v)
    return d


# ---- norms over rows -------------------------------------------------------------

BF16, F32, F16 = L.DTYPE_BF16, L.DTYPE_F32, L.DTYPE_F16


def _norm(**kw):
    return _set(L.LayerNormDesc(), dict(rows=8, inner=8, outer_stride=0, inner_stride=64, channels=64, x_dtype=BF16,
                                        y_dtype=BF16, param_dtype=F32, norm=1, eps=1e-5), kw)


def _norm_fwd(d, x=at(0), y=at(1), w=at(2), b=at(3), st=at(4)):
    return L.load().terra_swin_layer_norm(x, y, None if d is None else ctypes.byref(d), w, b, st, None)


NORM_DESCS = [
    (dict(x_dtype=L.DTYPE_U8), -2, "f32, bf16 or f16"),
    (dict(y_dtype=F16), -2, "f32, bf16 or f16"),
    (dict(param_dtype=7), -2, "f32, bf16 or f16"),
    (dict(rows=-1), -3, "rows must be"),
    (dict(rows=1 << 31), -3, "at most"),
    (dict(channels=0), -3, "channels > 0"),
    (dict(channels=(1 << 24) + 1), -5, "channels"),
    (dict(norm=0), -3, "unknown norm"),
    (dict(norm=3), -3, "unknown norm"),
    (dict(inner=0), -3, "inner"),
    (dict(inner=1 << 31), -3, "inner"),
    (dict(inner_stride=-1), -3, "strides"),
    (dict(outer_stride=1 << 40), -3, "strides"),
    (dict(eps=-1.0), -3, "eps"),
    (dict(eps=float("nan")), -3, "eps"),
]


@pytest.mark.parametrize("kw,code,text", NORM_DESCS)
def test_layer_norm_refuses_descriptors(kw, code, text):
    d = _norm(**kw)
    assert _norm_fwd(d) == code and text in L.last_error()
    assert L.load().terra_swin_layer_norm_workspace(ctypes.byref(d)) == code
    assert _norm_bwd(d) == code and text in L.last_error()


@pytest.mark.parametrize("kw,code,text", [
    (dict(d=None), -1, "desc"),
    (dict(x=None), -1, "x is NULL"),
    (dict(y=None), -1, "y is NULL"),
    (dict(x=at(0, 1)), -4, "x is not aligned"),
    (dict(y=at(1, 1)), -4, "y is not aligned"),
    (dict(w=at(2, 2)), -4, "weight"),
    (dict(b=at(3, 1)), -4, "bias"),
    (dict(st=at(4, 4)), -4, "statistics"),
    (dict(y=at(0)), -3, "overlap"),
    (dict(y=at(0, 1022)), -3, "overlap"),
    (dict(st=at(0, 8)), -3, "statistics"),
    (dict(st=at(1, 8)), -3, "statistics"),
])
def test_layer_norm_refuses_pointers(kw, code, text):
    kw = dict(kw)
    assert _norm_fwd(kw.pop("d", _norm()), **kw) == code, L.last_error()
    assert text in L.last_error()


def _norm_bwd(d, dy=at(0), x=at(1), st=at(2), dx=at(3), w=at(4), dw=at(5), db=at(6), work=at(7)):
    return L.load().terra_swin_layer_norm_bwd(dy, x, st, dx, ctypes.byref(d), w, dw, db, work, None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(dy=None), -1, "dy is NULL"),
    (dict(x=None), -1, "x is NULL"),
    (dict(st=None), -1, "statistics"),
    (dict(work=None), -1, "workspace"),
    (dict(dy=at(0, 1)), -4, "dy is not aligned"),
    (dict(dx=at(3, 1)), -4, "dx is not aligned"),
    (dict(dw=at(5, 2)), -4, "dweight"),
    (dict(db=at(6, 2)), -4, "dbias"),
    (dict(work=at(7, 2)), -4, "workspace"),
    (dict(st=at(2, 4)), -4, "statistics"),
    (dict(dx=at(0)), -3, "overlap"),
    (dict(dx=at(1)), -3, "overlap"),
    (dict(dx=at(2)), -3, "overlap"),
])
def test_layer_norm_backward_refuses(kw, code, text):
    assert _norm_bwd(_norm(), **kw) == code, L.last_error()
    assert text in L.last_error()


def test_layer_norm_of_no_rows_needs_nothing():
    assert _norm_fwd(_norm(rows=0), None, None, None, None, None) == 0
    assert _norm_bwd(_norm(rows=0), None, None, None, None, None, None, None, None) == 0
    assert _norm_bwd(_norm(), None, None, None, None, None, None, None, None) == 0  # no gradient is asked for
    assert L.load().terra_swin_layer_norm_workspace(ctypes.byref(_norm(rows=0))) == 0


def test_layer_norm_workspace_covers_the_sizes():
    for rows in (1, 3, 100, 5000, 1 << 20, (1 << 31) - 1):
        for C in (1, 64, 190, 192, 1000, 4096, 8192, 20000, 1 << 24):
            for x, y in ((BF16, BF16), (F32, F32), (F32, BF16), (F16, F32)):
                n = L.load().terra_swin_layer_norm_workspace(ctypes.byref(_norm(rows=rows, channels=C, x_dtype=x, y_dtype=y)))
                assert 2 * C <= n <= 1 << 27, (rows, C, n)


# ---- rotary positions ------------------------------------------------------------


def _rot(**kw):
    return _set(L.RotaryDesc(), dict(tokens=6, inner=6, position_tokens=3, x_outer_stride=0, x_inner_stride=256,
                                     x_head_stride=64, y_outer_stride=0, y_inner_stride=256, y_head_stride=64, heads=4,
                                     head_dim=64, dim=32, axes=1, dtype=BF16, position_bits=64, interleaved=0, inverse=0,
                                     amplitude=1.0), kw)


def _rotary(d, x=at(0), y=at(1), pos=at(2), turns=at(3)):
    return L.load().terra_swin_rotary(x, y, pos, turns, None if d is None else ctypes.byref(d), None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(dtype=L.DTYPE_U8), -2, "rotary supports"),
    (dict(position_bits=16), -2, "32 or 64"),
    (dict(tokens=-1), -3, "tokens"),
    (dict(tokens=1 << 31), -3, "tokens"),
    (dict(heads=0), -3, "heads"),
    (dict(heads=65536), -3, "heads"),
    (dict(head_dim=0), -3, "heads"),
    (dict(dim=0), -3, "even"),
    (dict(dim=33), -3, "even"),
    (dict(dim=66), -3, "even"),
    (dict(axes=0), -3, "axes"),
    (dict(axes=3), -3, "axes"),
    (dict(inner=0), -3, "inner"),
    (dict(position_tokens=0), -3, "position_tokens"),
    (dict(position_tokens=4), -3, "position_tokens"),
    (dict(x_head_stride=-1), -3, "strides"),
    (dict(y_inner_stride=1 << 40), -3, "strides"),
    (dict(y_head_stride=0), -3, "share a place"),
    (dict(y_inner_stride=0), -3, "share a place"),
    (dict(inner=3), -3, "share a place"),
])
def test_rotary_refuses_descriptors(kw, code, text):
    assert _rotary(_rot(**kw)) == code, L.last_error()
    assert text in L.last_error()


@pytest.mark.parametrize("kw,code,text", [
    (dict(d=None), -1, "desc"),
    (dict(x=None), -1, "NULL"),
    (dict(y=None), -1, "NULL"),
    (dict(pos=None), -1, "NULL"),
    (dict(turns=None), -1, "NULL"),
    (dict(x=at(0, 1)), -4, "aligned"),
    (dict(pos=at(2, 4)), -4, "positions"),
    (dict(turns=at(3, 4)), -4, "turns"),
    (dict(y=at(0, 16)), -3, "overlap"),
    (dict(y=at(0), d=_rot(y_inner_stride=512)), -3, "overlap"),
])
def test_rotary_refuses_pointers(kw, code, text):
    kw = dict(kw)
    assert _rotary(kw.pop("d", _rot()), **kw) == code, L.last_error()
    assert text in L.last_error()


def test_rotary_of_no_tokens_needs_nothing():
    assert _rotary(_rot(tokens=0), None, None, None, None) == 0


# ---- the update of the parameters --------------------------------------------------


def _grads(*rows):
    return (L.TensorList * max(len(rows), 1))(*[L.TensorList(p.value if p else None, n, t) for p, n, t in rows])


@pytest.mark.parametrize("rows,kw,code,text", [
    ([(at(0), 8, L.DTYPE_U8)], {}, -2, "f32, bf16 or f16"),
    ([(at(0), -1, F32)], {}, -3, "elements"),
    ([(at(0), 1 << 35, F32)], {}, -3, "elements"),
    ([(None, 8, F32)], {}, -1, "NULL"),
    ([(at(0, 2), 8, F32)], {}, -4, "aligned"),
    ([(at(0), 8, F32)], dict(result=None), -1, "result"),
    ([(at(0), 8, F32)], dict(work=None), -1, "workspace"),
    ([(at(0), 8, F32)], dict(work=at(8, 4)), -4, "aligned"),
    ([(at(0), 8, F32)], dict(max_norm=float("nan")), -3, "NaN"),
    ([(at(0), 8, F32)], dict(work=at(0, 8)), -3, "overlap"),
    ([(at(0), 8, F32)], dict(result=at(0, 28)), -3, "overlap"),
    ([(at(0), 8, F32)], dict(result=at(8, 4)), -3, "overlap"),
])
def test_gradient_norm_refuses(rows, kw, code, text):
    kw = {**dict(max_norm=1.0, result=at(9), work=at(8)), **kw}
    st = L.load().terra_swin_gradient_norm(_grads(*rows), len(rows), kw["max_norm"], kw["result"], kw["work"], None)
    assert st == code, L.last_error()
    assert text in L.last_error()


def test_gradient_norm_workspace():
    f = L.load().terra_swin_gradient_norm_workspace
    assert f(_grads(), 0) == 0 and f(None, 0) == 0
    assert f(None, 1) == -1 and f(_grads(), -1) == -3
    assert f(_grads((at(0), 0, F32), (at(1), 1, BF16), (at(2), 100000, F16)), 3) >= 2


def _adam(**kw):
    return _set(L.AdamWDesc(), dict(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.01, step=1), kw)


def _tensor(i=0, **kw):
    t = dict(param=at(8 * i), grad=at(8 * i + 1), exp_avg=at(8 * i + 2), exp_avg_sq=at(8 * i + 3), scales=None, numel=64,
             index=i, param_dtype=F32, grad_dtype=F32)
    t.update(kw)
    return L.AdamWTensor(**t)


def _adamw(tensors, d):
    return L.load().terra_swin_adamw((L.AdamWTensor * max(len(tensors), 1))(*tensors), len(tensors),
                                     None if d is None else ctypes.byref(d), None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(beta1=1.0), -3, "betas"),
    (dict(beta2=-0.1), -3, "betas"),
    (dict(beta1=float("nan")), -3, "betas"),
    (dict(eps=-1.0), -3, "eps"),
    (dict(weight_decay=-1.0), -3, "weight_decay"),
    (dict(lr=float("nan")), -3, "lr"),
    (dict(step=0), -3, "step"),
    (dict(step_ptr=at(50, 4)), -4, "aligned"),
    (dict(lr_ptr=at(50, 2)), -4, "aligned"),
    (dict(grad_factor=at(50, 1)), -4, "aligned"),
    (dict(found_inf=at(50, 1)), -4, "aligned"),
    (dict(seed=at(50, 4)), -4, "aligned"),
])
def test_adamw_refuses_options(kw, code, text):
    assert _adamw([_tensor()], _adam(**kw)) == code, L.last_error()
    assert text in L.last_error()


@pytest.mark.parametrize("tensors,code,text", [
    ([_tensor(param_dtype=L.DTYPE_U8)], -2, "f32, bf16 or f16"),
    ([_tensor(param_dtype=BF16, grad_dtype=F16)], -2, "f32, bf16 or f16"),
    ([_tensor(numel=-1)], -3, "elements"),
    ([_tensor(numel=1 << 35)], -3, "elements"),
    ([_tensor(scales=at(40))], -1, "seed"),
    ([_tensor(param=None)], -1, "NULL"),
    ([_tensor(grad=None)], -1, "NULL"),
    ([_tensor(exp_avg=None)], -1, "NULL"),
    ([_tensor(exp_avg_sq=None)], -1, "NULL"),
    ([_tensor(param=at(0, 2))], -4, "aligned"),
    ([_tensor(grad=at(1, 2))], -4, "aligned"),
    ([_tensor(exp_avg=at(2, 2))], -4, "aligned"),
    ([_tensor(grad=at(0))], -3, "overlap"),
    ([_tensor(exp_avg=at(3, 4))], -3, "overlap"),
    ([_tensor(0), _tensor(1), _tensor(0)], -3, "overlap"),
    ([_tensor(0), _tensor(1, param=at(0, 252))], -3, "overlap"),
    ([_tensor(0), _tensor(1, grad=at(2, 4))], -3, "overlap"),
    ([_tensor(0), _tensor(1, param_dtype=BF16, exp_avg=at(3))], -3, "overlap"),
])
def test_adamw_refuses_tensors(tensors, code, text):
    assert _adamw(tensors, _adam()) == code, L.last_error()
    assert text in L.last_error()


def test_adamw_of_nothing():
    assert _adamw([], None) == -1
    assert _adamw([], _adam()) == 0
    assert _adamw([_tensor(numel=0, param=None, grad=None, exp_avg=None, exp_avg_sq=None)], _adam()) == 0
    assert L.load().terra_swin_adamw(None, 1, ctypes.byref(_adam()), None) == -1
    assert L.load().terra_swin_adamw(None, -1, ctypes.byref(_adam()), None) == -3


class TestWrappers:
    """CPU tensors and bad arguments raise before anything is launched."""

    def test_cpu_tensors(self):
        x, p = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int64)
        m = kernels.moments(x)
        for call in (lambda: kernels.layer_norm(x, Norm()), lambda: autograd.layer_norm(x, Norm()),
                     lambda: kernels.layer_norm_backward(x, x, Norm(), torch.zeros(4, 2)),
                     lambda: kernels.rotary(x.view(4, 1, 8), Rotary(8), p), lambda: autograd.rotary(x.view(4, 1, 8), Rotary(8), p),
                     lambda: kernels.gradient_norm([x]), lambda: kernels.adamw_step([x], [x.clone()], [m], 1)):
            with pytest.raises(RuntimeError, match="ROCm devices only"):
                call()

    def test_rows_of_two_strides(self):
        rows = lambda t, dims=1: kernels._two_level_rows(t, dims, "x")  # noqa: E731
        x = torch.zeros(4, 6, 10)
        assert rows(x) == (24, 24, 240, 10)
        assert rows(x[:, :4]) == (16, 4, 60, 10)
        assert rows(x[:, ::2]) == (12, 12, 240, 20)
        assert rows(x[:, 1:2]) == (4, 4, 240, 60)
        assert rows(x.transpose(0, 1)) == (24, 4, 10, 60)
        assert rows(x[0, 0]) == (1, 1, 10, 10)
        assert rows(x, 2) == (4, 4, 240, 60)
        assert rows(x[:1, :1].expand(4, 6, 10)) == (24, 24, 0, 0)
        with pytest.raises(ValueError, match="at most two strides"):
            rows(torch.zeros(4, 6, 5, 10)[:, :4, :3])

    def test_rotary_options(self):
        for kw in (dict(dim=7), dict(dim=0), dict(dim=8, axes=3), dict(dim=8, base=0.0), dict(dim=8, factor=-1.0),
                   dict(dim=8, scaling="other"), dict(dim=8, scaling="yarn", factor=2.0)):
            with pytest.raises(ValueError):
                Rotary(**kw)

    @pytest.mark.parametrize("kw", [dict(dim=16), dict(dim=16, axes=2), dict(dim=2, scaling="ntk", factor=3.0),
                                    dict(dim=64, scaling="linear", factor=4.0), dict(dim=64, scaling="ntk", factor=8.0),
                                    dict(dim=64, scaling="yarn", factor=16.0, original_length=4096),
                                    dict(dim=64, base=5e5, scaling="yarn", factor=0.5, original_length=100)])
    def test_rotary_rates(self, kw):
        from oracle import training as tr

        rates, amplitude = tr.rates(**kw)
        r = Rotary(**kw)
        torch.testing.assert_close(r.rates, rates, rtol=1e-14, atol=0)
        assert r.amplitude == pytest.approx(amplitude, rel=1e-14)
        assert Rotary(**kw, amplitude=2.0).amplitude == 2.0

    def test_rotary_copies(self):
        import copy
        import pickle

        r = Rotary(8, device="cpu")
        for other in (copy.deepcopy(r), pickle.loads(pickle.dumps(r))):
            assert torch.equal(other.rates, r.rates) and other.dim == 8

    def test_moments(self):
        p = torch.zeros(10, 60).t()
        m = kernels.moments(p)
        assert m.exp_avg.dtype == torch.float32 and m.exp_avg.stride() == p.stride() and m.scales is None
        m = kernels.moments(p, 8)
        assert m.exp_avg.dtype == torch.float8_e4m3fn and m.exp_avg_sq.stride() == p.stride()
        assert tuple(m.scales.shape) == (2, 3)
        with pytest.raises(ValueError, match="32 bits or in 8"):
            kernels.moments(p, 16)

    def test_values_of_moments(self):
        p = torch.zeros(7, 100)
        codes = torch.arange(700) % 120
        m = kernels.Moments(codes.to(torch.uint8).view(torch.float8_e4m3fn).view(7, 100),
                            codes.flip(0).to(torch.uint8).view(torch.float8_e4m3fn).view(7, 100),
                            torch.tensor([[1.0, 2.0, 4.0], [0.5, 0.25, 8.0]]))
        from oracle import training as tr

        values, block = tr.e4m3_values(), torch.arange(700) // 256
        first, second = m.values()
        assert torch.equal(first.double().view(-1), values[codes] * m.scales[0].double()[block])
        torch.testing.assert_close(second.double().view(-1), (values[codes.flip(0)] * m.scales[1].double()[block]) ** 2)
        assert first.shape == p.shape

    def test_step_arguments(self):
        x = torch.zeros(4)
        with pytest.raises(ValueError, match="as many moments"):
            kernels.adamw_step([x], [x], [], 1)
        with pytest.raises(ValueError, match="stream"):
            kernels.adamw_step([x], [x], [kernels.moments(x)], 1, stream=-1)
        with pytest.raises(ValueError, match="max_norm"):
            kernels.gradient_norm([x], max_norm=0.0)
        with pytest.raises(ValueError, match="one gradient"):
            kernels.gradient_norm([])


def test_host_module():
    """It loads against this torch and takes descriptors of the library's size alone."""
    module = L.load_training()
    assert module.NormCall(bytes(_norm()), 0) is not None and module.RotaryCall(bytes(_rot())) is not None
    for call in (lambda: module.NormCall(bytes(_norm())[:-1], 0), lambda: module.RotaryCall(bytes(8))):
        with pytest.raises(RuntimeError, match="descriptor of"):
            call()
