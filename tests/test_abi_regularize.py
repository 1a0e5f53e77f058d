"""Argument checks of the regularised training operators (on the CPU, no
kernel runs): the C entry points and the tensor-level wrappers."""
import ctypes

import pytest
import torch

import terra_amd._lib as L
from terra_amd import kernels
from terra_amd.kernels import Norm, WindowGeometry

A = 1 << 20


def at(i, off=0):
    return ctypes.c_void_p(A * (i + 1) * 64 + off)


F32P = ctypes.c_void_p


def test_descriptor_mirrors_the_header():
    assert ctypes.sizeof(L.ResidualNormDesc) == 5 * 8 + 10 * 4 + 60 + 4  # 4: tail padding to 8 bytes
    assert (L.NORM_NONE, L.NORM_LAYER, L.NORM_RMS) == (0, 1, 2)


def _drop(x=at(0), y=at(1), dt=L.DTYPE_BF16, rows=4, C=64, stride=64, p=0.1, seed=at(9)):
    return L.load().terra_swin_dropout(x, y, dt, rows, C, stride, p, seed, 0, None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(dt=L.DTYPE_U8), -2, "dropout supports"),
    (dict(rows=-1), -3, "rows must be"),
    (dict(C=0, stride=0), -3, "columns > 0"),
    (dict(rows=1 << 31), -3, "at most"),
    (dict(C=1 << 27, stride=1 << 27), -3, "at most"),
    (dict(stride=63), -3, "row stride"),
    (dict(p=-0.1), -3, "probability"),
    (dict(p=1.5), -3, "probability"),
    (dict(p=float("nan")), -3, "probability"),
    (dict(seed=None), -1, "seed"),
    (dict(seed=at(9, 4)), -4, "seed"),
    (dict(x=None), -1, "NULL"),
    (dict(y=None), -1, "NULL"),
    (dict(x=at(0, 1)), -4, "aligned"),
    (dict(y=at(0, 2)), -3, "overlap"),
    (dict(y=at(0), stride=72), -3, "overlap"),
])
def test_dropout_refuses(kw, code, text):
    assert _drop(**kw) == code, L.last_error()
    assert text in L.last_error()


def test_dropout_of_no_rows_needs_nothing():
    assert _drop(rows=0, x=None, y=None) == 0
    assert L.load().terra_swin_gelu_dropout(None, None, 0, 0, 8, 0.0, None, 0, None) == 0
    assert L.load().terra_swin_gelu_dropout_bwd(None, None, None, 0, 0, 8, 0.0, None, 0, None, None, None) == 0


def _gelu_bwd(da=at(0), h=at(1), dh=at(2), dt=L.DTYPE_F32, rows=4, C=64, p=0.1, seed=at(9), sums=at(3), work=at(4)):
    return L.load().terra_swin_gelu_dropout_bwd(da, h, dh, dt, rows, C, p, seed, 0, sums, work, None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(dt=7), -2, "dropout supports"),
    (dict(p=2.0), -3, "probability"),
    (dict(seed=None), -1, "seed"),
    (dict(h=None), -1, "NULL"),
    (dict(dh=at(0, 4)), -3, "overlap"),
    (dict(dh=at(1, 4)), -3, "overlap"),
    (dict(dh=at(2, 2)), -4, "aligned"),
    (dict(work=None), -1, "workspace"),
    (dict(sums=at(3, 2)), -4, "column_sums"),
])
def test_gelu_dropout_backward_refuses(kw, code, text):
    assert _gelu_bwd(**kw) == code, L.last_error()
    assert text in L.last_error()


def test_gelu_dropout_refuses_overlap_and_sizes():
    lib = L.load()
    assert lib.terra_swin_gelu_dropout(at(0), at(0, 16), 0, 4, 64, 0.0, None, 0, None) == -3
    assert lib.terra_swin_gelu_dropout_workspace(-1, 8) == -3
    assert lib.terra_swin_gelu_dropout_workspace(8, 0) == -3
    assert lib.terra_swin_gelu_dropout_workspace(0, 8) == 0
    for rows, C in ((1, 8), (100000, 768), (1, (1 << 27) - 1), ((1 << 31) - 1, 8192), ((1 << 31) - 1, (1 << 27) - 1)):
        assert C <= lib.terra_swin_gelu_dropout_workspace(rows, C) <= 1 << 28


def _desc(**kw):
    d = L.ResidualNormDesc()
    vals = dict(rows=8, channels=64, h_stride=64, x_stride=64, gate_rows=1, p=0.1, h_dtype=L.DTYPE_BF16,
                x_dtype=L.DTYPE_F32, post_norm=1, next_norm=2, post_eps=1e-5, next_eps=1e-5, residual_scale=1.0)
    vals.update(kw)
    for k, v in vals.items():
        setattr(d, k, v)
    return d


def _fwd(desc, h=at(0), x=at(1), y=at(2), z=at(3), pw=at(4), pb=at(5), gate=at(6), nw=at(7), nb=at(8), seed=at(9)):
    return L.load().terra_swin_residual_norm(h, x, y, z, None if desc is None else ctypes.byref(desc), pw, pb, gate, nw, nb,
                                             seed, None)


DESCS = [
    (dict(h_dtype=L.DTYPE_F32, x_dtype=L.DTYPE_BF16), -2, "h is bf16"),
    (dict(h_dtype=L.DTYPE_F16, x_dtype=L.DTYPE_BF16), -2, "h is bf16"),
    (dict(h_dtype=L.DTYPE_U8), -2, "h is bf16"),
    (dict(rows=-1), -3, "rows must be"),
    (dict(channels=0), -3, "channels > 0"),
    (dict(channels=8193, h_stride=8193, x_stride=8193), -5, "8192"),
    (dict(rows=1 << 31), -3, "at most"),
    (dict(post_norm=3), -3, "unknown norm"),
    (dict(next_norm=-1), -3, "unknown norm"),
    (dict(gate_rows=-1), -3, "gate rows"),
    (dict(gate_rows=3), -3, "gate rows"),
    (dict(gate_rows=1 << 32), -3, "gate rows"),
    (dict(h_stride=63), -3, "row stride"),
    (dict(x_stride=63), -3, "row stride"),
    (dict(p=1.01), -3, "probability"),
    (dict(windows=1), -3, "must be positive"),
]


@pytest.mark.parametrize("kw,code,text", DESCS)
def test_residual_norm_refuses_descriptors(kw, code, text):
    assert _fwd(_desc(**kw)) == code, L.last_error()
    assert text in L.last_error()
    if "p" not in kw:
        assert L.load().terra_swin_residual_norm_workspace(ctypes.byref(_desc(**kw))) == code


@pytest.mark.parametrize("kw,code,text", [
    (dict(desc=None), -1, "desc"),
    (dict(h=None), -1, "h is NULL"),
    (dict(x=None), -1, "x is NULL"),
    (dict(y=None), -1, "y is NULL"),
    (dict(z=None), -1, "z is NULL"),
    (dict(gate=None), -1, "gate is NULL"),
    (dict(seed=None), -1, "seed"),
    (dict(h=at(0, 1)), -4, "aligned"),
    (dict(x=at(1, 2)), -4, "aligned"),
    (dict(pw=at(4, 2)), -4, "parameter"),
    (dict(y=at(1)), -3, "y must not overlap x"),
    (dict(y=at(0)), -3, "y must not overlap h"),
    (dict(z=at(0)), -3, "z must not overlap h"),
    (dict(z=at(2, 16)), -3, "z must not overlap y"),
])
def test_residual_norm_refuses_pointers(kw, code, text):
    kw = dict(kw)
    desc = kw.pop("desc", _desc())
    assert _fwd(desc, **kw) == code, L.last_error()
    assert text in L.last_error()


def test_residual_norm_refuses_a_geometry_of_another_grid():
    d = _desc(windows=1, rows=256)
    d.geom = WindowGeometry(1, 16, 16, 32, 8).to_c()
    assert _fwd(d) == -3 and "grid" in L.last_error()
    d.geom = WindowGeometry(1, 16, 24, 64, 8).to_c()
    assert _fwd(d) == -3 and "grid" in L.last_error()
    d.geom = WindowGeometry(1, 16, 16, 64, 7).to_c()
    assert _fwd(d) == -3 and "multiple of window" in L.last_error()


def _bwd(desc, h=at(0), x=at(1), dy=at(2), dz=at(3), dh=at(10), dx=at(11), gate=at(6), seed=at(9), dpw=at(12), dpb=at(13),
         dg=at(14), dnw=at(15), dnb=at(16), work=at(17)):
    return L.load().terra_swin_residual_norm_bwd(h, x, dy, dz, dh, dx, ctypes.byref(desc), at(4), at(5), gate, at(7), seed,
                                                 dpw, dpb, dg, dnw, dnb, work, None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(dh=None), -1, "dh is NULL"),
    (dict(dx=None), -1, "dx is NULL"),
    (dict(work=None), -1, "workspace"),
    (dict(seed=None), -1, "seed"),
    (dict(gate=None), -1, "gate is NULL"),
    (dict(dx=at(2)), -3, "dx must not overlap dy"),
    (dict(dh=at(0)), -3, "dh must not overlap h"),
    (dict(dh=at(3)), -3, "dh must not overlap dz"),
    (dict(dx=at(10)), -3, "dx must not overlap dh"),
    (dict(dnb=at(16, 2)), -4, "gradient"),
    (dict(dz=at(3, 1)), -4, "dz is not aligned"),
])
def test_residual_norm_backward_refuses(kw, code, text):
    assert _bwd(_desc(), **kw) == code, L.last_error()
    assert text in L.last_error()


@pytest.mark.parametrize("kw,text", [
    (dict(post_norm=0), "post-norm that"),
    (dict(next_norm=0), "next norm that"),
    (dict(gate_rows=0), "gate that"),
])
def test_residual_norm_backward_refuses_gradients_of_what_is_not_there(kw, text):
    assert _bwd(_desc(**kw)) == -3
    assert text in L.last_error()


def test_residual_norm_workspace_covers_the_sizes():
    lib = L.load()
    for rows in (1, 3, 100, 5000, 1 << 20, (1 << 31) - 2):
        for C in (1, 64, 192, 1000, 2000, 8192):
            for gates in (0, 1, 2, rows):
                if gates and rows % gates:
                    continue
                n = lib.terra_swin_residual_norm_workspace(ctypes.byref(_desc(rows=rows, channels=C, h_stride=C, x_stride=C,
                                                                             gate_rows=gates)))
                assert 0 < n <= 1 << 27 and n >= 4 * C, (rows, C, gates, n)


class TestWrappers:
    """CPU tensors and bad arguments raise before anything is launched."""

    def test_cpu_tensors(self):
        x = torch.zeros(4, 8)
        for call in (lambda: kernels.dropout(x, 0.1, None), lambda: kernels.gelu_dropout(x, 0.1, None),
                     lambda: kernels.gelu_dropout_backward(x, x, 0.1, None), lambda: kernels.residual_norm(x, x),
                     lambda: kernels.residual_norm_backward(x, x, x, None)):
            with pytest.raises(RuntimeError, match="ROCm devices only"):
                call()

    def test_dropout_arguments(self):
        x = torch.zeros(4, 8)
        for p in (-0.1, 1.1, float("nan")):
            with pytest.raises(ValueError, match="probability"):
                kernels._dropout_args(x, p, None, 0)
        for stream in (-1, 1 << 32):
            with pytest.raises(ValueError, match="stream"):
                kernels._dropout_args(x, 0.0, None, stream)
        with pytest.raises(ValueError, match="needs a seed"):
            kernels._dropout_args(x, 0.1, None, 0)
        for seed in (torch.zeros(1), torch.zeros(2, dtype=torch.int64), torch.zeros(1, dtype=torch.int64, device="meta")):
            with pytest.raises(ValueError, match="one int64"):
                kernels._dropout_args(x, 0.1, seed, 0)

    def test_token_rows(self):
        x = torch.zeros(4, 6, 10)
        assert kernels._token_rows(x, "x") == (24, 10, 10)
        assert kernels._token_rows(x[..., :3], "x") == (24, 3, 10)
        assert kernels._token_rows(x[:, :1, 2:5], "x") == (4, 3, 60)
        assert kernels._token_rows(x[0, 0], "x") == (1, 10, 10)
        assert kernels._token_rows(x[:0], "x") == (0, 10, 10)
        assert kernels._token_rows(torch.zeros(3, 0), "x") == (0, 0, 0)
        assert kernels._token_rows(x[:, ::2], "x") == (12, 10, 20)
        for bad in (x.transpose(1, 2), x[:, :4], x[:1, :1].expand(4, 6, 10), x[..., ::2]):
            with pytest.raises(ValueError, match="unit channel stride"):
                kernels._token_rows(bad, "x")
        with pytest.raises(ValueError, match="scalar"):
            kernels._token_rows(torch.zeros(()), "x")

    def test_norm_of(self):
        ln = torch.nn.LayerNorm(8, eps=1e-3)
        n = Norm.of(ln)
        assert n.weight is ln.weight and n.bias is ln.bias and n.eps == 1e-3 and not n.rms
        n = Norm.of(torch.nn.RMSNorm(8, eps=1e-4))
        assert n.rms and n.bias is None and n.eps == 1e-4
        assert Norm.of(torch.nn.RMSNorm(8)).eps == torch.finfo(torch.float32).eps
        assert Norm.of(None) is None
        for bad in (torch.nn.LayerNorm((2, 8)), torch.nn.Identity(), torch.nn.BatchNorm1d(8)):
            with pytest.raises(TypeError, match="LayerNorm or nn.RMSNorm"):
                Norm.of(bad)


def test_autograd_node_module():
    """The host module loads against this torch and takes descriptors of the library's size alone."""
    module = L.load_binding()
    d = L.ResidualNormDesc()
    assert module.Call(bytes(d), True, 0) is not None
    with pytest.raises(RuntimeError, match="descriptor of"):
        module.Call(bytes(d)[:-1], True, 0)
