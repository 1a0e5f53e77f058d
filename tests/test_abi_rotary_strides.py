"""Strides of terra_swin_rotary's output (on the CPU, no kernel runs): layouts in
which two threads would write one place are refused, all others are not."""
import ctypes
import itertools

import pytest

import terra_amd._lib as L

A = 1 << 24


def _call(heads, tokens, groups, strides, head_dim=8, same=False):
    d = L.RotaryDesc()
    for k, v in dict(tokens=tokens * groups, inner=tokens, position_tokens=tokens * groups, heads=heads, head_dim=head_dim, dim=head_dim,
                     axes=1, dtype=L.DTYPE_F32, position_bits=32, amplitude=1.0, x_head_stride=head_dim,
                     x_inner_stride=heads * head_dim, x_outer_stride=tokens * heads * head_dim).items():
        setattr(d, k, v)
    for k, v in strides.items():
        setattr(d, f"y_{k}_stride", v)
        if same:
            setattr(d, f"x_{k}_stride", v)
    at = [ctypes.c_void_p(A * i * 64) for i in (1, 1 if same else 2, 3, 4)]
    return L.load().terra_swin_rotary(*at, ctypes.byref(d), None)


def _shared(heads, tokens, groups, head_dim, head, inner, outer):
    """Whether two elements share a place, by counting them."""
    places = [o * outer + i * inner + h * head + e
              for o in range(groups) for i in range(tokens) for h in range(heads) for e in range(head_dim)]
    return len(set(places)) < len(places)


@pytest.mark.parametrize("same", [False, True])
@pytest.mark.parametrize("kw", [dict(head=7, inner=64, outer=512),     # heads over each other
                                dict(head=8, inner=16, outer=512),     # tokens over the heads of others
                                dict(head=8, inner=31, outer=512),
                                dict(head=8, inner=32, outer=96),      # groups over tokens of others
                                dict(head=8, inner=8, outer=512)])     # a diagonal: as many steps a head as a token
def test_outputs_that_lie_over_themselves(kw, same):
    assert _shared(4, 6, 2, 8, **kw)
    assert _call(4, 6, 2, kw, same=same) == -3, L.last_error()
    assert "share a place" in L.last_error()


@pytest.mark.parametrize("order", list(itertools.permutations(("head", "inner", "outer"))))
@pytest.mark.parametrize("gap", [0, 5])
def test_packed_and_padded_layouts_of_any_order(order, gap):
    """Refused for no stride: the call gets as far as its launch (on the CPU; with a device it would run)."""
    import torch

    if torch.cuda.is_available():
        pytest.skip("these addresses are not memory")
    sizes, strides, step = dict(head=4, inner=6, outer=2), {}, 8 + gap
    for name in order:
        strides[name] = step
        step = step * sizes[name] + gap
    assert not _shared(4, 6, 2, 8, **strides)
    assert _call(4, 6, 2, strides) != -3, L.last_error()


def test_strides_of_what_is_there_once_do_not_matter():
    import torch

    if torch.cuda.is_available():
        pytest.skip("these addresses are not memory")
    assert _call(1, 6, 1, dict(head=3, inner=8, outer=0)) != -3, L.last_error()
    assert _call(4, 1, 2, dict(head=8, inner=1, outer=32)) != -3, L.last_error()
    assert _call(4, 1, 2, dict(head=8, inner=1, outer=31)) == -3


def test_products_past_64_bits():
    import torch

    if torch.cuda.is_available():
        pytest.skip("these addresses are not memory")
    big = (1 << 40) - 1
    assert _call(65535, 1 << 15, 2, dict(head=big, inner=big - 1, outer=big - 2)) == -3
