"""The positions that WindowAttention(rotary=...) turns its heads by: where
they come from when a module is built without memory, moved, copied, loaded, or
given positions of its own."""
import copy
import io
import pickle

import pytest
import torch

from terra_amd.attention import WindowAttention
from terra_amd.transformer import SequentialSwinTransformer

ROWS_AND_COLUMNS = [[i, j] for i in range(3) for j in range(5)]


def _attn(**kw):
    return WindowAttention(32, (3, 5), 2, rotary=True, **kw)


def _meta(**kw):
    with torch.device("meta"):
        return _attn(**kw)


@pytest.mark.parametrize("bias", [True, False])
def test_parameters_assigned_from_a_state_dict(bias):
    m = _meta(use_relative_position_bias=bias)
    m.load_state_dict(_attn(use_relative_position_bias=bias).state_dict(), assign=True)
    assert m.token_positions.tolist() == ROWS_AND_COLUMNS
    m.to("cpu").double()
    assert m.token_positions.tolist() == ROWS_AND_COLUMNS and m.token_positions.dtype == torch.int32


def test_memory_given_without_a_state_dict(monkeypatch):
    """to_empty, of a module with memory or without, then an initialisation by hand."""
    empty = torch.empty_like
    monkeypatch.setattr(torch, "empty_like", lambda t, **kw: empty(t, **kw).fill_(77))  # as unwritten memory may be
    for m in (_meta(), _attn()):
        m = m.to_empty(device="cpu")
        with torch.no_grad():
            for p in m.parameters():
                p.zero_()
        assert m.token_positions.tolist() == ROWS_AND_COLUMNS


def test_on_meta():
    m = _meta()
    assert m.token_positions.is_meta and m.token_positions.shape == (15, 2)
    assert m.to_empty(device="cpu").token_positions.tolist() == ROWS_AND_COLUMNS
    m = _attn().to("meta")
    assert m.token_positions.is_meta and m.to_empty(device="cpu").token_positions.tolist() == ROWS_AND_COLUMNS


@pytest.mark.parametrize("how", ["assigned", "written"])
def test_positions_of_ones_own_stay(how):
    own = torch.tensor(ROWS_AND_COLUMNS, dtype=torch.int32) * 3 - 7
    m = _attn()
    if how == "assigned":
        m.token_positions = own.clone()
    else:
        m.token_positions.copy_(own)
    m.load_state_dict(_attn().state_dict())
    assert torch.equal(m.token_positions, own)
    f = io.BytesIO()
    torch.save(m, f)
    f.seek(0)
    for other in (m.to("cpu"), m.half(), copy.deepcopy(m), pickle.loads(pickle.dumps(m)),
                  torch.load(f, weights_only=False)):  # of a file that this test wrote
        other.load_state_dict(_attn().state_dict())
        assert torch.equal(other.token_positions, own)
    other.token_positions += 1
    assert torch.equal(other.token_positions, own + 1) and torch.equal(m.token_positions, own)


def test_positions_set_before_the_first_state_dict_stay():
    own = torch.tensor(ROWS_AND_COLUMNS, dtype=torch.int32) + 5
    m = _meta().to_empty(device="cpu")
    m.token_positions = own
    m.load_state_dict(_attn().state_dict())
    assert torch.equal(m.token_positions, own)


def test_in_no_state_dict_and_only_where_there_is_rotary():
    m, off = _attn(), WindowAttention(32, (3, 5), 2)
    assert m.state_dict().keys() == off.state_dict().keys()
    assert m.token_positions.tolist() == ROWS_AND_COLUMNS
    assert not hasattr(off, "token_positions")
    with torch.inference_mode():
        assert not _attn().token_positions.is_inference()


def test_a_module_pickled_with_the_positions_as_a_buffer():
    old = SequentialSwinTransformer(0, 6, 6, 32, window_size=3, num_heads=2, rotary=True)
    attn = old.attn
    for name in ("_positions", "_unloaded"):
        del attn.__dict__[name]
    held = torch.arange(18, dtype=torch.int32).view(9, 2)
    attn._buffers["token_positions"] = held
    attn._non_persistent_buffers_set.add("token_positions")
    for new in (pickle.loads(pickle.dumps(old)), copy.deepcopy(old)):
        assert torch.equal(new.attn.token_positions, held)
        assert "token_positions" not in dict(new.named_buffers())
        assert new.to("cpu").attn.state_dict().keys() == attn.state_dict().keys()
