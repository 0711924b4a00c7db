"""Host side of the 8-bit activations: what is refused, and the format's own arithmetic."""
import numpy as np
import pytest
import torch

import _act8_ref as ref
from detmatch_amd import _lib, act8


def test_host_tensors_are_refused():
    with pytest.raises(_lib.DetMatchHipError):
        act8.pack(torch.zeros(3, 32))


def test_types_and_shapes_are_refused():
    with pytest.raises(TypeError):
        act8.pack(torch.zeros(3, 32, dtype=torch.float64))
    with pytest.raises(ValueError):
        act8.pack(torch.zeros(()))
    with pytest.raises(ValueError):
        act8.pack(torch.zeros(3, 0))
    with pytest.raises(TypeError):
        act8.unpack(torch.zeros(3, 32, dtype=torch.uint8))


def test_entry_points_check_their_arguments():
    L = _lib.lib()
    bad = 1                                   # DM_ERR_INVALID_ARG, before any pointer is looked at
    assert L.dm_act8_pack(None, 3, 4, 32, 32, None, None, None) == bad
    assert L.dm_act8_pack(None, 0, 4, 0, 32, None, None, None) == bad
    assert L.dm_act8_pack(None, 0, 4, 32, 31, None, None, None) == bad
    assert L.dm_act8_pack(None, 0, -1, 32, 32, None, None, None) == bad
    assert L.dm_act8_pack(None, 0, 4, 32, 32, None, None, None) == bad
    assert L.dm_act8_pack(None, 0, 0, 32, 32, None, None, None) == 0
    assert L.dm_act8_unpack(None, None, 4, 32, None, 0, None) == bad
    assert L.dm_act8_unpack(None, None, 0, 32, None, 0, None) == 0


def test_row_views_copy_only_what_has_no_unit_stride():
    x = torch.arange(24.0).view(4, 6)
    assert act8.rows_view(x).data_ptr() == x.data_ptr()
    assert act8.rows_view(x[:, :4]).stride() == (6, 1)
    assert act8.rows_view(x.t()).is_contiguous()
    assert act8.rows_view(x[:1].expand(3, 6)).is_contiguous()
    assert act8.rows_view(x.view(2, 2, 6)).shape == (4, 6)
    assert act8.row_stride(act8.rows_view(x[1:2, :3])) == 3
    assert act8.rows_view(x[:, :1]).shape == (4, 1)


def test_reference_rounding_agrees_with_torch():
    """The listed codes are torch's float8_e4m3fn, and nearest-even is its cast."""
    bits = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn)
    assert np.array_equal(bits.double().numpy() if hasattr(bits, 'double') else bits.float().numpy(), ref.CODES)
    z = torch.from_numpy(np.random.RandomState(0).uniform(-448, 448, (64, 32)))
    z[:, 0] = 448.0                            # e = 0
    code, e = ref.pack(z)
    assert (e == 0).all()
    assert np.array_equal(code, z.float().to(torch.float8_e4m3fn).view(torch.uint8).numpy())
