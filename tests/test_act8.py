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


def test_linear_refuses_what_it_cannot_take():
    x, w = torch.zeros(4, 16), torch.zeros(8, 16)
    with pytest.raises(_lib.DetMatchHipError):
        act8.linear(x, w)
    with pytest.raises(ValueError):
        act8.linear(x, torch.zeros(8, 15))
    with pytest.raises(ValueError):
        act8.linear(x, w[0])
    with pytest.raises(ValueError):
        act8.linear(x, w, torch.zeros(7))
    with pytest.raises(ValueError):
        act8.linear(torch.zeros(4, 0), torch.zeros(8, 0))
    with pytest.raises(TypeError):
        act8.linear(x, w.half())
    with pytest.raises(TypeError):
        act8.linear(x.double(), w.double())
    with pytest.raises(TypeError):
        act8.linear(x, w, torch.zeros(8, dtype=torch.bfloat16))


def test_gemm_entry_checks_its_arguments():
    L = _lib.lib()
    p = 4096                                  # an aligned address that no check looks behind
    bad, workspace = 1, 2

    def call(form=0, dtype=1, a=p, lda=64, b=p, ldb=64, exps=None, bias=None, relu=0, m=8, n=8, k=64, c=p, bits=None, rowsum=None):
        return L.dm_act8_gemm(form, dtype, a, lda, b, ldb, 0, exps, bias, relu, m, n, k, c, bits, rowsum, None, 0, None)

    assert call(form=3) == bad and call(form=-1) == bad and call(dtype=3) == bad
    assert call(m=0) == bad and call(n=-1) == bad and call(k=0) == bad
    assert call(a=None) == bad and call(b=None) == bad and call(c=None) == bad
    assert call(lda=63) == bad and call(ldb=56) == bad
    assert call(form=2) == bad and call(exps=p) == bad and call(rowsum=p) == bad
    assert call(form=2, exps=p, relu=1) == bad and call(form=2, exps=p, bias=p) == bad
    assert call(form=2, exps=p, ldb=40) == bad and call(form=2, exps=p, b=p + 8) == bad
    assert L.dm_act8_gemm_workspace_bytes(0, 1, p, 8192, p, 8192, 0, 64, 64, 8192) > 0
    assert call(lda=8192, ldb=8192, k=8192) == workspace
    assert L.dm_act8_gemm_workspace_bytes(0, 1, p, 64, p, 64, 0, 0, 64, 64) == 0
    assert L.dm_act8_mask_rows(p, 1, 4, 12, 12, None, p, 12, None) == bad and L.dm_act8_mask_rows(p, 1, 4, 12, 8, None, p, 16, None) == bad
    assert L.dm_act8_mask_rows(None, 1, 0, 12, 12, None, None, 16, None) == 0


def test_unpack_refuses_codes_that_do_not_fit_their_shape():
    codes, exps = torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8)
    for c, e, shape in ((codes, exps, (4, 65)), (codes, exps, (5, 64)), (codes, exps, (4, 32)), (codes[:, ::2], exps, (4, 32)),
                        (codes, exps[:, :1], (4, 64)), (codes.int(), exps, (4, 64)), (codes, exps.int(), (4, 64)), (codes[:3], exps, (4, 64))):
        with pytest.raises(ValueError):
            act8.unpack(act8.Act8(c, e, shape, torch.float32))
    with pytest.raises(_lib.DetMatchHipError):
        act8.unpack(act8.Act8(codes, exps, (2, 2, 40), torch.float32))
