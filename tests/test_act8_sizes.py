"""Sizes that a kernel's 32-bit arithmetic does not hold are refused at the C entries (before any pointer is looked at)."""
from detmatch_amd import _lib, act8

P, BAD, LAST = 4096, 1, (1 << 31) - 1        # an aligned address; DM_ERR_INVALID_ARG; the largest int


def _gemm(form, m, n, k, lda, ldb, exps=None):
    return _lib.lib().dm_act8_gemm(form, 1, P, lda, P, ldb, 0, exps, None, 0, m, n, k, P, None, None, P, 1 << 62, None)


def test_sizes_next_to_the_largest_int_are_refused():
    L = _lib.lib()
    for size in (LAST, LAST - 62, act8._MAX + 1):
        assert _gemm(0, size, 8, 8, 8, 8) == BAD and _gemm(0, 8, 8, size, 1 << 32, 1 << 32) == BAD
        assert _gemm(1, 8, size, 8, 8, 1 << 32) == BAD and _gemm(2, size, 8, 8, 1 << 32, 32, P) == BAD
        for m, n, k in ((size, 8, 8), (8, size, 8), (8, 8, size)):
            assert L.dm_act8_gemm_workspace_bytes(0, 1, P, 1 << 32, P, 1 << 32, 0, m, n, k) == 0
        assert L.dm_act8_mask_rows(P, 1, 4, size, 1 << 32, None, P, (size + 7) // 8 * 8 if size < LAST - 7 else LAST - 7, None) == BAD
