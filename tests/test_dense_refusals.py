"""Batches that the linear layers refuse, without a GPU: a refused call never reaches a kernel."""
import ctypes as C

import pytest

from dlrm_amd import _capi

P = 1 << 20        # a made-up device address on a 16-byte boundary, never dereferenced
LIMIT = (1 << 31) - (1 << 20)


@pytest.mark.parametrize("N,K", [(1, 64), (8, 13), (64, 64)])        # one output, few inputs, a matrix product
@pytest.mark.parametrize("M", [LIMIT + 1, (1 << 31) - 1, 1 << 31, 1 << 40])
def test_too_many_rows(M, N, K):
    """The kernels' row numbers are 32-bit: the strides over the batch would pass their end."""
    L = _capi.lib()
    f = _capi.LinearDesc()
    f.M, f.N, f.K = M, N, K
    f.d_x, f.x_ld, f.d_w, f.w_ld, f.d_y, f.y_ld = P, K, P, K, P, N
    b = _capi.LinearBwdDesc()
    b.M, b.N, b.K = M, N, K
    b.d_dz, b.dz_ld, b.d_w, b.w_ld, b.d_x, b.x_ld, b.d_dx, b.dx_ld, b.d_dw, b.dw_ld = P, N, P, K, P, K, P, K, P, K
    for rc in (L.dlrm_linear_forward(C.byref(f), None), L.dlrm_linear_backward_data(C.byref(b), None),
               L.dlrm_linear_backward_weight(C.byref(b), C.c_void_p(P), C.c_size_t(1 << 62), None)):
        assert rc == 1 and "M too large" in L.dlrm_last_error().decode()


def test_too_many_rows_of_a_checkpoint():
    L = _capi.lib()
    b = _capi.LinearBwdDesc()
    b.M, b.N, b.K = 1 << 31, 4, 32
    b.d_dz, b.dz_ld, b.d_dw, b.dw_ld, b.x8 = P, 4, P, 32, _capi.Act8Desc(P, 32, P, 1)
    assert L.dlrm_linear_backward_weight(C.byref(b), C.c_void_p(P), C.c_size_t(1 << 62), None) == 1
    assert "M too large" in L.dlrm_last_error().decode()
