"""The weight gradient from an 8-bit checkpoint in every tile of its kernel, with and without columns of dz that the operand's end
cuts through, and through the static scratch where that caps the row ranges.

Tolerance of the products of random values, U = 2^-24: a matrix instruction adds 16 products of one of dz's three pieces to its
accumulator and is off by at most one step (2 U) of a number no larger than sum |dz x|, so a range of R rows is off by 6 R / 16
of them at most; then the ranges are added.  A column sum of dz is a chain of at most R / 8 additions in a thread, 16 across
threads and the ranges."""
import ctypes as C

import pytest
import torch

from tests import norm_ref
from tests.norm_ref import U

CASES = [  # M, N, K and the tile that the time model takes for them
    (2048, 256, 512, (64, 64)), (2702, 67, 290, (64, 64)), (1099, 224, 683, (64, 128)), (593, 491, 526, (64, 128)),
    (1856, 824, 196, (128, 128)), (731, 777, 597, (128, 128)), (1260, 1076, 985, (128, 256)), (1670, 803, 897, (128, 256)),
    (9828, 587, 212, (128, 256)), (8191, 1022, 1021, (128, 256))]


class Shape(C.Structure):
    _fields_ = [("tm", C.c_int), ("tn", C.c_int), ("ranges", C.c_int), ("rows", C.c_int), ("bytes", C.c_size_t)]


def shape(M, N, K, max_bytes=0):
    """dlrm::wgrad8_shape of the library"""
    from dlrm_amd import _capi
    f = _capi.lib()._ZN4dlrm12wgrad8_shapeEliim
    f.restype, f.argtypes = Shape, [C.c_int64, C.c_int, C.c_int, C.c_size_t]
    return f(M, N, K, max_bytes)


def test_the_cases_reach_every_kernel():
    """A change of the rule that takes the tile shows here, not as a kernel that no test runs any more."""
    for M, N, K, tile in CASES:
        s = shape(M, N, K)
        assert (s.tm, s.tn) == tile and s.ranges > 1 and s.rows % 32 == 0, (M, N, K)
    assert {(t, N % 4 != 0) for _, N, _, t in CASES} == {(t, cut) for t in [(64, 64), (64, 128), (128, 128), (128, 256)]
                                                         for cut in (False, True)}


def test_ranges_that_the_static_scratch_caps():
    from dlrm_amd import ops
    cap = 40 << 20
    for M, N, K in STATIC:
        free, capped = shape(M, N, K), shape(M, N, K, cap)
        assert free.ranges > capped.ranges and free.bytes > cap >= capped.ranges * 4 * (N * K + N)
        assert ops.linear_backward_weight_workspace_bytes(M, N, K, True) == free.bytes
    assert {shape(*s, cap).ranges > 1 for s in STATIC} == {False, True}


STATIC = [(8191, 1022, 1021), (4099, 2310, 2300)]


def one_row_a_column(M, N, K, seed):
    """x with one non-zero element in every column, a power of two, and dz whose elements fill their 24 bits: every element of the
    product is one element of dz times that power, to the bit."""
    from dlrm_amd import ops
    g = torch.Generator().manual_seed(seed)
    rows = torch.randint(0, M, (K,), generator=g)
    per = shape(M, N, K).rows
    edges = [0, M - 1, per - 1, per, M - M % 16 - 1, M - M % 16]
    rows[torch.randperm(K, generator=g)[:len(edges)]] = torch.tensor([min(e, M - 1) for e in edges])
    value = torch.pow(2.0, torch.randint(-2, 3, (K,), generator=g)) * (1 - 2 * torch.randint(0, 2, (K,), generator=g))
    x = torch.zeros(M, K)
    x[rows, torch.arange(K)] = value
    a = ops.act8_pack(x.cuda())
    assert torch.equal(ops.act8_unpack(a).cpu(), x)
    dz = torch.randn(M, N, generator=g)
    return dz, a, (dz[rows] * value[:, None]).t()


@pytest.mark.gpu
@pytest.mark.parametrize("pad", [0, 1])
@pytest.mark.parametrize("M,N,K,tile", CASES)
def test_every_element_to_the_bit(M, N, K, tile, pad):
    from dlrm_amd import ops
    dz, a, want = one_row_a_column(M, N, K, M + pad)
    d = torch.full((M, N + pad), float("nan"), device="cuda")[:, :N]
    d.copy_(dz)
    dw, _, _ = ops.linear_backward_weight(d, a, want_db=False)
    assert torch.equal(dw.cpu(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", STATIC)
def test_static_scratch_with_capped_ranges(M, N, K):
    from dlrm_amd import ops
    dz, a, want = one_row_a_column(M, N, K, 3)
    dw, db = torch.empty((N, K), device="cuda"), torch.empty(N, device="cuda")
    ops.linear_backward_weight_static(dz.cuda(), a, dw, db)
    assert torch.equal(dw.cpu(), want)
    s = shape(M, N, K, 40 << 20)
    assert ((db.cpu().double() - dz.double().sum(0)).abs() <= (s.rows / 8 + 18 + s.ranges) * U * dz.double().abs().sum(0)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K,tile", CASES)
def test_random_values(M, N, K, tile):
    from dlrm_amd import ops
    g = torch.Generator().manual_seed(M + N + K)
    x = torch.relu(torch.randn(M, K, generator=g) * torch.exp(0.7 * torch.randn(K, generator=g)))
    a = ops.act8_pack(x.cuda())
    x = norm_ref.unpack8(a.codes.cpu(), a.exps.cpu(), K)
    dz = torch.randn(M, N, generator=g) * torch.exp(2 * torch.randn(M, 1, generator=g))
    dw, db, ws = ops.linear_backward_weight(dz.cuda(), a)
    dz, s = dz.double(), shape(M, N, K)
    assert ((dw.cpu().double() - dz.t() @ x).abs() <= (6 * s.rows / 16 + s.ranges + 4) * U * (dz.abs().t() @ x) + 1e-45).all()
    assert ((db.cpu().double() - dz.sum(0)).abs() <= (s.rows / 8 + 18 + s.ranges) * U * dz.abs().sum(0)).all()
    again, _, _ = ops.linear_backward_weight(dz.float().cuda(), a, workspace=ws, want_db=False)
    assert torch.equal(again, dw)
