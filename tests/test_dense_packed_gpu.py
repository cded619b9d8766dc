"""The products of a linear layer on packed matrices of odd widths (rows on 4-byte boundaries only) against the same products on
copies whose rows are padded to 16 bytes: the same values in the same order, so the same bits.  Operands that end with their
buffer, and views whose rows end before it."""
import pytest
import torch

pytestmark = pytest.mark.gpu

SHAPES = [(130, 130, 130), (300, 1024, 479), (300, 479, 1024), (513, 131, 259), (64, 33, 129), (1000, 257, 67), (97, 66, 98)]


def packed(v):
    return v.clone()


def padded(v):
    ld = (v.shape[1] + 31) // 32 * 32 + 4
    buf = torch.zeros((v.shape[0], ld), device="cuda")
    buf[:, :v.shape[1]] = v
    return buf[:, :v.shape[1]]


def inside(v):
    """a view of a wider buffer, one column in"""
    buf = torch.full((v.shape[0], v.shape[1] + 3), float("nan"), device="cuda")
    buf[:, 1:1 + v.shape[1]] = v
    return buf[:, 1:1 + v.shape[1]]


@pytest.mark.parametrize("mode", [1, 2])
@pytest.mark.parametrize("layout", [packed, inside])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_packed_rows_give_the_padded_rows_bits(M, N, K, layout, mode):
    from dlrm_amd import ops
    g = torch.Generator().manual_seed(M + N * K)
    x, w, dz = (torch.randn(s, generator=g).cuda() for s in ((M, K), (N, K), (M, N)))
    b = torch.randn(N, generator=g).cuda()
    old = ops.get_gemm_mode()
    ops.set_gemm_mode(mode)
    try:
        def three(f):
            y = ops.linear_forward(f(x), f(w), b, True, out=torch.empty((M, N), device="cuda"))
            dx = ops.linear_backward_data(f(dz), f(w), out=torch.empty((M, K), device="cuda"))
            dw, db, _ = ops.linear_backward_weight(f(dz), f(x), dw=torch.empty((N, K), device="cuda"))
            return y, dx, dw, db
        for got, want in zip(three(layout), three(padded)):
            assert torch.isfinite(want).all() and torch.equal(got, want)
    finally:
        ops.set_gemm_mode(old)
