"""The products of a linear layer on operands whose rows lie so far apart that a tile of them spans 2^32 bytes or more, against the
same products on packed copies: the same values in the same order, so the same bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

# elements from row to row: 128 rows just past 2^32 bytes, on 16-byte boundaries and off them; 127 rows past 2^31 elements
WIDE = [8460004, 8460003, 16909324]
# 16 rows past 2^32 bytes (operands whose rows are reduction steps)
WIDEST = [71582800, 71582803]


@pytest.fixture(scope="module")
def room():
    buf = torch.empty(3_000_000_000, device="cuda")
    yield buf
    del buf
    torch.cuda.empty_cache()


def far(room, v, ld):
    assert v.shape[0] * ld <= room.numel()
    view = room.as_strided(v.shape, (ld, 1))
    view.copy_(v)
    return view


def rand(*shape, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).cuda()


@pytest.fixture(params=[0, 1, 2])
def mode(request):
    from dlrm_amd import ops
    old = ops.get_gemm_mode()
    ops.set_gemm_mode(request.param)
    yield request.param
    ops.set_gemm_mode(old)


def padded(v):
    """rows on 16-byte boundaries, readable up to a whole reduction step"""
    buf = torch.zeros((v.shape[0], (v.shape[1] + 31) // 32 * 32), device="cuda")
    buf[:, :v.shape[1]] = v
    return buf[:, :v.shape[1]]


@pytest.mark.parametrize("K", [64, 70])
@pytest.mark.parametrize("ld", WIDE)
def test_forward(room, mode, ld, K):
    from dlrm_amd import ops
    x, w, b = rand(131, K, seed=1), padded(rand(140, K, seed=2)), rand(140, seed=3)
    want = ops.linear_forward(padded(x), w, b, True)
    assert torch.equal(ops.linear_forward(far(room, x, ld), w, b, True), want)
    assert torch.equal(ops.linear_forward(padded(x), far(room, w, ld), b, True), want)


@pytest.mark.parametrize("ld", WIDE + WIDEST)
def test_data_gradient(room, mode, ld):
    from dlrm_amd import ops
    dz, w = rand(131, 38, seed=4), rand(38, 130, seed=5)
    want = ops.linear_backward_data(dz, w)
    if ld in WIDE:
        assert torch.equal(ops.linear_backward_data(far(room, dz, ld), w), want)
    assert torch.equal(ops.linear_backward_data(dz, far(room, w, ld)), want)


@pytest.mark.parametrize("ld", WIDEST)
def test_weight_gradient(room, mode, ld):
    from dlrm_amd import ops
    dz, x = rand(41, 70, seed=6), rand(41, 130, seed=7)
    want, want_b, _ = ops.linear_backward_weight(dz, x)
    for which in (0, 1):                        # (one of them at a time: they would take the same memory)
        dw, db, _ = ops.linear_backward_weight(far(room, dz, ld) if which == 0 else dz, far(room, x, ld) if which == 1 else x)
        assert torch.equal(dw, want) and torch.equal(db, want_b)


def test_weights_split_beforehand(room):
    """Rows too far apart for the kernel of weights that were split beforehand: the product without those weights' planes."""
    from dlrm_amd import ops
    old = ops.get_gemm_mode()
    ops.set_gemm_mode(2)
    try:
        x, w = rand(300, 64, seed=8), rand(128 * 128, 64, seed=9)
        want = ops.linear_forward(x, w, None, False)
        assert torch.equal(ops.linear_forward(far(room, x, 8460004), w, None, False, w_planes=ops.SplitWeights(w)), want)
    finally:
        ops.set_gemm_mode(old)
