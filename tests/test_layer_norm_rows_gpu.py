"""Layer norm over batches in which every team of lanes takes several rows, the last turn with teams that have none: what a
training batch does in rows of every width that a wave or less holds.

Parameter gradients, U = 2^-24: an element d xh is off by at most 4 U of itself, and the additions are a chain of the turns of a
team (3 here), the teams of a workgroup (64 at most), every 32nd of at most 1024 workgroups and 32 groups of those: at most 3 + 64
+ 32 + 32 + 4 = 135 U of the magnitudes' sum.  Everything else as in test_layer_norm_gpu.py, whose bounds do not depend on the
number of rows."""
import pytest
import torch

from tests import norm_ref
from tests.norm_ref import U
from tests.test_layer_norm_gpu import DTYPES, HALF, close, inputs, strided

pytestmark = pytest.mark.gpu

# Backward launches hold 512 workgroups (float32 rows of 257 to 8192) or 1024, of as many rows as teams of 4 to 64 lanes
# (bf16 rows of more than 512: 128) fit into 256 threads
BACKWARD = [(65601, 16), (65601, 24), (33001, 50), (16501, 100), (8203, 200), (4101, 300), (4103, 480), (2055, 1000)]
# forward launches 4096, or 2048 where a lane has 16 elements
FORWARD = [(262211, 16), (131101, 30), (65603, 60), (32801, 101), (16411, 250), (16403, 500), (8211, 1000)]


def rows_per_turn(N, bf16):
    """Rows that a backward launch of the most workgroups takes at a time"""
    piece = 8 if bf16 else 4
    lanes = 4
    while lanes < (128 if bf16 else 64) and lanes * piece < N:
        lanes *= 2
    return (512 if not bf16 and N > 256 else 1024) * (256 // lanes)


@pytest.mark.parametrize("dtype", DTYPES, ids=list(DTYPES))
@pytest.mark.parametrize("kept", [False, True], ids=["from_x", "from_8"])
@pytest.mark.parametrize("mask", [None, "y", "y8"])
@pytest.mark.parametrize("M,N", BACKWARD)
def test_backward(M, N, mask, kept, dtype):
    from dlrm_amd import ops
    bf16, dtype = dtype == "bf16", DTYPES[dtype]
    turn = rows_per_turn(N, bf16)
    assert turn < M <= 3 * turn and M % turn % 4 != 0
    x, gamma, beta, dy = inputs(M, N, dtype, seed=31)
    y_ref, xh, mean, rstd = norm_ref.norm(x.double(), gamma.double(), beta.double(), 1e-5, True)
    y, mean, rstd = y_ref.to(dtype), mean.float(), rstd.float()
    d_x, _ = strided(x, 3)
    d_y, _ = strided(y, 3)
    if kept:
        source = ops.act8_pack(xh.float().cuda())
        xh = norm_ref.unpack8(source.codes.cpu(), source.exps.cpu(), N)
    else:
        source, xh = d_x, (x.double() - mean.double()[:, None]) * rstd.double()[:, None]
    dx_ref, dg_ref, db_ref, d = norm_ref.norm_grad(dy.double(), xh, rstd.double(), gamma.double(), None if mask is None else y > 0)
    d_dy, _ = strided(dy, 3)
    out, buf = strided(torch.zeros_like(dy), 3)
    top = torch.zeros(1, device="cuda")
    args = dict(mean=None if kept else mean.cuda(), gamma=gamma.cuda(),
                relu_mask={None: None, "y": d_y, "y8": ops.act8_pack(d_y)}[mask])
    dx, dgamma, dbeta, ws = ops.layer_norm_backward(d_dy, source, rstd.cuda(), out=out, dx_absmax=top, **args)
    gd = (d * gamma).abs()
    room = 64 * U * rstd.double()[:, None] * (gd + gd.mean(1, keepdim=True) + xh.abs() * (gd * xh.abs()).mean(1, keepdim=True))
    close(dx, dx_ref, (room + HALF[dtype] * dx_ref.abs() + 1e-30) * (1 + HALF[dtype]))
    close(dgamma, dg_ref, 135 * U * (d * xh).abs().sum(0) + 1e-30)
    close(dbeta, db_ref, 135 * U * d.abs().sum(0) + 1e-30)
    assert top.item() == dx.float().abs().max().item()
    again = ops.layer_norm_backward(d_dy, source, rstd.cuda(), out=d_dy, workspace=ws, **args)
    assert all(torch.equal(a, b) for a, b in zip(again[:3], (dx, dgamma, dbeta)))      # the same bits, also in place
    out.fill_(7.0)
    assert (buf == 7.0).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=list(DTYPES))
@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("M,N", FORWARD)
def test_forward(M, N, relu, dtype):
    from dlrm_amd import ops
    dtype = DTYPES[dtype]
    x, gamma, beta, _ = inputs(M, N, dtype, seed=32)
    y_ref, xh, mean, rstd = norm_ref.norm(x.double(), gamma.double(), beta.double(), 1e-5, relu)
    d_x, _ = strided(x, 3)
    out, buf = strided(torch.zeros_like(x), 3)
    top = torch.zeros(1, device="cuda")
    y, m, r = ops.layer_norm_forward(d_x, gamma.cuda(), beta.cuda(), relu=relu, out=out, y_absmax=top)
    size = x.double().abs().mean(1)
    close(m, mean, 50 * U * size)
    close(r, rstd, 30 * U * rstd + rstd * (50 * U * size * rstd) ** 2)
    room_xh = 34 * U * xh.abs() + (rstd * 50 * U * size)[:, None]
    room = room_xh * gamma.double().abs() + 2 * U * ((xh * gamma).abs() + beta.double().abs()) + HALF[dtype] * y_ref.abs() + 1e-30
    close(y, y_ref, room * (1 + HALF[dtype]))
    assert top.item() == y.float().abs().max().item()
    xhat8, y8 = ops.Act8.empty(M, N), ops.Act8.empty(M, N)
    y2, _, r2 = ops.layer_norm_forward(d_x, gamma.cuda(), beta.cuda(), relu=relu, out=d_x, xhat8=xhat8, y8=y8)
    assert torch.equal(r2, r) and torch.equal(y2, y)
    of_y = ops.act8_pack(y)
    assert torch.equal(y8.codes, of_y.codes) and torch.equal(y8.exps, of_y.exps)
    step = torch.pow(2.0, (xhat8.exps.cpu().double() - 127)).repeat_interleave(32, 1)[:, :N]
    close(ops.act8_unpack(xhat8), xh, step / 2 + room_xh)
    out.fill_(7.0)
    assert (buf == 7.0).all()
