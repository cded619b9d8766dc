"""8-bit activation checkpoints on the GPU: packing and unpacking bit for bit against the float64 form, and the linear
layer's backward pass that reads them.

Packing is exact arithmetic (division by a power of two, one rounding to an integer), so codes and exponents are compared
for equality.  Weight gradient, element by element: dz is cut into three bf16 pieces that miss at most 2^-26 of an element,
products are exact and every accumulator adds at most 3 M of them in float32 in two levels (the rows of a range, at most a
few thousand, inside the matrix pipe 16 at a time; then the ranges), so with U = 2^-24 the error is below
(3 * rows of a range / 16 + ranges + 4) U sum |dz x| in the worst case; rounding errors of either sign make it the square
root of that in practice, and 64 U sum |dz x| holds for the at most 4099 rows used here with a factor above two to spare
against the worst case of 16-deep additions (3 * 256 / 16 + 17 + 4 = 69 for the longest range, all errors of one sign)."""
import pytest
import torch

from tests import norm_ref
from tests.norm_ref import U

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def strided(v, pad, fill=7.0):
    """device copy of a CPU tensor whose rows are `pad` elements apart, and the buffer around it"""
    buf = torch.full((v.shape[0] + 1, v.shape[1] + pad), fill, dtype=v.dtype, device="cuda")
    view = buf[:-1, :v.shape[1]]
    view.copy_(v)
    return view, buf


def values(M, N, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + 31 * M + N)
    v = torch.randn(M, N, generator=g) * torch.exp(3 * torch.randn(M, 1, generator=g))
    v *= torch.rand(M, N, generator=g) > 0.2
    return v.to(dtype)


@pytest.mark.parametrize("dtype", DTYPES, ids=list(DTYPES))
@pytest.mark.parametrize("pad", [0, 1, 8])
@pytest.mark.parametrize("M,N", [(1, 1), (1, 31), (3, 32), (5, 33), (9, 64), (2, 100), (70, 128), (257, 479), (33, 1024), (3, 2077),
                                 (2, 9001)])
def test_pack_and_unpack(M, N, pad, dtype):
    from dlrm_amd import ops
    v = values(M, N, DTYPES[dtype])
    x, _ = strided(v, pad)
    a = ops.act8_pack(x)
    codes, exps = norm_ref.pack8(v.double())
    assert torch.equal(a.codes.cpu(), codes) and torch.equal(a.exps.cpu(), exps)
    want = norm_ref.unpack8(codes, exps, N)
    for out_dtype in DTYPES.values():
        out, buf = strided(torch.zeros(M, N, dtype=out_dtype), pad)
        got = ops.act8_unpack(a, out=out)
        assert torch.equal(got.cpu().double(), want)
        out.fill_(7.0)
        assert (buf == 7.0).all()          # nothing outside the view was written


def test_values_where_the_rule_turns():
    from dlrm_amd import ops
    rows = [torch.zeros(32),
            torch.linspace(0, 127.4, 32), torch.linspace(0, 127.5, 32), torch.linspace(-127.49999, 3, 32),
            torch.arange(32) + 0.5, torch.arange(32) * 1e-45, torch.full((32,), 2.0 ** -120), torch.full((32,), 2.0 ** -119),
            torch.full((32,), torch.finfo(torch.float32).max), torch.full((32,), -torch.finfo(torch.float32).max),
            torch.cat([torch.tensor([float("inf"), -1.0, 1.0, 0.0]), torch.zeros(28)]),
            torch.cat([torch.tensor([float("nan"), -1.0, 1.0]), torch.ones(29)]),
            torch.cat([torch.tensor([-float("inf")]), -torch.ones(31)]),
            torch.cat([torch.tensor([100.0, 0.49, 0.5, 0.51, -0.49, -0.5, -0.51, 1e-30, -1e-30]), torch.zeros(23)])]
    v = torch.stack([r.float() for r in rows])
    v = torch.cat([v, v.flip(0)], 1)                    # each next to another block
    a = ops.act8_pack(v.cuda())
    codes, exps = norm_ref.pack8(v.double())
    assert torch.equal(a.exps.cpu(), exps)
    finite = torch.isfinite(v)
    assert torch.equal(a.codes.cpu()[finite], codes[finite])
    got, want = ops.act8_unpack(a).cpu().double(), norm_ref.unpack8(codes, exps, 64)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(), want.nan_to_num())
    assert torch.equal(norm_ref.positive8(a.codes.cpu(), 64)[finite], (v > 0)[finite])


def test_no_rows():
    from dlrm_amd import ops
    a = ops.act8_pack(torch.empty((0, 40), device="cuda"))
    assert a.shape == (0, 40) and ops.act8_unpack(a).shape == (0, 40)


def checkpoint(M, K, seed=0):
    """A ReLU output, its checkpoint on the device and the values that stands for."""
    from dlrm_amd import ops
    g = torch.Generator().manual_seed(seed + 17 * M + K)
    x = torch.relu(torch.randn(M, K, generator=g) * torch.exp(0.7 * torch.randn(K, generator=g)))
    a = ops.act8_pack(x.cuda())
    return x, a, norm_ref.unpack8(a.codes.cpu(), a.exps.cpu(), K)


SHAPES = [(1, 1, 1), (1, 7, 5), (31, 4, 33), (32, 64, 64), (33, 65, 31), (70, 1, 300), (130, 130, 130), (257, 512, 13), (300, 1024, 479),
          (2048, 256, 512), (4099, 96, 100), (1030, 200, 1056)]


@pytest.mark.parametrize("pad", [0, 1, 4])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_weight_gradient(M, N, K, pad):
    from dlrm_amd import ops
    _, a, x = checkpoint(M, K)
    g = torch.Generator().manual_seed(M + N)
    dz = torch.randn(M, N, generator=g) * torch.exp(2 * torch.randn(M, 1, generator=g))
    d, _ = strided(dz, pad)
    out, buf = strided(torch.zeros(N, K), pad)
    dw, db, ws = ops.linear_backward_weight(d, a, dw=out)
    want = dz.double().t() @ x
    room = 64 * U * (dz.double().abs().t() @ x.abs()) + 1e-45
    assert ((dw.cpu().double() - want).abs() <= room).all()
    assert ((db.cpu().double() - dz.double().sum(0)).abs() <= 64 * U * dz.double().abs().sum(0)).all()
    again, _, _ = ops.linear_backward_weight(d, a, workspace=ws, want_db=False)
    assert torch.equal(again, dw)                      # a fixed order of additions
    out.fill_(7.0)
    assert (buf == 7.0).all()


@pytest.mark.parametrize("mode", [0, 1, 2])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_data_gradient_masked_by_a_checkpoint(M, N, K, mode):
    """The codes in the mask's place give the bits that the activation itself gives, in every evaluation of the product."""
    from dlrm_amd import ops
    x, a, _ = checkpoint(M, K, seed=5)
    x[0, 0] = 1e-30                                     # rounds to zero and is positive
    a = ops.act8_pack(x.cuda())
    g = torch.Generator().manual_seed(M * N)
    dz, w = torch.randn(M, N, generator=g).cuda(), torch.randn(N, K, generator=g).cuda()
    old = ops.get_gemm_mode()
    ops.set_gemm_mode(mode)
    try:
        for ld in (0, 1):                               # rows of dx on 16 bytes, or not
            out, buf = strided(torch.zeros(M, K), ld)
            got = ops.linear_backward_data(dz, w, relu_mask=a, out=out)
            same, _ = strided(torch.zeros(M, K), ld)    # (rows of the same alignment: the same kernel)
            assert torch.equal(got, ops.linear_backward_data(dz, w, relu_mask=x.cuda(), out=same))
            out.fill_(7.0)
            assert (buf == 7.0).all()
    finally:
        ops.set_gemm_mode(old)


def test_data_gradient_with_weight_planes():
    """... and on weights that were split beforehand."""
    from dlrm_amd import ops
    M, N, K = 4096, 1024, 1024
    x, a, _ = checkpoint(M, K, seed=6)
    g = torch.Generator().manual_seed(1)
    dz, w = torch.randn(M, N, generator=g).cuda(), torch.randn(N, K, generator=g).cuda()
    planes = ops.SplitWeights(w)
    old = ops.get_gemm_mode()
    ops.set_gemm_mode(2)
    try:
        got = ops.linear_backward_data(dz, w, relu_mask=a, w_planes=planes)
        assert torch.equal(got, ops.linear_backward_data(dz, w, relu_mask=x.cuda(), w_planes=planes))
    finally:
        ops.set_gemm_mode(old)


@pytest.mark.parametrize("M,N,K", [(9300, 520, 700), (9300, 518, 701), (22100, 300, 200), (22101, 299, 193), (32800, 60, 500),
                                   (32811, 59, 499)])
def test_weight_gradient_of_every_tile(M, N, K):
    """Batches that give the wide tiles enough row ranges (of up to 576 rows): 3 * 36 matrix additions a range, at most 64 ranges
    here, so 180 U sum |dz x|."""
    from dlrm_amd import ops
    _, a, x = checkpoint(M, K)
    g = torch.Generator().manual_seed(M + N)
    dz = torch.randn(M, N, generator=g) * torch.exp(2 * torch.randn(M, 1, generator=g))
    dw, db, _ = ops.linear_backward_weight(dz.cuda(), a)
    want = dz.double().t() @ x
    assert ((dw.cpu().double() - want).abs() <= 180 * U * (dz.double().abs().t() @ x.abs())).all()
    assert ((db.cpu().double() - dz.double().sum(0)).abs() <= 180 * U * dz.double().abs().sum(0)).all()


def test_weight_gradient_of_wide_values():
    """Columns and samples many decades apart, blocks of zeros, a block that holds a NaN: its columns alone see it."""
    from dlrm_amd import ops
    M, N, K = 200, 70, 160
    g = torch.Generator().manual_seed(9)
    x = torch.randn(M, K, generator=g) * torch.exp(8 * torch.randn(K, generator=g))
    x[:, 64:96] = 0
    dz = torch.randn(M, N, generator=g) * torch.exp(8 * torch.randn(M, 1, generator=g))
    a = ops.act8_pack(x.cuda())
    v = norm_ref.unpack8(a.codes.cpu(), a.exps.cpu(), K)
    dw, _, _ = ops.linear_backward_weight(dz.cuda(), a)
    room = 64 * U * (dz.double().abs().t() @ v.abs())
    assert ((dw.cpu().double() - dz.double().t() @ v).abs() <= room).all()
    x[3, 100] = float("nan")
    bad, _, _ = ops.linear_backward_weight(dz.cuda(), ops.act8_pack(x.cuda()))
    assert torch.isnan(bad[:, 96:128]).all()
    assert torch.equal(bad[:, :96], dw[:, :96]) and torch.equal(bad[:, 128:], dw[:, 128:])


def test_weight_gradient_static_scratch():
    from dlrm_amd import ops
    _, a, _ = checkpoint(300, 64)
    dz = torch.randn(300, 40, generator=torch.Generator().manual_seed(2)).cuda()
    dw, db = torch.empty((40, 64), device="cuda"), torch.empty(40, device="cuda")
    ops.linear_backward_weight_static(dz, a, dw, db)
    want, want_b, _ = ops.linear_backward_weight(dz, a)
    assert torch.equal(dw, want) and torch.equal(db, want_b)


def test_checkpoint_of_another_shape_is_refused():
    from dlrm_amd import ops
    a = ops.act8_pack(torch.ones((8, 40), device="cuda"))
    with pytest.raises(ValueError):
        ops.linear_backward_weight(torch.ones((9, 4), device="cuda"), a)
    with pytest.raises(ValueError):
        ops.linear_backward_data(torch.ones((8, 4), device="cuda"), torch.ones((4, 41), device="cuda"), relu_mask=a)
    with pytest.raises(ValueError):
        ops.act8_pack(torch.ones((8, 41), device="cuda"), out=a)
    with pytest.raises(TypeError):
        ops.act8_pack(torch.ones((8, 40), device="cuda", dtype=torch.float16))
    with pytest.raises(ValueError):
        ops.act8_pack(torch.ones((40, 8), device="cuda").t())


def test_offsets_past_32_bits():
    """More than 2^32 codes: the last rows are what a call on them alone gives.  Small whole numbers, so every sum is exact."""
    from dlrm_amd import ops
    M, K, N, tail = (1 << 22) + 77, 1024, 4, 300
    x = torch.zeros((M, K), dtype=torch.bfloat16, device="cuda")
    x[-tail:] = torch.randint(-8, 9, (tail, K), device="cuda").to(torch.bfloat16)
    a = ops.act8_pack(x)
    last = ops.act8_pack(x[-tail:])
    assert torch.equal(a.codes[-tail:], last.codes) and torch.equal(a.exps[-tail:], last.exps)
    assert not a.codes[:tail].any()
    back = ops.act8_unpack(a, dtype=torch.bfloat16)
    assert torch.equal(back[-tail:], x[-tail:]) and not back[:tail].any()
    del back
    dz = torch.zeros((M, N), device="cuda")
    dz[-tail:] = torch.randint(-3, 4, (tail, N), device="cuda").float()
    dw, db, _ = ops.linear_backward_weight(dz, a)
    want, want_b, _ = ops.linear_backward_weight(dz[-tail:], last)
    assert want.any() and torch.equal(dw, want) and torch.equal(db, want_b)
