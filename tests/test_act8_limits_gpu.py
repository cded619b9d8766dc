"""The weight gradient from an 8-bit checkpoint at the ends of its ranges of sizes.  Small whole numbers, so that every sum is exact."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_weight_gradient_of_the_most_rows():
    """2^31 - 1 rows: 256 ranges of 2^23 rows, the last of which would end at 2^31."""
    from dlrm_amd import ops
    M, N, K, part = (1 << 31) - 1, 4, 13, 300
    g = torch.Generator().manual_seed(1)
    dz = torch.zeros((M, N), device="cuda")
    codes = torch.zeros((M, 32), dtype=torch.int8, device="cuda")
    exps = torch.full((M, 1), 127, dtype=torch.uint8, device="cuda")       # (steps of one)
    want, want_b = torch.zeros(N, K), torch.zeros(N)
    for at in (0, 1 << 30, M - part):
        d = torch.randint(-3, 4, (part, N), generator=g).float()
        c = torch.randint(-8, 9, (part, K), generator=g)
        dz[at:at + part] = d.cuda()
        codes[at:at + part, :K] = c.to(torch.int8).cuda()
        want, want_b = want + d.t() @ c.float(), want_b + d.sum(0)
    dw, db, _ = ops.linear_backward_weight(dz, ops.Act8(codes, exps, K))
    assert torch.equal(dw.cpu(), want) and torch.equal(db.cpu(), want_b)
    del dz, codes, exps
    torch.cuda.empty_cache()
