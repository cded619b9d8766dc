"""A recorded step owns the memory that its entries point to, also what the operators allocated while they were recorded."""
import gc
import weakref

import pytest
import torch

from dlrm_amd import ops
from dlrm_amd.plan import StepRecorder


def test_results_of_recorded_operators_live_as_long_as_the_plan():
    refs = []

    def made(*shape):
        t = torch.empty(shape)
        refs.append(weakref.ref(t))
        return t

    @ops._op
    def one(x):
        return made(3)

    @ops._op
    def several(x, out=None):
        a = ops.Act8(made(2, 64).to(torch.int8), torch.zeros((2, 2), dtype=torch.uint8), 40)
        refs[-1] = weakref.ref(a.codes)
        return made(4), a, None, 3, made(5)

    x = torch.zeros(1)
    rec = StepRecorder(x, x)
    with rec:
        one(x)
        several(x)
    gc.collect()
    assert len(refs) == 4 and all(r() is not None for r in refs)
    del rec
    gc.collect()
    assert all(r() is None for r in refs)
    one(x), several(x)                              # without a recorder nothing is held
    gc.collect()
    assert all(r() is None for r in refs)


@pytest.mark.gpu
def test_replay_writes_no_memory_of_others():
    """Outputs and workspaces left to the operators and dropped by the caller: tensors of the same sizes that are made afterwards
    stay as they are."""
    M, N, K = 300, 96, 160
    g = torch.Generator().manual_seed(1)
    x, dy, inner = (torch.randn(M, n, generator=g).cuda() for n in (N, N, K))
    rstd = torch.rand(M, generator=g).cuda()
    dw, want = torch.zeros((N, K), device="cuda"), torch.zeros((N, K), device="cuda")
    idx = torch.zeros(1, dtype=torch.int64, device="cuda")

    def step(dw):
        xh = ops.act8_pack(x)
        dx, _, _, _ = ops.layer_norm_backward(dy, xh, rstd)
        ops.linear_backward_weight(dx, ops.act8_pack(inner), dw=dw)

    step(want)
    rec = StepRecorder(idx, idx)
    with rec:
        step(dw)
    gc.collect()
    others = []
    for nbytes in (M * N, M * N * 4, M * K, M * 3, M * 5, N * 4, ops.layer_norm_backward_workspace_bytes(M, N),
                   ops.linear_backward_weight_workspace_bytes(M, N, K, True)):
        others += [torch.full((nbytes,), 77, dtype=torch.uint8, device="cuda") for _ in range(4)]
    for _ in range(3):
        rec.plan.run(0, rec.size)
        torch.cuda.synchronize()
        assert torch.equal(dw, want) and all((t == 77).all() for t in others)
        dw.zero_()
