"""What the linear layer's backward pass refuses beside an 8-bit checkpoint: operands of other types and shapes, whose launch would
read or write outside them.  Without a GPU: the tensors live on the CPU, and a call that gets past its checks ends in `launched`."""
import pytest
import torch

from dlrm_amd import _capi, ops

M, N, K = 6, 5, 40


@pytest.fixture
def launched(monkeypatch):
    calls = []
    monkeypatch.setattr(ops, "_device_of", lambda t: t.get_device())
    monkeypatch.setattr(ops, "_require_cuda", lambda *t: None)
    monkeypatch.setattr(ops, "_emit", lambda name, *args: calls.append((name,) + args))

    class Lib:
        @staticmethod
        def dlrm_linear_backward_weight_static(d, stream):
            calls.append(("static", d))
            return 0
    lib = _capi.lib()
    for n in ("dlrm_linear_backward_weight_act8_workspace_bytes", "dlrm_linear_backward_weight_workspace_bytes"):
        setattr(Lib, n, getattr(lib, n))
    monkeypatch.setattr(_capi, "lib", lambda: Lib)
    monkeypatch.setattr(ops, "_stream", lambda: None)
    return calls


def act8(rows=M, cols=K):
    nb = (cols + 31) // 32
    return ops.Act8(torch.zeros((rows, 32 * nb), dtype=torch.int8), torch.zeros((rows, nb), dtype=torch.uint8), cols)


def f32(*shape):
    return torch.zeros(shape)


BAD_DZ = [f32(M, N).bfloat16(), f32(M, N).double(), f32(M + 1, N), f32(N, M).t(), f32(M * N)]


@pytest.mark.parametrize("static", [False, True])
def test_weight_gradient(launched, static):
    def call(dz=f32(M, N), x=act8(), dw=f32(N, K), db=f32(N), **kw):
        return (ops.linear_backward_weight_static if static else ops.linear_backward_weight)(dz, x, dw, db, **kw)
    bad = [dict(dz=t) for t in BAD_DZ]
    bad += [dict(dw=t) for t in (f32(N, K).bfloat16(), f32(N, K - 1), f32(N - 1, K), f32(K, N).t(), f32(N * K))]
    bad += [dict(db=t) for t in (f32(N).double(), f32(N - 1), f32(2 * N)[::2])]
    if not static:
        bad += [dict(workspace=torch.zeros(1, dtype=torch.uint8).expand(1 << 20))]
    for kw in bad:
        with pytest.raises((TypeError, ValueError)):
            call(**kw)
    assert launched == []
    call()
    call(db=None, dw=f32(N, K + 3)[:, :K], dz=f32(M, N + 1)[:, 1:])
    assert len(launched) == 2


def test_data_gradient(launched):
    def call(dz=f32(M, N), w=f32(N, K), relu_mask=act8(), **kw):
        return ops.linear_backward_data(dz, w, relu_mask=relu_mask, **kw)
    bad = [dict(dz=t) for t in BAD_DZ]
    bad += [dict(w=t) for t in (f32(N, K).bfloat16(), f32(N, K + 1), f32(N + 1, K), f32(K, N).t())]
    bad += [dict(out=t) for t in (f32(M, K).bfloat16(), f32(M, K - 1), f32(M - 1, K), f32(K, M).t())]
    bad += [dict(relu_mask=act8(M + 1)), dict(relu_mask=act8(cols=K + 1))]
    for kw in bad:
        with pytest.raises((TypeError, ValueError)):
            call(**kw)
    assert launched == []
    assert call().shape == (M, K)
    call(out=f32(M, K + 3)[:, :K], w=f32(N, K + 1)[:, :K])
    assert len(launched) == 2
