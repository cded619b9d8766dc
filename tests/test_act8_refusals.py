"""What the 8-bit checkpoints and the layer norm refuse, and the float64 form of the checkpoint that the GPU tests compare
with: everything here runs without a GPU (a refused call never reaches a kernel)."""
import ctypes as C

import pytest
import torch

from dlrm_amd import _capi, ops
from tests import norm_ref

P = 1 << 20        # a made-up device address on a 16-byte boundary, never dereferenced


def refused(rc, word):
    assert rc == 1
    assert word in _capi.lib().dlrm_last_error().decode(), _capi.lib().dlrm_last_error()


def act8(codes=P, ld=64, exps=P, exps_ld=2):
    return _capi.Act8Desc(codes, ld, exps, exps_ld)


@pytest.mark.parametrize("entry", ["pack", "unpack"])
def test_pack_refuses(entry):
    L = _capi.lib()

    def call(x=P, dtype=0, rows=4, cols=40, ld=40, a=act8()):
        a = None if a is None else C.byref(a)
        if entry == "pack":
            return L.dlrm_act8_pack(C.c_void_p(x), C.c_int32(dtype), C.c_int64(rows), C.c_int32(cols), C.c_int64(ld), a, None)
        return L.dlrm_act8_unpack(a, C.c_int64(rows), C.c_int32(cols), C.c_void_p(x), C.c_int32(dtype), C.c_int64(ld), None)

    refused(call(a=None), "NULL")
    refused(call(dtype=2), "dtype")
    refused(call(rows=-1), "shape")
    refused(call(cols=0), "shape")
    refused(call(ld=39), "shape")
    refused(call(x=0), "NULL")
    refused(call(x=P + 2), "aligned")
    refused(call(a=act8(codes=0)), "NULL")
    refused(call(a=act8(exps=0)), "NULL")
    refused(call(a=act8(codes=P + 8)), "16-byte")
    refused(call(a=act8(ld=72)), "16-byte")
    refused(call(a=act8(ld=48)), "too small")          # 40 columns are two blocks: 64 codes
    refused(call(a=act8(exps_ld=1)), "too small")
    assert call(x=0, rows=0) == 0                      # no rows: nothing to do


def norm_desc(**kw):
    d = _capi.LayerNormDesc()
    d.M, d.N, d.dtype, d.eps = 4, 40, 0, 1e-5
    d.d_x, d.x_ld, d.d_y, d.y_ld = P, 40, P, 40
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def test_layer_norm_forward_refuses():
    L = _capi.lib()

    def call(**kw):
        return L.dlrm_layer_norm_forward(C.byref(norm_desc(**kw)), None)

    refused(L.dlrm_layer_norm_forward(None, None), "NULL")
    refused(call(M=-1), "shape")
    refused(call(N=0), "shape")
    refused(call(dtype=7), "dtype")
    refused(call(act=2), "act")
    refused(call(eps=-1.0), "eps")
    refused(call(eps=float("nan")), "eps")
    refused(call(d_x=0), "NULL")
    refused(call(d_y=0), "NULL")
    refused(call(x_ld=39), "leading")
    refused(call(y_ld=0), "leading")
    refused(call(d_x=P + 1), "aligned")
    refused(call(xhat8=act8(ld=32)), "too small")
    refused(call(y8=act8(codes=P + 4)), "16-byte")
    assert call(M=0, d_x=0, d_y=0) == 0


def test_layer_norm_backward_refuses():
    L = _capi.lib()

    def call(ws=P, nbytes=1 << 30, **kw):
        d = _capi.LayerNormBwdDesc()
        d.M, d.N = 4, 40
        d.d_x = d.d_dy = d.d_dx = d.d_mean = d.d_rstd = d.d_dgamma = P
        d.x_ld = d.dy_ld = d.dx_ld = d.relu_mask_ld = 40
        for k, v in kw.items():
            setattr(d, k, v)
        return L.dlrm_layer_norm_backward(C.byref(d), C.c_void_p(ws), C.c_size_t(nbytes), None)

    refused(L.dlrm_layer_norm_backward(None, None, C.c_size_t(0), None), "NULL")
    refused(call(M=-3), "shape")
    refused(call(dtype=3), "dtype")
    refused(call(d_dy=0), "NULL")
    refused(call(d_rstd=0), "NULL")
    refused(call(d_dx=0), "NULL")
    refused(call(d_x=0), "exactly one")
    refused(call(xhat8=act8()), "exactly one")
    refused(call(d_mean=0), "means")
    refused(call(d_relu_mask=P, relu_mask8=act8()), "two ReLU masks")
    refused(call(dx_ld=39), "leading")
    refused(call(d_relu_mask=P, relu_mask_ld=39), "leading")
    refused(call(d_dy=P + 2), "aligned")
    refused(call(d_x=0, d_mean=0, xhat8=act8(ld=32)), "too small")
    refused(call(relu_mask8=act8(exps=0)), "NULL")
    refused(call(ws=0), "workspace")
    refused(call(nbytes=16), "workspace")
    refused(call(ws=P + 8), "aligned")
    refused(L.dlrm_layer_norm_backward_workspace_bytes(C.c_int64(4), 8, None), "NULL")


def test_linear_backward_refuses_mixed_operands():
    L = _capi.lib()
    d = _capi.LinearBwdDesc()
    d.M, d.N, d.K = 4, 8, 40
    d.d_dz, d.dz_ld, d.d_w, d.w_ld, d.d_x, d.x_ld = P, 8, P, 40, P, 40
    d.d_dx, d.dx_ld, d.d_dw, d.dw_ld = P, 40, P, 40
    d.x8 = act8()
    refused(L.dlrm_linear_backward_weight(C.byref(d), C.c_void_p(P), C.c_size_t(1 << 30), None), "both")
    d.d_x = 0
    d.x8 = act8(ld=32)
    refused(L.dlrm_linear_backward_weight(C.byref(d), C.c_void_p(P), C.c_size_t(1 << 30), None), "too small")
    d.x8, d.K, d.dw_ld = act8(ld=1 << 31, exps_ld=1 << 26), (1 << 30) + 1, 1 << 31
    refused(L.dlrm_linear_backward_weight(C.byref(d), C.c_void_p(P), C.c_size_t(1 << 62), None), "2^30")
    d.x8, d.K, d.dw_ld = act8(ld=(1 << 24) + 16), 40, 40
    refused(L.dlrm_linear_backward_weight(C.byref(d), C.c_void_p(P), C.c_size_t(1 << 30), None), "2^24")
    d.x8 = act8(codes=0)
    refused(L.dlrm_linear_backward_weight(C.byref(d), C.c_void_p(P), C.c_size_t(1 << 30), None), "NULL")
    d.d_relu_mask, d.relu_mask_ld, d.relu_mask8 = P, 40, act8()
    refused(L.dlrm_linear_backward_data(C.byref(d), None), "two ReLU masks")
    d.d_relu_mask, d.relu_mask8 = 0, act8(exps_ld=1)
    refused(L.dlrm_linear_backward_data(C.byref(d), None), "too small")


def test_plan_entries_refuse_null():
    L = _capi.lib()
    plan = C.c_void_p()
    _capi.check(L.dlrm_plan_create(C.byref(plan)))
    assert L.dlrm_plan_add_layer_norm_forward(plan, None) == -1
    assert L.dlrm_plan_add_layer_norm_backward(plan, None, None, C.c_size_t(0)) == -1
    assert L.dlrm_plan_add_act8_pack(plan, None, C.c_int32(0), C.c_int64(0), C.c_int32(1), C.c_int64(1), None) == -1
    assert L.dlrm_plan_add_act8_unpack(plan, None, C.c_int64(0), C.c_int32(1), None, C.c_int32(0), C.c_int64(1)) == -1
    assert L.dlrm_plan_size(plan) == 0
    L.dlrm_plan_destroy(plan)


def test_python_layer_refuses():
    codes, exps = torch.zeros((3, 64), dtype=torch.int8), torch.zeros((3, 2), dtype=torch.uint8)
    with pytest.raises(TypeError):
        ops.Act8(codes.float(), exps, 40)
    with pytest.raises(TypeError):
        ops.Act8(codes, exps.to(torch.int8), 40)
    with pytest.raises(ValueError):
        ops.Act8(codes, exps, 65)
    with pytest.raises(ValueError):
        ops.Act8(codes[:, :40], exps, 40)
    with pytest.raises(ValueError):
        ops.Act8(codes, exps[:2], 40)
    with pytest.raises(ValueError):
        ops.Act8(codes.t().contiguous().t(), exps, 40)
    with pytest.raises(ValueError):
        ops.Act8(torch.zeros((3, 72), dtype=torch.int8), exps, 40)         # rows of 72 codes: not on 16-byte boundaries
    with pytest.raises(ValueError):
        ops.Act8(torch.zeros((3, 80), dtype=torch.int8)[:, 8:], exps, 40)
    a = ops.Act8(codes, exps, 40)
    assert a.shape == (3, 40)
    x = torch.zeros((3, 40))
    for call in (lambda: ops.act8_pack(x), lambda: ops.act8_unpack(a, out=x), lambda: ops.layer_norm_forward(x),
                 lambda: ops.layer_norm_backward(x, x, torch.zeros(3), torch.zeros(3)),
                 lambda: ops.linear_backward_weight(x, a)):
        with pytest.raises(_capi.DlrmError, match="device tensors"):
            call()


def test_reference_checkpoint():
    """The float64 form itself: half a step, the smallest step that fits, the mark of small positive values."""
    g = torch.Generator().manual_seed(3)
    v = torch.randn(50, 70, generator=g) * torch.exp(6 * torch.randn(50, 1, generator=g))
    v[0] = 0
    v[1, 3] = float("inf")
    v[2, 40] = float("nan")
    v[3, :32] = torch.linspace(0, 127.4, 32)
    v[4, :32] = torch.linspace(0, 127.5, 32)           # the largest rounds to 128: the next step
    v[5] = 1e-42
    v = v.double()
    codes, exps = norm_ref.pack8(v)
    back = norm_ref.unpack8(codes, exps, 70)
    assert (back[0] == 0).all() and (codes[0] == 0).all()
    assert torch.isnan(back[1, :32]).all() and torch.isfinite(back[1, 32:]).all()
    assert torch.isnan(back[2, 32:64]).all() and torch.isfinite(back[2, 64:]).all()
    assert exps[3, 0] == 127 and exps[4, 0] == 128
    assert (back[5] == 0).all() and (codes[5, :70] == -128).all() and (codes[5, 70:] == 0).all()
    ok = ~torch.isnan(back)
    step = torch.pow(2.0, (exps.long() - 127).double()).repeat_interleave(32, 1)[:, :70]
    assert ((back - v).abs() <= step / 2)[ok].all()
    assert (norm_ref.positive8(codes, 70) == (v > 0))[ok].all()
    big = v[6:].abs().reshape(44, -1)
    assert torch.isfinite(big).all()
    low = (exps[6:].long() > 1)
    blocks = torch.nn.functional.pad(v[6:].abs(), (0, 26)).view(44, 3, 32).amax(2)
    assert (blocks >= 63.75 * torch.pow(2.0, (exps[6:].long() - 127).double()))[low].all()


@pytest.mark.parametrize("option", [dict(norm=True), dict(keep8=True)])
def test_the_c_hosted_model_refuses(option):
    """The step hosted in C has neither: it must not train another model than the one asked for."""
    from dlrm_amd.cmodel import CModel
    from dlrm_amd.model import DLRMConfig
    with pytest.raises(ValueError, match="C-hosted"):
        CModel(DLRMConfig.mlperf(**option), 64)
