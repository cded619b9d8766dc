"""Two ranks on the CPU (gloo) train normalised layers with 8-bit checkpoints to the parameters that one process reaches with the
whole batch: gamma and beta are all-reduced with the other dense gradients.  Operators: tests/cpu_ops_shim.py, and the float64 forms
of tests/norm_ref.py for the norm and the checkpoints.  A gradient is summed in another order, so parameters agree to a few 1e-7 of
the largest; 1e-5 as in the other sharded tests."""
import os

import numpy as np
import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from tests import cpu_ops_shim, norm_ref
from tests.test_distributed_cpu import _free_port


def install(ops):
    cpu_ops_shim.install(ops)
    plain_weight, plain_data = ops.linear_backward_weight, ops.linear_backward_data

    def values(a):
        return norm_ref.unpack8(a.codes, a.exps, a.cols) if isinstance(a, ops.Act8) else a.double()

    def act8_pack(x, out=None):
        codes, exps = norm_ref.pack8(x.double())
        out.codes.copy_(codes)
        out.exps.copy_(exps)
        return out

    def layer_norm_forward(x, gamma, beta, eps, relu, out, mean=None, rstd=None, want_stats=True, xhat8=None, y8=None):
        y, xh, m, r = norm_ref.norm(x.double(), gamma.double(), beta.double(), eps, relu)
        for to, v in ((out, y), (mean, m), (rstd, r)):
            if to is not None:
                to.copy_(v)
        for a, v in ((xhat8, xh.float()), (y8, out)):
            if a is not None:
                act8_pack(v, out=a)

    def layer_norm_backward(dy, x, rstd, mean, gamma, relu_mask, out, dgamma, dbeta, workspace):
        xh = values(x) if mean is None else (x.double() - mean.double()[:, None]) * rstd.double()[:, None]
        mask = norm_ref.positive8(relu_mask.codes, relu_mask.cols) if isinstance(relu_mask, ops.Act8) else relu_mask > 0
        dx, dg, db, _ = norm_ref.norm_grad(dy.double(), xh, rstd.double(), gamma.double(), mask)
        for to, v in ((out, dx), (dgamma, dg), (dbeta, db)):
            to.copy_(v)
        return out, dgamma, dbeta, workspace

    def linear_backward_weight(dz, x, **kw):
        return plain_weight(dz, values(x).float(), **kw)

    def linear_backward_data(dz, w, relu_mask=None, out=None):
        if isinstance(relu_mask, ops.Act8):
            relu_mask = norm_ref.positive8(relu_mask.codes, relu_mask.cols).float()
        return plain_data(dz, w, relu_mask=relu_mask, out=out)

    for f in (act8_pack, layer_norm_forward, layer_norm_backward, linear_backward_weight, linear_backward_data):
        setattr(ops, f.__name__, f)


def _worker(rank, world, port, norm, keep8, ret):
    os.environ["MASTER_ADDR"] = "127.0.0.1"
    os.environ["MASTER_PORT"] = str(port)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        from dlrm_amd import ops
        from dlrm_amd.model import DLRM, DLRMConfig
        from tests.oracle_model import make_batch
        install(ops)
        cfg = DLRMConfig(table_rows=[50, 7, 300, 20], dim=16, dense_in=13, bottom=[33, 24, 16], top=[40, 61, 1], lr=0.05, lookups=2,
                         norm=norm, keep8=keep8)
        Bl, L = 6, cfg.lookups
        Bg = Bl * world
        m = DLRM(cfg, Bl, device="cpu", rank=rank, world=world, seed=4)
        one = DLRM(cfg, Bg, device="cpu", seed=4, plan=m.plan)               # (the features in the same order)
        assert torch.equal(m.params, one.params)
        rng, start = np.random.default_rng(7), one.params.clone()
        for _ in range(3):
            dense, idx, off, labels = make_batch(rng, cfg, Bg)

            def ids(tables):
                picked = np.concatenate([idx[t * Bg * L:(t + 1) * Bg * L] for t in tables])
                return torch.from_numpy(picked), torch.arange(len(tables) * Bg + 1) * L
            dense, labels, part = torch.from_numpy(dense), torch.from_numpy(labels), slice(rank * Bl, (rank + 1) * Bl)
            m.load_batch(dense[part], labels[part])
            loss = m.train_step(*ids(m.local_table_ids)).clone()
            dist.all_reduce(loss)
            one.load_batch(dense, labels)
            want = one.train_step(*ids(one.local_table_ids))
            assert abs(loss.item() - want.item()) <= 1e-5 * abs(want.item())
        for a, b in zip(m.bottom.gamma + m.bottom.beta + m.top.gamma + m.top.beta, one.bottom.gamma + one.bottom.beta + one.top.gamma +
                        one.top.beta):
            assert float((a - b).abs().max()) <= 1e-5 * float(b.abs().max())
        assert float((m.params - one.params).abs().max()) <= 1e-5 * float(one.params.abs().max())
        assert float((one.params - start).abs().max()) > 1e-3
        ret[rank] = True
    finally:
        dist.destroy_process_group()


@pytest.mark.parametrize("norm,keep8", [(True, False), (False, True), (True, True)])
def test_two_ranks_train_as_one_process(norm, keep8):
    ret = mp.get_context("spawn").Manager().dict()
    mp.spawn(_worker, args=(2, _free_port(), norm, keep8, ret), nprocs=2, join=True)
    assert dict(ret) == {0: True, 1: True}
