"""The model with normalised hidden layers and with 8-bit activation checkpoints: the dense gradients of a train step against the
same step in float64, whose backward pass takes the values of the checkpoints that the step left (they are part of what is
computed, not an error of it).  Tolerance: every product, norm and interaction on the way is within a few 1e-6 of its own
tensor's largest value (the operators' tests), at most eight of them follow each other: 2e-5 of a gradient's largest value."""
import numpy as np
import pytest
import torch

from tests import norm_ref
from tests.oracle_model import make_batch

pytestmark = pytest.mark.gpu


def config(interaction, norm, keep8):
    from dlrm_amd.model import DLRMConfig
    if interaction == "dot":
        return DLRMConfig(table_rows=[50, 3, 1000, 7], dim=16, dense_in=13, bottom=[64, 40, 16], top=[96, 61, 33, 1], lr=0.01, norm=norm,
                          keep8=keep8)
    return DLRMConfig(table_rows=[500] * 3, dim=32, dense_in=20, bottom=[48, 32], top=[32, 17, 1], interaction="cat", loss="mse",
                      pooling="mean", lookups=3, lr=0.01, norm=norm, keep8=keep8)


def run_step(cfg, B=53, **kw):
    from dlrm_amd.model import DLRM
    m = DLRM(cfg, B, seed=3, **kw)
    g = torch.Generator().manual_seed(4)
    for v in m.bottom.beta + m.top.beta:                # (parameters that the start leaves at zero and one)
        v.copy_(0.2 * torch.randn(v.shape, generator=g))
    for v in m.bottom.gamma + m.top.gamma:
        v.copy_(1 + 0.2 * torch.randn(v.shape, generator=g))
    before = m.params.clone()
    dense, idx, off, labels = make_batch(np.random.default_rng(5), cfg, B)
    m.load_batch(torch.from_numpy(dense).cuda(), torch.from_numpy(labels).cuda())
    loss = m.train_step(torch.from_numpy(idx).cuda(), torch.from_numpy(off).cuda())
    torch.cuda.synchronize()
    return m, before, loss.item()


class Reference:
    """A stack in float64 on the parameters a step started with."""

    def __init__(self, stack, before, model):
        def at_start(t):
            return before.as_strided(t.shape, t.stride(), t.storage_offset()).cpu().double()
        self.stack = stack
        self.W, self.b = [at_start(t) for t in stack.W], [at_start(t) for t in stack.b]
        self.g, self.e = [at_start(t) for t in stack.gamma], [at_start(t) for t in stack.beta]

    def forward(self, x):
        s = self.stack
        self.inputs, self.xh, self.rstd = [x], [], []
        for i in range(s.n_layers):
            z = x @ self.W[i].t() + self.b[i]
            if i + 1 < s.n_layers and s.norm:
                x, xh, _, rstd = norm_ref.norm(z, self.g[i], self.e[i], s.norm_eps, True)
                self.xh.append(xh)
                self.rstd.append(rstd)
            else:
                x = z.clamp_min(0) if s.last_relu or i + 1 < s.n_layers else z
            self.inputs.append(x)
        return x

    def backward(self, dz):
        """(gradients by name, gradient of the input)"""
        s, out = self.stack, {}
        for i in reversed(range(s.n_layers)):
            kept = self.inputs[i]
            if i > 0 and s.keep8:
                kept = norm_ref.unpack8(s.y8[i - 1].codes.cpu(), s.y8[i - 1].exps.cpu(), s.y8[i - 1].cols)
                positive = norm_ref.positive8(s.y8[i - 1].codes.cpu(), s.y8[i - 1].cols)
            else:
                positive = kept > 0
            out["W", i], out["b", i] = dz.t() @ kept, dz.sum(0)
            dx = dz @ self.W[i]
            if i == 0:
                return out, dx
            if s.norm:
                xh = self.xh[i - 1]
                if s.keep8:
                    xh = norm_ref.unpack8(s.xhat8[i - 1].codes.cpu(), s.xhat8[i - 1].exps.cpu(), s.xhat8[i - 1].cols)
                dz, out["g", i - 1], out["e", i - 1], _ = norm_ref.norm_grad(dx, xh, self.rstd[i - 1], self.g[i - 1], positive)
            else:
                dz = torch.where(positive, dx, torch.zeros_like(dx))


def check(ref, grads):
    s = ref.stack
    of = {"W": s.dW, "b": s.db, "g": s.dgamma, "e": s.dbeta}
    assert len(grads) == sum(len(v) for v in of.values())
    for (kind, i), want in grads.items():
        got = of[kind][i].cpu().double()
        assert float((got - want).abs().max()) <= 2e-5 * float(want.abs().max()), (kind, i)


@pytest.mark.parametrize("wgrad_stream", [False, True])
@pytest.mark.parametrize("interaction", ["dot", "cat"])
@pytest.mark.parametrize("norm,keep8", [(True, False), (False, True), (True, True)])
def test_gradients(norm, keep8, interaction, wgrad_stream):
    cfg = config(interaction, norm, keep8)
    m, before, loss = run_step(cfg, wgrad_stream=wgrad_stream)
    B, D, F = m.B, cfg.dim, cfg.num_features
    bottom, top = Reference(m.bottom, before, m), Reference(m.top, before, m)
    x0 = bottom.forward(m.x_dense[:, :cfg.dense_in].cpu().double())
    n0 = x0.shape[1]
    pooled = m.feat[:, n0:n0 + cfg.num_tables * D].cpu().double()
    feat = torch.cat([x0, pooled], 1)
    if interaction == "dot":
        f = feat.view(B, F, D)
        li, lj = torch.tril_indices(F, F, -1)
        logit = top.forward(torch.cat([x0, torch.bmm(f, f.transpose(1, 2).contiguous())[:, li, lj]], 1))
    else:
        logit = top.forward(feat)
    t = m.labels.cpu().double().view(-1, 1)
    if cfg.loss == "bce":
        want_loss = torch.nn.functional.binary_cross_entropy_with_logits(logit, t).item()
        dz = (torch.sigmoid(logit) - t) / B
    else:
        want_loss = ((logit - t) ** 2).mean().item()
        dz = 2 * (logit - t) / B
    assert abs(loss - want_loss) <= 1e-5 * abs(want_loss)
    assert float((m.pred.cpu().double() - logit).abs().max()) <= 1e-5 * float(logit.abs().max())
    grads, dinter = top.backward(dz)
    check(top, grads)
    if interaction == "dot":
        S = torch.zeros(B, F, F, dtype=torch.float64)
        S[:, li, lj] = dinter[:, D:]
        d0 = dinter[:, :D] + torch.bmm(S + S.transpose(1, 2), f)[:, 0]
    else:
        d0 = dinter[:, :n0]
    grads, _ = bottom.backward(torch.where(x0 > 0, d0, torch.zeros_like(d0)))
    check(bottom, grads)
    assert torch.equal(m.params, before - cfg.lr * m.grads) or float((m.params - (before - cfg.lr * m.grads)).abs().max()) <= 2e-7 * float(
        before.abs().max())


@pytest.mark.parametrize("norm,keep8", [(True, False), (False, True), (True, True)])
def test_replayed_step_has_the_direct_steps_bits(norm, keep8):
    from dlrm_amd.model import DLRM
    cfg, B, got = config("dot", norm, keep8), 53, []
    for replay in (False, True):
        m = DLRM(cfg, B, seed=3, replay=replay)
        rng = np.random.default_rng(6)
        for _ in range(3):
            dense, idx, off, labels = make_batch(rng, cfg, B)
            m.load_batch(torch.from_numpy(dense).cuda(), torch.from_numpy(labels).cuda())
            loss = m.train_step(torch.from_numpy(idx).cuda(), torch.from_numpy(off).cuda())
        torch.cuda.synchronize()
        got.append((m.params.clone(), m.weight.clone(), loss.clone()))
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_hidden_outputs_share_two_buffers():
    from dlrm_amd.model import DLRM
    cfg = config("dot", True, True)
    m = DLRM(cfg, 8, seed=1)
    assert len({t.data_ptr() for t in m.top_acts[:-1]}) == 2 and m.top_acts[0].data_ptr() == m.top_acts[2].data_ptr()
    # inference leaves no checkpoints behind and predicts what the training forward does
    dense, idx, off, labels = make_batch(np.random.default_rng(5), cfg, 8)
    m.load_batch(torch.from_numpy(dense).cuda(), torch.from_numpy(labels).cuda())
    for a in m.top.y8 + m.top.xhat8:
        a.codes.fill_(5)
    pred = m.forward(torch.from_numpy(idx).cuda(), torch.from_numpy(off).cuda()).clone()
    torch.cuda.synchronize()
    assert all((a.codes == 5).all() for a in m.top.y8 + m.top.xhat8)
    m.train_step(torch.from_numpy(idx).cuda(), torch.from_numpy(off).cuda())
    assert torch.equal(m.pred, pred)
