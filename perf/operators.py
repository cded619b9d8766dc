"""What the operators of a normalised MLP layer with 8-bit activation checkpoints are measured on.

Four kinds of pass:
  norm         layer norm over the rows of a [M, N] activation (optional ReLU behind it, optional 8-bit checkpoints)
  norm_grad    its backward pass: input gradient and the two parameter gradients
  checkpoint   an activation into 8 bits and back
  linear_grad  a linear layer's backward pass from the 8-bit checkpoint of its input

An 8-bit checkpoint of a [M, N] tensor holds one signed byte per element and one exponent byte per 32 consecutive columns
of a row: value = code * 2^(exponent - 127).  Code -128 is a positive value that rounds to zero.
"""
import math

import torch

own = False

DEV = "cuda"
EPS = 1e-5


# ------------------------------------------------------------------------------------------------ cases


def listed():
    return [
        # one sample scored by a served model: the widest layer of the Criteo Terabyte top MLP
        dict(name="norm serve one row", op="norm", M=1, N=1024, pad=0, dtype="f32", relu=True, keep=False),
        # pooled vectors of a Criteo Kaggle batch (26 tables x 2048 samples), 16 wide
        dict(name="norm pooled 16 wide", op="norm", M=53248, N=16, pad=0, dtype="f32", relu=False, keep=False),
        # the interaction's 479 columns, rows packed without padding, in bf16
        dict(name="norm bf16 479 wide", op="norm", M=8191, N=479, pad=0, dtype="bf16", relu=False, keep=False),
        # a training step's first top layer at the full batch: both checkpoints leave with the same pass
        dict(name="norm train 65536", op="norm", M=65536, N=1024, pad=0, dtype="f32", relu=True, keep=True),
        # a bottom layer's backward pass at the batch one GPU of eight gets
        dict(name="norm_grad 8192", op="norm_grad", M=8192, N=512, pad=0, dtype="f32", relu=False, keep=False),
        # few, very long rows
        dict(name="norm_grad long bf16", op="norm_grad", M=33, N=16384, pad=0, dtype="bf16", relu=True, keep=False),
        # the full batch again, from the checkpoints that the forward pass left
        dict(name="norm_grad kept 65536", op="norm_grad", M=65536, N=1024, pad=0, dtype="f32", relu=True, keep=True),
        # the interaction's output of a small batch, rows padded to 480 floats
        dict(name="checkpoint 2048 x 479", op="checkpoint", M=2048, N=479, pad=1, dtype="f32"),
        # a whole activation of the full batch
        dict(name="checkpoint bf16 65536", op="checkpoint", M=65536, N=1024, pad=0, dtype="bf16"),
        # Criteo Kaggle's top layer: weight and data gradients
        dict(name="linear_grad 2048", op="linear_grad", M=2048, N=256, K=512, data=True),
        # the first top layer of the Terabyte model at an odd batch: its input is 479 wide
        dict(name="linear_grad 479 in", op="linear_grad", M=16381, N=1024, K=479, data=True),
        # the largest layer at the full batch: the weight gradient alone
        dict(name="linear_grad 65536", op="linear_grad", M=65536, N=1024, K=1024, data=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm_grad", "checkpoint", "linear_grad"])
    if op == "linear_grad":
        M, N, K = _log(rng, 1, 65536), _log(rng, 1, 1024), _log(rng, 13, 1024)
        return dict(op=op, M=M, N=N, K=K, data=rng.random() < 0.5)
    N = _log(rng, 16, 16384)
    M = _log(rng, 1, min(65536, (64 << 20) // N))
    case = dict(op=op, M=M, N=N, pad=rng.choice([0, 0, 1, 8, 37]), dtype=rng.choice(["f32", "bf16"]))
    if op != "checkpoint":
        case.update(relu=rng.random() < 0.5, keep=rng.random() < 0.5)
    return case


def _blocks(n):
    return -(-n // 32)


def work(case):
    M, N = case["M"], case["N"]
    s = 2 if case.get("dtype") == "bf16" else 4
    if case["op"] == "linear_grad":
        K = case["K"]
        products = 2 if case["data"] else 1
        # dz and the checkpoint read, dW and db written; for the data gradient W read and dx written as well
        b = 4 * M * N + M * (K + _blocks(K)) + 4 * N * K + 4 * N
        if case["data"]:
            b += 4 * N * K + 4 * M * K
        return {"bytes": b, "flops": 2 * M * N * K * products}
    kept = M * (N + _blocks(N))
    if case["op"] == "checkpoint":
        return {"bytes": 2 * M * N * s + 2 * kept, "flops": 4 * M * N}
    if case["op"] == "norm":
        stats = 4 * M if case["keep"] else 8 * M
        return {"bytes": 2 * M * N * s + 8 * N + stats + (2 * kept if case["keep"] else 0), "flops": 9 * M * N}
    source = kept + 4 * M if case["keep"] else M * N * s + 8 * M
    mask = (M * N * (1 if case["keep"] else s)) if case["relu"] else 0
    return {"bytes": source + mask + 2 * M * N * s + 12 * N, "flops": 13 * M * N}


# ------------------------------------------------------------------------------------------------ inputs


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) * 2 + 1)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _rows(M, N, pad, dtype):
    """[M, N] view of rows that are `pad` elements apart from each other's end."""
    return torch.empty((M, N + pad), dtype=dtype, device=DEV)[:, :N]


def _activation(g, M, N, pad, dtype):
    """What a linear layer hands to its norm: columns of different spread, an offset per row, a few larger values."""
    x = _rows(M, N, pad, dtype)
    v = _randn(g, M, N)
    v *= torch.exp(0.3 * _randn(g, N))
    v += 0.5 * _randn(g, M, 1)
    v *= torch.where(torch.rand(M, N, generator=g, device=DEV) < 1e-3, 4.0, 1.0)
    x.copy_(v)
    return x


def _to8(v):
    """The 8-bit checkpoint of float32 values [M, N]: codes int8 [M, 32 * blocks] and exponents uint8 [M, blocks]."""
    M, N = v.shape
    nb = _blocks(N)
    u = torch.zeros((M, nb * 32), dtype=torch.float32, device=v.device)
    u[:, :N] = v
    u = u.view(M, nb, 32)
    bits = u.abs().amax(2).contiguous().view(torch.int32)
    e = (((bits + 0x10000) >> 23) - 6).clamp_min(1)
    q = torch.round(u * ((254 - e) << 23).view(torch.float32)[:, :, None])
    q = torch.where((q == 0) & (u > 0), -128.0, q)
    return q.view(M, nb * 32).to(torch.int8), e.to(torch.uint8)


def _from8(codes, exps, N):
    """The values a checkpoint stands for, float32 [M, N]."""
    M, nb = exps.shape
    q = codes.to(torch.float32)
    q = torch.where(codes == -128, 0.0, q)
    step = (exps.to(torch.int32) << 23).view(torch.float32)
    return (q.view(M, nb, 32) * step[:, :, None]).view(M, nb * 32)[:, :N]


def _positive(codes, N):
    return ((codes > 0) | (codes == -128))[:, :N]


def prepare(case, seed):
    g = _gen(seed)
    M, N = case["M"], case["N"]
    if case["op"] == "linear_grad":
        K = case["K"]
        x = torch.relu(_randn(g, M, K) * torch.exp(0.5 * _randn(g, K)))
        codes, exps = _to8(x)
        del x
        # a loss gradient: every sample its own size, a third of it cut by the ReLU behind this layer
        dz = _randn(g, M, N) * torch.exp(_randn(g, M, 1)) / M
        dz *= torch.rand(M, N, generator=g, device=DEV) > 1 / 3
        w = _randn(g, N, K) * (2.0 / (N + K)) ** 0.5
        return dict(case=case, codes=codes, exps=exps, dz=dz, w=w, dw=torch.empty_like(w), db=torch.empty(N, device=DEV),
                    dx=torch.empty((M, K), device=DEV) if case["data"] else None)
    dtype = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
    pad = case["pad"]
    x = _activation(g, M, N, pad, dtype)
    s = dict(case=case, x=x)
    if case["op"] == "checkpoint":
        s["codes"] = torch.empty((M, 32 * _blocks(N)), dtype=torch.int8, device=DEV)
        s["exps"] = torch.empty((M, _blocks(N)), dtype=torch.uint8, device=DEV)
        s["out"] = _rows(M, N, pad, dtype)
        return s
    s["gamma"] = 1.0 + 0.1 * _randn(g, N)
    s["beta"] = 0.1 * _randn(g, N)
    s["out"] = _rows(M, N, pad, dtype)
    s["mean"], s["rstd"] = torch.empty(M, device=DEV), torch.empty(M, device=DEV)
    if case["op"] == "norm":
        if case["keep"]:
            for k in ("xhat", "y"):
                s[k + "_codes"] = torch.empty((M, 32 * _blocks(N)), dtype=torch.int8, device=DEV)
                s[k + "_exps"] = torch.empty((M, _blocks(N)), dtype=torch.uint8, device=DEV)
        return s
    dy = _rows(M, N, pad, dtype)
    dy.copy_(_randn(g, M, N) * torch.exp(_randn(g, M, 1)) / M)
    s.update(dy=dy, dgamma=torch.empty(N, device=DEV), dbeta=torch.empty(N, device=DEV))
    xhat, mean, rstd = _normalised(x)
    s["mean"].copy_(mean[:, 0])
    s["rstd"].copy_(rstd[:, 0])
    y = xhat * s["gamma"] + s["beta"]
    if case["relu"]:
        y = torch.relu(y)
    if case["keep"]:
        s["xhat_codes"], s["xhat_exps"] = _to8(xhat)
        s["y_codes"], s["y_exps"] = _to8(y.to(dtype).float())
        del s["x"]
    else:
        s["y"] = _rows(M, N, pad, dtype)
        s["y"].copy_(y)
    return s


# ------------------------------------------------------------------------------------------------ the passes


def _normalised(x):
    x = x.float()
    mean = x.sum(1, keepdim=True) / x.shape[1]
    d = x - mean
    rstd = 1.0 / torch.sqrt((d * d).sum(1, keepdim=True) / x.shape[1] + EPS)
    return d * rstd, mean, rstd


def _plain_norm(s):
    case, N = s["case"], s["case"]["N"]
    xhat, mean, rstd = _normalised(s["x"])
    y = xhat * s["gamma"] + s["beta"]
    if case["relu"]:
        y = torch.clamp_min(y, 0.0)
    y = y.to(s["x"].dtype)
    out = dict(y=y, rstd=rstd[:, 0])
    if case["keep"]:
        out["xhat8"] = _from8(*_to8(xhat), N).to(torch.bfloat16)
        out["y8"] = _from8(*_to8(y.float()), N).to(torch.bfloat16)
    else:
        out["mean"] = mean[:, 0]
    return out


def _plain_norm_grad(s):
    case, N = s["case"], s["case"]["N"]
    rstd = s["rstd"][:, None]
    if case["keep"]:
        xhat = _from8(s["xhat_codes"], s["xhat_exps"], N)
    else:
        xhat = (s["x"].float() - s["mean"][:, None]) * rstd
    d = s["dy"].float()
    if case["relu"]:
        d = torch.where(_positive(s["y_codes"], N) if case["keep"] else s["y"] > 0, d, 0.0)
    gd = d * s["gamma"]
    c1 = gd.sum(1, keepdim=True) / N
    c2 = (gd * xhat).sum(1, keepdim=True) / N
    dx = rstd * (gd - c1 - xhat * c2)
    return dict(dx=dx.to(s["dy"].dtype), dgamma=(d * xhat).sum(0), dbeta=d.sum(0))


def _plain_linear_grad(s):
    K = s["case"]["K"]
    out = dict(dw=s["dz"].t() @ _from8(s["codes"], s["exps"], K), db=s["dz"].sum(0))
    if s["case"]["data"]:
        out["dx"] = torch.where(_positive(s["codes"], K), s["dz"] @ s["w"], 0.0)
    return out


def _run_own(s):
    from dlrm_amd import ops
    case, N = s["case"], s["case"]["N"]
    if case["op"] == "norm":
        if not case["keep"]:
            y, mean, rstd = ops.layer_norm_forward(s["x"], s["gamma"], s["beta"], eps=EPS, relu=case["relu"], out=s["out"],
                                                   mean=s["mean"], rstd=s["rstd"])
            return dict(y=y, rstd=rstd, mean=mean)
        xhat8 = ops.Act8(s["xhat_codes"], s["xhat_exps"], N)
        y8 = ops.Act8(s["y_codes"], s["y_exps"], N)
        y, _, rstd = ops.layer_norm_forward(s["x"], s["gamma"], s["beta"], eps=EPS, relu=case["relu"], out=s["out"],
                                            mean=s["mean"], rstd=s["rstd"], xhat8=xhat8, y8=y8)
        return dict(y=y, rstd=rstd, xhat8=ops.act8_unpack(xhat8, dtype=torch.bfloat16),
                    y8=ops.act8_unpack(y8, dtype=torch.bfloat16))
    if case["op"] == "norm_grad":
        if case["keep"]:
            x = ops.Act8(s["xhat_codes"], s["xhat_exps"], N)
            mask = ops.Act8(s["y_codes"], s["y_exps"], N)
        else:
            x, mask = s["x"], s["y"]
        dx, dgamma, dbeta, s["ws"] = ops.layer_norm_backward(
            s["dy"], x, s["rstd"], mean=None if case["keep"] else s["mean"], gamma=s["gamma"],
            relu_mask=mask if case["relu"] else None, out=s["out"], dgamma=s["dgamma"], dbeta=s["dbeta"],
            workspace=s.get("ws"))
        return dict(dx=dx, dgamma=dgamma, dbeta=dbeta)
    if case["op"] == "checkpoint":
        a = ops.act8_pack(s["x"], out=ops.Act8(s["codes"], s["exps"], N))
        return ops.act8_unpack(a, out=s["out"])
    x8 = ops.Act8(s["codes"], s["exps"], case["K"])
    dw, db, s["ws"] = ops.linear_backward_weight(s["dz"], x8, dw=s["dw"], db=s["db"], workspace=s.get("ws"))
    out = dict(dw=dw, db=db)
    if case["data"]:
        out["dx"] = ops.linear_backward_data(s["dz"], s["w"], relu_mask=x8, out=s["dx"])
    return out


def run(state):
    if own:
        return _run_own(state)
    op = state["case"]["op"]
    if op == "norm":
        return _plain_norm(state)
    if op == "norm_grad":
        return _plain_norm_grad(state)
    if op == "checkpoint":
        return _from8(*_to8(state["x"].float()), state["case"]["N"]).to(state["x"].dtype)
    return _plain_linear_grad(state)


# ------------------------------------------------------------------------------------------------ 64 bits


def _values64(codes, exps, N):
    """code * 2^(exponent - 127), column by column of a block."""
    block = torch.arange(N, device=codes.device) // 32
    q = codes[:, :N].double()
    return torch.where(codes[:, :N] == -128, 0.0, torch.ldexp(q, exps[:, block].long() - 127))


def _rounded64(v):
    """Every value to the nearest multiple of its block's step, ties to the even one; the step is the smallest power of two
    with max |v| below 127.5 steps."""
    M, N = v.shape
    nb = _blocks(N)
    u = torch.nn.functional.pad(v, (0, nb * 32 - N)).view(M, nb, 32)
    frac, e = torch.frexp(u.abs().amax(2, keepdim=True))
    e = torch.clamp_min(torch.where(frac < 127.5 / 128, e - 7, e - 6), -126)
    return torch.ldexp(torch.round(torch.ldexp(u, -e)), e).view(M, nb * 32)[:, :N]


def exact(case, seed):
    s = prepare(case, seed)
    N = case["N"]
    if case["op"] == "checkpoint":
        return _rounded64(s["x"].double())
    if case["op"] == "linear_grad":
        K = case["K"]
        dz = s["dz"].double()
        out = dict(dw=torch.mm(dz.t(), _values64(s["codes"], s["exps"], K)), db=dz.sum(0))
        if case["data"]:
            c = s["codes"][:, :K]
            out["dx"] = torch.mm(dz, s["w"].double()).masked_fill_(~((c > 0) | (c == -128)), 0.0)
        return out
    gamma, beta = s["gamma"].double(), s["beta"].double()
    if case["op"] == "norm":
        x = s["x"].double()
        var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
        rstd = (var + EPS).rsqrt()
        xhat = (x - mean).mul_(rstd)
        y = torch.addcmul(beta, xhat, gamma)
        if case["relu"]:
            y.clamp_min_(0)
        out = dict(y=y, rstd=rstd.flatten())
        if case["keep"]:
            out["xhat8"], out["y8"] = _rounded64(xhat), _rounded64(y)
        else:
            out["mean"] = mean.flatten()
        return out
    rstd = s["rstd"].double()[:, None]
    if case["keep"]:
        xhat = _values64(s["xhat_codes"], s["xhat_exps"], N)
        positive = (s["y_codes"][:, :N] > 0) | (s["y_codes"][:, :N] == -128)
    else:
        xhat = (s["x"].double() - s["mean"].double()[:, None]) * rstd
        positive = s["y"] > 0
    d = s["dy"].double()
    if case["relu"]:
        d = d * positive
    gd = d * gamma
    dx = rstd * (gd - gd.mean(1, keepdim=True) - xhat * (gd * xhat).mean(1, keepdim=True))
    return dict(dx=dx, dgamma=(d * xhat).sum(0), dbeta=d.sum(0))
