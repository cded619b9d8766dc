"""Layer norm forward and backward on the GPU against float64, element by element.

Tolerances, with U = 2^-24 (half a float32 step, relative).  A row's sums are chains of at most 32 additions in a lane (40 in
the longest row here) followed by at most 10 across lanes, so a sum is off by at most 50 U times the sum of magnitudes.
  mean   50 U mean|x|
  rstd   the squares' sum and the mean's error (whose first-order share is zero: deviations add up to nothing) give 25 U + 4 U
  xh     34 U |xh| + rstd * 50 U mean|x|;  y one product and one sum more, and its own rounding where it is bf16
  dx     two such sums, three products:  64 U rstd (|gd| + mean|gd| + |xh| mean|gd xh|), and the rounding of dx
  dgamma, dbeta   chains of the rows of a team, the teams of a workgroup, the workgroups: at most 160 U times the magnitudes'
         sum for the up to 4099 rows used here
A checkpoint's value is within half a step (its block's largest magnitude / 127) of the value it was made from."""
import pytest
import torch

from tests import norm_ref
from tests.norm_ref import U

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}      # half a step of the stored type
SHAPES = [(1, 1), (1, 16), (3, 2), (3, 17), (5, 31), (37, 32), (65, 33), (2, 64), (1000, 128), (9, 255), (33, 479), (4, 512),
          (131, 1000), (3, 1024), (17, 1300), (2, 2048), (5, 2049), (3, 4096), (2, 5000), (3, 8192), (2, 8200), (2, 16384), (3, 16385),
          (1, 40001),
          # workgroups of 3, 5, 6, 10, 14 and 15 waves, with more rows than workgroups
          (1300, 1030), (1100, 1201), (770, 2263), (513, 2856), (258, 5029), (257, 6714), (259, 11167), (300, 15300)]


def strided(v, pad, fill=7.0):
    buf = torch.full((v.shape[0] + 1, v.shape[1] + pad), fill, dtype=v.dtype, device="cuda")
    view = buf[:-1, :v.shape[1]]
    view.copy_(v)
    return view, buf


def inputs(M, N, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + 1009 * M + N)
    x = (torch.randn(M, N, generator=g) * torch.exp(0.5 * torch.randn(N, generator=g)) + torch.randn(M, 1, generator=g)).to(dtype)
    gamma, beta = 1 + 0.3 * torch.randn(N, generator=g), 0.3 * torch.randn(N, generator=g)
    dy = (torch.randn(M, N, generator=g) * torch.exp(torch.randn(M, 1, generator=g))).to(dtype)
    return x, gamma, beta, dy


def close(got, want, room):
    """got == want within room, element by element"""
    err = (got.detach().cpu().double() - want).abs()
    assert (err <= room).all(), "off by up to %.3g of what is allowed" % float((err / room).nan_to_num(0).max())


@pytest.mark.parametrize("dtype", DTYPES, ids=list(DTYPES))
@pytest.mark.parametrize("pad", [0, 1, 8])
@pytest.mark.parametrize("M,N", SHAPES)
def test_forward(M, N, pad, dtype):
    from dlrm_amd import ops
    dtype = DTYPES[dtype]
    relu, plain = (M + N) % 2 == 0, N % 3 == 0
    x, gamma, beta, _ = inputs(M, N, dtype)
    g, b = (torch.ones(N), torch.zeros(N)) if plain else (gamma, beta)
    y_ref, xh, mean, rstd = norm_ref.norm(x.double(), g.double(), b.double(), 1e-5, relu)
    d_x, _ = strided(x, pad)
    out, buf = strided(torch.zeros_like(x), pad)
    d_max = torch.zeros(1, device="cuda")
    y, m, r = ops.layer_norm_forward(d_x, None if plain else gamma.cuda(), None if plain else beta.cuda(), relu=relu, out=out,
                                     y_absmax=d_max)
    size = x.double().abs().mean(1)
    close(m, mean, 50 * U * size)
    close(r, rstd, 30 * U * rstd + U * rstd * (50 * U * size * rstd) ** 2 / U)
    room_xh = 34 * U * xh.abs() + (rstd * 50 * U * size)[:, None]
    room = room_xh * g.double().abs() + 2 * U * ((xh * g).abs() + b.double().abs()) + HALF[dtype] * y_ref.abs() + 1e-30
    if dtype == torch.bfloat16:
        room = room * (1 + HALF[dtype])
    close(y, y_ref, room)
    assert d_max.item() == y.float().abs().max().item()
    # the same call with checkpoints: the same y, y8 = the checkpoint of y, xh8 within half a step of xh
    xhat8, y8 = ops.Act8.empty(M, N), ops.Act8.empty(M, N)
    out2, _ = strided(torch.zeros_like(x), pad)         # (rows of the same alignment: the same kernel)
    y2, _, r2 = ops.layer_norm_forward(d_x, None if plain else gamma.cuda(), None if plain else beta.cuda(), relu=relu, out=out2,
                                       xhat8=xhat8, y8=y8)
    assert torch.equal(y2, y) and torch.equal(r2, r)
    of_y = ops.act8_pack(y)
    assert torch.equal(y8.codes, of_y.codes) and torch.equal(y8.exps, of_y.exps)
    step = torch.pow(2.0, (xhat8.exps.cpu().double() - 127)).repeat_interleave(32, 1)[:, :N]
    close(ops.act8_unpack(xhat8), xh, step / 2 + room_xh)
    assert (xhat8.codes.cpu()[:, N:] == 0).all() and (y8.codes.cpu()[:, N:] == 0).all()
    out.fill_(7.0)
    assert (buf == 7.0).all()
    # in place
    y3, none_m, none_r = ops.layer_norm_forward(d_x, None if plain else gamma.cuda(), None if plain else beta.cuda(), relu=relu,
                                                out=d_x, want_stats=False)
    assert torch.equal(y3, y2) and none_m is None and none_r is None


@pytest.mark.parametrize("dtype", DTYPES, ids=list(DTYPES))
@pytest.mark.parametrize("pad", [0, 1, 8])
@pytest.mark.parametrize("kept", [False, True], ids=["from_x", "from_8"])
@pytest.mark.parametrize("M,N", SHAPES + [(4099, 24), (4099, 65)])
def test_backward(M, N, kept, pad, dtype):
    from dlrm_amd import ops
    dtype = DTYPES[dtype]
    x, gamma, beta, dy = inputs(M, N, dtype, seed=1)
    masks = {0: None, 1: "y", 2: "y8"}
    kind = masks[(M + N + pad) % 3]
    plain = N % 5 == 0
    g = torch.ones(N) if plain else gamma
    y_ref, xh, mean, rstd = norm_ref.norm(x.double(), gamma.double(), beta.double(), 1e-5, True)
    y = y_ref.to(dtype)
    mean, rstd = mean.float(), rstd.float()
    d_x, _ = strided(x, pad)
    d_y, _ = strided(y, pad)
    if kept:
        xhat8 = ops.act8_pack(xh.float().cuda())
        source, xh = xhat8, norm_ref.unpack8(xhat8.codes.cpu(), xhat8.exps.cpu(), N)
    else:
        source, xh = d_x, (x.double() - mean.double()[:, None]) * rstd.double()[:, None]
    relu_mask = {None: None, "y": d_y, "y8": ops.act8_pack(d_y)}[kind]
    dx_ref, dg_ref, db_ref, d = norm_ref.norm_grad(dy.double(), xh, rstd.double(), g.double(), None if kind is None else y > 0)
    d_dy, _ = strided(dy, pad)
    out, buf = strided(torch.zeros_like(dy), pad)
    d_max = torch.zeros(1, device="cuda")
    args = dict(mean=None if kept else mean.cuda(), gamma=None if plain else gamma.cuda(), relu_mask=relu_mask)
    dx, dgamma, dbeta, ws = ops.layer_norm_backward(d_dy, source, rstd.cuda(), out=out, dx_absmax=d_max, **args)
    gd = (d * g).abs()
    room = 64 * U * rstd.double()[:, None] * (gd + gd.mean(1, keepdim=True) + xh.abs() * (gd * xh.abs()).mean(1, keepdim=True))
    close(dx, dx_ref, (room + HALF[dtype] * dx_ref.abs() + 1e-30) * (1 + HALF[dtype]))
    close(dgamma, dg_ref, 160 * U * (d * xh).abs().sum(0) + 1e-30)
    close(dbeta, db_ref, 160 * U * d.abs().sum(0) + 1e-30)
    assert d_max.item() == dx.float().abs().max().item()
    kept_dx = dx.clone()
    # one parameter's gradient alone, none, the same bits again, in place
    only_b = torch.full((N,), 7.0, device="cuda")
    out2, _ = strided(torch.zeros_like(dy), pad)        # (rows of the same alignment: the same kernel)
    dx2, dg2, db2, ws = ops.layer_norm_backward(d_dy, source, rstd.cuda(), out=out2, dbeta=only_b, want_params=False, workspace=ws, **args)
    assert torch.equal(dx2, kept_dx) and dg2 is None and torch.equal(db2, dbeta)
    dx3, _, _, _ = ops.layer_norm_backward(d_dy, source, rstd.cuda(), out=d_dy, workspace=ws, dgamma=torch.empty(N, device="cuda"), **args)
    assert torch.equal(dx3, kept_dx)
    out.fill_(7.0)
    assert (buf == 7.0).all()


@pytest.mark.parametrize("M,N", [(1, 24), (33, 24), (5, 100), (1025, 256), (3, 300), (2, 1500), (1, 1500)])
def test_in_place_with_maxima(M, N):
    """The output over the input, in batches whose last rows do not fill a workgroup: its largest magnitude is that of the rows."""
    from dlrm_amd import ops
    x, gamma, beta, dy = (t.cuda() for t in inputs(M, N, torch.float32, seed=17))
    y, mean, rstd = ops.layer_norm_forward(x, gamma * 1e-3, beta * 1e-3)
    dx, _, _, _ = ops.layer_norm_backward(dy, x, rstd, mean=mean, gamma=gamma * 1e-3)
    for _ in range(5):
        top, into = torch.zeros(1, device="cuda"), x.clone()
        ops.layer_norm_forward(into, gamma * 1e-3, beta * 1e-3, out=into, y_absmax=top)
        assert torch.equal(into, y) and top.item() == y.abs().max().item()
        top, into = torch.zeros(1, device="cuda"), dy.clone()
        ops.layer_norm_backward(into, x, rstd, mean=mean, gamma=gamma * 1e-3, out=into, dx_absmax=top)
        assert torch.equal(into, dx) and top.item() == dx.abs().max().item()


def test_gradient_against_differences():
    """dx, dgamma and dbeta against central differences of the float64 forward formula, contracted with random directions: the
    differences of a loss L = sum(y r) with a step of 1e-5 are exact to about 1e-9 of the gradients' size, the kernel's own
    rounding (64 U of sums of magnitudes) is what is left."""
    from dlrm_amd import ops
    M, N = 7, 130
    x, gamma, beta, r = inputs(M, N, torch.float32, seed=4)
    x64, g64, b64 = x.double(), gamma.double(), beta.double()

    def loss(xx, gg, bb):
        y, _, _, _ = norm_ref.norm(xx, gg, bb, 1e-5, True)
        return float((y * r.double()).sum())

    y, mean, rstd = ops.layer_norm_forward(x.cuda(), gamma.cuda(), beta.cuda(), relu=True)
    dx, dg, db, _ = ops.layer_norm_backward(r.cuda(), x.cuda(), rstd, mean=mean, gamma=gamma.cuda(), relu_mask=y)
    gen = torch.Generator().manual_seed(8)
    # (no element of y is so near zero that the steps carry it across the kink)
    assert norm_ref.norm(x64, g64, b64, 1e-5, False)[0].abs().min() > 1e-4
    for grad, at in ((dx, 0), (dg, 1), (db, 2)):
        for _ in range(5):
            v = torch.randn(grad.shape, generator=gen).double()
            v /= v.abs().max()
            h = 1e-5
            ends = []
            for s in (h, -h):
                p = [x64, g64, b64]
                p[at] = p[at] + s * v
                ends.append(loss(*p))
            diff = (ends[0] - ends[1]) / (2 * h)
            got = float((grad.cpu().double() * v).sum())
            assert abs(got - diff) <= 1e-5 * float((grad.cpu().double() * v).abs().sum())


def test_large_offset():
    """Rows far from zero: deviations are squared after the mean is known."""
    from dlrm_amd import ops
    g = torch.Generator().manual_seed(5)
    x = (torch.randn(20, 640, generator=g) + 4096.0)
    y, mean, rstd = ops.layer_norm_forward(x.cuda())
    ref, xh, m, r = norm_ref.norm(x.double(), torch.ones(640).double(), torch.zeros(640).double(), 1e-5, False)
    close(mean, m, 50 * U * m.abs())
    close(y, ref, 40 * U * ref.abs() + (r * 50 * U * m.abs())[:, None])


def test_constant_rows_and_zeros():
    from dlrm_amd import ops
    x = torch.full((5, 300), 2.5, device="cuda")
    x[1] = 0
    y, mean, rstd = ops.layer_norm_forward(x, beta=torch.full((300,), 0.5, device="cuda"))
    assert (y == 0.5).all() and torch.equal(mean, x[:, 0])
    assert ((rstd.double().cpu() - 1e-5 ** -0.5).abs() <= 4 * U * 1e-5 ** -0.5 + 1e-5 ** -0.5 * 2.0 ** -24).all()


def test_values_that_are_not_numbers_stay_in_their_row():
    from dlrm_amd import ops
    x, gamma, beta, dy = inputs(6, 200, torch.float32, seed=7)
    clean, m0, r0 = ops.layer_norm_forward(x.cuda(), gamma.cuda(), beta.cuda(), relu=True)
    bad = x.clone()
    bad[1, 5], bad[3, 199] = float("nan"), float("inf")
    y, m, r = ops.layer_norm_forward(bad.cuda(), gamma.cuda(), beta.cuda(), relu=True)
    keep = [0, 2, 4, 5]
    assert torch.equal(y[keep], clean[keep]) and torch.equal(r[keep], r0[keep])
    assert torch.isnan(y[1]).all() and torch.isnan(y[3]).all()
    # gradients that the ReLU cuts off may be anything
    wild = torch.where(clean.cpu() > 0, dy, torch.full_like(dy, float("nan")))
    a = ops.layer_norm_backward(dy.cuda(), x.cuda(), r0, mean=m0, gamma=gamma.cuda(), relu_mask=clean)
    for mask in (clean, ops.act8_pack(clean)):
        b = ops.layer_norm_backward(wild.cuda(), x.cuda(), r0, mean=m0, gamma=gamma.cuda(), relu_mask=mask)
        assert all(torch.equal(p, q) for p, q in zip(a[:3], b[:3]))
    # a row that the ReLU cuts off altogether
    none = clean.clone()
    none[2] = 0
    c = ops.layer_norm_backward(dy.cuda(), x.cuda(), r0, mean=m0, gamma=gamma.cuda(), relu_mask=none)
    assert (c[0][2] == 0).all() and torch.isfinite(c[1]).all()


def test_no_rows():
    from dlrm_amd import ops
    x = torch.empty((0, 24), device="cuda")
    y, mean, rstd = ops.layer_norm_forward(x, relu=True, xhat8=ops.Act8.empty(0, 24))
    assert y.shape == (0, 24) and mean.shape == (0,)
    dg = torch.full((24,), 7.0, device="cuda")
    dx, dg, db, _ = ops.layer_norm_backward(x, x, rstd, mean=mean, dgamma=dg)
    assert dx.shape == (0, 24) and (dg == 0).all() and (db == 0).all()


def test_refusals_before_a_launch():
    from dlrm_amd import ops
    x = torch.ones((4, 40), device="cuda")
    v = torch.ones(40, device="cuda")
    s = torch.ones(4, device="cuda")
    a = ops.act8_pack(x)
    bad = [lambda: ops.layer_norm_forward(x.t()), lambda: ops.layer_norm_forward(x[:1].expand(4, 40)),
           lambda: ops.layer_norm_forward(x, gamma=v[:39]), lambda: ops.layer_norm_forward(x, beta=v.double()),
           lambda: ops.layer_norm_forward(x, out=x[:3]), lambda: ops.layer_norm_forward(x, out=x.bfloat16()),
           lambda: ops.layer_norm_forward(x, mean=s[:3]), lambda: ops.layer_norm_forward(x, xhat8=x),
           lambda: ops.layer_norm_forward(x, y8=ops.Act8.empty(5, 40)), lambda: ops.layer_norm_forward(x.half()),
           lambda: ops.layer_norm_forward(x, eps=-1.0),
           lambda: ops.layer_norm_backward(x, x, s), lambda: ops.layer_norm_backward(x, a, s, mean=s),
           lambda: ops.layer_norm_backward(x, x.bfloat16(), s, mean=s), lambda: ops.layer_norm_backward(x, x[:3], s, mean=s),
           lambda: ops.layer_norm_backward(x, a, s, relu_mask=x[:, :39]), lambda: ops.layer_norm_backward(x, a, v),
           lambda: ops.layer_norm_backward(x, a, s, workspace=torch.empty(1, dtype=torch.uint8, device="cuda").expand(1 << 20)),
           lambda: ops.layer_norm_backward(x, a, s, dgamma=s), lambda: ops.layer_norm_backward(x, ops.Act8.empty(4, 41), s)]
    from dlrm_amd._capi import DlrmError
    for call in bad:
        with pytest.raises((TypeError, ValueError, DlrmError)):
            call()


def test_graph_replays():
    """Forward with checkpoints, backward and the linear layer's backward pass from them captured once and replayed with new
    inputs, eager work of the same buffers' program and synchronizations between the replays: every replay has the eager bits."""
    from dlrm_amd import ops
    M, N, K = 300, 96, 160
    x, gamma, beta, dy = inputs(M, N, torch.float32, seed=11)
    sx, sdy, sin = torch.zeros((M, N), device="cuda"), torch.zeros((M, N), device="cuda"), torch.zeros((M, K), device="cuda")
    gamma, beta = gamma.cuda(), beta.cuda()
    xhat8, y8, in8 = ops.Act8.empty(M, N), ops.Act8.empty(M, N), ops.Act8.empty(M, K)
    buf = dict(y=torch.empty((M, N), device="cuda"), rstd=torch.empty(M, device="cuda"), mean=torch.empty(M, device="cuda"),
               dx=torch.empty((M, N), device="cuda"), dg=torch.empty(N, device="cuda"), db=torch.empty(N, device="cuda"),
               dw=torch.empty((N, K), device="cuda"), dwb=torch.empty(N, device="cuda"))
    ws1 = torch.empty(ops.layer_norm_backward_workspace_bytes(M, N), dtype=torch.uint8, device="cuda")
    ws2 = torch.empty(ops.linear_backward_weight_workspace_bytes(M, N, K, True), dtype=torch.uint8, device="cuda")

    def step():
        ops.act8_pack(sin, out=in8)
        ops.layer_norm_forward(sx, gamma, beta, relu=True, out=buf["y"], mean=buf["mean"], rstd=buf["rstd"], xhat8=xhat8, y8=y8)
        ops.layer_norm_backward(sdy, xhat8, buf["rstd"], gamma=gamma, relu_mask=y8, out=buf["dx"], dgamma=buf["dg"], dbeta=buf["db"],
                                workspace=ws1)
        ops.linear_backward_weight(buf["dx"], in8, dw=buf["dw"], db=buf["dwb"], workspace=ws2)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for k in range(4):
        g = torch.Generator().manual_seed(k)
        sx.copy_(torch.randn(M, N, generator=g))
        sdy.copy_(torch.randn(M, N, generator=g))
        sin.copy_(torch.randn(M, K, generator=g))
        step()
        torch.cuda.synchronize()
        want = {n: t.clone() for n, t in buf.items()}
        for t in buf.values():
            t.fill_(-1.0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(buf[n], want[n]) for n in buf), k


def test_recorded_step():
    """The operators handed to a recorded step and replayed from it."""
    from dlrm_amd import ops
    from dlrm_amd.plan import StepRecorder
    M, N = 70, 48
    x, gamma, beta, dy = (t.cuda() for t in inputs(M, N, torch.float32, seed=12))
    y, mean, rstd = torch.empty_like(x), torch.empty(M, device="cuda"), torch.empty(M, device="cuda")
    xhat8, y8 = ops.Act8.empty(M, N), ops.Act8.empty(M, N)
    dx, dg, db, back = torch.empty_like(x), torch.empty(N, device="cuda"), torch.empty(N, device="cuda"), torch.empty_like(x)
    ws = torch.empty(ops.layer_norm_backward_workspace_bytes(M, N), dtype=torch.uint8, device="cuda")
    idx = torch.zeros(1, dtype=torch.int64, device="cuda")

    def step():
        ops.layer_norm_forward(x, gamma, beta, relu=True, out=y, mean=mean, rstd=rstd, xhat8=xhat8)
        ops.act8_pack(y, out=y8)
        ops.layer_norm_backward(dy, xhat8, rstd, gamma=gamma, relu_mask=y8, out=dx, dgamma=dg, dbeta=db, workspace=ws)
        ops.act8_unpack(y8, out=back)

    step()
    want = [t.clone() for t in (y, dx, dg, db, back)]
    rec = StepRecorder(idx, idx)
    with rec:
        step()
    assert rec.size == 4 and [rec.plan.op_name(i) for i in range(4)] == ["layer_norm_forward", "act8_pack", "layer_norm_backward",
                                                                         "act8_unpack"]
    for t in (y, dx, dg, db, back):
        t.fill_(-1.0)
    rec.plan.run(0, 4)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip((y, dx, dg, db, back), want))


def test_another_stream():
    from dlrm_amd import ops
    x, gamma, beta, dy = (t.cuda() for t in inputs(500, 300, torch.float32, seed=13))
    y, mean, rstd = ops.layer_norm_forward(x, gamma, beta)
    want = ops.layer_norm_backward(dy, x, rstd, mean=mean, gamma=gamma)[:3]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        y2, m2, r2 = ops.layer_norm_forward(x, gamma, beta)
        got = ops.layer_norm_backward(dy, x, r2, mean=m2, gamma=gamma)[:3]
    s.synchronize()
    assert torch.equal(y, y2) and all(torch.equal(a, b) for a, b in zip(want, got))


def test_normalised_layers_train_from_checkpoints():
    """Two layers Linear -> norm -> ReLU and a last linear one, as a training step would run them: forward, then backward from the
    8-bit checkpoints alone (inputs, normalised rows, outputs), against float64 with the same checkpoints' values.  Every tensor is
    the result of at most four products and two norms, each within a few 1e-6 of its own largest value."""
    from dlrm_amd import ops
    M, sizes = 700, [40, 128, 96, 8]
    g = torch.Generator().manual_seed(21)
    W = [torch.randn(n, k, generator=g) / k ** 0.5 for k, n in zip(sizes[:-1], sizes[1:])]
    B = [0.1 * torch.randn(n, generator=g) for n in sizes[1:]]
    G = [1 + 0.1 * torch.randn(n, generator=g) for n in sizes[1:-1]]
    E = [0.1 * torch.randn(n, generator=g) for n in sizes[1:-1]]
    x0, dout = torch.randn(M, sizes[0], generator=g), torch.randn(M, sizes[-1], generator=g) / M
    dev = [t.cuda() for t in W], [t.cuda() for t in B], [t.cuda() for t in G], [t.cuda() for t in E]

    x, kept_in, kept_xh, rstds = x0.cuda(), [ops.act8_pack(x0.cuda())], [], []
    for i in range(2):
        z = ops.linear_forward(x, dev[0][i], dev[1][i], False)
        xhat8, y8 = ops.Act8.empty(*z.shape), ops.Act8.empty(*z.shape)
        x, _, rstd = ops.layer_norm_forward(z, dev[2][i], dev[3][i], relu=True, out=z, xhat8=xhat8, y8=y8)
        kept_in.append(y8)
        kept_xh.append(xhat8)
        rstds.append(rstd)
    out = ops.linear_forward(x, dev[0][2], dev[1][2], False)

    grads, dz, ws = {}, dout.cuda(), None
    for i in reversed(range(3)):
        if i < 2:
            dz, grads["g%d" % i], grads["e%d" % i], _ = ops.layer_norm_backward(dz, kept_xh[i], rstds[i], gamma=dev[2][i],
                                                                               relu_mask=kept_in[i + 1])
        grads["w%d" % i], grads["b%d" % i], ws = ops.linear_backward_weight(dz, kept_in[i], workspace=ws)
        dz = ops.linear_backward_data(dz, dev[0][i])
    grads["x"] = dz
    torch.cuda.synchronize()

    ref, y = {}, x0.double()
    for i in range(2):
        y, _, _, _ = norm_ref.norm(y @ W[i].double().t() + B[i].double(), G[i].double(), E[i].double(), 1e-5, True)
    y = y @ W[2].double().t() + B[2].double()
    dz = dout.double()

    def of(a):
        return norm_ref.unpack8(a.codes.cpu(), a.exps.cpu(), a.cols)

    for i in reversed(range(3)):
        if i < 2:
            mask = norm_ref.positive8(kept_in[i + 1].codes.cpu(), kept_in[i + 1].cols)
            dz, ref["g%d" % i], ref["e%d" % i], _ = norm_ref.norm_grad(dz, of(kept_xh[i]), rstds[i].cpu().double(), G[i].double(), mask)
        ref["w%d" % i], ref["b%d" % i] = dz.t() @ of(kept_in[i]), dz.sum(0)
        dz = dz @ W[i].double()
    ref["x"] = dz
    assert float((out.cpu().double() - y).abs().max()) <= 1e-5 * float(y.abs().max())
    for n in ref:
        assert float((grads[n].cpu().double() - ref[n]).abs().max()) <= 1e-5 * float(ref[n].abs().max()), n


def test_offsets_past_32_bits():
    """More than 2^32 elements, and rows 2^31 elements apart: the last rows are what a call on them alone gives."""
    from dlrm_amd import ops
    M, N, tail = (1 << 22) + 77, 1024, 300
    x = torch.zeros((M, N), dtype=torch.bfloat16, device="cuda")
    x[-tail:] = torch.randn(tail, N, device="cuda").to(torch.bfloat16)
    xhat8 = ops.Act8.empty(M, N)
    y, mean, rstd = ops.layer_norm_forward(x, relu=True, xhat8=xhat8)
    a8 = ops.Act8.empty(tail, N)
    ya, ma, ra = ops.layer_norm_forward(x[-tail:], relu=True, xhat8=a8)
    assert torch.equal(y[-tail:], ya) and torch.equal(mean[-tail:], ma) and torch.equal(rstd[-tail:], ra)
    assert torch.equal(xhat8.codes[-tail:], a8.codes) and torch.equal(xhat8.exps[-tail:], a8.exps)
    for source, short, m, s in ((x, x[-tail:], mean, ma), (xhat8, a8, None, None)):
        dx, _, db, _ = ops.layer_norm_backward(x, source, rstd, mean=m, relu_mask=y, want_params=False)
        dxa, _, _, _ = ops.layer_norm_backward(x[-tail:], short, ra, mean=s, relu_mask=ya, want_params=False)
        assert torch.equal(dx[-tail:], dxa) and not dx[:tail].any()
        del dx
    del y, xhat8
    apart = x.view(-1).as_strided((2, 64), ((1 << 31) + 8, 1))
    apart.copy_(torch.randn(2, 64, device="cuda"))
    near = apart.clone()
    assert torch.equal(ops.layer_norm_forward(apart, out=apart)[0], ops.layer_norm_forward(near)[0])
