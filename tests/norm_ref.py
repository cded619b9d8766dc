"""Plain float64 forms of layer norm and of the 8-bit activation checkpoint, on the CPU."""
import torch

U = 2.0 ** -24      # half a step of a float32 value, relative


def pack8(v):
    """Codes int8 [M, 32 blocks], exponents uint8 [M, blocks] of a float64 [M, N] whose values are float32 numbers."""
    M, N = v.shape
    nb = (N + 31) // 32
    u = torch.zeros((M, nb * 32), dtype=torch.float64)
    u[:, :N] = v
    u = u.view(M, nb, 32)
    amax = u.abs().amax(2)
    bad = ~torch.isfinite(u).all(2)
    e = torch.ones((M, nb), dtype=torch.int64)
    while True:
        up = ~bad & (e < 248) & (amax >= 127.5 * torch.pow(2.0, (e - 127).double()))
        if not up.any():
            break
        e += up
    step = torch.pow(2.0, (e - 127).double())
    q = torch.round(torch.where(bad[:, :, None], torch.zeros_like(u), u) / step[:, :, None]).clamp(-127, 127)
    q = torch.where((q == 0) & (u > 0), torch.full_like(q, -128.0), q)
    e[bad] = 255
    return q.view(M, nb * 32).to(torch.int8), e.to(torch.uint8)


def unpack8(codes, exps, N):
    nb = exps.shape[1]
    q = codes[:, :nb * 32].double()
    q = torch.where(q == -128, torch.zeros_like(q), q).view(-1, nb, 32)
    step = torch.pow(2.0, (exps.long() - 127).double())
    step = torch.where(exps == 255, torch.full_like(step, float("nan")), step)
    return (q * step[:, :, None]).reshape(-1, nb * 32)[:, :N]


def positive8(codes, N):
    return ((codes > 0) | (codes == -128))[:, :N]


def norm(x, gamma, beta, eps, relu):
    """(y, xh, mean, rstd) of float64 rows."""
    mean = x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + eps)
    xh = (x - mean) * rstd
    y = xh * gamma + beta
    return (torch.where(y < 0, torch.zeros_like(y), y) if relu else y), xh, mean[:, 0], rstd[:, 0]


def norm_grad(dy, xh, rstd, gamma, mask):
    """(dx, dgamma, dbeta, d) of float64 rows; mask: bool or None."""
    d = dy if mask is None else torch.where(mask, dy, torch.zeros_like(dy))
    gd = d * gamma
    dx = rstd[:, None] * (gd - gd.mean(1, keepdim=True) - xh * (gd * xh).mean(1, keepdim=True))
    return dx, (d * xh).sum(0), d.sum(0), d
