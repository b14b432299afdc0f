"""Plain 64-bit statements of MXFP4 and of the expert layer, for tests."""

import torch

GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def quantize(x):
    """(codes one a byte [M, K], scale bytes [M, K / 32]) of x, by the nearest grid point (ties to the even code)."""
    b = x.double().unflatten(1, (-1, 32))
    amax = b.abs().amax(2, keepdim=True)
    bad = ~torch.isfinite(amax)
    amax = torch.where(bad, 0.0, amax)
    e = torch.where(amax > 0, torch.frexp(amax).exponent - 3, -127).clamp(min=-127)
    v = torch.where(bad, 0.0, b) * torch.ldexp(torch.ones_like(amax), -e)
    d = (v.abs().clamp(max=6.0).unsqueeze(-1) - GRID.to(x.device)).abs()
    near = d == d.amin(-1, keepdim=True)  # one point, or two on a tie
    idx = torch.arange(8, device=x.device)
    code = torch.where(near, idx + 16 * (idx % 2), 99).amin(-1) % 16  # the even one of two
    code = code + 8 * torch.signbit(torch.where(bad, 0.0, b)).long()
    byte = torch.where(bad, 255, e + 127).squeeze(2)
    return code.flatten(1).to(torch.uint8), byte.to(torch.uint8)


def values(code, byte):
    """What codes [..., K] under scale bytes [..., K / 32] stand for, float64."""
    grid = GRID.to(code.device)
    v = torch.where(code >= 8, -1.0, 1.0) * grid[(code & 7).long()]
    s = torch.where(byte == 255, torch.nan, torch.ldexp(torch.ones(byte.shape, dtype=torch.float64, device=byte.device),
                                                        byte.int() - 127))
    return (v.unflatten(-1, (-1, 32)) * s.unsqueeze(-1)).flatten(-2)


def pack(code):
    return code[..., 0::2] | (code[..., 1::2] << 4)


def unpack(q):
    return torch.stack((q & 15, q >> 4), -1).flatten(-2)


def block_fp8(w, s):
    """e4m3 [E, R, K] under scales [E, ceil(R / 128), ceil(K / 128)], float64."""
    r, k = w.shape[-2:]
    return w.double() * s.double().repeat_interleave(128, -2)[..., :r, :].repeat_interleave(128, -1)[..., :k]


def route(logits, top_k, renormalize=True):
    """(ids, weights): the largest logits, ties to the lower index; -inf and NaN never (id -1, weight 0)."""
    z = logits.double()
    z = torch.where(torch.isnan(z), -torch.inf, z)
    order = torch.sort(-z, dim=1, stable=True).indices[:, :top_k]
    l = z.gather(1, order)
    top = torch.where(l[:, :1] > -torch.inf, l[:, :1], 0.0)
    ex = torch.where(l > -torch.inf, torch.exp(l - top), 0.0)
    total = ex.sum(1, keepdim=True) if renormalize else torch.exp(z - top).sum(1, keepdim=True)
    return torch.where(l > -torch.inf, order, -1), torch.where(total > 0, ex / total, 0.0)


def moe(x, ids, weights, w13, w2):
    """(y, bound on the kernel's error before y's own rounding), float64; w13 [E, 2 I, H], w2 [E, H, I] dequantized.

    The bound: fp32 sums of n products carry at most (n / 8 + 64) 2^-23 of the sum of magnitudes (two truncated MMA
    steps per 16, the scale products, 8 warps); silu adds 2^-20; h and x go to f16 (half a step: 2^-11, and x is
    exact but for 2^-25 of its block's largest value)."""
    x = x.double()
    i = w2.shape[2]
    y, bound = torch.zeros_like(x), torch.zeros_like(x)
    for t in range(x.shape[0]):
        for j in range(ids.shape[1]):
            e = int(ids[t, j])
            if not 0 <= e < w13.shape[0]:
                continue
            gu, size = w13[e] @ x[t], w13[e].abs() @ x[t].abs()
            err = size * ((x.shape[1] / 8 + 64) * 2.0 ** -23 + 2.0 ** -25)
            g, u = gu[:i], gu[i:]
            s = g * torch.sigmoid(g)
            h = s * u
            dh = 1.1 * err[:i] * u.abs() + (s.abs() + 1.1 * err[:i]) * err[i:] + h.abs() * (2.0 ** -20 + 2.0 ** -11)
            p = float(weights[t, j])
            y[t] += p * (w2[e] @ h)
            a = w2[e].abs()
            bound[t] += abs(p) * (a @ dh + a @ h.abs() * ((i / 8 + 64) * 2.0 ** -23))
    return y, bound
