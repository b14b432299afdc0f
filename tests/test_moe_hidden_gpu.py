"""The expert layer's hidden values keep more than 16 bits' worth of digits.

Weights and activations are small integers and every gate is large enough
that silu(g) = g in fp32 (exp(-g) < 2^-25), so that h = g u is an integer of up
to 21 bits.  A row of W2 takes the difference of two of them, which is exact in
fp32: y is that difference, rounded once to its type.  An h in f16 or bf16 is
off by up to 2^-12 or 2^-9 of itself, many times the difference's last bit.
"""

import pytest
import torch

import blockfp8_b200 as bf
import mx_reference as R

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA GPU"),
]

DEV = "cuda"
LEVELS = torch.tensor([0, 1, 2, 3, 4, 6])  # integers that e2m1 and e4m3 hold


def _weights(fmt, w):
    """Integers [E, rows, K] as the layer takes them, every scale 1."""
    e, rows, k = w.shape
    if fmt == "fp8":
        return [w.float().to(torch.float8_e4m3fn), torch.ones(e, -(-rows // 128), -(-k // 128), device=DEV)]
    code = torch.zeros_like(w, dtype=torch.uint8)
    for c, v in ((2, 1), (4, 2), (5, 3), (6, 4), (7, 6)):
        code = torch.where(w.abs() == v, c, code)
    code = (code + 8 * (w < 0).to(torch.uint8)).to(torch.uint8)
    byte = torch.full((e, rows, k // 32), 127, dtype=torch.uint8, device=DEV)
    return [R.pack(code), bf.tile_mxfp4_scales(byte)]


def _layer(fmt, t, e, h, i, seed):
    g = torch.Generator().manual_seed(seed)
    pick = lambda *shape: LEVELS[torch.randint(0, 6, shape, generator=g)]  # noqa: E731
    x = torch.randint(1, 4, (t, h), generator=g)
    w1, w3 = pick(e, i, h).clamp(min=1), pick(e, i, h) * (1 - 2 * torch.randint(0, 2, (e, i, h), generator=g))
    half = i // 2  # columns c and c + half differ in one weight of W3 alone
    w1[:, half:], w3[:, half:] = w1[:, :half], w3[:, :half]
    w3[:, half:, 0] = torch.where(w3[:, half:, 0] == 1, 2, 1)
    w2 = torch.zeros(e, h, i, dtype=torch.long)
    row = torch.arange(h)
    w2[:, row, row * 7 % half], w2[:, row, row * 7 % half + half] = 1, -1
    w13 = torch.cat((w1, w3), 1).to(DEV)
    w2 = w2.to(DEV)
    return x.to(DEV), w13, w2, _weights(fmt, w13) + _weights(fmt, w2)


def _expected(x, ids, w13, w2):
    i = w2.shape[2]
    y = torch.zeros(x.shape, dtype=torch.float64, device=DEV)
    largest = 0.0
    for t in range(x.shape[0]):
        for e in ids[t].tolist():
            gu = w13[e].double() @ x[t].double()
            h = gu[:i] * gu[i:]
            assert gu[:i].min() > 18  # exp(-g) < 2^-25
            largest = max(largest, float(h.abs().max()))
            y[t] += w2[e].double() @ h
    assert 2 ** 13 < largest < 2 ** 21
    return y


def _check(fmt, t, e, k, h, i, dtype):
    x, w13, w2, args = _layer(fmt, t, e, h, i, seed=t + i)
    ids = torch.stack([torch.randperm(e, generator=torch.Generator().manual_seed(9 + n))[:k] for n in range(t)])
    ids = ids.to(torch.int32).to(DEV)
    y = bf.moe_experts(x.to(dtype), ids, torch.ones(t, k, device=DEV), *args)
    want = _expected(x, ids, w13, w2)
    assert want.abs().max() < 65504
    assert torch.equal(y, want.to(dtype))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("fmt", ["fp8", "mxfp4"])
@pytest.mark.parametrize("t,e,k,h,i", [(1, 1, 1, 32, 64), (1, 8, 8, 64, 160), (3, 4, 2, 96, 320), (8, 5, 3, 64, 1120),
                                       (2, 2, 1, 64, 4160)])
def test_a_few_tokens(fmt, t, e, k, h, i, dtype):
    _check(fmt, t, e, k, h, i, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("fmt", ["fp8", "mxfp4"])
@pytest.mark.parametrize("t,e,k,h,i", [(9, 4, 2, 64, 128), (20, 3, 1, 128, 2112), (64, 16, 4, 64, 192)])
def test_a_batch(fmt, t, e, k, h, i, dtype):
    _check(fmt, t, e, k, h, i, dtype)
