"""The expert layer for a few tokens on a B200, in both weight formats.

Held to a 64-bit statement: every value within bf16's (fp16's) half step plus
the derived bound of mx_reference.moe, and the whole within half a step of its
norm (roundings are at most that each, and independent ones far less).
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


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


class Layer:
    """Random expert weights, as the kernels take them and dequantized."""

    def __init__(self, fmt, e, h, i, seed=0):
        g = _gen(seed)
        self.e, self.h, self.i = e, h, i
        self.args, self.dense = [], []
        for rows, k in ((2 * i, h), (h, i)):
            if fmt == "fp8":
                w = (torch.randn(e, rows, k, device=DEV, generator=g) * 90).clamp(-448, 448).to(torch.float8_e4m3fn)
                s = (0.5 + torch.rand(e, -(-rows // 128), -(-k // 128), device=DEV, generator=g)) / (90 * k ** 0.5)
                self.args += [w, s]
                self.dense.append(R.block_fp8(w, s))
            else:
                w = torch.randn(e * rows, k, device=DEV, generator=g) / k ** 0.5
                code, byte = (t.view(e, rows, -1) for t in R.quantize(w))
                self.args += [R.pack(code), bf.tile_mxfp4_scales(byte)]
                self.dense.append(R.values(code, byte))


def _x(t, h, seed, dtype=torch.bfloat16):
    return torch.randn(t, h, device=DEV, generator=_gen(seed)).to(dtype)


def _check(y, x, ids, weights, layer):
    ref, bound = R.moe(x, ids, weights, *layer.dense)
    step = torch.finfo(x.dtype).eps / 2
    err = (y.double() - ref).abs()
    assert y.dtype == x.dtype and torch.isfinite(y).all()
    assert (err <= ref.abs() * step + bound + 2.0 ** -25).all(), float((err / (ref.abs() * step + bound + 2.0 ** -25)).max())
    # f16 activations (2^-11 a value) beside the output's own rounding
    assert (y.double() - ref).norm() <= ref.norm() * max(step, 2.0 ** -10)


SIZES = [  # tokens, experts, top_k, H, I
    (1, 1, 1, 32, 32), (1, 4, 2, 128, 96), (1, 16, 8, 512, 256), (2, 5, 3, 160, 64), (3, 8, 1, 1056, 288),
    (7, 12, 4, 256, 160), (8, 32, 8, 1024, 384), (9, 3, 2, 544, 128), (16, 64, 6, 256, 512), (17, 4, 4, 512, 96),
    (33, 40, 5, 288, 224), (64, 6, 2, 256, 128), (64, 128, 8, 512, 128), (64, 17, 16, 96, 64),
]


@pytest.mark.parametrize("fmt", ["fp8", "mxfp4"])
@pytest.mark.parametrize("t,e,k,h,i", SIZES)
def test_moe(fmt, t, e, k, h, i):
    layer = Layer(fmt, e, h, i, seed=t + e)
    x = _x(t, h, seed=h)
    logits = torch.randn(t, e, device=DEV, generator=_gen(i))
    for renormalize in (True, False):
        y = bf.moe(x, logits, *layer.args, top_k=k, renormalize=renormalize)
        _check(y, x, *R.route(logits, k, renormalize), layer)
        assert torch.equal(y, bf.moe(x, logits, *layer.args, top_k=k, renormalize=renormalize))


@pytest.mark.parametrize("fmt", ["fp8", "mxfp4"])
@pytest.mark.parametrize("t,e,k,h,i", [(1, 8, 2, 8192, 64), (12, 4, 2, 8192, 96), (2, 3, 2, 64, 9248), (20, 3, 1, 128, 4160),
                                       (5, 512, 8, 96, 64)])
def test_moe_long_rows_and_many_experts(fmt, t, e, k, h, i):
    layer = Layer(fmt, e, h, i, seed=1)
    x = _x(t, h, seed=2)
    logits = torch.randn(t, e, device=DEV, generator=_gen(3))
    _check(bf.moe(x, logits, *layer.args, top_k=k), x, *R.route(logits, k), layer)


@pytest.mark.parametrize("fmt", ["fp8", "mxfp4"])
def test_types_and_views(fmt):
    layer = Layer(fmt, 6, 288, 160, seed=4)
    wide = _x(20, 512, 5, torch.float16)
    x = wide[2:15, 64:64 + 288]
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        logits = torch.randn(13, 6 + 3, device=DEV, generator=_gen(6)).to(dtype)[:, :6]  # rows with a stride
        y = bf.moe(x, logits, *layer.args, top_k=2)
        _check(y, x, *R.route(logits, 2), layer)
    w13, s13, w2, s2 = layer.args
    room = torch.zeros(6, w13.shape[1], w13.shape[2] + 32, dtype=torch.uint8, device=DEV)
    room[..., :w13.shape[2]] = w13.view(torch.uint8)
    padded = room.view(w13.dtype)[..., :w13.shape[2]]
    assert torch.equal(bf.moe(x, logits, padded, s13, w2, s2, top_k=2), y)


@pytest.mark.parametrize("fmt", ["fp8", "mxfp4"])
@pytest.mark.parametrize("t", [1, 8, 23, 64])
def test_every_token_to_one_expert(fmt, t):
    layer = Layer(fmt, 9, 256, 128, seed=7)
    x = _x(t, 256, 8)
    ids = torch.full((t, 1), 5, dtype=torch.int32, device=DEV)
    p = torch.rand(t, 1, device=DEV, generator=_gen(9))
    _check(bf.moe_experts(x, ids, p, *layer.args), x, ids, p, layer)


@pytest.mark.parametrize("fmt", ["fp8", "mxfp4"])
def test_ids_outside_and_repeated(fmt):
    layer = Layer(fmt, 5, 160, 96, seed=10)
    x = _x(6, 160, 11)
    ids = torch.tensor([[0, 0, 0], [-1, 2, 7], [-1, -1, -1], [4, 1, 4], [5, -7, 3], [2, 1, 0]], dtype=torch.int32, device=DEV)
    p = torch.tensor([[0.5, 0.25, 0.25], [9.0, 1.0, 9.0], [1.0, 1.0, 1.0], [-0.5, 2.0, 1.5], [3.0, 3.0, 1.0],
                      [0.0, 1.0, 0.0]], device=DEV)
    y = bf.moe_experts(x, ids, p, *layer.args)
    _check(y, x, ids, p, layer)
    assert (y[2] == 0).all()
    for t in range(6):  # one token alone, its expert perhaps three times
        _check(bf.moe_experts(x[t:t + 1], ids[t:t + 1], p[t:t + 1], *layer.args), x[t:t + 1], ids[t:t + 1], p[t:t + 1], layer)
    many = torch.full((1, 16), 3, dtype=torch.int32, device=DEV)
    layer16 = Layer(fmt, 16, 160, 96, seed=10)
    p16 = torch.rand(1, 16, device=DEV, generator=_gen(3))
    _check(bf.moe_experts(x[:1], many, p16, *layer16.args), x[:1], many, p16, layer16)
    none = torch.full((6, 3), -1, dtype=torch.int32, device=DEV)
    torch.empty(1 << 20, device=DEV).fill_(torch.nan)  # what the allocator hands out next
    y = bf.moe_experts(x, none, p, *layer.args)
    assert y.shape == x.shape and (y == 0).all()


def test_ties_and_masked_logits():
    layer = Layer("fp8", 40, 128, 64, seed=12)
    x = _x(7, 128, 13)
    inf, nan = torch.inf, torch.nan
    logits = torch.zeros(7, 40, device=DEV)                      # row 0: all equal, the first ones win
    logits[1] = torch.randint(0, 3, (40,), device=DEV, generator=_gen(14)).float()
    logits[2] = -inf                                             # nothing to choose: zeros
    logits[3] = -inf
    logits[3, 37] = -3.0                                         # one to choose
    logits[4] = nan
    logits[4, [3, 30]] = torch.tensor([1.0, 2.0], device=DEV)
    logits[5] = -0.0
    logits[5, 33] = 0.0                                          # equal to -0
    logits[6] = torch.finfo(torch.float32).min                   # the lowest value can be chosen
    for renormalize in (True, False):
        y = bf.moe(x, logits, *layer.args, top_k=4, renormalize=renormalize)
        ids, p = R.route(logits, 4, renormalize)
        assert ids[0].tolist() == ids[5].tolist() == ids[6].tolist() == [0, 1, 2, 3]
        assert ids[3].tolist() == [37, -1, -1, -1] and ids[4].tolist() == [30, 3, -1, -1]
        _check(y, x, ids, p, layer)
        assert (y[2] == 0).all()


def test_no_tokens():
    layer = Layer("fp8", 4, 64, 32, seed=1)
    x = torch.empty(0, 64, dtype=torch.bfloat16, device=DEV)
    assert bf.moe(x, torch.empty(0, 4, device=DEV), *layer.args, top_k=2).shape == (0, 64)


def test_values_far_apart():
    # activations over the whole of bf16's range beside ordinary ones
    layer = Layer("mxfp4", 4, 256, 128, seed=15)
    x = _x(5, 256, 16)
    x[0] *= 2.0 ** -100
    x[1] *= 2.0 ** 30
    x[2, ::7] *= 2.0 ** 12
    x[3] = 0
    x[4, :] = 2.0 ** -130
    logits = torch.randn(5, 4, device=DEV, generator=_gen(17))
    _check(bf.moe(x, logits, *layer.args, top_k=2), x, *R.route(logits, 2), layer)
    x[1, 3] = torch.nan
    y = bf.moe(x, logits, *layer.args, top_k=2)
    assert torch.isnan(y[1]).all() and torch.isfinite(y[[0, 2, 3, 4]]).all()


def test_streams_and_graphs():
    layer = Layer("fp8", 16, 512, 256, seed=18)
    xs = [_x(9, 512, 20 + s) for s in range(3)]
    ls = [torch.randn(9, 16, device=DEV, generator=_gen(30 + s)) for s in range(3)]
    want = [bf.moe(x, l, *layer.args, top_k=4) for x, l in zip(xs, ls)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(4):  # at the same time on two streams
        with torch.cuda.stream(side):
            got.append(bf.moe(xs[0], ls[0], *layer.args, top_k=4))
        got.append(bf.moe(xs[1], ls[1], *layer.args, top_k=4))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[n % 2]) for n, y in enumerate(got))
    graphs = []
    for s in range(2):  # two graphs of one pool, replayed in turn
        x, l = xs[s].clone(), ls[s].clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=graphs[0][0].pool() if graphs else None):
            y = bf.moe(x, l, *layer.args, top_k=4)
        graphs.append((graph, x, l, y))
    for n in (0, 1, 2, 1):
        for graph, x, l, y in graphs:
            x.copy_(xs[n])
            l.copy_(ls[n])
            graph.replay()
            assert torch.equal(y, want[n])


def test_layers_in_a_row_as_a_model_runs_them():
    """Norm, MXFP4 projection, router, experts and residual, twice, eagerly and captured: the same bits."""
    h, e = 512, 16
    layer = Layer("mxfp4", e, h, 192, seed=21)
    proj = bf.quantize_mxfp4(torch.randn(h, h, device=DEV, generator=_gen(22)) / h ** 0.5)
    router = torch.randn(e, h, device=DEV, generator=_gen(23)).bfloat16() / h ** 0.5
    x0 = _x(6, h, 24)

    def block(x):
        a = x + bf.linear_mxfp4(x, *proj)
        return a + bf.moe(a, a @ router.t(), *layer.args, top_k=4)

    def model(x):
        return block(block(x))

    want = model(x0)
    a = x0
    for _ in range(2):  # the same in 64 bits from each kernel's own inputs
        q = bf.dequantize_mxfp4(*bf.quantize_mxfp4(a)).double()
        ref = q @ bf.dequantize_mxfp4(*proj).double().t()
        lin = bf.linear_mxfp4(a, *proj)
        assert (lin.double() - ref).norm() <= ref.norm() * 2.0 ** -8
        b = a + lin
        logits = b @ router.t()
        y = bf.moe(b, logits, *layer.args, top_k=4)
        _check(y, b, *R.route(logits, 4), layer)
        a = b + y
    assert torch.equal(a, want)
    static = x0.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = model(static)
    graph.replay()
    assert torch.equal(out, want)
