"""MXFP4 and expert-layer entry points without a GPU: layouts and refusals."""

import ctypes

import pytest
import torch

import blockfp8_b200 as bf
import mx_reference as R
from blockfp8_b200 import _native

needs_native = pytest.mark.skipif(not bf.native_available(), reason="native libraries not built")

U8, F32, BF16, E4M3 = torch.uint8, torch.float32, torch.bfloat16, torch.float8_e4m3fn


@pytest.mark.parametrize("r,k", [(1, 32), (127, 96), (128, 128), (129, 160), (300, 1056)])
def test_scale_tiles(r, k):
    s = torch.randint(0, 256, (2, r, k // 32), dtype=U8)
    t = bf.tile_mxfp4_scales(s)
    assert t.shape == (2, -(-r // 128), -(-k // 128), 32, 16) and t.is_contiguous()
    assert torch.equal(bf.untile_mxfp4_scales(t, r, k), s)
    for row, b in ((0, 0), (r - 1, k // 32 - 1), (r // 2, k // 64)):
        assert t[1, row // 128, b // 4, row % 32, 4 * (row % 128 // 32) + b % 4] == s[1, row, b]
    assert t.long().sum() == s.long().sum()  # zeros past the matrix
    assert torch.equal(bf.tile_mxfp4_scales(s[0].view(torch.float8_e8m0fnu)), t[0])


def test_scale_tiles_refuse():
    with pytest.raises(ValueError):
        bf.tile_mxfp4_scales(torch.zeros(4))
    with pytest.raises(ValueError):
        bf.tile_mxfp4_scales(torch.zeros(4, 4))
    for shape in ((1, 1, 32, 16), (2, 1, 32, 15), (2, 1, 32)):
        with pytest.raises(ValueError):
            bf.untile_mxfp4_scales(torch.zeros(shape, dtype=U8), 130, 128)


def test_reference_codes_are_the_grid():
    x = torch.tensor([[0.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, -0.3, 6.0] + [0.0] * 21])
    code, byte = R.quantize(x)
    assert byte.item() == 127 and code[0, :11].tolist() == [0, 0, 2, 2, 4, 4, 6, 6, 7, 9, 7]


def _codes(rows, k):
    return torch.zeros(rows, k // 2, dtype=U8)


def _tiles(rows, k, *lead):
    return torch.zeros(*lead, -(-rows // 128), -(-k // 128), 32, 16, dtype=U8)


@needs_native
@pytest.mark.parametrize("call,reason", [
    (lambda: bf.quantize_mxfp4(torch.zeros(4, 64, dtype=BF16)), "CUDA tensors only"),
    (lambda: bf.quantize_mxfp4(torch.zeros(4, 64, dtype=torch.float64)), "x must be bfloat16"),
    (lambda: bf.quantize_mxfp4(torch.zeros(64, dtype=BF16)), "2-D"),
    (lambda: bf.quantize_mxfp4(torch.zeros(4, 48, dtype=BF16)), "multiple of 32"),
    (lambda: bf.quantize_mxfp4(torch.zeros(4, 0, dtype=BF16)), "multiple of 32"),
    (lambda: bf.quantize_mxfp4(torch.zeros(64, 4, dtype=BF16).t()[:, :32]), "row-major"),
    (lambda: bf.quantize_mxfp4(torch.zeros(4, 68, dtype=BF16)[:, :64]), "row-major"),
    (lambda: bf.quantize_mxfp4(torch.zeros(4, 72, dtype=BF16)[:, 4:68]), "row-major"),
    (lambda: bf.quantize_mxfp4(torch.zeros(1, 64, dtype=BF16).expand(4, 64)), "row-major"),
    (lambda: bf.dequantize_mxfp4(_codes(4, 64), _tiles(4, 64)), "CUDA tensors only"),
    (lambda: bf.dequantize_mxfp4(_codes(4, 64), _tiles(4, 64), torch.float16), "dtype"),
    (lambda: bf.dequantize_mxfp4(_codes(4, 64).float(), _tiles(4, 64)), "uint8"),
    (lambda: bf.dequantize_mxfp4(_codes(130, 64), _tiles(4, 64)), "scales"),
    (lambda: bf.dequantize_mxfp4(_codes(4, 160), _tiles(4, 64)), "scales"),
    (lambda: bf.dequantize_mxfp4(_codes(4, 64), torch.zeros(4, 2, dtype=U8)), "scales"),
    (lambda: bf.dequantize_mxfp4(_codes(4, 64), _tiles(4, 64, 2)[0].transpose(2, 3).contiguous().transpose(2, 3)), "contiguous"),
    (lambda: bf.gemm_mxfp4(_codes(4, 64), _tiles(4, 64), _codes(8, 64), _tiles(8, 64)), "CUDA tensors only"),
    (lambda: bf.gemm_mxfp4(_codes(4, 64), _tiles(4, 64), _codes(12, 64), _tiles(12, 64)), "multiple of 8"),
    (lambda: bf.gemm_mxfp4(_codes(4, 64), _tiles(4, 64), _codes(8, 96), _tiles(8, 96)), "K mismatch"),
    (lambda: bf.linear_mxfp4(torch.zeros(4, 64), _codes(8, 64), _tiles(8, 64)), "bfloat16 or float16"),
    (lambda: bf.linear_mxfp4(torch.zeros(4, 64, dtype=BF16), _codes(0, 64), _tiles(0, 64)), "multiple of 8"),
    (lambda: bf.linear_mxfp4(torch.zeros(4, 64, dtype=BF16), _codes(8, 64), _tiles(8, 64)), "CUDA tensors only"),
])
def test_mxfp4_refusals(call, reason):
    with pytest.raises(ValueError, match=reason):
        call()


def _layer(e=4, h=64, i=96, fmt="fp8"):
    if fmt == "fp8":
        return [torch.zeros(e, 2 * i, h, dtype=E4M3), torch.zeros(e, -(-2 * i // 128), -(-h // 128)),
                torch.zeros(e, h, i, dtype=E4M3), torch.zeros(e, -(-h // 128), -(-i // 128))]
    return [torch.zeros(e, 2 * i, h // 2, dtype=U8), _tiles(2 * i, h, e), torch.zeros(e, h, i // 2, dtype=U8), _tiles(h, i, e)]


def _moe(t=3, h=64, e=4, top_k=2, layer=None, x=None, logits=None):
    layer = layer or _layer(e, h)
    x = torch.zeros(t, h, dtype=BF16) if x is None else x
    logits = torch.zeros(t, e) if logits is None else logits
    return bf.moe(x, logits, *layer, top_k=top_k)


@needs_native
@pytest.mark.parametrize("call,reason", [
    (lambda: _moe(), "CUDA tensors only"),
    (lambda: _moe(layer=_layer(fmt="mxfp4")), "CUDA tensors only"),
    (lambda: _moe(t=65), "at most 64 tokens"),
    (lambda: _moe(h=48, layer=_layer(h=48)), "multiple of 32"),
    (lambda: _moe(h=8224, layer=_layer(h=8224)), "at most 8192"),
    (lambda: _moe(layer=_layer(i=40)), "multiple of 32"),
    (lambda: _moe(top_k=0), "top_k"),
    (lambda: _moe(top_k=5), "top_k"),
    (lambda: _moe(e=20, top_k=17), "top_k"),
    (lambda: _moe(e=513, layer=_layer()), "512 experts"),
    (lambda: _moe(e=5, layer=_layer(e=4)), "w13 must be"),
    (lambda: _moe(layer=_layer(h=96)), "w13 must be"),
    (lambda: _moe(x=torch.zeros(3, 64)), "bfloat16 or float16"),
    (lambda: _moe(x=torch.zeros(64, dtype=BF16)), "router_logits"),
    (lambda: _moe(x=torch.zeros(3, 68, dtype=BF16)[:, :64]), "row-major"),
    (lambda: _moe(logits=torch.zeros(4, 4)), "router_logits"),
    (lambda: _moe(logits=torch.zeros(3, 4, dtype=torch.float64)), "router_logits"),
    (lambda: _moe(logits=torch.zeros(4, 3).t()), "router_logits"),
    (lambda: _moe(logits=torch.zeros(1, 4).expand(3, 4)), "router_logits"),
    (lambda: _moe(layer=_layer()[:2] + _layer(fmt="mxfp4")[2:]), "w13 and w2|w2 must be|w13 must be"),
    (lambda: _moe(layer=[_layer()[0], _layer()[1][:, :1], *_layer()[2:]]), "scales of w13"),
    (lambda: _moe(layer=[*_layer()[:3], _layer()[3].double()]), "scales of w2"),
    (lambda: _moe(layer=[_layer()[0][:1].expand(4, -1, -1), *_layer()[1:]]), "overlap"),
    (lambda: _moe(layer=[_layer()[0].transpose(1, 2).contiguous().transpose(1, 2), *_layer()[1:]]), "rows"),
])
def test_moe_refusals(call, reason):
    with pytest.raises(ValueError, match=reason):
        call()


@needs_native
def test_moe_experts_refusals():
    x, layer = torch.zeros(3, 64, dtype=BF16), _layer()
    ids, p = torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, 2)
    for bad_ids, bad_p in ((ids.long(), p), (ids, p.double()), (ids[:2], p[:2]), (ids, p[:, :1]), (ids.t().contiguous().t(), p)):
        with pytest.raises(ValueError, match="topk_ids"):
            bf.moe_experts(x, bad_ids, bad_p, *layer)
    with pytest.raises(ValueError, match="CUDA tensors only"):
        bf.moe_experts(x, ids, p, *layer)
    with pytest.raises(ValueError, match="top_k"):
        bf.moe_experts(x, torch.zeros(3, 0, dtype=torch.int32), torch.zeros(3, 0), *layer)


@needs_native
def test_fakes_give_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x = torch.empty(5, 160, dtype=BF16)
        q, s = torch.ops.blockfp8_b200.quantize_mxfp4(x)
        assert q.shape == (5, 80) and s.shape == (1, 2, 32, 16)
        assert torch.ops.blockfp8_b200.dequantize_mxfp4(q, s, dtype=F32).dtype == F32
        assert torch.ops.blockfp8_b200.linear_mxfp4(x, torch.empty(24, 80, dtype=U8), torch.empty(1, 2, 32, 16, dtype=U8)).shape == (5, 24)


@needs_native
def test_c_abi_refuses_before_any_launch():
    lib = _native.capi()
    q = _native.Mxfp4QuantProblem(x=16, ldx=64, x_type=1, q=16, ldq=32, s=16, M=4, K=64)
    for field, value in (("K", 48), ("M", -1), ("x_type", 3), ("q", 8), ("ldq", 24), ("x", 8), ("s", None), ("ldx", 60)):
        bad = _native.Mxfp4QuantProblem.from_buffer_copy(q)
        setattr(bad, field, value)
        assert lib.bfp8_launch_mxfp4_quantize(ctypes.byref(bad), None) == _native.BFP8_EINVAL, field
    g = _native.Mxfp4GemmProblem(a=16, lda=32, sa=16, b=16, ldb=32, sb=16, c=16, ldc=8, M=4, N=8, K=64)
    for field, value in (("N", 12), ("K", 0), ("ldc", 4), ("c", None), ("b", 8), ("ldb", 16), ("sb", None)):
        bad = _native.Mxfp4GemmProblem.from_buffer_copy(g)
        setattr(bad, field, value)
        assert lib.bfp8_launch_mxfp4_gemm(ctypes.byref(bad), None) == _native.BFP8_EINVAL, field
    m = _native.MoeProblem(x=16, ldx=64, x_type=1, logits=16, ld_logits=4, logits_type=0, format=0, w13=16, w13_expert=64 * 192,
                           w13_row=64, s13=16, w2=16, w2_expert=64 * 96, w2_row=96, s2=16, y=16, ldy=64, T=3, H=64, I=96, E=4,
                           top_k=2)
    assert lib.bfp8_moe_workspace_bytes(ctypes.byref(m)) > 0
    for field, value in (("T", 0), ("T", 65), ("H", 16), ("I", 0), ("E", 513), ("top_k", 5), ("x_type", 0), ("format", 2),
                         ("logits", None), ("ids", 16), ("w13_row", 72), ("w2_expert", 8), ("y", None), ("s2", 8)):
        bad = _native.MoeProblem.from_buffer_copy(m)
        setattr(bad, field, value)
        assert lib.bfp8_moe_workspace_bytes(ctypes.byref(bad)) == _native.BFP8_EINVAL, field
        assert lib.bfp8_launch_moe(ctypes.byref(bad), 256, None) == _native.BFP8_EINVAL, field
    assert lib.bfp8_launch_moe(ctypes.byref(m), 8, None) == _native.BFP8_EINVAL  # workspace alignment


@needs_native
@pytest.mark.parametrize("fmt", [0, 1])
def test_every_allowed_layer_has_a_layout(fmt):
    """Shared memory holds some layout of every size that the checks let through."""
    lib = _native.capi()
    m = _native.MoeProblem(x=16, ldx=8192, x_type=1, logits=16, ld_logits=512, logits_type=0, format=fmt, w13=16,
                           w13_expert=1 << 36, w13_row=1 << 15, s13=16, w2=16, w2_expert=1 << 36, w2_row=1 << 15, s2=16, y=16, ldy=8192)
    for m.T in (1, 2, 7, 8, 9, 16, 17, 33, 64):
        for m.H in (32, 96, 1024, 2880, 4096, 4128, 7168, 8160, 8192):
            for m.I in (32, 128, 1408, 2880, 4096, 4128, 14336, 16384 + 32):
                for m.E in (1, 4, 128, 512):
                    for m.top_k in {1, min(8, m.E), min(16, m.E)}:
                        assert lib.bfp8_moe_workspace_bytes(ctypes.byref(m)) > 0, (m.T, m.H, m.I, m.E, m.top_k)


@needs_native
def test_c_abi_refuses_sizes_past_its_integers():
    """Sizes whose tile and unit counts would leave 32 bits are refused with a reason, before any launch."""
    lib = _native.capi()
    big = 2 ** 31 - 32  # (K + 127) / 128 would overflow
    q = _native.Mxfp4QuantProblem(x=16, ldx=big, x_type=1, q=16, ldq=big // 2, s=16, M=4, K=big)
    assert lib.bfp8_launch_mxfp4_quantize(ctypes.byref(q), None) == _native.BFP8_EINVAL
    q = _native.Mxfp4QuantProblem(x=16, ldx=64, x_type=1, q=16, ldq=32, s=16, M=2 ** 31 - 1, K=64)
    assert lib.bfp8_launch_mxfp4_quantize(ctypes.byref(q), None) == _native.BFP8_EINVAL
    d = _native.Mxfp4DequantProblem(q=16, ldq=big // 2, s=16, y=16, ldy=big, y_type=1, M=4, K=big)
    assert lib.bfp8_launch_mxfp4_dequantize(ctypes.byref(d), None) == _native.BFP8_EINVAL
    for sizes in ({"K": big}, {"M": 2 ** 31 - 1}, {"N": 2 ** 31 - 8}):
        g = _native.Mxfp4GemmProblem(a=16, lda=big // 2, sa=16, b=16, ldb=big // 2, sb=16, c=16, ldc=2 ** 31, M=4, N=8, K=64)
        for name, value in sizes.items():
            setattr(g, name, value)
        assert lib.bfp8_launch_mxfp4_gemm(ctypes.byref(g), None) == _native.BFP8_EINVAL, sizes
    g = _native.Mxfp4GemmProblem(a=16, lda=big, b=16, ldb=big // 2, sb=16, c=16, ldc=8, M=4, N=8, K=big, a_type=1)
    assert lib.bfp8_launch_mxfp4_gemm(ctypes.byref(g), None) == _native.BFP8_EINVAL

    def layer(**sizes):
        m = _native.MoeProblem(x=16, ldx=32, x_type=1, logits=16, ld_logits=16, logits_type=0, format=0, w13=16,
                               w13_expert=1 << 40, w13_row=32, s13=16, w2=16, w2_expert=1 << 40, w2_row=1 << 32, s2=16,
                               y=16, ldy=32, T=1, H=32, I=64, E=16, top_k=1)
        for name, value in sizes.items():
            setattr(m, name, value)
        return lib.bfp8_moe_workspace_bytes(ctypes.byref(m))

    assert layer() > 0 and layer(I=1 << 24) > 0
    assert layer(I=(1 << 24) + 32) == _native.BFP8_EINVAL
    assert layer(I=1 << 30) == _native.BFP8_EINVAL  # 2 I leaves 32 bits
    # 64 x 16 pairs in chunks of their own: as many units as 2^31
    assert layer(I=1 << 24, T=64, top_k=16) == _native.BFP8_EINVAL
    assert b"units" in lib.bfp8_last_error()
