"""Forms of the expert layer's calls: ragged rows of work, expert stacks with
strides, and the C ABI."""

import ctypes

import pytest
import torch

import blockfp8_b200 as bf
import mx_reference as R
from blockfp8_b200 import _native
from test_moe_gpu import DEV, Layer, _check, _gen, _x

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA GPU"),
]


@pytest.mark.parametrize("fmt", ["fp8", "mxfp4"])
@pytest.mark.parametrize("t,e,k,h,i", [(16, 3, 2, 288, 1056), (64, 7, 4, 416, 1504), (33, 5, 5, 96, 4128)])
def test_last_row_of_units_leaves_groups_without_work(fmt, t, e, k, h, i):
    """Batches have two producer warps.  The last row of a CTA's units has work for some of its four groups,
    so that one producer is done while the other still fills its slots: no wait gives up, and every call has
    the same bits."""
    layer = Layer(fmt, e, h, i, seed=31)
    x, logits = _x(t, h, 32), torch.randn(t, e, device=DEV, generator=_gen(33))
    want = bf.moe(x, logits, *layer.args, top_k=k)
    _check(want, x, *R.route(logits, k), layer)
    for _ in range(200):
        y = bf.moe(x, logits, *layer.args, top_k=k)
    assert torch.equal(y, want)
    assert _native.device_status() == 0


@pytest.mark.parametrize("fmt", ["fp8", "mxfp4"])
@pytest.mark.parametrize("t,e,k,h,i", [
    (8, 3, 1, 8192, 96),    # few tokens that do not fit half an SM
    (3, 5, 1, 8192, 4160),  # and K ranges
    (7, 2, 1, 96, 160),     # pairs 0-3 and 4-6 of one expert
    (4, 2, 2, 64, 2080),    # every expert has pairs in both halves
    (5, 2, 1, 128, 4128),
    (8, 2, 2, 160, 96),     # more than eight pairs, experts with all eight tokens
    (6, 1, 1, 64, 4224),
])
def test_few_tokens_in_every_layout(fmt, t, e, k, h, i):
    layer = Layer(fmt, e, h, i, seed=41)
    x, logits = _x(t, h, 42), torch.randn(t, e, device=DEV, generator=_gen(43))
    _check(bf.moe(x, logits, *layer.args, top_k=k), x, *R.route(logits, k), layer)


@pytest.mark.parametrize("fmt", ["fp8", "mxfp4"])
def test_busy_and_quiet_experts_side_by_side(fmt):
    """Chunks of one to eight pairs in every order, so that CTAs' shares begin inside and between them."""
    t, h, i = 64, 96, 416
    layer = Layer(fmt, 40, h, i, seed=51)
    x = _x(t, h, 52)
    g = torch.Generator().manual_seed(53)
    for n in (1, 2, 5, 12, 40):
        ids = torch.randint(0, n, (t, 3), generator=g).to(torch.int32).to(DEV)
        p = torch.rand(t, 3, device=DEV, generator=_gen(54))
        _check(bf.moe_experts(x, ids, p, *layer.args), x, ids, p, layer)


def test_what_the_launch_refuses_is_a_value_error():
    """A limit that the C ABI alone checks (units of one launch); nothing is launched or touched."""
    e, h, i = 16, 32, 1 << 24
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 24 GB")
    u8, fp8 = torch.uint8, torch.float8_e4m3fn
    w13 = torch.empty(e, 2 * i, h, dtype=u8, device=DEV).view(fp8)
    w2 = torch.empty(e, h, i, dtype=u8, device=DEV).view(fp8)
    scales = torch.empty(e, 2 * i // 128, 1, device=DEV), torch.empty(e, 1, i // 128, device=DEV)
    x = torch.zeros(64, h, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError, match="units"):
        bf.moe(x, torch.zeros(64, e, device=DEV), w13, scales[0], w2, scales[1], top_k=16)
    del w13, w2
    torch.cuda.empty_cache()


@pytest.mark.parametrize("fmt", ["fp8", "mxfp4"])
@pytest.mark.parametrize("t", [3, 20])
@pytest.mark.parametrize("h,i", [(160, 96), (288, 416), (2880, 64)])
def test_expert_stacks_with_a_stride_between_experts(fmt, t, h, i):
    """Every other expert of a stack, and padded rows, where rows end inside a 128-byte column: what is read
    past a row's end is another row or nothing, and never counts (it is NaN here)."""
    layer = Layer(fmt, 4, h, i, seed=61)
    x, logits = _x(t, h, 62), torch.randn(t, 4, device=DEV, generator=_gen(63))
    want = bf.moe(x, logits, *layer.args, top_k=2)
    _check(want, x, *R.route(logits, 2), layer)
    w13, s13, w2, s2 = layer.args
    nan = 0x7F  # e4m3's NaN; an MXFP4 byte of 6 and -6 otherwise

    def apart(w, pad):
        room = torch.full((8, w.shape[1], w.shape[2] + pad), nan, dtype=torch.uint8, device=DEV)
        room[::2, :, : w.shape[2]] = w.view(torch.uint8)
        return room.view(w.dtype)[::2, :, : w.shape[2]]

    for pad in (0, 16, 48):
        y = bf.moe(x, logits, apart(w13, pad), s13, apart(w2, pad), s2, top_k=2)
        assert torch.equal(y, want)
    # the last rows of an allocation, nothing behind them
    flat = torch.full((w2.numel() + 64,), nan, dtype=torch.uint8, device=DEV)
    flat[64:] = w2.view(torch.uint8).flatten()
    assert torch.equal(bf.moe(x, logits, w13, s13, flat[64:].view(w2.dtype).view(w2.shape), s2, top_k=2), want)


@pytest.mark.parametrize("fmt", ["fp8", "mxfp4"])
@pytest.mark.parametrize("t,routed", [(2, False), (20, False), (2, True), (20, True)])
def test_c_abi_launches_the_layer(fmt, t, routed):
    lib = _native.capi()
    e, h, i, k = 6, 288, 160, 3
    layer = Layer(fmt, e, h, i, seed=71)
    x, logits = _x(t, h, 72), torch.randn(t, e, device=DEV, generator=_gen(73))
    w13, s13, w2, s2 = layer.args
    ids, p = R.route(logits, k)
    ids, p = ids.to(torch.int32).contiguous(), p.float().contiguous()
    wide = torch.full((t, h + 8), 7.0, dtype=x.dtype, device=DEV)
    m = _native.MoeProblem(x=x.data_ptr(), ldx=h, x_type=1, renormalize=1, format=int(fmt == "mxfp4"),
                           w13=w13.data_ptr(), w13_expert=w13.stride(0), w13_row=w13.stride(1), s13=s13.data_ptr(),
                           w2=w2.data_ptr(), w2_expert=w2.stride(0), w2_row=w2.stride(1), s2=s2.data_ptr(),
                           y=wide.data_ptr(), ldy=h + 8, T=t, H=h, I=i, E=e, top_k=k)
    if routed:
        m.ids, m.weights = ids.data_ptr(), p.data_ptr()
    else:
        m.logits, m.ld_logits, m.logits_type = logits.data_ptr(), e, 0
    size = lib.bfp8_moe_workspace_bytes(ctypes.byref(m))
    room = torch.full((size + 4096,), 0xAB, dtype=torch.uint8, device=DEV)  # any contents, and nothing written behind it
    status = lib.bfp8_launch_moe(ctypes.byref(m), room.data_ptr(), torch.cuda.current_stream().cuda_stream)
    assert status == 0, lib.bfp8_last_error()
    torch.cuda.synchronize()
    want = bf.moe_experts(x, ids, p, *layer.args) if routed else bf.moe(x, logits, *layer.args, top_k=k)
    assert torch.equal(wide[:, :h], want) and (wide[:, h:] == 7.0).all() and (room[size:] == 0xAB).all()
    _check(want, x, ids, p, layer)
