"""Forms of the expert layer's calls: ragged rows of work, expert stacks with
strides, and the C ABI."""

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
