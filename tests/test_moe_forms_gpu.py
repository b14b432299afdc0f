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
