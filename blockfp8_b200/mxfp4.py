"""MXFP4 linear layers: 4-bit weights and activations beside block FP8.

OCP microscaling, 4 bit: e2m1 codes (magnitudes 0, 0.5, 1, 1.5, 2, 3, 4, 6)
with one power-of-two scale per 32 consecutive values of a row.

    e    = max(floor(log2(amax)) - 2, -127)         scale byte = e + 127
    code = e2m1(x * 2^-e)    to nearest, ties to even, at most 6 in magnitude

A block that holds an infinity or a NaN reads back as NaN throughout.

  codes   [R, K / 2]  uint8, row-major, value 2j in the low nibble of byte j
  scales  [ceil(R / 128), ceil(K / 128), 32, 16]  uint8, the tensor cores'
          operand order: row r of a 128-row tile at [r % 32], its four bytes
          of a 128-wide K tile at 4 (r / 32); zeros past the matrix.
          tile_mxfp4_scales / untile_mxfp4_scales convert from and to the
          plain [R, K / 32] of checkpoints.

K is a multiple of 32, N of 8.  The kernels check their arguments themselves
(ValueError) and run on CUDA tensors only.  No reference counterpart: the
reference's formats are block FP8 alone (blockfp8/layout.py:1-35).
"""

import torch

from . import _native
from .layout import cdiv

__all__ = ["dequantize_mxfp4", "gemm_mxfp4", "linear_mxfp4", "quantize_mxfp4", "tile_mxfp4_scales",
           "untile_mxfp4_scales"]


class _Ops:
    """torch.ops.blockfp8_b200's operators, looked up once."""

    def __getattr__(self, name):
        if not _native.load_ops():
            raise RuntimeError(f"native extension not built ({_native.OPS_LIB} missing); "
                               "run python -m blockfp8_b200.build")
        op = getattr(torch.ops.blockfp8_b200, name).default
        setattr(self, name, op)
        return op


ops = _Ops()


def quantize_mxfp4(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x [M, K] bfloat16, float16 or float32 -> (codes, scales) in the layouts above."""
    return ops.quantize_mxfp4(x)


def dequantize_mxfp4(q: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values that the codes stand for, [M, K] bfloat16 or float32.  Exact in both for what quantize_mxfp4
    makes (scale bytes up to 252); under the bytes 253 and 254 codes of 4 and 6 (254: 2 and more) are infinite in
    both types."""
    return ops.dequantize_mxfp4(q, scales, dtype=dtype)


def gemm_mxfp4(a_q: torch.Tensor, a_scales: torch.Tensor, b_q: torch.Tensor, b_scales: torch.Tensor) -> torch.Tensor:
    """C [M, N] bfloat16 = A [M, K] @ B [N, K]^T, both MXFP4, accumulated in float32."""
    return ops.gemm_mxfp4(a_q, a_scales, b_q, b_scales)


def linear_mxfp4(x: torch.Tensor, b_q: torch.Tensor, b_scales: torch.Tensor) -> torch.Tensor:
    """x [M, K] bfloat16 or float16 @ MXFP4 weight^T in one call: gemm_mxfp4(*quantize_mxfp4(x), b_q, b_scales)."""
    return ops.linear_mxfp4(x, b_q, b_scales)


def tile_mxfp4_scales(scales: torch.Tensor) -> torch.Tensor:
    """Scale bytes [..., R, K / 32] (uint8 or float8_e8m0fnu) in the operand layout
    [..., ceil(R / 128), ceil(K / 128), 32, 16]; on any device, once per weight."""
    if scales.dim() < 2 or scales.element_size() != 1:
        raise ValueError(f"scales must be bytes [..., R, K / 32], got {scales.dtype} {tuple(scales.shape)}")
    *lead, r, kb = scales.shape
    rt, kt, n = cdiv(r, 128), cdiv(kb, 4), len(lead)
    s = torch.nn.functional.pad(scales.view(torch.uint8), (0, kt * 4 - kb, 0, rt * 128 - r))
    s = s.view(*lead, rt, 4, 32, kt, 4)  # tile, quarter, row of 32, K tile, block
    return s.permute(*range(n), n, n + 3, n + 2, n + 1, n + 4).reshape(*lead, rt, kt, 32, 16).contiguous()


def untile_mxfp4_scales(scales: torch.Tensor, rows: int, k: int) -> torch.Tensor:
    """The plain bytes [..., rows, k / 32] of scales in the operand layout."""
    *lead, rt, kt, a, b = scales.shape if scales.dim() >= 4 else (0, 0, 0, 0)
    if (a, b) != (32, 16) or (rt, kt) != (cdiv(rows, 128), cdiv(k, 128)) or k % 32:
        raise ValueError(f"scales of a [{rows}, {k}] matrix must be [..., {cdiv(rows, 128)}, {cdiv(k, 128)}, 32, 16], "
                         f"got {tuple(scales.shape)}")
    n = len(lead)
    s = scales.reshape(*lead, rt, kt, 32, 4, 4).permute(*range(n), n, n + 3, n + 2, n + 1, n + 4)
    return s.reshape(*lead, rt * 128, kt * 4)[..., :rows, : k // 32].contiguous()
