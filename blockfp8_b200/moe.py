"""A mixture-of-experts layer for a few tokens (decode), weights streamed once.

    y[t] = sum_j p[t, j] W2[e] (silu(W1[e] x[t]) * (W3[e] x[t])),   e = ids[t, j]

  x      [T, H]       bfloat16 or float16, 1 <= T <= 64; y has its type
  w13    [E, 2 I, H]  W1 (gate) over W3 (up);  w2 [E, H, I]
         block FP8:  float8_e4m3fn with float32 scales
                     [E, ceil(rows / 128), ceil(K / 128)]
         MXFP4:      uint8 codes [E, rows, K / 2] with scale tiles
                     [E, ceil(rows / 128), ceil(K / 128), 32, 16]

Activations are not quantized: at these sizes the weights are the traffic.  x
enters the products as f16 with one power of two per token and 128 values,
which holds bf16 exactly down to 2^-28 of the largest of them; h as two such
parts, 22 bits of each value (2^-39 of the largest at worst).  (The dense
block-FP8 linear quantizes its activations; a layer built from it differs by
that rounding.)
Three launches (two kernels that stream weights, and a small sum) and no
synchronisation; results do not depend on the order in which CTAs finish.
MXFP4 scales multiply fp32 sums before the activations' own powers of two do:
scale bytes above 230 (2^103) may overflow there although the result would not.  H and I are multiples of 32, H at most 8192, E at most
512, top_k at most 16.  The kernels check their arguments themselves
(ValueError).  No reference counterpart: the reference covers dense linears.
"""

import torch

from .mxfp4 import ops

__all__ = ["moe", "moe_experts"]


def moe(x: torch.Tensor, router_logits: torch.Tensor, w13: torch.Tensor, w13_scales: torch.Tensor, w2: torch.Tensor,
        w2_scales: torch.Tensor, top_k: int, renormalize: bool = True) -> torch.Tensor:
    """The layer from its router's logits [T, E] (float32, bfloat16 or float16).

    A token goes to its top_k largest logits, ties to the lower index; -inf
    and NaN are never chosen, so a token with no other logit gets zeros.  Its
    weights are the softmax over all experts, or over the chosen ones
    (renormalize)."""
    return ops.moe(x, router_logits, w13, w13_scales, w2, w2_scales, top_k, renormalize)


def moe_experts(x: torch.Tensor, topk_ids: torch.Tensor, topk_weights: torch.Tensor, w13: torch.Tensor,
                w13_scales: torch.Tensor, w2: torch.Tensor, w2_scales: torch.Tensor) -> torch.Tensor:
    """The layer after a router of the caller's: topk_ids [T, top_k] int32 and
    topk_weights [T, top_k] float32.  An id outside [0, E) adds nothing (a
    padded token, an expert of another rank); an id may repeat."""
    return ops.moe_experts(x, topk_ids, topk_weights, w13, w13_scales, w2, w2_scales)
