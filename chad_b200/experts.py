"""Layers with affine 4-bit weights around the attention: projections and routed experts.

The reference runs its models with weights in the same affine format as the cache
(tests/test_engine_kvquant.py:22-37): every projection is an mx.quantized_matmul, and its
mixture-of-experts layers are fused kernels over stacked quantized experts
(src/chad/mlx_moe_fused.py). Both are built here on the operators of `ops`, forward only: like
the attention, none of them records a gradient.
"""

from __future__ import annotations

from typing import Optional

import torch

from . import ops
from .ops import GROUP_SIZE, QuantTuple


def quantize_weight(weight: torch.Tensor, bits: int = 4,
                    dtype: Optional[torch.dtype] = None) -> QuantTuple:
    """(w, scales, biases) of a weight (..., N, K), K a multiple of 64: mx.quantize of a weight
    matrix. The groups run along K, so the rows are quantized as K/64 rows of one group. (8 bits to
    store a weight and `ops.dequantize` it; the products take 4.)"""
    *lead, k = weight.shape
    if k % GROUP_SIZE:
        raise ValueError(f"K {k} is not a multiple of {GROUP_SIZE}")
    w, s, b = ops.quantize(weight.reshape(-1, GROUP_SIZE), bits, scale_dtype=dtype)
    return (w.view(*lead, k * bits // 32), s.view(*lead, k // GROUP_SIZE),
            b.view(*lead, k // GROUP_SIZE))


class QuantizedLinear:
    """y = act(x W^T) with 4-bit weights: what an nn.QuantizedLinear of the reference's models
    computes. activation="swiglu" takes the concatenated gate and up projections."""

    def __init__(self, w_quant: QuantTuple, activation: Optional[str] = None):
        self.w_quant = tuple(w_quant)
        self.activation = activation

    @classmethod
    def from_weight(cls, weight: torch.Tensor, activation: Optional[str] = None,
                    dtype: Optional[torch.dtype] = None) -> "QuantizedLinear":
        return cls(quantize_weight(weight, dtype=dtype), activation)

    def __call__(self, x: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        return ops.quantized_matmul(x, self.w_quant, activation=self.activation, out=out)


class QuantizedExperts:
    """Routed feed-forward: top-k routing, gated first projection of the chosen experts, their
    second projection and the weighted sum back in token order.

    gate_up: 4-bit weights (E, 2F, K), the gate's F rows first; down: (E, K, F).
    """

    def __init__(self, gate_up: QuantTuple, down: QuantTuple, top_k: int, normalize: bool = True):
        e, f2, _ = gate_up[0].shape
        k = gate_up[1].shape[-1] * GROUP_SIZE
        if tuple(down[0].shape[:2]) != (e, k) or down[1].shape[-1] * GROUP_SIZE * 2 != f2:
            raise ValueError(f"down {tuple(down[0].shape)} does not match gate_up "
                             f"{tuple(gate_up[0].shape)}")
        if not 0 < top_k <= e:
            raise ValueError(f"top_k must be in 1..{e} (got {top_k})")
        self.gate_up = tuple(gate_up)
        self.down = tuple(down)
        self.top_k = top_k
        self.normalize = normalize

    @classmethod
    def from_weights(cls, gate_up: torch.Tensor, down: torch.Tensor, top_k: int,
                     normalize: bool = True,
                     dtype: Optional[torch.dtype] = None) -> "QuantizedExperts":
        return cls(quantize_weight(gate_up, dtype=dtype), quantize_weight(down, dtype=dtype),
                   top_k, normalize)

    def __call__(self, x: torch.Tensor, logits: torch.Tensor,
                 residual: Optional[torch.Tensor] = None) -> torch.Tensor:
        """x (T, K), router logits (T, E) -> (residual +) the experts' weighted sum (T, K)."""
        if x.dim() != 2 or logits.dim() != 2 or logits.shape[0] != x.shape[0]:
            raise ValueError(f"x {tuple(x.shape)} and logits {tuple(logits.shape)} must be (T, K) "
                             "and (T, E) of the same tokens")
        r = ops.route_topk(logits, self.top_k, normalize=self.normalize)
        h = ops.grouped_quantized_matmul(x, self.gate_up, r.offsets, rows=r.rows,
                                         activation="swiglu")
        y = ops.grouped_quantized_matmul(h, self.down, r.offsets)
        return ops.expert_combine(y, r.slots, r.weights, residual=residual)
