"""The PACKED MoE layer for at most 32 tokens: a decoding step's block, or one token.

:func:`llada_quant_b200.fused_moe.moe_layer` is laid out for hundreds of rows
per call (router, alignment, permute, expert GEMMs, combine).  With a few
tokens those launches cost more than the weights they read, so
:class:`FewTokenMoE` runs the layer in two: router, top-k and GEMM1, then GEMM2
and the combine.  ``moe_layer(..., impl="few")`` and ``fused_moe(...,
impl="few")`` reach the same kernels.

Numerics: weights ``q * s`` in fp32 without the rounding of each weight to
bf16, router logits and ``h`` in fp32 accuracy, one rounding of the output.
The layer for many tokens rounds all of these to bf16, so near-equal logits may
choose another expert here; a caller who needs its choice routes with
``ops.route`` and calls :meth:`FewTokenMoE.routed`.  CUDA only, no backward pass.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import ops
from .moe import PackedExperts


class FewTokenMoE:
    """One packed layer, checked once; calls then cost two launches and little host time.

    ``gate_w`` bf16 ``[E, H]`` (may be None for :meth:`routed` alone), ``bias`` fp32 ``[E]`` added to
    the logits (``-inf`` bars an expert), ``renormalize`` divides a token's weights by their sum.
    """

    def __init__(self, packed: PackedExperts, gate_w: Optional[torch.Tensor], top_k: int,
                 bias: Optional[torch.Tensor] = None, renormalize: bool = False) -> None:
        if not 1 <= top_k <= packed.num_experts:
            raise ValueError(f"top_k must be 1 to {packed.num_experts}, got {top_k}")
        ops._no_grad_through("the few-token layer", gate_w, bias)
        gate_w = None if gate_w is None else ops._aligned(gate_w)
        bias = None if bias is None else bias.to(torch.float32).contiguous()
        self._held = (packed, gate_w, bias)  # the descriptor has their addresses
        args = (packed.qw1, packed.sw1, packed.qw2, packed.sw2, top_k, packed.bits)
        self._layer = None if gate_w is None else ops.few_layer(*args, gate_w, bias, renormalize)
        self._routed = ops.few_layer(*args)
        self.top_k = top_k
        self.num_experts, self.hidden = packed.num_experts, packed.hidden
        self.device = packed.qw1.device

    def __call__(self, x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """x bf16 ``[T <= 32, H]`` -> (out bf16 ``[T, H]``, weights fp32 ``[T, k]``, ids int32 ``[T, k]``)."""
        x, weights, ids = self._outputs(x)
        return ops.few_call(self._layer, x, weights, ids), weights, ids

    def with_logits(self, x: torch.Tensor):
        """As a call, with the router's logits (bias added) fp32 ``[T, E]`` as the fourth."""
        x, weights, ids = self._outputs(x)
        logits = torch.empty(x.shape[0], self.num_experts, dtype=torch.float32, device=self.device)
        return ops.few_call(self._layer, x, weights, ids, logits), weights, ids, logits

    def _outputs(self, x: torch.Tensor):
        if self._layer is None:
            raise ValueError("this layer was made without gate_w: call routed(x, weights, ids)")
        x = ops.few_rows(x, self.hidden, self.device)
        T = x.shape[0]
        return (x, torch.empty(T, self.top_k, dtype=torch.float32, device=self.device),
                torch.empty(T, self.top_k, dtype=torch.int32, device=self.device))

    def routed(self, x: torch.Tensor, topk_weights: torch.Tensor, topk_ids: torch.Tensor) -> torch.Tensor:
        """The experts alone, with the caller's routing ``[T, k]``.  Ids outside ``[0, E)`` contribute
        nothing; an expert that a token names twice counts with the sum of the two weights."""
        x = ops.few_rows(x, self.hidden, self.device)
        w, ids = ops.few_routing(topk_weights, topk_ids, x.shape[0], self.top_k, self.num_experts, self.device)
        return ops.few_call(self._routed, x, w, ids)
