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
    """One packed layer, checked when it is made; calls then cost two launches and little host time.

    ``top_k`` is at most E.  ``gate_w`` bf16 ``[E, H]`` (may be None for :meth:`routed` alone), ``bias``
    fp32 ``[E]`` added to the logits (``-inf`` bars an expert), ``renormalize`` divides a token's weights
    by their sum.

    Calls see what the operands hold at the call.  A gate_w that is not contiguous and 16-byte aligned,
    and a bias of another type, are copied for every call.  An operand whose memory was exchanged
    (``module.to()``, ``parameter.data = ...``) is seen by the next call, which checks all of them again;
    until then the layer holds the memory that they had.
    """

    def __init__(self, packed: PackedExperts, gate_w: Optional[torch.Tensor], top_k: int,
                 bias: Optional[torch.Tensor] = None, renormalize: bool = False) -> None:
        if not 1 <= top_k <= packed.num_experts:
            raise ValueError(f"top_k must be 1 to {packed.num_experts}, got {top_k}")
        ops._no_grad_through("the few-token layer", gate_w, bias)
        self.top_k, self._renormalize = top_k, renormalize
        self._packed, self._gate, self._bias = packed, gate_w, bias
        given = (packed.qw1, packed.sw1, packed.qw2, packed.sw2, gate_w, bias)
        self._operands = tuple(t for t in given if t is not None)
        self._prepare()

    def _prepare(self) -> tuple:
        """The descriptors of the operands as they are now: (addresses, what keeps them alive, layer, routed layer);
        no layer where the router's operands have to be copied."""
        p = self._packed
        at = [t.data_ptr() for t in self._operands]
        # (an alias owns its storage even where the operand gets another: no address of `at` is given away)
        held = [t.detach() for t in self._operands]
        layer = None
        if self._gate is not None:
            layer, copies = self._router()
            if copies:
                layer = None
        routed = ops.few_layer(p.qw1, p.sw1, p.qw2, p.sw2, self.top_k, p.bits)
        self._ready = ready = (at, held, layer, routed)
        self.num_experts, self.hidden, self.device = p.num_experts, p.hidden, p.qw1.device
        return ready

    def _router(self) -> tuple:
        """The layer's descriptor, and the copies that it points at where gate_w or bias cannot be read as it is."""
        p = self._packed
        gate_w = ops._aligned(self._gate.detach())
        bias = None if self._bias is None else self._bias.detach().to(torch.float32).contiguous()
        layer = ops.few_layer(p.qw1, p.sw1, p.qw2, p.sw2, self.top_k, p.bits, gate_w, bias, self._renormalize)
        pairs = ((gate_w, self._gate), (bias, self._bias))
        return layer, [t for t, given in pairs if t is not None and t.data_ptr() != given.data_ptr()]

    def _checked(self) -> tuple:
        ready = self._ready
        return ready if [t.data_ptr() for t in self._operands] == ready[0] else self._prepare()

    def _layer(self) -> tuple:
        """(descriptor, what has to live until the call).  Copies are made for each call, in its stream's order and in its
        graph, so that it sees what the operands hold then."""
        ready = self._checked()
        return (ready[2], ready[1]) if ready[2] is not None or self._gate is None else self._router()

    def __call__(self, x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """x bf16 ``[T <= 32, H]`` -> (out bf16 ``[T, H]``, weights fp32 ``[T, k]``, ids int32 ``[T, k]``)."""
        layer, held = self._layer()
        x, weights, ids = self._outputs(x)
        return ops.few_call(layer, x, weights, ids), weights, ids

    def with_logits(self, x: torch.Tensor):
        """As a call, with the router's logits (bias added) fp32 ``[T, E]`` as the fourth."""
        layer, held = self._layer()
        x, weights, ids = self._outputs(x)
        logits = torch.empty(x.shape[0], self.num_experts, dtype=torch.float32, device=self.device)
        out = ops.few_call(layer, x, weights, ids, logits)
        return out, weights, ids, logits if self._bias is None else logits.add_(self._bias.detach())

    def _outputs(self, x: torch.Tensor):
        if self._gate is None:
            raise ValueError("this layer was made without gate_w: call routed(x, weights, ids)")
        x = ops.few_rows(x, self.hidden, self.device)
        T = x.shape[0]
        return (x, torch.empty(T, self.top_k, dtype=torch.float32, device=self.device),
                torch.empty(T, self.top_k, dtype=torch.int32, device=self.device))

    def routed(self, x: torch.Tensor, topk_weights: torch.Tensor, topk_ids: torch.Tensor) -> torch.Tensor:
        """The experts alone, with the caller's routing ``[T, k]``.  Ids outside ``[0, E)`` contribute
        nothing; an expert that a token names twice counts with the sum of the two weights."""
        at, held, layer, routed = self._checked()
        x = ops.few_rows(x, self.hidden, self.device)
        w, ids = ops.few_routing(topk_weights, topk_ids, x.shape[0], self.top_k, self.num_experts, self.device)
        return ops.few_call(routed, x, w, ids)
