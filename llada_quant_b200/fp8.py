"""8-bit floating point (e4m3) with one scale per block of 128: quantizer, product, linear module.

Rows carry one fp32 scale per 128 values, weights one per 128 x 128 block, and
both operands of the product stay in 8 bits: ``out = sum over blocks of
(row scale * weight scale) * (codes . codes)``, fp32 sums, one rounding.  It
stands beside :class:`llada_quant_b200.linear.QuantLinear`, whose integer
weights meet bf16 rows: :class:`Fp8Linear` reads half the bytes of bf16 and,
with many rows, multiplies at the tensor cores' 8-bit rate.  CUDA only, no
backward pass.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Union

import torch
import torch.nn as nn

from . import ops

BLOCK = ops.FP8_BLOCK


@dataclass(slots=True)
class Fp8Tensor:
    """e4m3 ``codes [M, K]`` and fp32 ``scale [ceil(M / block_rows), ceil(K / 128)]``: value = code * scale."""

    codes: torch.Tensor
    scale: torch.Tensor
    block_rows: int

    @property
    def shape(self) -> torch.Size:
        return self.codes.shape

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        M, K = self.codes.shape
        wide = self.scale.repeat_interleave(self.block_rows, 0)[:M].repeat_interleave(BLOCK, 1)[:, :K]
        return (self.codes.to(torch.float32) * wide).to(dtype)

    def storage_bytes(self) -> int:
        return self.codes.numel() + self.scale.numel() * 4


def quantize_fp8(x: torch.Tensor, block_rows: int = 1) -> Fp8Tensor:
    """x ``[M, K]`` (fp32, fp16 or bf16) to e4m3: ``block_rows`` 1 for rows, 128 for weights.

    ``scale = amax / 448`` of the block and ``code`` the e4m3 nearest to ``x * 448 / amax`` (ties to
    even); amax is taken as at least ``448 * 2**-60``.  For fp32 values the quotient is that of fp32
    steps, within ``2**-23`` of it, so a value that close to the border of two codes may get either.  A block
    with a NaN or an infinity dequantizes to NaN.
    """
    codes, scale = ops._fp8_quantize_impl(x, block_rows)
    return Fp8Tensor(codes, scale, block_rows)


def fp8_linear(x: Union[torch.Tensor, Fp8Tensor], weight: Fp8Tensor, bias: Optional[torch.Tensor] = None,
               out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``x . weight^T + bias``: x ``[M, K]`` values (quantized on the way as by :func:`quantize_fp8`) or an
    :class:`Fp8Tensor` of rows; weight ``[N, K]`` in 128 x 128 blocks; K a multiple of 16."""
    return _multiply(ops.Fp8Weight(_weight(weight).codes, weight.scale, bias, out_dtype), x)


def _weight(w: Fp8Tensor) -> Fp8Tensor:
    if w.block_rows != BLOCK:
        raise ValueError("the weight needs one scale per 128 x 128 block")
    return w


def _multiply(w: ops.Fp8Weight, x: Union[torch.Tensor, Fp8Tensor]) -> torch.Tensor:
    if not isinstance(x, Fp8Tensor):
        return w.multiply(x)
    if x.block_rows != 1:
        raise ValueError("the rows need one scale per 128 values of a row")
    return w.multiply(x.codes, x.scale)


class Fp8Linear(nn.Module):
    """Linear layer on e4m3 weights: ``qweight`` uint8 ``[out, in]`` (the codes' bytes), ``scale`` fp32
    ``[ceil(out / 128), ceil(in / 128)]``, ``bias`` of ``compute_dtype`` or None.  Calls see what the buffers
    hold at the call; a bias of another type, or a buffer that is not contiguous and 16-byte aligned, is
    copied for every call.

    The codes are bytes, not float8, so that ``module.half()`` and the like leave them alone.  ``scale`` they
    round, and a scale that is not fp32 is refused: cast a model before its layers are quantized, or load the
    scales again after it.
    """

    def __init__(self, in_features: int, out_features: int, bias: bool = False,
                 compute_dtype: torch.dtype = torch.bfloat16) -> None:
        super().__init__()
        self._sizes(in_features, out_features, compute_dtype)
        self.register_buffer("qweight", torch.zeros(out_features, in_features, dtype=torch.uint8))
        self.register_buffer("scale", torch.ones(ops.fp8_groups(out_features), ops.fp8_groups(in_features)))
        self.register_buffer("bias", torch.zeros(out_features, dtype=compute_dtype) if bias else None)

    def _sizes(self, in_features: int, out_features: int, compute_dtype: torch.dtype) -> None:
        if in_features < 16 or in_features % 16 != 0 or out_features < 1:
            raise ValueError(f"Fp8Linear needs in_features in multiples of 16, got {in_features} -> {out_features}")
        if compute_dtype not in (torch.float32, torch.float16, torch.bfloat16):
            raise ValueError(f"compute_dtype must be fp32, fp16 or bf16, got {compute_dtype}")
        self.in_features = in_features
        self.out_features = out_features
        self.compute_dtype = compute_dtype
        self._ready = None

    @classmethod
    def from_codes(cls, weight: Fp8Tensor, bias: Optional[torch.Tensor] = None,
                   compute_dtype: torch.dtype = torch.bfloat16) -> "Fp8Linear":
        """A layer over codes that are there already (no copy where their rows are whole and aligned)."""
        N, K = _weight(weight).shape
        m = cls.__new__(cls)
        nn.Module.__init__(m)
        m._sizes(K, N, compute_dtype)
        held = ops.Fp8Weight(weight.codes, weight.scale, bias, compute_dtype)
        m.register_buffer("qweight", held.codes.view(torch.uint8).contiguous())
        m.register_buffer("scale", held.scale)
        m.register_buffer("bias", held.bias)
        return m

    @classmethod
    def from_linear(cls, linear: nn.Linear, compute_dtype: torch.dtype = torch.bfloat16) -> "Fp8Linear":
        """Quantize a linear layer's weight on its GPU."""
        w = linear.weight.detach()
        if w.dtype not in (torch.float32, torch.float16, torch.bfloat16):
            w = w.to(torch.float32)
        bias = None if linear.bias is None else linear.bias.detach()
        return cls.from_codes(quantize_fp8(w, BLOCK), bias, compute_dtype)

    @property
    def weight(self) -> Fp8Tensor:
        return Fp8Tensor(self.qweight.view(torch.float8_e4m3fn), self.scale, BLOCK)

    def dequantize_weight(self) -> torch.Tensor:
        return self.weight.dequantize(self.compute_dtype)

    def storage_bytes(self) -> int:
        tensors = [self.qweight, self.scale] + ([self.bias] if self.bias is not None else [])
        return sum(t.numel() * t.element_size() for t in tensors)

    def extra_repr(self) -> str:
        return f"{self.in_features} -> {self.out_features}, e4m3 codes, blocks of {BLOCK}"

    def __getstate__(self):
        return {**self.__dict__, "_ready": None}  # addresses do not outlive the object

    def __setattr__(self, name, value) -> None:
        if name in ("qweight", "scale", "bias"):
            self.__dict__["_ready"] = None  # (it would keep the old buffer's memory until the next call)
        super().__setattr__(name, value)

    def _apply(self, fn, recurse=True):
        self._ready = None
        return super()._apply(fn, recurse)

    def _load_from_state_dict(self, *args, **kwargs) -> None:
        self._ready = None
        super()._load_from_state_dict(*args, **kwargs)

    def _multiplier(self) -> ops.Fp8Weight:
        """The checked operand of the buffers as they are now, kept until one is replaced.  An operand that copied one of
        them serves this call alone: the next sees what the buffer holds then, in its own stream's order and graph."""
        b, r = self._buffers, self._ready
        q, s, bias = b["qweight"], b["scale"], b["bias"]
        at = (q.data_ptr(), s.data_ptr(), 0 if bias is None else bias.data_ptr())
        if r is None or r[0] is not q or r[1] is not s or r[2] is not bias or r[3] != at or r[4].dtype is not self.compute_dtype:
            w = ops.Fp8Weight(q.view(torch.float8_e4m3fn), s, bias, self.compute_dtype)
            self._ready = None if w.copied else (q, s, bias, at, w)
            return w
        return r[4]

    def forward(self, x: Union[torch.Tensor, Fp8Tensor]) -> torch.Tensor:
        """x ``[..., in]`` (any of fp32, fp16, bf16) or an :class:`Fp8Tensor` ``[M, in]`` -> ``[..., out]``."""
        w = self._multiplier()
        if isinstance(x, Fp8Tensor) or x.dim() == 2:
            return _multiply(w, x)
        return w.multiply(x.reshape(-1, x.shape[-1])).reshape(*x.shape[:-1], self.out_features)
