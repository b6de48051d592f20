"""Projections in 8 bits: a layer whose four products (q/k/v, output, gate/up, down) take rows of float8_e4m3 numbers with a power-of-two
scale to each 128 features, on both sides (``csrc/gemm_fp8.cu``).

The weights are rounded once, when they are bound; the tokens' rows where they arise: in the norm before a product
(``rmsnorm_fp8``), behind attention, and in the gated product itself, whose activation leaves in 8 bits for the down projection
(``swiglu_fp8``).  What lies between stays as it is: the residual sum in float32, q, k, v, the cache and attention in
bfloat16, every sum in float32.  The reference keeps its weights in 16 bits (gpu_decoder.cu:15-61).

A model says so with ``"projection_dtype": "float8_e4m3"`` in its ``config.json`` (its layers) and ``"output_projection_dtype"``
(the projection over the vocabulary); its tensors are stored as ever.
"""
from __future__ import annotations

from typing import Optional

import torch

from .. import kernels
from ..config.registry import register_part
from ..weights.loader import TensorSource
from . import matmul_backend
from .attention import GQAttention
from .base import ResidualStream
from .linear import Linear
from .mlp import ACTIVATIONS, SwiGLU
from .norm import RMSNorm

FEW_TOKENS = 16         # up to here q, k and v stay float32 sums, which the rotation (and attention of single tokens) takes with the bias


def _need_bfloat16(dtype: torch.dtype) -> None:
    if dtype != torch.bfloat16:
        raise ValueError(f"projections in 8 bits belong to a bfloat16 engine, got {dtype}")


def rows_in_8_bits(x: torch.Tensor) -> kernels.Fp8Rows:
    out = kernels.fp8_rows(x.shape[0], x.shape[1], x.device)
    kernels.quantize_fp8(x, out)
    return out


class Fp8Linear(Linear):
    """``Linear`` with its weights in 8 bits (``rows``); its input is ``kernels.Fp8Rows``."""
    rows: Optional[kernels.Fp8Rows] = None

    def bind(self, source: TensorSource, dtype: torch.dtype, device: torch.device) -> None:
        _need_bfloat16(dtype)
        self.rows = kernels.fp8_rows(self.out_features, self.in_features, device)
        at = 0
        for stem, n in self.pieces:                # a piece at a time: none is held twice
            self._round(source.get(f"{stem}{self.weight_suffix}").to(device=device), at)
            at += n
        if self.has_bias:
            bs = [source.get(f"{stem}{self.bias_suffix}").to(device=device, dtype=torch.float32) for stem, _ in self.pieces]
            self.bias = (torch.cat(bs, dim=0) if len(bs) > 1 else bs[0]).contiguous()

    def bind_tensor(self, weight: torch.Tensor) -> None:
        """An already prepared weight (a tied output projection's embedding table), rounded here."""
        _need_bfloat16(weight.dtype)
        self.rows = kernels.fp8_rows(self.out_features, self.in_features, weight.device)
        self._round(weight, 0)

    def _round(self, weight: torch.Tensor, at: int) -> None:
        if weight.dtype not in (torch.bfloat16, torch.float32):
            weight = weight.float()                # (float16 as it is stored)
        n = weight.shape[0]
        kernels.quantize_fp8(weight.contiguous(), kernels.Fp8Rows(self.rows.q[at:at + n], self.rows.s[at:at + n]))
        torch.cuda.current_stream(weight.device).synchronize()      # the products read them ahead of what is before them on the stream

    def forward(self, x: kernels.Fp8Rows, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        return self._product(x, self.bias, out_dtype or torch.bfloat16)

    def forward_partial(self, x: kernels.Fp8Rows, with_bias: bool = True) -> torch.Tensor:
        return self._product(x, self.bias if with_bias else None, torch.bfloat16)

    def sums(self, x: kernels.Fp8Rows) -> torch.Tensor:
        """float32 [1, T, N] without the bias, in the form of partial sums."""
        return self._product(x, None, torch.float32).unsqueeze(0)

    def _product(self, x: kernels.Fp8Rows, bias: Optional[torch.Tensor], dtype: torch.dtype) -> torch.Tensor:
        out = torch.empty((x.q.shape[0], self.out_features), dtype=dtype, device=x.q.device)
        kernels.gemm_fp8(x, self.rows, bias, out, resident=True)
        matmul_backend.counters["own"] += 1
        return out


@register_part("norm", "rmsnorm_fp8")
class RMSNormFp8(RMSNorm):
    """``rmsnorm`` whose output leaves as rows in 8 bits, for products that take them."""

    def native_params(self):
        return dict(super().native_params(), kind="rmsnorm_fp8")

    def forward(self, stream: ResidualStream, out_dtype: torch.dtype, rows: Optional[torch.Tensor] = None) -> kernels.Fp8Rows:
        stream.settle()
        out = kernels.fp8_rows(stream.x.shape[0] if rows is None else rows.numel(), self.size, stream.x.device)
        kernels.add_rmsnorm_fp8(stream.x, stream.delta, self.weight, out, self.eps, rows=rows, write_back=rows is None,
                                delta_scale=stream.delta_scale)
        if rows is None:
            stream.clear()
        return out


@register_part("mixer", "gq_attention_fp8")
class GQAttentionFp8(GQAttention):
    """``gq_attention`` with its two projections in 8 bits, its input too."""

    def __init__(self, *args, **kw):
        super().__init__(*args, **kw)
        self.qkv = Fp8Linear(self.qkv.in_features, self.qkv.pieces, bias=self.qkv.has_bias)
        self.out = Fp8Linear(self.out.in_features, self.out.pieces, bias=self.out.has_bias)

    def native_params(self):
        answer = super().native_params()
        return answer and dict(answer, kind="gq_attention_fp8", wqkv=self.qkv.rows, wo=self.out.rows)

    def _few_token_sums(self, x: kernels.Fp8Rows) -> Optional[torch.Tensor]:
        return self.qkv.sums(x) if x.q.shape[0] <= FEW_TOKENS else None

    def _out_product(self, attn: torch.Tensor) -> torch.Tensor:
        return self.out.forward_partial(rows_in_8_bits(attn))


@register_part("feed_forward", "swiglu_fp8")
class SwiGLUFp8(SwiGLU):
    """``swiglu`` (silu or gelu_tanh) with its products in 8 bits: one from the norm's rows to the activation's, one from those to the
    branch's output."""

    def __init__(self, *args, **kw):
        super().__init__(*args, **kw)
        if self.activation == "clamped":
            raise ValueError("feed-forward in 8 bits: the activation must be 'silu' or 'gelu_tanh'")
        self.gate_up = Fp8Linear(self.gate_up.in_features, self.gate_up.pieces, bias=self.has_bias, weight_suffix=self.gate_up.weight_suffix,
                                 bias_suffix=self.gate_up.bias_suffix)
        self.down = Fp8Linear(self.down.in_features, self.down.pieces, bias=self.has_bias, weight_suffix=self.down.weight_suffix,
                              bias_suffix=self.down.bias_suffix)

    def native_params(self):
        answer = super().native_params()
        return answer and dict(answer, kind="swiglu_fp8", wgu=self.gate_up.rows, wd=self.down.rows)

    def _products(self, x: kernels.Fp8Rows) -> torch.Tensor:
        h = kernels.fp8_rows(x.q.shape[0], self.intermediate_size, x.q.device)
        kernels.gemm_fp8_gated(x, self.gate_up.rows, self.gate_up.bias, h, ACTIVATIONS[self.activation], resident=True)
        matmul_backend.counters["own"] += 1
        return self._down(h)
