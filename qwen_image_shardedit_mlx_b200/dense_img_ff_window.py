"""Dense image MLP from q6 layers, with the reference's LoRA rules.

Mirrors shardedit_mlx/dense_img_ff_window.py: ``materialize_dense_linear``
dequantises a q6 layer once (here on the GPU dequant kernel) and folds
several adapters into the dense weight (:93-153); a single adapter stays
additive (:95-118); ``DenseFeedForward`` runs dense Linear math with the
optional additive adapters (:32-67); ``materialize_dense_img_ff`` builds one
from an ``img_ff``-shaped module and reports the dense bytes (:156-196).

This is the dense comparator of the q6 path (library GEMMs on dequantised
weights), kept for A/B checks and for callers that trade HBM for speed.
``DenseFeedForward.fused`` / ``.half`` run the same MLP, and the feed-forward
half of a block around it, on this library's dense kernels (dense.py), with
gradients: what fine-tuning a materialised layer needs.
"""

from __future__ import annotations

import torch
import torch.nn.functional as F

from qwen_image_shardedit_mlx_b200.dense import dense_linear, layer_norm_modulate
from qwen_image_shardedit_mlx_b200.lora import LoRAAdapter, iter_adapters, lora_delta_weight
from qwen_image_shardedit_mlx_b200.q6_metal_mlp import DenseLinearWeights, dequantize_linear, quantized_linear_spec


class DenseFeedForward:
    """img_ff replacement: dense Linear math matching QwenFeedForward."""

    def __init__(self, mlp_in: DenseLinearWeights, mlp_out: DenseLinearWeights, *,
                 mlp_in_lora: tuple[torch.Tensor, torch.Tensor, float] | None = None,
                 mlp_out_lora: tuple[torch.Tensor, torch.Tensor, float] | None = None) -> None:
        self.mlp_in = mlp_in
        self.mlp_out = mlp_out
        self.mlp_in_lora = mlp_in_lora
        self.mlp_out_lora = mlp_out_lora

    @staticmethod
    def _linear(hidden: torch.Tensor, weights: DenseLinearWeights,
                lora: tuple[torch.Tensor, torch.Tensor, float] | None) -> torch.Tensor:
        out = hidden @ weights.weight.T
        if weights.bias is not None:
            out = out + weights.bias
        if lora is not None:
            a, b, scale = lora
            out = out + scale * ((hidden @ a) @ b)
        return out

    def __call__(self, hidden: torch.Tensor) -> torch.Tensor:
        hidden = self._linear(hidden, self.mlp_in, self.mlp_in_lora)
        hidden = F.gelu(hidden, approximate="tanh")
        return self._linear(hidden, self.mlp_out, self.mlp_out_lora)

    def fused(self, hidden: torch.Tensor, *, residual: torch.Tensor | None = None,
              gate: torch.Tensor | None = None) -> torch.Tensor:
        """``residual + gate * ff(hidden)`` in two launches of ``dense_linear``
        (bias and GELU, then bias, gate and residual, in the epilogues);
        differentiable in hidden, the weights, the biases, the gate and the
        residual.  bf16 or fp16.  An additive adapter does not fit the epilogue:
        fold it into the weight first (``materialize_dense_img_ff(fold_single=True)``)."""

        if self.mlp_in_lora is not None or self.mlp_out_lora is not None:
            raise ValueError("fused() takes no additive LoRA: materialise with fold_single=True")
        mid = dense_linear(hidden, self.mlp_in.weight, self.mlp_in.bias, activation="gelu_tanh")
        return dense_linear(mid, self.mlp_out.weight, self.mlp_out.bias, residual=residual, gate=gate)

    def half(self, x: torch.Tensor, shift: torch.Tensor, scale: torch.Tensor, gate: torch.Tensor, *,
             eps: float = 1e-6) -> torch.Tensor:
        """The feed-forward half of a block, ``x + gate * ff(LayerNorm(x) * (1 + scale) + shift)``
        (benchmarks/profile_qwen_block.py:262-301), differentiable in x, the
        modulation vectors ([D], or [S, D] with one set per sample) and the
        weights."""

        return self.fused(layer_norm_modulate(x, shift, scale, eps=eps), residual=x, gate=gate)


def _nbytes(t: torch.Tensor | None) -> int:
    return 0 if t is None else t.numel() * t.element_size()


def _dense_nbytes(w: DenseLinearWeights) -> int:
    return _nbytes(w.weight) + _nbytes(w.bias)


def materialize_dense_linear(layer: torch.nn.Module, *, dtype: torch.dtype = torch.bfloat16,
                             fold_single: bool = False) -> DenseLinearWeights:
    """Dequantise a q6 layer; with two or more adapters fold sum s_i (A_i B_i)^T
    into the weight (the reference keeps a single adapter additive;
    ``fold_single`` folds that one too)."""

    dense = dequantize_linear(quantized_linear_spec(layer), dtype=dtype)
    adapters = list(iter_adapters(layer))
    if len(adapters) >= (1 if fold_single else 2):
        delta = lora_delta_weight(adapters, dtype=torch.float32)
        if tuple(delta.shape) != tuple(dense.weight.shape):
            raise ValueError(f"LoRA delta shape {tuple(delta.shape)} != weight shape {tuple(dense.weight.shape)}")
        dense = DenseLinearWeights(weight=(dense.weight.to(torch.float32) + delta.to(dense.weight.device)).to(dtype),
                                   bias=dense.bias)
    return dense


def _additive(layer: torch.nn.Module, dtype: torch.dtype) -> tuple[torch.Tensor, torch.Tensor, float] | None:
    adapters: list[LoRAAdapter] = list(iter_adapters(layer))
    if len(adapters) != 1:
        return None
    ad = adapters[0]
    return ad.lora_A.to(dtype), ad.lora_B.to(dtype), float(ad.scale)


def materialize_dense_img_ff(img_ff: torch.nn.Module, *, dtype: torch.dtype = torch.bfloat16,
                             fold_single: bool = False) -> tuple[DenseFeedForward, int]:
    """Dequantise one feed-forward's mlp_in / mlp_out into a DenseFeedForward;
    returns it with the dense weight bytes.  ``fold_single`` folds a layer's only
    adapter into its weight instead of keeping it additive."""

    mlp_in = materialize_dense_linear(img_ff.mlp_in, dtype=dtype, fold_single=fold_single)
    mlp_out = materialize_dense_linear(img_ff.mlp_out, dtype=dtype, fold_single=fold_single)
    dense = DenseFeedForward(mlp_in, mlp_out,
                             mlp_in_lora=None if fold_single else _additive(img_ff.mlp_in, dtype),
                             mlp_out_lora=None if fold_single else _additive(img_ff.mlp_out, dtype))
    return dense, _dense_nbytes(mlp_in) + _dense_nbytes(mlp_out)
