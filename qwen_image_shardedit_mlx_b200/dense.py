"""Dense 16-bit linear and layer norm with gradients.

The trainable twins of what the q6 block computes around its packed weights:

* ``dense_linear``: ``residual + gate * act(x @ W^T + bias)`` with the epilogue
  of ``q6_linear`` over a dense bf16 / fp16 weight (a materialised feed-forward
  layer, an embedding or a modulation projection), from one row to long ones.
* ``layer_norm`` / ``layer_norm_modulate``: an affine norm, or the adaLN form
  ``LayerNorm(x) * (1 + scale) + shift`` with one vector pair per sample; bf16,
  fp16 or fp32 rows of any width.

Both differentiate through ``torch.autograd`` and have functional forms
(``*_forward`` / ``*_backward``) that launch the same kernels without it.  Inputs
with a forward-mode tangent are refused.  The functional forms may be captured in a
CUDA graph.  A differentiable call under
capture, and the backward pass of an earlier one, are refused: autograd would
run parts of it on the streams that it recorded for the leaves, outside the
capture.

Tensors must live on one CUDA device; kernels are ordered on its current
stream, nothing synchronises, and equal calls give equal bits.  The checks, the
allocations and the autograd nodes are native (csrc/q6_torch.cpp, the extension
module ``_q6torch``), the kernels libq6b200.so's.
"""

from __future__ import annotations

from collections.abc import Sequence
from types import ModuleType
from typing import NamedTuple

import torch

from qwen_image_shardedit_mlx_b200 import _lib

ACTIVATIONS = {None: _lib.Q6_ACT_NONE, "gelu_tanh": _lib.Q6_ACT_GELU_TANH, "silu": _lib.Q6_ACT_SILU}
_LINEAR_OUTPUTS = {"x": _lib.Q6_GRAD_X, "weight": _lib.Q6_GRAD_W, "bias": _lib.Q6_GRAD_BIAS, "gate": _lib.Q6_GRAD_GATE}

_module: ModuleType | None = None


def _native() -> ModuleType:
    """The extension module (loaded at the first call; there is no fallback)."""

    global _module
    if _module is None:
        _lib.lib()  # a clear error where the library is not built
        try:
            from qwen_image_shardedit_mlx_b200 import _q6torch
        except ImportError as e:
            raise RuntimeError("the extension module _q6torch is not built; run "
                               f"`python -m qwen_image_shardedit_mlx_b200.build` ({e})") from e
        _module = _q6torch
    return _module


def _activation(name: str | None) -> int:
    try:
        return ACTIVATIONS[name]
    except (KeyError, TypeError):
        raise ValueError(f"activation must be one of {tuple(ACTIVATIONS)}, got {name!r}") from None


# ----------------------------------------------------------------------------- linear


class DenseGrads(NamedTuple):
    """Gradients of ``dense_linear`` (None where not asked for); the residual's is ``dy`` itself."""

    x: torch.Tensor | None
    weight: torch.Tensor | None
    bias: torch.Tensor | None
    gate: torch.Tensor | None


def dense_linear(
    x: torch.Tensor,
    weight: torch.Tensor,
    bias: torch.Tensor | None = None,
    *,
    activation: str | None = None,
    residual: torch.Tensor | None = None,
    gate: torch.Tensor | None = None,
) -> torch.Tensor:
    """``residual + gate * act(x @ W^T + bias)`` for x [..., K] and a dense weight [N, K]; returns [..., N].

    bf16 or fp16, every tensor in x's dtype; sums in fp32, one rounding at the
    output.  ``activation`` is None, "gelu_tanh" or "silu".  ``gate`` is [N], or
    [S, N] with S the leading size of x (one vector per sample); ``residual``
    has the output's shape.  Differentiable in every tensor (once).  x, the
    weight, the residual and the gate may be strided views; an operand whose
    address or row stride is no multiple of 16 bytes is copied to an aligned
    layout first.
    """

    return _native().dense_linear(x, weight, bias, _activation(activation), residual, gate)


def dense_linear_forward(
    x: torch.Tensor,
    weight: torch.Tensor,
    bias: torch.Tensor | None = None,
    *,
    activation: str | None = None,
    residual: torch.Tensor | None = None,
    gate: torch.Tensor | None = None,
    save_preact: bool = False,
) -> tuple[torch.Tensor, torch.Tensor | None]:
    """(y, preact): ``dense_linear`` without autograd.  With ``save_preact`` the
    second value is ``x @ W^T + bias`` for ``dense_linear_backward``, in fp16
    (whatever x's dtype, held at the largest fp16 value, beyond which the slope of
    every activation is 0 or 1), or in fp32 when a gate is given; else None."""

    return _native().dense_linear_forward(x, weight, bias, _activation(activation), residual, gate, save_preact)


def dense_linear_backward(
    dy: torch.Tensor,
    x: torch.Tensor | None,
    weight: torch.Tensor | None,
    *,
    preact: torch.Tensor | None = None,
    activation: str | None = None,
    gate: torch.Tensor | None = None,
    outputs: Sequence[str] = ("x", "weight", "bias"),
) -> DenseGrads:
    """Gradients of ``dense_linear`` for the output gradient ``dy``.

    ``outputs`` names what to compute ("x", "weight", "bias", "gate").  ``x``
    may be None without "weight", ``weight`` may be None without "x".
    ``preact`` is the forward's, needed with an activation or for "gate".  The
    weight's and the x gradient multiply the gradient of the pre-activation
    rounded to the tensors' dtype (in fp16 with that type's range: beyond 65504 it is
    infinite); all sums are held in fp32.
    """

    want = 0
    for name in outputs:
        if name not in _LINEAR_OUTPUTS:
            raise ValueError(f"outputs must be among {tuple(_LINEAR_OUTPUTS)}; got {tuple(outputs)}")
        want |= _LINEAR_OUTPUTS[name]
    return DenseGrads(*_native().dense_linear_backward(dy, x, weight, preact, _activation(activation), gate, want))


# ------------------------------------------------------------------------- layer norm


class NormGrads(NamedTuple):
    """Gradients of a layer norm (None where not asked for)."""

    x: torch.Tensor | None
    weight: torch.Tensor | None
    bias: torch.Tensor | None


def _vectors_1d(weight: torch.Tensor | None, bias: torch.Tensor | None) -> None:
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and t.dim() != 1:
            raise ValueError(f"{name} must be 1-D, got {tuple(t.shape)}")


def _pair(shift: torch.Tensor, scale: torch.Tensor) -> None:
    if shift is None or scale is None:
        raise ValueError("layer_norm_modulate needs shift and scale")


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, *,
               eps: float = 1e-6) -> torch.Tensor:
    """``LayerNorm(x) * weight + bias`` over the last axis (bf16, fp16 or fp32).

    ``weight`` and ``bias`` ([D], either may be None) are in x's dtype or in
    fp32.  Statistics and sums are held in fp32, the output is rounded once.
    Differentiable in every tensor (once).
    """

    _vectors_1d(weight, bias)
    return _native().layer_norm(x, weight, bias, eps, 0)


def layer_norm_modulate(x: torch.Tensor, shift: torch.Tensor, scale: torch.Tensor, *, eps: float = 1e-6) -> torch.Tensor:
    """``LayerNorm(x) * (1 + scale) + shift`` over the last axis: the block's adaLN
    modulate, differentiable, for any width.  ``shift`` / ``scale`` are [D], or
    [S, D] with S the leading size of x (one pair per sample; strided views of a
    modulation output are read in place)."""

    _pair(shift, scale)
    return _native().layer_norm(x, scale, shift, eps, _lib.Q6_NORM_ONE_PLUS)


def layer_norm_forward(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, *,
                       eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(y, mean, rstd): ``layer_norm`` without autograd; mean and rstd are fp32 [rows]."""

    _vectors_1d(weight, bias)
    return _native().layer_norm_forward(x, weight, bias, eps, 0)


def layer_norm_modulate_forward(x: torch.Tensor, shift: torch.Tensor, scale: torch.Tensor, *,
                                eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(y, mean, rstd): ``layer_norm_modulate`` without autograd."""

    _pair(shift, scale)
    return _native().layer_norm_forward(x, scale, shift, eps, _lib.Q6_NORM_ONE_PLUS)


def _norm_backward(dy, x, weight, mean, rstd, outputs, flags) -> NormGrads:
    want = set(outputs)
    if not want <= {"x", "weight", "bias"}:
        raise ValueError(f"outputs must be among x, weight, bias; got {tuple(outputs)}")
    return NormGrads(*_native().layer_norm_backward(dy, x, weight, mean, rstd, flags, "x" in want, "weight" in want,
                                                    "bias" in want))


def layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, weight: torch.Tensor | None, mean: torch.Tensor,
                        rstd: torch.Tensor, *, outputs: Sequence[str] = ("x", "weight", "bias")) -> NormGrads:
    """Gradients of ``layer_norm`` from its forward's statistics.  The vectors'
    gradients have the weight's shape and dtype ([D] in x's dtype without one)."""

    return _norm_backward(dy, x, weight, mean, rstd, outputs, 0)


def layer_norm_modulate_backward(dy: torch.Tensor, x: torch.Tensor, scale: torch.Tensor, mean: torch.Tensor,
                                 rstd: torch.Tensor, *,
                                 outputs: Sequence[str] = ("x", "weight", "bias")) -> NormGrads:
    """Gradients of ``layer_norm_modulate``: "weight" names the scale's, "bias" the shift's."""

    return _norm_backward(dy, x, scale, mean, rstd, outputs, _lib.Q6_NORM_ONE_PLUS)
