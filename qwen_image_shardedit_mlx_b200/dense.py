"""Dense 16-bit linear and layer norm with gradients.

The trainable twins of what the q6 block computes around its packed weights:

* ``dense_linear``: ``residual + gate * act(x @ W^T + bias)`` with the epilogue
  of ``q6_linear`` over a dense bf16 / fp16 weight (a materialised feed-forward
  layer, an embedding or a modulation projection), from one row to long ones.
* ``layer_norm`` / ``layer_norm_modulate``: an affine norm, or the adaLN form
  ``LayerNorm(x) * (1 + scale) + shift`` with one vector pair per sample; bf16,
  fp16 or fp32 rows of any width.

Both differentiate through ``torch.autograd`` and have functional forms
(``*_forward`` / ``*_backward``) that launch the same kernels without it.  The
functional forms may be captured in a CUDA graph.  A differentiable call under
capture is refused: its backward pass would run on the streams that autograd
recorded for the leaves, outside the capture.

Tensors must live on one CUDA device; kernels are ordered on its current
stream, nothing synchronises, and equal calls give equal bits.
"""

from __future__ import annotations

from collections.abc import Sequence
from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from qwen_image_shardedit_mlx_b200 import _lib
from qwen_image_shardedit_mlx_b200.ops import _ptr, _require_cuda

ACTIVATIONS = {None: _lib.Q6_ACT_NONE, "gelu_tanh": _lib.Q6_ACT_GELU_TANH, "silu": _lib.Q6_ACT_SILU}
_DTYPES = {torch.bfloat16: _lib.Q6_DTYPE_BF16, torch.float16: _lib.Q6_DTYPE_F16, torch.float32: _lib.Q6_DTYPE_F32}


class _on:
    """Make ``device`` current for a launch (a no-op when it already is)."""

    __slots__ = ("guard", "stream")

    def __init__(self, device: torch.device) -> None:
        self.guard = None if device.index == torch.cuda.current_device() else torch.cuda.device(device)
        self.stream = 0

    def __enter__(self) -> "_on":
        if self.guard is not None:
            self.guard.__enter__()
        self.stream = torch.cuda.current_stream().cuda_stream
        return self

    def __exit__(self, *exc) -> None:
        if self.guard is not None:
            self.guard.__exit__(*exc)


def _rows(t: torch.Tensor, width: int) -> tuple[torch.Tensor, int]:
    """``t`` as [rows, width] with contiguous columns, and its row stride in
    elements (a copy only where the layout does not allow that)."""

    if t.is_contiguous():
        return t, width
    t2 = t.reshape(-1, width)
    rows = t2.shape[0]
    if (width > 1 and t2.stride(1) != 1) or (rows > 1 and t2.stride(0) < width):
        return t2.contiguous(), width
    return t2, (t2.stride(0) if rows > 1 else width)


def _vectors(t: torch.Tensor, width: int) -> tuple[torch.Tensor, int]:
    """[width] or [S, width] vectors with contiguous elements and the stride between them."""

    t, ld = _rows(t, width)
    return t, ld


def _sample_rows(name: str, t: torch.Tensor, x: torch.Tensor, width: int) -> int:
    """Rows that share one vector of ``t``: [width] or [1, width] (all rows), or
    [S, width] / [S, 1, ..., width] with S the leading size of ``x``."""

    leading = x.shape[:-1]
    m = 1
    for v in leading:
        m *= v
    if t.shape[-1:] != (width,) or any(v != 1 for v in t.shape[1:-1]):
        raise ValueError(f"{name} must be [{width}] or [samples, {width}], got {tuple(t.shape)}")
    if t.dim() == 1 or t.shape[0] == 1:
        return m
    if not leading or t.shape[0] != leading[0]:
        raise ValueError(f"{name} {tuple(t.shape)} does not match the samples of x {tuple(x.shape)}")
    return m // t.shape[0]


def _pack_bit(ptr: int, ld: int, bit: int) -> int:
    return bit if ptr % 16 or ld % 8 else 0


def _workspace(nbytes: int, device: torch.device) -> torch.Tensor | None:
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _refuse_capture(what: str) -> None:
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"{what} cannot be captured in a CUDA graph with gradients: capture {what}_forward and "
                           f"{what}_backward, or call it under torch.no_grad()")


# ----------------------------------------------------------------------------- linear


class DenseGrads(NamedTuple):
    """Gradients of ``dense_linear`` (None where not asked for); the residual's is ``dy`` itself."""

    x: torch.Tensor | None
    weight: torch.Tensor | None
    bias: torch.Tensor | None
    gate: torch.Tensor | None


def _check_linear(x, weight, bias, activation, residual, gate) -> int:
    """Validate the operands of a dense linear; returns the rows per gate vector."""

    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {tuple(ACTIVATIONS)}, got {activation!r}")
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"dense_linear takes bfloat16 or float16, got {x.dtype}")
    if weight.dim() != 2 or x.dim() < 1:
        raise ValueError(f"weight must be 2-D and x at least 1-D, got {tuple(weight.shape)}, {tuple(x.shape)}")
    n, k = weight.shape
    if n == 0 or k == 0:
        raise ValueError(f"weight must not be empty, got {tuple(weight.shape)}")
    if x.shape[-1] != k:
        raise ValueError(f"x in_features {x.shape[-1]} != weight in_features {k}")
    for name, t in (("weight", weight), ("bias", bias), ("residual", residual), ("gate", gate)):
        if t is not None and t.dtype != x.dtype:
            raise ValueError(f"{name} is {t.dtype}, x is {x.dtype}")
    if bias is not None and bias.shape != (n,):
        raise ValueError(f"bias must be ({n},), got {tuple(bias.shape)}")
    if residual is not None and residual.shape != x.shape[:-1] + (n,):
        raise ValueError(f"residual must be {tuple(x.shape[:-1]) + (n,)}, got {tuple(residual.shape)}")
    rows = x.numel() // k
    return rows if gate is None else _sample_rows("gate", gate, x, n)


def _linear_forward(x, weight, bias, activation, residual, gate, save_preact):
    rows_per_gate = _check_linear(x, weight, bias, activation, residual, gate)
    dev = _require_cuda(x, weight, bias, residual, gate)
    n, k = weight.shape
    shape = x.shape[:-1] + (n,)
    with _on(dev) as here:
        y = torch.empty(shape, dtype=x.dtype, device=dev)
        # the gate's gradient sums act(z) itself: rounded to 16 bits, z would cost it as much as its own rounding
        zdt = x.dtype if gate is None else torch.float32
        z = torch.empty(shape, dtype=zdt, device=dev) if save_preact else None
        m = x.numel() // k
        if m == 0:
            return y, z
        x2, ldx = _rows(x, k)
        w2, ldw = _rows(weight, k)
        r2, ldr = _rows(residual, n) if residual is not None else (None, n)
        g2, ldg = _vectors(gate, n) if gate is not None else (None, n)
        b2 = None if bias is None else bias.contiguous()
        xp, wp = x2.data_ptr(), w2.data_ptr()
        lib = _lib.lib()
        nbytes = lib.q6_dense_linear_workspace_bytes(
            m, n, k, _pack_bit(xp, ldx, _lib.Q6_PACK_X) | _pack_bit(wp, ldw, _lib.Q6_PACK_W))
        ws = _workspace(nbytes, dev)
        _lib.check(
            lib.q6_dense_linear(xp, ldx, wp, ldw, _ptr(b2), _ptr(g2), ldg, rows_per_gate, _ptr(r2), ldr,
                                y.data_ptr(), _ptr(z), _DTYPES[zdt], m, n, k, _DTYPES[x.dtype], ACTIVATIONS[activation], _ptr(ws),
                                nbytes, here.stream), "q6_dense_linear")
    return y, z


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
    second value is ``x @ W^T + bias`` (in x's dtype, or in fp32 when a gate is
    given), which ``dense_linear_backward`` takes; else None."""

    with torch.no_grad():
        return _linear_forward(x, weight, bias, activation, residual, gate, save_preact)


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
    rounded to the tensors' dtype; all sums are held in fp32.
    """

    want = set(outputs)
    if not want <= {"x", "weight", "bias", "gate"}:
        raise ValueError(f"outputs must be among x, weight, bias, gate; got {tuple(outputs)}")
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {tuple(ACTIVATIONS)}, got {activation!r}")
    if dy.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"dense_linear_backward takes bfloat16 or float16, got {dy.dtype}")
    if ("weight" in want and x is None) or ("x" in want and weight is None):
        raise ValueError("the weight's gradient needs x, the gradient of x needs weight")
    if preact is None and want and (activation is not None or "gate" in want):
        raise ValueError("preact is needed with an activation or for the gate's gradient")
    if "gate" in want and gate is None:
        raise ValueError("the gate's gradient needs gate")
    n = dy.shape[-1] if dy.dim() else 0
    if n == 0 or (weight is not None and (weight.dim() != 2 or weight.shape[0] != n or weight.shape[1] == 0)):
        raise ValueError(f"dy {tuple(dy.shape)} does not match weight {None if weight is None else tuple(weight.shape)}")
    k = weight.shape[1] if weight is not None else x.shape[-1] if x is not None else 1
    if x is not None and (x.shape != dy.shape[:-1] + (k,) or k == 0):
        raise ValueError(f"x {tuple(x.shape)} does not match dy {tuple(dy.shape)} and {k} in_features")
    if preact is not None and preact.shape != dy.shape:
        raise ValueError(f"preact must be {tuple(dy.shape)}, got {tuple(preact.shape)}")
    for name, t in (("x", x), ("weight", weight), ("preact", preact), ("gate", gate)):
        if t is not None and t.dtype != dy.dtype and not (t is preact and t.dtype == torch.float32):
            raise ValueError(f"{name} is {t.dtype}, dy is {dy.dtype}")
    m = dy.numel() // n
    rows_per_gate = m if gate is None else _sample_rows("gate", gate, dy, n)
    dev = _require_cuda(dy, x, weight, preact, gate)
    with torch.no_grad(), _on(dev) as here:
        def new(shape):
            return (torch.zeros if m == 0 else torch.empty)(shape, dtype=dy.dtype, device=dev)

        dx = new(dy.shape[:-1] + (k,)) if "x" in want else None
        dw = new((n, k)) if "weight" in want else None
        db = new((n,)) if "bias" in want else None
        dg = new(gate.shape) if "gate" in want else None
        if m == 0 or not want:
            return DenseGrads(dx, dw, db, dg)
        dy2, ldy = _rows(dy, n)
        x2, ldx = _rows(x, k) if dw is not None else (None, k)
        w2, ldw = _rows(weight, k) if dx is not None else (None, k)
        g2, ldg = _vectors(gate, n) if gate is not None else (None, n)
        z2 = None if preact is None else preact.contiguous()
        dyp, xp, wp = dy2.data_ptr(), _ptr(x2), _ptr(w2)
        bits = ((_lib.Q6_GRAD_X if dx is not None else 0) | (_lib.Q6_GRAD_W if dw is not None else 0)
                | (_lib.Q6_GRAD_BIAS if db is not None else 0) | (_lib.Q6_GRAD_GATE if dg is not None else 0))
        pack = (_pack_bit(xp or 0, ldx, _lib.Q6_PACK_X) | _pack_bit(wp or 0, ldw, _lib.Q6_PACK_W)
                | _pack_bit(dyp, ldy, _lib.Q6_PACK_DY))
        act, lib = ACTIVATIONS[activation], _lib.lib()
        nbytes = lib.q6_dense_linear_grad_workspace_bytes(m, n, k, rows_per_gate, act, int(gate is not None), bits, pack)
        ws = _workspace(nbytes, dev)
        _lib.check(
            lib.q6_dense_linear_grad(dyp, ldy, xp, ldx, wp, ldw, _ptr(z2),
                                     _DTYPES[dy.dtype if z2 is None else z2.dtype], _ptr(g2), ldg, rows_per_gate, _ptr(dx),
                                     _ptr(dw), _ptr(db), _ptr(dg), m, n, k, _DTYPES[dy.dtype], act, _ptr(ws), nbytes,
                                     here.stream), "q6_dense_linear_grad")
    return DenseGrads(dx, dw, db, dg)


class _DenseLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, gate, residual, activation):
        need_x, need_w, need_b, need_g = ctx.needs_input_grad[:4]
        save = need_g or (activation is not None and (need_x or need_w or need_b))
        y, z = _linear_forward(x, weight, bias, activation, residual, gate, save)
        ctx.activation = activation
        ctx.save_for_backward(x if need_w else None, weight if need_x else None, z, gate)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, z, gate = ctx.saved_tensors
        needs = ctx.needs_input_grad
        want = [name for name, need in zip(("x", "weight", "bias", "gate"), needs) if need]
        g = dense_linear_backward(dy, x, weight, preact=z, activation=ctx.activation, gate=gate, outputs=want)
        return g.x, g.weight, g.bias, g.gate, dy if needs[4] else None, None


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

    if torch.is_grad_enabled() and (
            x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)
            or (gate is not None and gate.requires_grad) or (residual is not None and residual.requires_grad)):
        if x.is_cuda:
            _refuse_capture("dense_linear")
        return _DenseLinear.apply(x, weight, bias, gate, residual, activation)
    return _linear_forward(x, weight, bias, activation, residual, gate, False)[0]


# ------------------------------------------------------------------------- layer norm


class NormGrads(NamedTuple):
    """Gradients of a layer norm (None where not asked for)."""

    x: torch.Tensor | None
    weight: torch.Tensor | None
    bias: torch.Tensor | None


def _check_norm(x, weight, bias, eps) -> tuple[int, int]:
    """Validate the operands of a layer norm; returns (D, rows per vector)."""

    if x.dtype not in _DTYPES:
        raise ValueError(f"layer_norm takes bfloat16, float16 or float32, got {x.dtype}")
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError(f"x must have a last axis of at least one value, got {tuple(x.shape)}")
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative, got {eps}")
    d = x.shape[-1]
    rows = x.numel() // d
    if weight is not None and bias is not None and (weight.dtype != bias.dtype or weight.shape != bias.shape):
        raise ValueError(f"the two vectors must agree, got {weight.dtype} {tuple(weight.shape)} and "
                         f"{bias.dtype} {tuple(bias.shape)}")
    v = weight if weight is not None else bias
    if v is None:
        return d, rows
    if v.dtype != x.dtype and v.dtype != torch.float32:
        raise ValueError(f"the vectors must be {x.dtype} or float32, got {v.dtype}")
    return d, _sample_rows("the vectors", v, x, d)


def _norm_vectors(weight, bias, d):
    """Both vectors with one stride between samples (copied to a dense layout if they differ)."""

    w2, ldv = _vectors(weight, d) if weight is not None else (None, d)
    b2, ldb = _vectors(bias, d) if bias is not None else (None, ldv)
    if weight is None:
        ldv = ldb
    if ldb != ldv:
        w2, b2, ldv = w2.contiguous(), b2.contiguous(), d
    return w2, b2, ldv


def _norm_forward(x, weight, bias, eps, flags, stats):
    d, rows_per_vec = _check_norm(x, weight, bias, eps)
    dev = _require_cuda(x, weight, bias)
    m = x.numel() // d
    with _on(dev) as here:
        y = torch.empty(x.shape, dtype=x.dtype, device=dev)
        mean = rstd = None
        if stats:
            mean, rstd = torch.empty((2, m), dtype=torch.float32, device=dev).unbind(0)
        if m == 0:
            return y, mean, rstd
        x2, ldx = _rows(x, d)
        w2, b2, ldv = _norm_vectors(weight, bias, d)
        v = weight if weight is not None else bias
        vdt = x.dtype if v is None else v.dtype
        _lib.check(
            _lib.lib().q6_layer_norm(x2.data_ptr(), ldx, _ptr(w2), _ptr(b2), ldv, rows_per_vec, y.data_ptr(),
                                     _ptr(mean), _ptr(rstd), m, d, eps, _DTYPES[x.dtype], _DTYPES[vdt], flags,
                                     here.stream), "q6_layer_norm")
    return y, mean, rstd


def _norm_backward(dy, x, weight, mean, rstd, vec_shape, vec_dtype, flags, want):
    if x.dtype not in _DTYPES or dy.dtype != x.dtype or dy.shape != x.shape or x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError(f"dy {dy.dtype} {tuple(dy.shape)} does not match x {x.dtype} {tuple(x.shape)}")
    d = x.shape[-1]
    m = x.numel() // d
    for name, t in (("mean", mean), ("rstd", rstd)):
        if t.dtype != torch.float32 or t.numel() != m:
            raise ValueError(f"{name} must hold {m} float32 values, got {t.dtype} {tuple(t.shape)}")
    if weight is not None and weight.dtype != x.dtype and weight.dtype != torch.float32:
        raise ValueError(f"the weight must be {x.dtype} or float32, got {weight.dtype}")
    dev = _require_cuda(dy, x, weight, mean, rstd)
    like = torch.empty(vec_shape, dtype=vec_dtype, device="meta") if weight is None else weight
    rows_per_vec = _sample_rows("the vectors", like, x, d)
    with torch.no_grad(), _on(dev) as here:
        def new(shape, dtype):
            return (torch.zeros if m == 0 else torch.empty)(shape, dtype=dtype, device=dev)

        dx = new(x.shape, x.dtype) if "x" in want else None
        dw = new(vec_shape, vec_dtype) if "weight" in want else None
        db = new(vec_shape, vec_dtype) if "bias" in want else None
        if m == 0 or not want:
            return NormGrads(dx, dw, db)
        x2, ldx = _rows(x, d)
        dy2, ldy = _rows(dy, d)
        w2, ldv = _vectors(weight, d) if weight is not None else (None, d)
        bits = (_lib.Q6_GRAD_W if dw is not None else 0) | (_lib.Q6_GRAD_BIAS if db is not None else 0)
        lib, dt = _lib.lib(), _DTYPES[x.dtype]
        nbytes = lib.q6_layer_norm_grad_workspace_bytes(m, d, rows_per_vec, dt, bits) if bits else 0
        ws = _workspace(nbytes, dev)
        _lib.check(
            lib.q6_layer_norm_grad(dy2.data_ptr(), ldy, x2.data_ptr(), ldx, _ptr(w2), ldv, rows_per_vec,
                                   mean.contiguous().data_ptr(), rstd.contiguous().data_ptr(), _ptr(dx), _ptr(dw),
                                   _ptr(db), m, d, dt, _DTYPES[vec_dtype], flags, _ptr(ws), nbytes, here.stream),
            "q6_layer_norm_grad")
    return NormGrads(dx, dw, db)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, flags):
        y, mean, rstd = _norm_forward(x, weight, bias, eps, flags, True)
        ctx.flags = flags
        v = weight if weight is not None else bias
        ctx.vec = (x.shape[-1:], x.dtype) if v is None else (v.shape, v.dtype)
        ctx.save_for_backward(x, weight, mean, rstd)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, mean, rstd = ctx.saved_tensors
        want = [name for name, need in zip(("x", "weight", "bias"), ctx.needs_input_grad) if need]
        g = _norm_backward(dy, x, weight, mean, rstd, *ctx.vec, ctx.flags, want)
        return g.x, g.weight, g.bias, None, None


def _norm(what, x, weight, bias, eps, flags):
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        if x.is_cuda:
            _refuse_capture(what)
        return _LayerNorm.apply(x, weight, bias, float(eps), flags)
    return _norm_forward(x, weight, bias, float(eps), flags, False)[0]


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, *,
               eps: float = 1e-6) -> torch.Tensor:
    """``LayerNorm(x) * weight + bias`` over the last axis (bf16, fp16 or fp32).

    ``weight`` and ``bias`` ([D], either may be None) are in x's dtype or in
    fp32.  Statistics and sums are held in fp32, the output is rounded once.
    Differentiable in every tensor (once).
    """

    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and t.dim() != 1:
            raise ValueError(f"{name} must be 1-D, got {tuple(t.shape)}")
    return _norm("layer_norm", x, weight, bias, eps, 0)


def layer_norm_modulate(x: torch.Tensor, shift: torch.Tensor, scale: torch.Tensor, *, eps: float = 1e-6) -> torch.Tensor:
    """``LayerNorm(x) * (1 + scale) + shift`` over the last axis: the block's adaLN
    modulate, differentiable, for any width.  ``shift`` / ``scale`` are [D], or
    [S, D] with S the leading size of x (one pair per sample; strided views of a
    modulation output are read in place)."""

    if shift is None or scale is None:
        raise ValueError("layer_norm_modulate needs shift and scale")
    return _norm("layer_norm_modulate", x, scale, shift, eps, _lib.Q6_NORM_ONE_PLUS)


def layer_norm_forward(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, *,
                       eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(y, mean, rstd): ``layer_norm`` without autograd; mean and rstd are fp32 [rows]."""

    with torch.no_grad():
        return _norm_forward(x, weight, bias, float(eps), 0, True)


def layer_norm_modulate_forward(x: torch.Tensor, shift: torch.Tensor, scale: torch.Tensor, *,
                                eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(y, mean, rstd): ``layer_norm_modulate`` without autograd."""

    with torch.no_grad():
        return _norm_forward(x, scale, shift, float(eps), _lib.Q6_NORM_ONE_PLUS, True)


def layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, weight: torch.Tensor | None, mean: torch.Tensor,
                        rstd: torch.Tensor, *, outputs: Sequence[str] = ("x", "weight", "bias")) -> NormGrads:
    """Gradients of ``layer_norm`` from its forward's statistics.  The vectors'
    gradients have the weight's shape and dtype ([D] in x's dtype without one)."""

    _check_outputs(outputs)
    shape, dtype = (x.shape[-1:], x.dtype) if weight is None else (weight.shape, weight.dtype)
    return _norm_backward(dy, x, weight, mean, rstd, shape, dtype, 0, set(outputs))


def layer_norm_modulate_backward(dy: torch.Tensor, x: torch.Tensor, scale: torch.Tensor, mean: torch.Tensor,
                                 rstd: torch.Tensor, *,
                                 outputs: Sequence[str] = ("x", "weight", "bias")) -> NormGrads:
    """Gradients of ``layer_norm_modulate``: "weight" names the scale's, "bias" the shift's."""

    _check_outputs(outputs)
    return _norm_backward(dy, x, scale, mean, rstd, scale.shape, scale.dtype, _lib.Q6_NORM_ONE_PLUS, set(outputs))


def _check_outputs(outputs) -> None:
    if not set(outputs) <= {"x", "weight", "bias"}:
        raise ValueError(f"outputs must be among x, weight, bias; got {tuple(outputs)}")
