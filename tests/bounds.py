"""Values in 64 bits with a bound on how far a kernel's value may be from them.

``B(v, e)`` holds a tensor ``v`` and an elementwise error bound ``e``.  The
operations below propagate both through the operators' formulas by first-order
error analysis with absolute values (worst case, no statistics):

* a rounding to dtype t adds half a step, ``eps(t) / 2 * |v|`` (and half the
  smallest subnormal);
* a sum of n products held in fp32 adds at most ``n * 2^-23 * sum |a b|``
  (each addition rounds or truncates a partial sum no larger than that sum);
* an fp32 elementwise step adds a few 2^-24 of its result, the approximate
  exp and divide of the activations under 2^-20.
"""

from __future__ import annotations

import math

import torch

F32 = 2.0 ** -23


class B:
    def __init__(self, v: torch.Tensor, e: torch.Tensor | float = 0.0) -> None:
        self.v = v.double()
        self.e = torch.zeros_like(self.v) + e if not isinstance(e, torch.Tensor) else e.double().expand_as(self.v)

    def __add__(self, o: "B") -> "B":
        v = self.v + o.v
        return B(v, self.e.expand_as(v) + o.e.expand_as(v) + 2.0 ** -24 * v.abs())

    def __neg__(self) -> "B":
        return B(-self.v, self.e)

    def __sub__(self, o: "B") -> "B":
        return self + (-o)

    def __mul__(self, o: "B") -> "B":
        v = self.v * o.v
        return B(v, self.v.abs() * o.e + self.e * o.v.abs() + self.e * o.e + 2.0 ** -24 * v.abs())

    def reshape(self, *shape) -> "B":
        return B(self.v.reshape(*shape), self.e.reshape(*shape))

    def t(self) -> "B":
        return B(self.v.t(), self.e.t())

    def sum(self, dim: int) -> "B":
        n = self.v.shape[dim]
        return B(self.v.sum(dim), self.e.sum(dim) + n * F32 * self.v.abs().sum(dim))

    def mean(self) -> "B":
        """Mean over the last axis, kept."""
        n = self.v.shape[-1]
        s = self.sum(-1)
        return B((s.v / n).unsqueeze(-1), (s.e / n).unsqueeze(-1) + 2.0 ** -23 * (s.v / n).abs().unsqueeze(-1))

    def round(self, dtype: torch.dtype) -> "B":
        fi = torch.finfo(dtype)
        half = fi.eps / 2
        return B(self.v, self.e + half * (self.v.abs() + self.e) + fi.tiny * fi.eps / 2)

    def check(self, got: torch.Tensor, what: str, floor: float = 1e-30) -> None:
        """``got`` lies within the bound everywhere."""
        assert got.shape == self.v.shape, (what, tuple(got.shape), tuple(self.v.shape))
        off = (got.double() - self.v).abs()
        ratio = (off / (self.e + floor)).max().item() if off.numel() else 0.0
        assert math.isfinite(ratio) and ratio <= 1.0, f"{what}: {ratio:.3g} times the bound"


def mm(a: B, b: B) -> B:
    """a @ b with fp32 sums."""
    k = a.v.shape[-1]
    mag = a.v.abs() @ b.v.abs()
    return B(a.v @ b.v, a.v.abs() @ b.e + a.e @ b.v.abs() + a.e @ b.e + k * F32 * mag)


K2, C = 2.0 * math.sqrt(2.0 / math.pi), 0.044715


def act_value(z: torch.Tensor, name: str | None) -> torch.Tensor:
    if name == "gelu_tanh":
        return z * torch.sigmoid(K2 * (z + C * z ** 3))
    if name == "silu":
        return z * torch.sigmoid(z)
    return z


def slope_value(z: torch.Tensor, name: str | None) -> torch.Tensor:
    if name == "gelu_tanh":
        s = torch.sigmoid(K2 * (z + C * z ** 3))
        return s + z * s * (1 - s) * K2 * (1 + 3 * C * z * z)
    if name == "silu":
        s = torch.sigmoid(z)
        return s + z * s * (1 - s)
    return torch.ones_like(z)


def act(z: B, name: str | None) -> B:
    if name is None:
        return z
    v = act_value(z.v, name)
    return B(v, 1.13 * z.e + 2.0 ** -20 * (v.abs() + z.v.abs() * 2.0 ** -10))  # |act'| <= 1.13 for both


def slope(z: B, name: str | None) -> B:
    if name is None:
        return B(torch.ones_like(z.v))
    return B(slope_value(z.v, name), 0.85 * z.e + 2.0 ** -19)  # |act''| <= 0.80 (GELU-tanh), 0.5 (SiLU)


def linear(x: B, w: B, b: B | None, name: str | None, gate: B | None, res: B | None, dtype) -> tuple[B, B]:
    """(y, pre-activation in fp32); gate broadcasts against the rows."""
    z = mm(x, w.t())
    if b is not None:
        z = z + b
    y = act(z, name)
    if gate is not None:
        y = gate * y
    if res is not None:
        y = res + y
    return y.round(dtype), z


def linear_grads(dy: B, x: B, w: B, z: B, name: str | None, gate: B | None, dtype, groups: int):
    """(dx, dw, db, dgate) for rows in ``groups`` equal runs with a gate each; ``z`` as saved (rounded)."""
    t = dy * gate if gate is not None else dy
    dz = t * slope(z, name) if name is not None else t
    # without an activation or gate the products read dy itself
    dz16 = dz.round(dtype) if (name is not None or gate is not None) else dz
    n = dy.v.shape[-1]
    dg = (dy * act(z, name)).reshape(groups, -1, n).sum(1)
    return mm(dz16, w).round(dtype), mm(dz16.t(), x).round(dtype), dz.sum(0).round(dtype), dg.round(dtype)


def norm(x: B, w: B | None, b: B | None, eps: float, dtype) -> tuple[B, B, B]:
    """(y, xh, rstd) of a layer norm; w and b broadcast against the rows."""
    c = x - x.mean()
    var = (c * c).mean()
    s = var.v + eps
    low = (s - var.e).clamp_min(torch.finfo(torch.float64).tiny)
    rstd = B(s.rsqrt(), 0.5 * var.e / (low * low.sqrt()) + 2.0 ** -22 * s.rsqrt())
    xh = c * rstd
    y = xh if w is None else xh * w
    if b is not None:
        y = y + b
    return y.round(dtype), xh, rstd


def norm_grads(dy: B, xh: B, rstd: B, w: B | None, dtype, vec_dtype, groups: int):
    """(dx, dweight, dbias) with the rows in ``groups`` equal runs with a vector each."""
    a = dy if w is None else dy * w
    dx = rstd * (a - a.mean() - xh * (a * xh).mean())
    d = dy.v.shape[-1]
    dw = (dy * xh).reshape(groups, -1, d).sum(1)
    db = dy.reshape(groups, -1, d).sum(1)
    return dx.round(dtype), dw.round(vec_dtype), db.round(vec_dtype)
