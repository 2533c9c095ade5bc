"""The dense linear's and the layer norm's checks of their arguments, on the CPU,
and the reference formulas of bounds.py against differences."""

from __future__ import annotations

import pytest
import torch

import bounds
from qwen_image_shardedit_mlx_b200 import _lib, dense

BF = torch.bfloat16


def t(*shape, dtype=BF):
    return torch.zeros(shape, dtype=dtype)


@pytest.mark.parametrize("kw,match", [
    (dict(x=t(4, 8, dtype=torch.float32)), "bfloat16 or float16"),
    (dict(x=t(4, 9)), "in_features"),
    (dict(weight=t(6, 8, 1)), "2-D"),
    (dict(weight=t(0, 8)), "empty"),
    (dict(weight=t(6, 8, dtype=torch.float16)), "weight is"),
    (dict(bias=t(5)), "bias must be"),
    (dict(bias=t(6, dtype=torch.float32)), "bias is"),
    (dict(activation="relu"), "activation"),
    (dict(residual=t(4, 5)), "residual must be"),
    (dict(residual=t(1, 6)), "residual must be"),
    (dict(gate=t(7)), "gate must be"),
    (dict(gate=t(3, 6)), "samples"),
    (dict(gate=t(2, 2, 6)), "gate must be"),
    (dict(), "CUDA"),
])
def test_linear_refuses(kw, match):
    args = dict(x=t(4, 8), weight=t(6, 8), bias=None, activation=None, residual=None, gate=None) | kw
    x, w, b = args.pop("x"), args.pop("weight"), args.pop("bias")
    with pytest.raises((ValueError, RuntimeError), match=match):
        dense.dense_linear(x, w, b, **args)
    with pytest.raises((ValueError, RuntimeError), match=match):
        dense.dense_linear(x, w.requires_grad_(True), b, **args)


@pytest.mark.parametrize("kw,match", [
    (dict(outputs=("y",)), "among"),
    (dict(x=None), "needs x"),
    (dict(weight=None), "needs weight"),
    (dict(activation="silu"), "preact"),
    (dict(preact=t(4, 6)), "preact is"),
    (dict(outputs=("gate",), preact=t(4, 6, dtype=torch.float16)), "needs gate"),
    (dict(preact=t(4, 5, dtype=torch.float16)), "preact must be"),
    (dict(x=t(5, 8)), "does not match"),
    (dict(weight=t(7, 8)), "does not match"),
    (dict(x=t(4, 8, dtype=torch.float16)), "x is"),
    (dict(dy=t(4, 6, dtype=torch.float32)), "bfloat16 or float16"),
    (dict(), "CUDA"),
])
def test_linear_backward_refuses(kw, match):
    args = dict(dy=t(4, 6), x=t(4, 8), weight=t(6, 8)) | kw
    with pytest.raises((ValueError, RuntimeError), match=match):
        dense.dense_linear_backward(args.pop("dy"), args.pop("x"), args.pop("weight"), **args)


@pytest.mark.parametrize("kw,match", [
    (dict(x=t(4, 8, dtype=torch.float64)), "bfloat16, float16 or float32"),
    (dict(x=t(4, 0)), "at least one"),
    (dict(weight=t(7)), r"\[8\]"),
    (dict(weight=t(8, dtype=torch.float16)), "float32"),
    (dict(weight=t(1, 8)), "1-D"),
    (dict(weight=t(8), bias=t(8, dtype=torch.float32)), "agree"),
    (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps"),
    (dict(), "CUDA"),
])
def test_norm_refuses(kw, match):
    args = dict(x=t(4, 8), weight=None, bias=None, eps=1e-6) | kw
    with pytest.raises((ValueError, RuntimeError), match=match):
        dense.layer_norm(args["x"], args["weight"], args["bias"], eps=args["eps"])


def test_modulate_refuses():
    for shift, scale, match in ((t(3, 8), t(3, 8), "samples"), (t(8), t(2, 8), "agree"), (None, t(8), "needs"),
                                (t(2, 8), t(2, 8), "CUDA")):
        with pytest.raises((ValueError, RuntimeError), match=match):
            dense.layer_norm_modulate(t(2, 4, 8), shift, scale)
    stats = torch.zeros(8)
    for kw, match in ((dict(outputs=("scale",)), "among"), (dict(mean=torch.zeros(7)), "mean"), (dict(), "CUDA")):
        args = dict(mean=stats, outputs=("x",)) | kw
        with pytest.raises((ValueError, RuntimeError), match=match):
            dense.layer_norm_modulate_backward(t(2, 4, 8), t(2, 4, 8), t(2, 8), args["mean"], stats,
                                               outputs=args["outputs"])


def test_c_entries_refuse_before_the_device():
    lib, inv, uns, al, wsp = (_lib.lib(), _lib.Q6_ERR_INVALID_ARGUMENT, _lib.Q6_ERR_UNSUPPORTED,
                              _lib.Q6_ERR_ALIGNMENT, _lib.Q6_ERR_WORKSPACE)

    def linear(**kw):
        a = dict(x=256, ldx=64, w=256, ldw=64, bias=None, gate=None, ldg=0, rpg=4, res=None, ldr=0, y=256, pre=None,
                 pdt=0, M=4, N=32, K=64, dtype=0, act=0, ws=None, wsb=0, stream=None) | kw
        return lib.q6_dense_linear(*a.values())

    assert linear(x=None) == inv and linear(w=None) == inv and linear(y=None) == inv
    assert linear(M=0) == inv and linear(N=0) == inv and linear(K=-1) == inv and linear(M=1 << 31) == inv
    assert linear(ldx=63) == inv and linear(ldw=60) == inv and linear(res=256, ldr=31) == inv
    assert linear(rpg=3) == inv and linear(rpg=0) == inv and linear(rpg=2, gate=256, ldg=16) == inv
    assert linear(act=3) == inv and linear(act=-1) == inv
    assert linear(dtype=2) == uns and linear(pre=256, pdt=0) == uns and linear(pre=258, pdt=2) == al
    assert linear(x=257) == al and linear(y=255) == al and linear(ws=128, wsb=1 << 30) == al
    assert linear(M=40, rpg=40, x=258) == wsp  # an operand off its 16 bytes is copied: the workspace must hold it
    assert lib.q6_dense_linear_workspace_bytes(40, 32, 64, _lib.Q6_PACK_X) >= 40 * 64 * 2
    assert lib.q6_dense_linear_workspace_bytes(0, 32, 64, 0) == 0

    def grad(**kw):
        a = dict(dy=256, ldy=32, x=256, ldx=64, w=256, ldw=64, pre=None, pdt=1, gate=None, ldg=0, rpg=4, dx=256, dw=256,
                 db=256, dg=None, M=4, N=32, K=64, dtype=1, act=0, ws=None, wsb=0, stream=None) | kw
        return lib.q6_dense_linear_grad(*a.values())

    assert grad(dy=None) == inv and grad(x=None) == inv and grad(w=None) == inv
    assert grad(act=1) == inv and grad(dg=256) == inv and grad(dg=256, pre=256) == inv
    assert grad(ldy=31) == inv and grad(rpg=5) == inv and grad(dtype=2) == uns
    assert grad() == wsp and grad(dw=129) == al
    assert grad(dx=None, dw=None, db=None) == _lib.Q6_OK  # nothing asked for

    def norm(**kw):
        a = dict(x=256, ldx=64, w=256, b=256, ldv=64, rpv=4, y=256, mean=None, rstd=None, M=4, D=64, eps=1e-6, dtype=0,
                 vdt=0, flags=0, stream=None) | kw
        return lib.q6_layer_norm(*a.values())

    assert norm(x=None) == inv and norm(y=None) == inv and norm(mean=256) == inv and norm(D=0) == inv
    assert norm(ldx=63) == inv and norm(rpv=3) == inv and norm(rpv=2, ldv=8) == inv and norm(flags=2) == inv
    assert norm(eps=-1.0) == inv and norm(eps=float("nan")) == inv
    assert norm(dtype=3) == uns and norm(vdt=1) == uns
    assert norm(y=255) == al and norm(vdt=2, w=258) == al

    def ngrad(**kw):
        a = dict(dy=256, ldy=64, x=256, ldx=64, w=256, ldv=64, rpv=4, mean=256, rstd=256, dx=256, dw=256, db=256, M=4,
                 D=64, dtype=2, vdt=2, flags=1, ws=None, wsb=0, stream=None) | kw
        return lib.q6_layer_norm_grad(*a.values())

    assert ngrad(dy=None) == inv and ngrad(mean=None) == inv and ngrad(rstd=None) == inv and ngrad(ldy=10) == inv
    assert ngrad(M=4096, rpv=4096) == wsp and ngrad(dx=258) == al
    assert ngrad(dx=None, dw=None, db=None) == _lib.Q6_OK
    assert lib.q6_layer_norm_grad_workspace_bytes(4, 64, 3, 2, 6) == 0


@pytest.mark.parametrize("name", [None, "gelu_tanh", "silu"])
def test_reference_gradients_against_differences(name):
    g = torch.Generator().manual_seed(0)
    x, w, b, gate, dy = (torch.randn(s, generator=g, dtype=torch.float64) for s in
                         ((6, 5), (7, 5), (7,), (6, 7), (6, 7)))
    gate = gate[:1].expand(6, 7).clone()

    def loss(x, w, b, gate):
        return (dy * gate * bounds.act_value(x @ w.t() + b, name)).sum()

    z = bounds.B(x @ w.t() + b)
    got = bounds.linear_grads(bounds.B(dy), bounds.B(x), bounds.B(w), z, name, bounds.B(gate), torch.float64, 1)
    h = 1e-5
    for i, arg in enumerate((x, w, b, gate)):
        v = torch.randn(arg.shape, generator=g, dtype=torch.float64)
        if i == 3:
            v = v[:1].expand_as(arg)
        lo, hi = [x, w, b, gate], [x, w, b, gate]
        lo[i], hi[i] = arg - h * v, arg + h * v
        diff = (loss(*hi) - loss(*lo)) / (2 * h)
        want = (got[i].v.reshape(-1, *v.shape[1:] if i < 3 and v.dim() > 1 else (v.shape[-1],)) *
                (v if i < 3 else v[:1])).sum()
        assert abs(diff - want) < 1e-7 * max(1.0, abs(want))


def test_reference_norm_gradients_against_differences():
    g = torch.Generator().manual_seed(1)
    x, dy = (torch.randn((4, 9), generator=g, dtype=torch.float64) for _ in range(2))
    w, b = (torch.randn((9,), generator=g, dtype=torch.float64) for _ in range(2))

    def loss(x, w, b):
        return (dy * (torch.nn.functional.layer_norm(x, (9,), eps=1e-6) * w + b)).sum()

    bw = bounds.B(w.expand(4, 9))
    _, xh, rstd = bounds.norm(bounds.B(x), bw, bounds.B(b.expand(4, 9)), 1e-6, torch.float64)
    got = bounds.norm_grads(bounds.B(dy), xh, rstd, bw, torch.float64, torch.float64, 1)
    h = 1e-5
    for i, arg in enumerate((x, w, b)):
        v = torch.randn(arg.shape, generator=g, dtype=torch.float64)
        lo, hi = [x, w, b], [x, w, b]
        lo[i], hi[i] = arg - h * v, arg + h * v
        diff = (loss(*hi) - loss(*lo)) / (2 * h)
        assert abs(diff - (got[i].v.reshape(v.shape) * v).sum()) < 1e-7


def test_no_samples_with_a_vector_each():
    """A batch of no samples carries no vectors either: checked like any other call."""
    with pytest.raises(RuntimeError, match="CUDA"):
        dense.dense_linear(t(0, 4, 8), t(6, 8), gate=t(0, 6))
    with pytest.raises(RuntimeError, match="CUDA"):
        dense.dense_linear_backward(t(0, 4, 6), t(0, 4, 8), t(6, 8), gate=t(0, 6), outputs=("x",))
    with pytest.raises(RuntimeError, match="CUDA"):
        dense.layer_norm_modulate(t(0, 4, 8), t(0, 8), t(0, 8))
    with pytest.raises(ValueError, match="samples"):
        dense.dense_linear(t(2, 4, 8), t(6, 8), gate=t(0, 6))


def test_forward_mode_tangents_are_refused():
    """Without a derivative of its own a call must not drop a tangent: torch would read it as zero."""
    fw = torch.autograd.forward_ad

    def refused(f):
        with pytest.raises(RuntimeError, match="forward-mode"):
            f()

    x, w, b, r, g = t(4, 8), t(6, 8), t(6), t(4, 6), t(6)
    with fw.dual_level():
        for i in range(5):
            for leaf in (False, True):  # with and without a gradient beside the tangent
                a = [v.clone().requires_grad_(leaf) for v in (x, w, b, r, g)]
                a[i] = fw.make_dual(a[i], torch.ones_like(a[i]))
                refused(lambda: dense.dense_linear(a[0], a[1], a[2], residual=a[3], gate=a[4]))
                with torch.no_grad():
                    refused(lambda: dense.dense_linear(a[0], a[1], a[2], residual=a[3], gate=a[4]))
            refused(lambda: dense.dense_linear_forward(a[0], a[1], a[2], residual=a[3], gate=a[4]))
        dy, z = t(4, 6), t(4, 6, dtype=torch.float16)
        for i in range(5):
            a = [v.clone() for v in (dy, x, w, z, g)]
            a[i] = fw.make_dual(a[i], torch.ones_like(a[i]))
            refused(lambda: dense.dense_linear_backward(*a[:3], preact=a[3], gate=a[4]))
        for i in range(3):
            for leaf in (False, True):
                a = [v.clone().requires_grad_(leaf) for v in (x, t(8), t(8))]
                a[i] = fw.make_dual(a[i], torch.ones_like(a[i]))
                refused(lambda: dense.layer_norm(*a))
                refused(lambda: dense.layer_norm_modulate(*a))
            refused(lambda: dense.layer_norm_forward(*a))
            refused(lambda: dense.layer_norm_modulate_forward(*a))
        stats = torch.zeros(4)
        for i in range(5):
            a = [v.clone() for v in (x, x, t(8), stats, stats)]
            a[i] = fw.make_dual(a[i], torch.ones_like(a[i]))
            refused(lambda: dense.layer_norm_backward(*a))
            refused(lambda: dense.layer_norm_modulate_backward(*a))
