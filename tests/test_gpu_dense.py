"""The dense linear and the layer norm against 64-bit formulas, with elementwise
bounds from error analysis (bounds.py)."""

from __future__ import annotations

import math

import pytest
import torch

import bounds
from bounds import B
from qwen_image_shardedit_mlx_b200 import _lib, dense, ops

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


@pytest.fixture(autouse=True)
def _no_device_error():
    yield
    assert ops.device_error() == 0


def rand(shape, dtype, seed, std=1.0, mean=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * std + mean).to(dtype)


def rows_of(t, width):
    return t.reshape(-1, width)


def spread(vec, rows):
    """[S, N] vectors over the rows of S equal runs, as [rows, N]."""
    return vec.repeat_interleave(rows // vec.shape[0], 0)


def make_linear(samples, rows, k, n, dtype, *, bias=True, gate=True, residual=True, seed=0):
    x = rand((samples, rows, k), dtype, seed)
    w = rand((n, k), dtype, seed + 1, 1.0 / math.sqrt(k))
    b = rand((n,), dtype, seed + 2, 0.5) if bias else None
    g = rand((samples, n), dtype, seed + 3) if gate else None
    r = rand((samples, rows, n), dtype, seed + 4) if residual else None
    dy = rand((samples, rows, n), dtype, seed + 5)
    return x, w, b, g, r, dy


def check_linear(x, w, b, g, r, dy, activation):
    """Forward and every gradient of one call against the bounds."""
    dtype, (n, k) = x.dtype, w.shape
    m = x.numel() // k
    leaves = [t for t in (x, w, b, g, r) if t is not None]
    for t in leaves:
        t.requires_grad_(True)
    y = dense.dense_linear(x, w, b, activation=activation, residual=r, gate=g)
    grads = dict(zip([name for name, t in zip("xwbgr", (x, w, b, g, r)) if t is not None],
                     torch.autograd.grad(y, leaves, dy)))
    for t in leaves:
        t.requires_grad_(False)
    plain = dense.dense_linear(x, w, b, activation=activation, residual=r, gate=g)
    assert torch.equal(plain, y)  # with and without gradients: the same bits
    groups = 1 if g is None else g.reshape(-1, n).shape[0]
    bx, bw = B(rows_of(x, k)), B(w)
    bb = None if b is None else B(b)
    bg = None if g is None else B(spread(g.reshape(-1, n), m))
    br = None if r is None else B(rows_of(r, n))
    ry, rz = bounds.linear(bx, bw, bb, activation, bg, br, dtype)
    ry.check(rows_of(y, n), "y")
    bdy = B(rows_of(dy, n))
    dx, dw, db, dg = bounds.linear_grads(bdy, bx, bw, rz.round(torch.float16 if g is None else torch.float32), activation, bg,
                                          dtype, groups)
    dx.check(rows_of(grads["x"], k), "dx")
    dw.check(grads["w"], "dw")
    if b is not None:
        db.check(grads["b"], "db")
    if g is not None:
        dg.check(grads["g"].reshape(groups, n), "dgate")
    if r is not None:
        assert torch.equal(grads["r"], dy)
    return y, grads


LINEAR = [
    # samples, rows, k, n
    (1, 1, 64, 64), (1, 1, 1, 1), (1, 3, 7, 5), (2, 5, 33, 17), (1, 16, 128, 256), (3, 11, 72, 40),
    (1, 64, 256, 192), (2, 65, 200, 129), (1, 130, 1001, 77), (4, 64, 520, 264), (1, 257, 136, 392),
    (2, 333, 1001, 777), (1, 300, 2056, 1032), (1, 512, 768, 1536), (1, 2, 4104, 24), (1, 1000, 8, 2048),
    (1, 4, 1536, 6144), (1, 640, 640, 640),
]


@pytest.mark.parametrize("shape", LINEAR, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("dtype,activation", [("bf16", "gelu_tanh"), ("fp16", "silu"), ("bf16", None)])
def test_linear_and_gradients(shape, dtype, activation):
    check_linear(*make_linear(*shape, DT[dtype]), activation)


@pytest.mark.parametrize("mask", range(8))
def test_linear_optional_operands(mask):
    args = make_linear(2, 40, 96, 136, torch.bfloat16, bias=bool(mask & 1), gate=bool(mask & 2),
                       residual=bool(mask & 4), seed=mask)
    check_linear(*args, None)
    check_linear(*args, "gelu_tanh")


@pytest.mark.parametrize("m", [1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 96, 127, 128, 129, 191,
                               192, 193, 255, 256, 257])
def test_linear_every_row_count(m):
    x, w, b, g, r, dy = make_linear(1, m, 320, 272, torch.bfloat16, seed=m)
    check_linear(x, w, b, g, r, dy, "silu")


@pytest.mark.parametrize("m", range(1, 18))
@pytest.mark.parametrize("k,n", [(328, 264), (333, 57), (2048, 24)])
def test_linear_few_rows(m, k, n):
    # one and two tiles of rows, aligned and not, a gate per row; at 17 the other path
    x, w, b, g, r, dy = make_linear(m, 1, k, n, torch.bfloat16, seed=m)
    check_linear(x, w, b, g, r, dy, "gelu_tanh")
    x, w, b, g, r, dy = make_linear(1, m, k, n + 1, torch.float16, seed=m, gate=False)
    check_linear(x, w, b, g, r, dy, None)


@pytest.mark.parametrize("k,n", [(6144, 136), (6145, 136), (6143, 40), (4096, 8192), (4096, 8193)])
def test_linear_nine_rows_on_both_sides_of_the_rule(k, n):
    check_linear(*make_linear(3, 3, k, n, torch.bfloat16), "silu")


@pytest.mark.parametrize("k", [1, 2, 8, 15, 16, 24, 63, 64, 65, 127, 128, 136, 192, 1023])
def test_linear_every_contraction_length(k):
    check_linear(*make_linear(1, 72, k, 80, torch.float16, seed=k), None)
    check_linear(*make_linear(1, 3, k, 80, torch.bfloat16, seed=k), None)


PLANS = [f"{ct},{pair},{split}" for ct, pair in ((256, 1), (192, 1), (128, 1), (128, 0), (64, 0), (32, 0), (16, 0))
         for split in (1, 2, 3, 4, 8, 11)]


@pytest.mark.parametrize("plan", PLANS)
def test_linear_every_tile_shape_and_split(plan, monkeypatch):
    # every tile shape, alone and with the sum split, at sizes that
    # leave ragged tiles on every side, in every operand order (forward, dx, dw)
    monkeypatch.setenv("Q6_DENSE_PLAN", plan)
    check_linear(*make_linear(2, 150, 808, 696, torch.bfloat16), "gelu_tanh")
    check_linear(*make_linear(1, 515, 707, 773, torch.float16, gate=False), "silu")
    check_linear(*make_linear(1, 5, 1544, 264, torch.bfloat16), None)


@pytest.mark.parametrize("shape", [(1, 3456, 768, 3072), (2, 1728, 3072, 776), (1, 4099, 1031, 515), (3, 700, 520, 2056)],
                         ids=lambda s: "x".join(map(str, s)))
def test_linear_large(shape):
    check_linear(*make_linear(*shape, torch.bfloat16), "gelu_tanh")


def test_linear_strided_views_and_odd_addresses():
    dtype = torch.bfloat16
    base = rand((2, 70, 400), dtype, 1)
    wbase = rand((96, 300), dtype, 2, 0.1)
    dybase = rand((2, 70, 200), dtype, 3)
    for off in (0, 1, 8):
        x = base[:, :, off:off + 136].detach()
        w = wbase[:, off:off + 136].detach()
        gate = rand((2, 2, 6, 96 + off), dtype, 4)[:, 1, 2, off:].detach()
        res = base[:, :, off + 200:off + 296].detach()
        dy = dybase[:, :, off:off + 96]
        check_linear(x, w, None, gate, res, dy, "gelu_tanh")
    # transposed operands (columns not contiguous)
    check_linear(rand((136, 50), dtype, 5).t().detach(), rand((136, 48), dtype, 6, 0.1).t().detach(), None, None, None,
                 rand((48, 50), dtype, 7).t(), None)


def test_linear_expanded_output_gradient():
    x, w, b, _, _, _ = make_linear(1, 50, 64, 72, torch.bfloat16)
    w.requires_grad_(True)
    b.requires_grad_(True)
    dense.dense_linear(x, w, b).sum().backward()  # dy is an expanded scalar
    ones = torch.ones((50, 72), dtype=torch.bfloat16, device="cuda")
    ref = dense.dense_linear_backward(ones, x.reshape(50, 64), w.detach(), outputs=("weight", "bias"))
    assert torch.equal(w.grad, ref.weight) and torch.equal(b.grad, ref.bias)
    assert torch.equal(b.grad, torch.full_like(b, 50.0))


def test_linear_values_at_the_edges_of_the_type():
    # pre-activations far out: act saturates, its slope is 0 or 1, nothing turns into NaN
    for dtype, big in ((torch.bfloat16, 2.0 ** 100), (torch.float16, 3.0e4)):
        for activation in ("gelu_tanh", "silu"):
            x = torch.tensor([[big], [-big], [0.0], [30.0], [-30.0]], dtype=dtype, device="cuda")
            w = torch.ones((1, 1), dtype=dtype, device="cuda")
            y, z = dense.dense_linear_forward(x, w, activation=activation, save_preact=True)
            assert torch.equal(z.float(), x.float().clamp(-65504.0, 65504.0))
            assert torch.equal(y[:, 0].float().cpu(), torch.relu(x[:, 0].float()).cpu()) or torch.allclose(
                y[:, 0].float(), torch.relu(x[:, 0].float()), atol=1e-10, rtol=0)
            g = dense.dense_linear_backward(torch.ones_like(y), x, w, preact=z, activation=activation, outputs=("x",))
            want = torch.tensor([1.0, 0.0, 0.5, 1.0, 0.0], device="cuda")
            assert torch.allclose(g.x[:, 0].float(), want, atol=1e-10, rtol=0)


def test_linear_nan_and_infinity_stay_in_their_rows():
    x, w, b, _, r, _ = make_linear(1, 40, 72, 48, torch.bfloat16, gate=False)
    clean = dense.dense_linear(x, w, b, residual=r)
    bad = x.clone()
    bad[0, 7, 3] = float("nan")
    bad[0, 21, 70] = float("inf")
    y = dense.dense_linear(bad, w, b, residual=r)
    keep = [i for i in range(40) if i not in (7, 21)]
    assert torch.equal(y[0, keep], clean[0, keep])
    assert y[0, 7].isnan().all() and not y[0, 21].isfinite().any()


def test_linear_empty_rows():
    w = rand((24, 16), torch.bfloat16, 0).requires_grad_(True)
    b = rand((24,), torch.bfloat16, 1).requires_grad_(True)
    x = torch.empty((3, 0, 16), dtype=torch.bfloat16, device="cuda", requires_grad=True)
    y = dense.dense_linear(x, w, b, activation="silu")
    assert y.shape == (3, 0, 24)
    y.sum().backward()
    assert torch.equal(w.grad, torch.zeros_like(w)) and torch.equal(b.grad, torch.zeros_like(b))
    assert x.grad.shape == x.shape


def test_no_samples_with_a_vector_each():
    x = torch.empty((0, 5, 16), dtype=torch.bfloat16, device="cuda", requires_grad=True)
    w = rand((24, 16), torch.bfloat16, 1).requires_grad_(True)
    g = torch.empty((0, 24), dtype=torch.bfloat16, device="cuda", requires_grad=True)
    scale = torch.empty((0, 16), dtype=torch.bfloat16, device="cuda", requires_grad=True)
    y = dense.dense_linear(dense.layer_norm_modulate(x, scale, scale), w, activation="silu", gate=g)
    assert y.shape == (0, 5, 24)
    y.sum().backward()
    assert x.grad.shape == x.shape and g.grad.shape == g.shape and scale.grad.shape == scale.shape
    assert torch.equal(w.grad, torch.zeros_like(w))


def test_linear_partial_gradients_equal_the_whole():
    x, w, b, g, r, dy = make_linear(2, 50, 64, 88, torch.float16)
    y, z = dense.dense_linear_forward(x, w, b, activation="silu", residual=r, gate=g, save_preact=True)
    full = dense.dense_linear_backward(dy, x, w, preact=z, activation="silu", gate=g,
                                       outputs=("x", "weight", "bias", "gate"))
    for name in ("x", "weight", "bias", "gate"):
        one = dense.dense_linear_backward(dy, x if name == "weight" else None, w if name == "x" else None, preact=z,
                                          activation="silu", gate=g, outputs=(name,))
        assert torch.equal(getattr(one, name), getattr(full, name)), name
        assert all(getattr(one, o) is None for o in ("x", "weight", "bias", "gate") if o != name)
    for leaf in (x, w, b, g, r):  # autograd with one leaf at a time
        leaf.requires_grad_(True)
        got, = torch.autograd.grad(dense.dense_linear(x, w, b, activation="silu", residual=r, gate=g), leaf, dy)
        leaf.requires_grad_(False)
        want = {id(x): full.x, id(w): full.weight, id(b): full.bias, id(g): full.gate, id(r): dy}[id(leaf)]
        assert torch.equal(got, want)


def test_linear_gradient_against_differences():
    # directional difference of L = sum(dy * y) along v: the outputs' roundings
    # (half a step each, both sides) and the cubic term bound its error
    dtype, h = torch.float16, 2.0 ** -3
    x, w, b, g, r, dy = make_linear(1, 48, 64, 56, dtype, residual=False)
    w.requires_grad_(True)
    y = dense.dense_linear(x, w, b, activation="silu", gate=g)
    grad, = torch.autograd.grad(y, w, dy)
    w = w.detach()
    v = (torch.sign(grad.float()) * 2.0 ** -4).to(dtype)  # with the gradient, so that it is not lost in the roundings
    step = (v.float() * h).to(dtype)
    wp, wm = (w.float() + step.float()).to(dtype), (w.float() - step.float()).to(dtype)
    yp, ym = (dense.dense_linear(x, t, b, activation="silu", gate=g).double() for t in (wp, wm))
    moved = (wp.double() - wm.double()) / 2  # what the rounded weights moved by
    centre = (wp.double() + wm.double()) / 2
    diff = (dy.double() * (yp - ym)).sum() / 2
    want = (grad.double() * moved).sum()
    half = torch.finfo(dtype).eps / 2
    dzv = rows_of(x, 64).double() @ moved.t()
    rounding = (dy.double().abs() * half * (yp.abs() + ym.abs())).sum() / 2
    cubic = (dy.double().abs().reshape(-1, 56) * g.double().abs() * dzv.abs() ** 3).sum() / 6 * 0.35  # |silu'''| < 0.35
    shifted = (dy.double().abs().reshape(-1, 56) * g.double().abs() * 0.5 * dzv.abs()
               * (rows_of(x, 64).double() @ (centre - w.double()).t()).abs()).sum()  # |silu''| <= 0.5
    own = (moved.abs() * grad.double().abs()).sum() * 4 * half
    limit = rounding + cubic + shifted + own
    assert limit < 0.05 * want.abs()
    assert (diff - want).abs() <= limit


def test_linear_repeats_bit_for_bit_on_streams_and_in_graphs():
    x, w, b, g, r, dy = make_linear(2, 200, 264, 328, torch.bfloat16)

    def both():
        y, z = dense.dense_linear_forward(x, w, b, activation="gelu_tanh", residual=r, gate=g, save_preact=True)
        return [y, z, *dense.dense_linear_backward(dy, x, w, preact=z, activation="gelu_tanh", gate=g,
                                                   outputs=("x", "weight", "bias", "gate"))]

    first = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = both()
    again = both()  # at the same time
    torch.cuda.synchronize()
    for a, o, c in zip(first, other, again):
        assert torch.equal(a, o) and torch.equal(a, c)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = both()
        graphs.append((graph, out))
    x.copy_(rand(x.shape, x.dtype, 99))
    for graph, _ in graphs:
        graph.replay()
    want = both()
    torch.cuda.synchronize()
    for _, out in graphs:
        for a, o in zip(want, out):
            assert torch.equal(a, o)


def test_linear_capture_with_gradients_is_refused():
    x, w, b, _, _, _ = make_linear(1, 8, 16, 16, torch.bfloat16)
    w.requires_grad_(True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="dense_linear_forward"):
            dense.dense_linear(x, w, b)
        with torch.no_grad():
            y = dense.dense_linear(x, w, b)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, dense.dense_linear(x, w.detach(), b))


@pytest.mark.parametrize("m,k,n", [(5, 136, 72), (13, 130, 71), (300, 264, 520), (300, 263, 521), (96, 4096, 136), (96, 4096, 131)])
def test_output_in_place_of_the_residual(m, k, n):
    # the C entry may write y over the residual: few rows, whole and ragged blocks, split sums, odd widths
    lib = _lib.lib()
    x, w, b, _, _, _ = make_linear(1, m, k, n, torch.bfloat16, gate=False)
    r = rand((m, n), torch.bfloat16, 9)
    g = rand((n,), torch.bfloat16, 10)
    want = dense.dense_linear(x[0], w, b, activation="silu", gate=g, residual=r)
    pack = (_lib.Q6_PACK_X | _lib.Q6_PACK_W) if k % 8 else 0
    nbytes = lib.q6_dense_linear_workspace_bytes(m, n, k, pack)
    ws = torch.empty((max(nbytes, 1),), dtype=torch.uint8, device="cuda")
    status = lib.q6_dense_linear(x.data_ptr(), k, w.data_ptr(), k, b.data_ptr(), g.data_ptr(), n, m, r.data_ptr(), n,
                                 r.data_ptr(), None, _lib.Q6_DTYPE_F16, m, n, k, _lib.Q6_DTYPE_BF16, _lib.Q6_ACT_SILU,
                                 ws.data_ptr(), nbytes, torch.cuda.current_stream().cuda_stream)
    assert status == 0
    torch.cuda.synchronize()
    assert torch.equal(r, want)


def test_captured_backward_of_an_eager_call_is_refused():
    x, w, b, _, _, _ = make_linear(1, 12, 16, 16, torch.bfloat16)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for name, f in (("dense_linear_backward", lambda leaf: dense.dense_linear(x, w, leaf)),
                        ("layer_norm_backward", lambda leaf: dense.layer_norm(x, None, leaf))):
            leaf = b.detach().requires_grad_(True)
            y = f(leaf)
            dy = torch.ones_like(y)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                with pytest.raises(RuntimeError, match=name):
                    torch.autograd.grad(y, leaf, dy, retain_graph=True)
                z = dy + 1
            graph.replay()
            (grad,) = torch.autograd.grad(y, leaf, dy)  # outside a capture as ever
            assert torch.equal(grad, torch.full_like(b, 12.0)) and torch.equal(z, dy + 1)
    torch.cuda.current_stream().wait_stream(stream)


def test_linear_residual_rows_around_the_output_are_left_alone():
    x, w, b, _, _, _ = make_linear(1, 37, 40, 56, torch.bfloat16, gate=False)
    guard = torch.full((3, 37, 56), 7.0, dtype=torch.bfloat16, device="cuda")
    y = dense.dense_linear(x, w, b, residual=guard[1:2])
    assert torch.equal(guard, torch.full_like(guard, 7.0))
    ry, _ = bounds.linear(B(rows_of(x, 40)), B(w), B(b), None, None, B(rows_of(guard[1], 56)), torch.bfloat16)
    ry.check(rows_of(y, 56), "y")


# ------------------------------------------------------------------------- layer norm


def check_norm(x, w, b, dy, *, modulate, eps=1e-6):
    """Forward and gradients against the bounds; w / b are weight / bias, or scale / shift."""
    dtype, d = x.dtype, x.shape[-1]
    m = x.numel() // d
    leaves = [t for t in (x, w, b) if t is not None]
    for t in leaves:
        t.requires_grad_(True)
    y = dense.layer_norm_modulate(x, b, w, eps=eps) if modulate else dense.layer_norm(x, w, b, eps=eps)
    got = dict(zip([n for n, t in zip("xwb", (x, w, b)) if t is not None], torch.autograd.grad(y, leaves, dy)))
    for t in leaves:
        t.requires_grad_(False)
    plain = dense.layer_norm_modulate(x, b, w, eps=eps) if modulate else dense.layer_norm(x, w, b, eps=eps)
    assert torch.equal(plain, y)
    vec = w if w is not None else b
    groups = 1 if vec is None else vec.reshape(-1, d).shape[0]
    bw = None if w is None else B(spread(w.reshape(-1, d).double() + (1.0 if modulate else 0.0), m),
                                  2.0 ** -24 * 4 if modulate else 0.0)
    bb = None if b is None else B(spread(b.reshape(-1, d), m))
    ry, xh, rstd = bounds.norm(B(rows_of(x, d)), bw, bb, eps, dtype)
    ry.check(rows_of(y, d), "y")
    vdt = dtype if vec is None else vec.dtype
    dx, dw, db = bounds.norm_grads(B(rows_of(dy, d)), xh, rstd, bw, dtype, vdt, groups)
    dx.check(rows_of(got["x"], d), "dx")
    if w is not None:
        dw.check(got["w"].reshape(groups, d), "dweight")
    if b is not None:
        db.check(got["b"].reshape(groups, d), "dbias")


def make_norm(samples, rows, d, dtype, vec_dtype, *, per_sample, seed=0):
    x = rand((samples, rows, d), dtype, seed, 2.0, 0.5)
    shape = (samples, d) if per_sample else (d,)
    return x, rand(shape, vec_dtype, seed + 1, 0.3, 0.0 if per_sample else 1.0), rand(shape, vec_dtype, seed + 2, 0.3), \
        rand((samples, rows, d), dtype, seed + 3)


NORM = [(1, 1, 1), (1, 1, 8), (1, 5, 3), (2, 7, 33), (1, 9, 64), (3, 50, 100), (1, 333, 129), (2, 40, 256), (1, 17, 1001),
        (2, 21, 1024), (1, 64, 1152), (1, 70, 2048), (2, 33, 3072), (1, 12, 4096), (1, 5, 8192), (1, 3, 12288),
        (1, 2, 20001), (1, 2, 16384), (700, 1, 40), (1, 3000, 72), (5, 301, 128), (3, 1003, 16), (2, 259, 31), (1, 20003, 64)]


@pytest.mark.parametrize("shape", NORM, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("dtype,vec", [("bf16", "bf16"), ("fp16", "fp32"), ("fp32", "fp32")])
def test_norm_and_gradients(shape, dtype, vec):
    x, w, b, dy = make_norm(*shape, DT[dtype], DT[vec], per_sample=False)
    check_norm(x, w, b, dy, modulate=False)
    x, w, b, dy = make_norm(*shape, DT[dtype], DT[vec], per_sample=True, seed=5)
    check_norm(x, w, b, dy, modulate=True)


@pytest.mark.parametrize("dtype,vec", [("bf16", "fp32"), ("fp16", "fp16")])
def test_norm_other_vector_types(dtype, vec):
    for d in (72, 515, 1536):
        x, w, b, dy = make_norm(1, 40, d, DT[dtype], DT[vec], per_sample=False)
        check_norm(x, w, b, dy, modulate=False)
        check_norm(x, w, None, dy, modulate=False)
        check_norm(x, None, b, dy, modulate=False)
        check_norm(x, None, None, dy, modulate=False)


def test_norm_strided_views_and_odd_addresses():
    base = rand((2, 30, 700), torch.bfloat16, 1, 2.0)
    mod = rand((2, 2, 6, 264), torch.bfloat16, 2, 0.3)
    for off in (0, 1, 8):
        d = 256
        x, dy = base[:, :, off:off + d].detach(), base[:, :, off + 300:off + 300 + d]
        check_norm(x, mod[:, 1, 1, off:off + d].detach(), mod[:, 1, 0, off:off + d].detach(), dy, modulate=True)
        # scale and shift with different strides
        check_norm(x, mod[:, 1, 1, off:off + d].detach(), rand((2, d), torch.bfloat16, 3), dy, modulate=True)
    check_norm(rand((96, 20), torch.float32, 4).t().detach(), None, None, rand((96, 20), torch.float32, 5).t(),
               modulate=False)


def test_norm_constant_rows_and_offsets():
    x = torch.full((4, 257), 3.0, device="cuda")
    x[1] = 0.0
    dy = rand((4, 257), torch.float32, 1)
    check_norm(x, rand((257,), torch.float32, 2), rand((257,), torch.float32, 3), dy, modulate=False, eps=1e-5)
    # a mean far from zero: centred sums keep the variance
    x = rand((8, 3000), torch.float32, 4, 1.0, 1000.0)
    check_norm(x, None, None, rand((8, 3000), torch.float32, 5), modulate=False)


def test_norm_nan_stays_in_its_row():
    x = rand((9, 520), torch.bfloat16, 1)
    w = rand((520,), torch.bfloat16, 2)
    clean = dense.layer_norm(x, w)
    bad = x.clone()
    bad[4, 100] = float("nan")
    bad[6, 0] = float("inf")
    y = dense.layer_norm(bad, w)
    keep = [0, 1, 2, 3, 5, 7, 8]
    assert torch.equal(y[keep], clean[keep])
    assert y[4].isnan().all() and y[6].isnan().any()


def test_norm_empty_rows():
    x = torch.empty((0, 64), dtype=torch.bfloat16, device="cuda", requires_grad=True)
    w = rand((64,), torch.bfloat16, 1).requires_grad_(True)
    dense.layer_norm(x, w).sum().backward()
    assert torch.equal(w.grad, torch.zeros_like(w)) and x.grad.shape == (0, 64)


def test_norm_agrees_with_the_block_kernel():
    from qwen_image_shardedit_mlx_b200 import block

    x, scale, shift, _ = make_norm(1, 50, 1024, torch.bfloat16, torch.bfloat16, per_sample=True)
    ours = dense.layer_norm_modulate(x, shift, scale).float()
    theirs = block.layernorm_modulate(x, shift, scale).float()
    assert ((ours - theirs).abs() <= 2.0 ** -7 * theirs.abs() + 1e-6).all()  # a step of bf16: both round once


def test_norm_gradient_against_differences():
    x, w, b, dy = make_norm(1, 6, 40, torch.float32, torch.float32, per_sample=False)
    x = x.requires_grad_(True)
    grad, = torch.autograd.grad(dense.layer_norm(x, w, b), x, dy)
    x = x.detach()
    h = 2.0 ** -7
    v = torch.sign(grad)
    yp, ym = (dense.layer_norm(x + s * h * v, w, b).double() for s in (1.0, -1.0))
    diff = (dy.double() * (yp - ym)).sum() / (2 * h)
    want = (grad.double() * v.double()).sum()
    # roundings: y to within 64 fp32 steps of sums of 40 and of x + h v; curvature: third derivative of a
    # normalisation of rows with std ~2 is below 15 |v|^3 / std^3
    rounding = (dy.double().abs() * (yp.abs() + ym.abs() + 2.0)).sum() * 64 * 2.0 ** -24 / (2 * h)
    cubic = (dy.double().abs() * w.double().abs()).sum() * 15 * h * h / 6
    assert (diff - want).abs() <= rounding + cubic
    assert rounding + cubic < 0.05 * want.abs()


def test_norm_repeats_bit_for_bit_in_graphs():
    x, w, b, dy = make_norm(2, 300, 520, torch.bfloat16, torch.bfloat16, per_sample=True)

    def both():
        y, mean, rstd = dense.layer_norm_modulate_forward(x, b, w)
        return [y, mean, rstd, *dense.layer_norm_modulate_backward(dy, x, w, mean, rstd)]

    first = both()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    for a, o in zip(first, out):
        assert torch.equal(a, o)
    xg = x.clone().requires_grad_(True)
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        with pytest.raises(RuntimeError, match="layer_norm_modulate_forward"):
            dense.layer_norm_modulate(xg, b, w)


# ---------------------------------------------------- the operators as they are used together


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_feed_forward_half_forward_and_backward(dtype):
    """x + gate * fc2(gelu(fc1(LayerNorm(x) (1 + scale) + shift))), every gradient."""
    s, t, d, f = 2, 45, 96, 200
    x = rand((s, t, d), dtype, 1)
    scale, shift, gate = (rand((s, d), dtype, 2 + i, 0.3) for i in range(3))
    w1, b1 = rand((f, d), dtype, 6, d ** -0.5), rand((f,), dtype, 7, 0.1)
    w2, b2 = rand((d, f), dtype, 8, f ** -0.5), rand((d,), dtype, 9, 0.1)
    dy = rand((s, t, d), dtype, 10)
    leaves = [x, scale, shift, gate, w1, b1, w2, b2]
    for leaf in leaves:
        leaf.requires_grad_(True)
    h = dense.layer_norm_modulate(x, shift, scale)
    a = dense.dense_linear(h, w1, b1, activation="gelu_tanh")
    y = dense.dense_linear(a, w2, b2, residual=x, gate=gate)
    gx, gscale, gshift, ggate, gw1, gb1, gw2, gb2 = torch.autograd.grad(y, leaves, dy)
    m = s * t
    bx, bdy = B(rows_of(x.detach(), d)), B(rows_of(dy, d))
    bsc, bsh, bg = (B(spread(v.detach(), m)) for v in (scale, shift, gate))
    one = B(bsc.v + 1.0, 2.0 ** -22)
    bw1, bb1, bw2, bb2 = (B(v.detach()) for v in (w1, b1, w2, b2))
    rh, xh, rstd = bounds.norm(bx, one, bsh, 1e-6, dtype)
    ra, z1 = bounds.linear(rh, bw1, bb1, "gelu_tanh", None, None, dtype)
    ry, z2 = bounds.linear(ra, bw2, bb2, None, bg, bx, dtype)
    ry.check(rows_of(y.detach(), d), "y")
    da, dw2, db2, dgate = bounds.linear_grads(bdy, ra, bw2, z2.round(torch.float32), None, bg, dtype, s)
    dh, dw1, db1, _ = bounds.linear_grads(da, rh, bw1, z1.round(torch.float16), "gelu_tanh", None, dtype, s)
    dxn, dscale, dshift = bounds.norm_grads(dh, xh, rstd, one, dtype, dtype, s)
    dx = (dxn + bdy).round(dtype)
    for got, want, name in ((gx, dx, "dx"), (gscale, dscale, "dscale"), (gshift, dshift, "dshift"),
                            (ggate, dgate, "dgate"), (gw1, dw1, "dw1"), (gb1, db1, "db1"), (gw2, dw2, "dw2"),
                            (gb2, db2, "db2")):
        want.check(got.reshape(want.v.shape), name)


def make_ff(d=128, h=256, seed=0):
    from qwen_image_shardedit_mlx_b200 import QwenFeedForward

    return QwenFeedForward.random(d, h, generator=torch.Generator(device="cuda").manual_seed(seed))


def test_materialised_feed_forward_half_trains():
    from qwen_image_shardedit_mlx_b200.dense_img_ff_window import materialize_dense_img_ff

    s, t, d = 2, 40, 128
    ff, _ = materialize_dense_img_ff(make_ff())
    x, dy = rand((s, t, d), torch.bfloat16, 1), rand((s, t, d), torch.bfloat16, 2)
    shift, scale, gate = (rand((s, d), torch.bfloat16, 3 + i, 0.3) for i in range(3))
    weights = [ff.mlp_in.weight, ff.mlp_in.bias, ff.mlp_out.weight, ff.mlp_out.bias]
    leaves = [x, shift, scale, gate, *weights]
    for leaf in leaves:
        leaf.requires_grad_(True)
    y = ff.half(x, shift, scale, gate)
    grads = torch.autograd.grad(y, leaves, dy)
    # the same calls one by one, without autograd: the same bits
    with torch.no_grad():
        h, mean, rstd = dense.layer_norm_modulate_forward(x, shift, scale)
        a, z1 = dense.dense_linear_forward(h, weights[0], weights[1], activation="gelu_tanh", save_preact=True)
        out, z2 = dense.dense_linear_forward(a, weights[2], weights[3], residual=x, gate=gate, save_preact=True)
        g2 = dense.dense_linear_backward(dy, a, weights[2], preact=z2, gate=gate,
                                         outputs=("x", "weight", "bias", "gate"))
        g1 = dense.dense_linear_backward(g2.x, h, weights[0], preact=z1, activation="gelu_tanh")
        gn = dense.layer_norm_modulate_backward(g1.x, x, scale, mean, rstd)
    assert torch.equal(y, out)
    for got, want in zip(grads, (gn.x + dy, gn.bias, gn.weight, g2.gate, g1.weight, g1.bias, g2.weight, g2.bias)):
        assert torch.equal(got, want)
    # the unfused module rounds where the fused one does not: its own roundings (the
    # products' outputs, the bias sums, GELU) bound the distance
    with torch.no_grad():
        fused, plain = ff.fused(x).double(), ff(x).double()
    assert (fused - plain).norm() <= 4 * 2.0 ** -8 * plain.norm()


def test_materialised_feed_forward_with_an_adapter():
    from qwen_image_shardedit_mlx_b200.dense_img_ff_window import materialize_dense_img_ff
    from qwen_image_shardedit_mlx_b200.lora import iter_adapters, lora_delta_weight

    q6 = make_ff()
    a, b = rand((128, 32), torch.bfloat16, 5, 0.1), rand((32, 256), torch.bfloat16, 6, 0.1)
    q6.mlp_in.set_lora(a, b, 0.5)
    additive, _ = materialize_dense_img_ff(q6)
    x = rand((3, 128), torch.bfloat16, 7)
    with pytest.raises(ValueError, match="fold_single"):
        additive.fused(x)
    folded, _ = materialize_dense_img_ff(q6, fold_single=True)
    assert folded.mlp_in_lora is None
    q6.mlp_in.set_lora(None)
    base, _ = materialize_dense_img_ff(q6)
    q6.mlp_in.set_lora(a, b, 0.5)
    want = (base.mlp_in.weight.float() + lora_delta_weight(list(iter_adapters(q6.mlp_in)), dtype=torch.float32)
            ).to(torch.bfloat16)
    assert torch.equal(folded.mlp_in.weight, want)
    assert folded.fused(x).shape == (3, 128)


def test_second_derivatives_are_refused():
    x = rand((4, 16), torch.bfloat16, 1).requires_grad_(True)
    w = rand((8, 16), torch.bfloat16, 2).requires_grad_(True)
    for y in (dense.dense_linear(x, w, activation="silu"), dense.layer_norm(x)):
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.autograd.grad(y.sum(), x, create_graph=True)


def test_saved_tensors_changed_in_place_are_noticed():
    x = rand((4, 16), torch.bfloat16, 1)
    w = rand((8, 16), torch.bfloat16, 2).requires_grad_(True)
    y = dense.dense_linear(x, w)
    x.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_gradients_add_up_over_calls_that_share_leaves():
    x = rand((2, 24, 32), torch.bfloat16, 1)
    w = rand((32, 32), torch.bfloat16, 2, 0.2).requires_grad_(True)
    v = rand((32,), torch.float32, 3).requires_grad_(True)
    one, = torch.autograd.grad(dense.dense_linear(x, w).float().sum(), w)
    (dense.dense_linear(x, w).float().sum() + dense.dense_linear(x, w).float().sum()).backward()
    assert torch.equal(w.grad, one + one)
    h = dense.layer_norm(dense.dense_linear(dense.layer_norm(x, v), w), v)  # the same vector in two norms
    h.float().sum().backward()
    assert v.grad.shape == (32,) and v.grad.isfinite().all()


def test_operators_on_a_side_stream_with_tensors_of_another():
    x, w, b, g, r, dy = make_linear(2, 70, 136, 264, torch.bfloat16)
    ready = torch.cuda.Event()
    ready.record()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        side.wait_event(ready)
        w.requires_grad_(True)
        y = dense.dense_linear(x, w, b, activation="silu", residual=r, gate=g)
        n = dense.layer_norm(y, None, None)
        grad, = torch.autograd.grad(n, w, dy)
    torch.cuda.current_stream().wait_stream(side)
    y2 = dense.dense_linear(x, w, b, activation="silu", residual=r, gate=g)
    grad2, = torch.autograd.grad(dense.layer_norm(y2), w, dy)
    assert torch.equal(y, y2) and torch.equal(grad, grad2)


def test_rows_far_into_a_tensor_of_more_than_2_31_elements():
    # a view whose rows start past 2^31 elements: offsets are 64-bit
    d, rows = 1 << 20, 2100
    big = torch.zeros((rows, d), dtype=torch.bfloat16, device="cuda")
    x = big[rows - 3:, 5:5 + 264]
    x.copy_(rand((3, 264), torch.bfloat16, 1))
    near = x.contiguous()
    w = rand((72, 264), torch.bfloat16, 2, 0.1)
    assert torch.equal(dense.dense_linear(x, w), dense.dense_linear(near, w))
    assert torch.equal(dense.layer_norm(x), dense.layer_norm(near))
    wide = big[::700, :264]  # rows 7.3e8 elements apart
    wide.copy_(rand(wide.shape, torch.bfloat16, 3))
    pad = wide.contiguous()
    assert torch.equal(dense.layer_norm(wide), dense.layer_norm(pad))
    tall = torch.cat([wide.contiguous()] * 4)
    many = big[::175, 8:272]
    many.copy_(tall[:many.shape[0]] if many.shape[0] <= tall.shape[0] else many)
    assert torch.equal(dense.dense_linear(many, w), dense.dense_linear(many.contiguous(), w))


def test_outputs_of_more_than_2_31_elements():
    m, k, n = 131080, 8, 16400  # 2.15e9 outputs
    x, w = rand((m, k), torch.bfloat16, 1), rand((n, k), torch.bfloat16, 2)
    y = dense.dense_linear(x, w)
    for rows in (slice(0, 5), slice(m // 2, m // 2 + 5), slice(m - 5, m)):
        assert torch.equal(y[rows], dense.dense_linear(x[rows].contiguous(), w))
    del y
    d = 1 << 15
    x = torch.zeros((65600, d), dtype=torch.bfloat16, device="cuda")
    x[-3:] = rand((3, d), torch.bfloat16, 3)
    y = dense.layer_norm(x)
    assert torch.equal(y[-3:], dense.layer_norm(x[-3:].contiguous()))


def test_padded_batch_leaves_the_padding_alone():
    # rows behind the last one of a buffer stay as they were
    x, w, b, _, _, _ = make_linear(1, 45, 72, 96, torch.bfloat16, gate=False)
    y = dense.dense_linear(x[0, :37], w, b)
    after = torch.full((16, 96), 3.0, dtype=torch.bfloat16, device="cuda")
    assert y.shape == (37, 96) and torch.equal(after, torch.full_like(after, 3.0))
    assert torch.equal(y, dense.dense_linear(x, w, b)[0, :37])


@pytest.mark.parametrize("samples,rows", [(70000, 1), (300, 3), (64, 100)])
def test_many_vectors(samples, rows):
    x, w, b, dy = make_norm(samples, rows, 24, torch.bfloat16, torch.bfloat16, per_sample=True)
    check_norm(x, w, b, dy, modulate=True)


def test_many_gates():
    check_linear(*make_linear(700, 3, 40, 56, torch.bfloat16), "silu")
    check_linear(*make_linear(3000, 1, 8, 24, torch.float16), None)


def test_status_errors_have_the_library_class():
    from qwen_image_shardedit_mlx_b200._lib import Q6Error

    x = torch.zeros((2, 8), dtype=torch.bfloat16, device="cuda")
    huge = torch.zeros((1,), dtype=torch.bfloat16, device="cuda").expand((1 << 30) + 1, 1)[:, :1]
    with pytest.raises(Q6Error):
        dense.dense_linear_forward(huge, torch.zeros((1, 1), dtype=torch.bfloat16, device="cuda"))
    assert dense.dense_linear(x, x).shape == (2, 2)


def test_linear_nan_reaches_the_gradients():
    # a NaN pre-activation gives NaN gradients in its row, a large one does not
    x = rand((4, 16), torch.bfloat16, 1)
    w = torch.eye(16, dtype=torch.bfloat16, device="cuda")
    x[1, 3], x[2, 5] = float("nan"), 1e30
    y, z = dense.dense_linear_forward(x, w, activation="silu", save_preact=True)
    dx = dense.dense_linear_backward(torch.ones_like(y), x, w, preact=z, activation="silu", outputs=("x",)).x
    assert dx[1].isnan().all()  # every value of row 1 sums a product with the NaN
    assert dx[[0, 2, 3]].isfinite().all() and dx[2, 5] == 1.0
