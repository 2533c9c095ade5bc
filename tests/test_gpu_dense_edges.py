"""The dense linear and the layer norm at the ends of their range: row scales far
from one, guarded buffers, far strides, threads and saved-tensor hooks."""

from __future__ import annotations

import pytest
import torch
import torch.utils.checkpoint

import bounds
from bounds import B
from qwen_image_shardedit_mlx_b200 import _lib, dense, ops
from test_gpu_dense import DT, check_norm, rand, spread

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _no_device_error():
    yield
    assert ops.device_error() == 0


# row std, eps, std of dy: every input, output and statistic fits the types (the sum
# of squares of 4096 values of 1e17 is 4.1e37)
SCALES = [(1e13, 1e-6, 1.0), (1e15, 1e-6, 1.0), (1e17, 1e-6, 1.0), (1e17, 1e-6, 1e-24), (1e-14, 0.0, 1.0),
          (1e-17, 0.0, 1.0), (1e-17, 0.0, 1e18)]


@pytest.mark.parametrize("std,eps,dy_std", SCALES)
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("d", [64, 256, 264, 1001, 1024, 3000, 4096])
def test_norm_rows_of_any_scale(std, eps, dy_std, dtype, d):
    # a warp and several per row, with and without 16-byte accesses, one and two vectors
    for samples, modulate in ((1, False), (2, True)):
        x = rand((samples, 21, d), DT[dtype], d, std)
        # a part along xh, so that the gradient's third term counts
        dy = ((rand(x.shape, torch.float32, d + 1) + 0.5 * x.float().sign()) * dy_std).to(DT[dtype])
        shape = (samples, d) if modulate else (d,)
        w = rand(shape, DT[dtype], d + 2, 0.3, 0.0 if modulate else 1.0)
        b = rand(shape, DT[dtype], d + 3, 0.3)
        check_norm(x, w, b, dy, modulate=modulate, eps=eps)


def test_product_behind_a_kernel_of_several_seconds():
    """A product may be resident long before its inputs are ready (the kernel in front lets
    it start early): its pipeline's wait limits of 2 s must not count that time."""

    def bias_gradient(m):  # a gate per row of eight columns: one block adds m partial sums
        return dense.dense_linear_backward(torch.ones((m, 8), dtype=torch.bfloat16, device="cuda"), None, None,
                                           gate=torch.ones((m, 8), dtype=torch.bfloat16, device="cuda"),
                                           outputs=("bias",)).bias

    def milliseconds(m):
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        bias_gradient(m)
        end.record()
        end.synchronize()
        return start.elapsed_time(end)

    bias_gradient(1 << 22)
    m = min(int((1 << 24) * 3500.0 / milliseconds(1 << 24)), 1 << 29)
    if (ms := milliseconds(m)) < 2500.0:
        pytest.skip(f"the kernel in front takes {ms:.0f} ms only")
    for rows, n in ((40, 72), (700, 776)):
        x, w = rand((rows, 264), torch.bfloat16, rows), rand((n, 264), torch.bfloat16, n, 0.1)
        want = dense.dense_linear(x, w)
        db = bias_gradient(m)
        got = dense.dense_linear(x, w)  # nothing between the two launches
        torch.cuda.synchronize()
        assert ops.device_error() == 0
        assert torch.equal(got, want)
        assert (db.float() > 0).all()


class Guarded:
    """Buffers carved out of one filled allocation: what lies between them must stay."""

    FILL, GAP = 0xA5, 4096

    def __init__(self, nbytes):
        self.bytes = torch.full((nbytes,), self.FILL, dtype=torch.uint8, device="cuda")
        self.at, self.parts = self.GAP, []

    def take(self, nbytes, shift=0):
        """Address of ``nbytes`` bytes, ``shift`` past a multiple of 256."""
        start = self.at + (-(self.bytes.data_ptr() + self.at)) % 256 + shift
        self.at = start + nbytes + self.GAP
        assert self.at <= self.bytes.numel()
        self.parts.append((start, nbytes))
        return self.bytes.data_ptr() + start

    def value(self, address, like):
        """The buffer at ``address`` as a tensor of ``like``'s shape and type."""
        start = address - self.bytes.data_ptr()
        return self.bytes[start:start + like.numel() * like.element_size()].clone().view(like.dtype).reshape(like.shape)

    def check(self):
        outside = torch.ones_like(self.bytes, dtype=torch.bool)
        for start, nbytes in self.parts:
            outside[start:start + nbytes] = False
        assert (self.bytes[outside] == self.FILL).all()


def stream():
    return torch.cuda.current_stream().cuda_stream


# few rows, one and two row tiles; ragged tiles; split sums; operands that are copied
# first; single rows and columns
GUARD_LINEAR = [(1, 264, 72), (7, 133, 57), (13, 520, 24), (16, 1031, 1), (17, 72, 40), (45, 264, 136), (150, 707, 773),
                (300, 2056, 1032), (96, 4096, 131), (257, 8, 393), (515, 1, 9), (33, 63, 2050)]


@pytest.mark.parametrize("m,k,n", GUARD_LINEAR)
@pytest.mark.parametrize("shift", [0, 2])
@pytest.mark.parametrize("gated", [False, True])
def test_linear_writes_nothing_beside_its_buffers(m, k, n, shift, gated):
    lib, dtype = _lib.lib(), torch.bfloat16
    x, w, b, dy = (rand(s, dtype, i, std) for i, (s, std) in enumerate(
        (((m, k), 1.0), ((n, k), k ** -0.5), ((n,), 0.5), ((m, n), 1.0))))
    gates = 3 if gated and m % 3 == 0 else 1
    gate = rand((gates, n), dtype, 5) if gated else None
    xs = x.reshape(gates, -1, k)
    y, z = dense.dense_linear_forward(xs, w, b, activation="gelu_tanh", gate=gate, save_preact=True)
    outputs = ("x", "weight", "bias", "gate")[:4 if gated else 3]
    want = dense.dense_linear_backward(dy.reshape(gates, -1, n), xs, w, preact=z, activation="gelu_tanh", gate=gate,
                                       outputs=outputs)
    pack = sum(bit for bit, odd in ((_lib.Q6_PACK_X, k % 8), (_lib.Q6_PACK_W, k % 8), (_lib.Q6_PACK_DY, n % 8)) if odd)
    gate_args = (gate.data_ptr() if gated else None, n, m // gates)
    zt = _lib.Q6_DTYPE_F32 if gated else _lib.Q6_DTYPE_F16

    nbytes = lib.q6_dense_linear_workspace_bytes(m, n, k, pack)
    g = Guarded(nbytes + 8 * m * n + (1 << 16))
    py, pz, ws = g.take(2 * m * n, shift), g.take(z.element_size() * m * n, 2 * shift), g.take(nbytes)
    status = lib.q6_dense_linear(x.data_ptr(), k, w.data_ptr(), k, b.data_ptr(), *gate_args, None, 0, py, pz, zt, m, n, k,
                                 _lib.Q6_DTYPE_BF16, _lib.Q6_ACT_GELU_TANH, ws if nbytes else None, nbytes, stream())
    assert status == 0
    g.check()
    assert torch.equal(g.value(py, y), y) and torch.equal(g.value(pz, z), z)

    flags = _lib.Q6_GRAD_X | _lib.Q6_GRAD_W | _lib.Q6_GRAD_BIAS | (_lib.Q6_GRAD_GATE if gated else 0)
    nbytes = lib.q6_dense_linear_grad_workspace_bytes(m, n, k, m // gates, _lib.Q6_ACT_GELU_TANH, int(gated), flags, pack)
    g = Guarded(nbytes + 2 * (m * k + n * k + 4 * n) + (1 << 16))
    pdx, pdw, pdb = g.take(2 * m * k, shift), g.take(2 * n * k, shift), g.take(2 * n, shift)
    pdg = g.take(2 * n * gates, shift) if gated else None
    ws = g.take(nbytes)
    status = lib.q6_dense_linear_grad(dy.data_ptr(), n, x.data_ptr(), k, w.data_ptr(), k, z.data_ptr(), zt, *gate_args, pdx,
                                      pdw, pdb, pdg, m, n, k, _lib.Q6_DTYPE_BF16, _lib.Q6_ACT_GELU_TANH, ws, nbytes,
                                      stream())
    assert status == 0
    g.check()
    assert torch.equal(g.value(pdx, x), want.x.reshape(m, k)) and torch.equal(g.value(pdw, w), want.weight)
    assert torch.equal(g.value(pdb, b), want.bias)
    if gated:
        assert torch.equal(g.value(pdg, gate), want.gate)


@pytest.mark.parametrize("vecs,rows,d", [(1, 1, 1), (1, 5, 3), (2, 7, 33), (1, 37, 64), (3, 50, 100), (2, 40, 256),
                                         (1, 17, 1001), (2, 33, 1536), (1, 301, 128), (1, 5, 8200), (1, 2, 33001)])
@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_norm_writes_nothing_beside_its_buffers(vecs, rows, d, shift, dtype):
    lib, dt, m = _lib.lib(), DT[dtype], vecs * rows
    code = {"bf16": _lib.Q6_DTYPE_BF16, "fp32": _lib.Q6_DTYPE_F32}[dtype]
    size = dt.itemsize
    x, dy = rand((vecs, rows, d), dt, 1, 2.0), rand((vecs, rows, d), dt, 2)
    scale, bias = rand((vecs, d), dt, 3, 0.3), rand((vecs, d), dt, 4, 0.3)
    y, mean, rstd = dense.layer_norm_modulate_forward(x, bias, scale)
    g = Guarded(m * d * size + 8 * m + (1 << 16))
    py, pm, pr = g.take(m * d * size, shift * size), g.take(4 * m, shift * 4), g.take(4 * m)
    status = lib.q6_layer_norm(x.data_ptr(), d, scale.data_ptr(), bias.data_ptr(), d, rows, py, pm, pr, m, d, 1e-6, code,
                               code, _lib.Q6_NORM_ONE_PLUS, stream())
    assert status == 0
    g.check()
    # an odd address takes another kernel, with sums in another order: each within its own bound
    bx, bw, bb = B(x.reshape(m, d)), B(spread(scale.double() + 1.0, m), 2.0 ** -22), B(spread(bias, m))
    ry, xh, rs = bounds.norm(bx, bw, bb, 1e-6, dt)
    for p, ref, bound in ((py, y, ry), (pm, mean, bx.mean()), (pr, rstd, rs)):
        bound.check(g.value(p, ref).reshape(bound.v.shape), "forward")
        assert shift or torch.equal(g.value(p, ref), ref)

    want = dense.layer_norm_modulate_backward(dy, x, scale, mean, rstd)
    flags = _lib.Q6_GRAD_W | _lib.Q6_GRAD_BIAS
    nbytes = lib.q6_layer_norm_grad_workspace_bytes(m, d, rows, code, flags)
    g = Guarded(m * d * size + 2 * vecs * d * size + nbytes + (1 << 16))
    pdx, pdw, pdb = (g.take(v * d * size, shift * size) for v in (m, vecs, vecs))
    ws = g.take(nbytes)
    status = lib.q6_layer_norm_grad(dy.data_ptr(), d, x.data_ptr(), d, scale.data_ptr(), d, rows, mean.data_ptr(),
                                    rstd.data_ptr(), pdx, pdw, pdb, m, d, code, code, _lib.Q6_NORM_ONE_PLUS,
                                    ws if nbytes else None, nbytes, stream())
    assert status == 0
    g.check()
    dx, dw, db = bounds.norm_grads(B(dy.reshape(m, d)), xh, rs, bw, dt, dt, vecs)
    for p, ref, bound in ((pdx, want.x, dx), (pdw, want.weight, dw), (pdb, want.bias, db)):
        bound.check(g.value(p, ref).reshape(bound.v.shape), "backward")
        assert shift or torch.equal(g.value(p, ref), ref)


@pytest.mark.parametrize("off", [0, 8, 5])
def test_rows_of_every_operand_far_apart(off):
    """Operands whose rows pass 2^31 elements, through the tensor maps, the aligned copies
    (odd addresses), the strided residual and gates, and every gradient."""

    base = torch.zeros((2200, 1 << 20), dtype=torch.bfloat16, device="cuda")

    def far(rows, cols, at, seed, std=1.0):
        step = 2199 // (rows - 1)
        assert (rows - 1) * step << 20 > 1 << 31
        v = base[:(rows - 1) * step + 1:step, at + off:at + off + cols]
        v.copy_(rand((rows, cols), torch.bfloat16, seed, std))
        return v

    m, k, n = 21, 264, 136
    args = [far(m, k, 0, 1), far(n, k, 1000, 2, 0.1), far(m, n, 2000, 3), far(m, n, 3000, 4), far(m, n, 4000, 5)]
    near = [v.contiguous() for v in args]

    def passes(x, w, r, dy, g):
        out = []
        for act, gate in (("gelu_tanh", None), ("silu", g)):  # one vector, and one per row
            y, z = dense.dense_linear_forward(x, w, activation=act, residual=r, gate=gate, save_preact=True)
            outputs = ("x", "weight", "bias") + (("gate",) if gate is not None else ())
            out += [y, z, *dense.dense_linear_backward(dy, x, w, preact=z, activation=act, gate=gate, outputs=outputs)]
        out += dense.dense_linear_backward(dy, x, w)  # dy itself is the products' operand
        h, mean, rstd = dense.layer_norm_modulate_forward(r, g, dy)
        return out + [h, mean, rstd, *dense.layer_norm_modulate_backward(dy, r, g, mean, rstd)]

    got, want = passes(*args), passes(*near)
    for a, b in zip(got, want):
        assert (a is None) == (b is None)
        if a is not None:
            if off == 5 and a.shape == (m,):  # the norm's kernel without 16-byte accesses sums in another order
                assert (a - b).abs().max() <= n * 2.0 ** -23 * b.abs().max() * 4
            elif off == 5 and a.dtype == torch.bfloat16:
                assert (a.double() - b.double()).abs().max() <= 2.0 ** -7 * b.double().abs().max()
            else:
                assert torch.equal(a, b)
    if off == 5:
        for a, b in zip(got[:-6], want[:-6]):
            assert (a is None and b is None) or torch.equal(a, b)


def test_calls_from_several_threads():
    from concurrent.futures import ThreadPoolExecutor

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            x, w, b = (rand(s, torch.bfloat16, i + j) for j, s in enumerate(((3, 60 + i, 136), (200, 136), (136,))))
            leaves = [v.requires_grad_(True) for v in (x, w, b)]
            out = []
            for _ in range(8):
                y = dense.dense_linear(dense.layer_norm(x, b, b), w, activation="silu")
                out.append([y.detach(), *torch.autograd.grad(y.float().sum(), leaves)])
            torch.cuda.current_stream().synchronize()
        return out

    with ThreadPoolExecutor(4) as pool:
        together = list(pool.map(work, range(8)))
    for i, runs in enumerate(together):
        alone = work(i)[0]
        for run in runs:
            assert all(torch.equal(a, b) for a, b in zip(run, alone))


def test_saved_tensor_hooks_and_recomputation():
    x, w, b, gate = (rand(s, torch.bfloat16, i) for i, s in enumerate(((2, 40, 72), (136, 72), (136,), (2, 136))))
    leaves = [v.requires_grad_(True) for v in (x, w, b, gate)]
    dy = rand((2, 40, 136), torch.bfloat16, 9)

    def half(x, w, b, gate):
        return dense.dense_linear(dense.layer_norm(x), w, b, activation="gelu_tanh", gate=gate)

    want = torch.autograd.grad(half(*leaves), leaves, dy)
    with torch.autograd.graph.save_on_cpu():
        y = half(*leaves)
    kept = torch.autograd.grad(y, leaves, dy)
    again = torch.autograd.grad(torch.utils.checkpoint.checkpoint(half, *leaves, use_reentrant=False), leaves, dy)
    for a, b_, c in zip(want, kept, again):
        assert torch.equal(a, b_) and torch.equal(a, c)


def test_function_transforms_are_refused():
    """torch.func wraps tensors: a call must not compute without the wrapper's derivative or batch."""

    x, w = rand((4, 16), torch.bfloat16, 1), rand((8, 16), torch.bfloat16, 2)
    for f in (lambda v: dense.dense_linear(v, w).float().sum(), lambda v: dense.layer_norm(v).float().sum()):
        with pytest.raises(RuntimeError):
            torch.func.grad(f)(x)
        with pytest.raises(RuntimeError):
            torch.func.jvp(f, (x,), (torch.ones_like(x),))
        with pytest.raises(RuntimeError):
            torch.func.vmap(f)(x)
    assert dense.dense_linear(x, w).shape == (4, 8)  # and nothing of it lingers


def test_tensors_that_stand_for_their_negative():
    # the imaginary part of a conjugate is a view with a sign to apply; one column of it needs no copy
    both = torch.view_as_complex(rand((6, 1, 2), torch.float32, 1)).conj()
    x, plain = both.imag, both.imag.resolve_neg()
    assert x.is_neg() and not plain.is_neg()
    zeros, ones = torch.zeros((6, 1), device="cuda"), torch.ones((6, 1), device="cuda")
    b = rand((1,), torch.float32, 2)
    for call in (lambda v: dense.layer_norm_forward(v, b, b), lambda v: dense.layer_norm_modulate_forward(ones, v, v),
                 lambda v: dense.layer_norm_backward(v, ones, None, zeros[:, 0], ones[:, 0]),
                 lambda v: dense.layer_norm_backward(ones, ones, None, v, v)):
        for got, want in zip(call(x), call(plain)):
            assert (got is None and want is None) or torch.equal(got, want)
    w, flipped = rand((24, 16), torch.bfloat16, 3), torch._neg_view(rand((24, 16), torch.bfloat16, 3))
    a = rand((40, 16), torch.bfloat16, 4)
    assert torch.equal(dense.dense_linear(a, flipped, flipped[:, 0]), dense.dense_linear(a, -w, -w[:, 0]))
    dy, z = rand((40, 24), torch.bfloat16, 5), rand((40, 24), torch.float32, 6)
    for got, want in zip(dense.dense_linear_backward(torch._neg_view(dy), a, w, preact=torch._neg_view(z), activation="silu"),
                         dense.dense_linear_backward(-dy, a, w, preact=-z, activation="silu")):
        assert (got is None and want is None) or torch.equal(got, want)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("d", [1, 3, 7, 13, 14, 56, 61, 120, 224, 480, 960, 1001, 1920, 3000, 3072, 4097, 7680, 8192])
def test_norm_constant_rows_have_no_spread(dtype, d):
    """A row of one value (padding, a fill with the type's lowest value): its sums are exact
    in fp32 (at most 11 bits a value, 2^13 of them), so its mean is that value and its
    output the bias alone."""

    fi = torch.finfo(DT[dtype])
    big = 2.0 ** 60 if dtype == "bf16" else fi.max
    values = [0.0, 1.0, -3.0, 1.0 + fi.eps, 255.0, -1000.0, 2.0 ** 15 * (2 - fi.eps), -big, big / 3, big / 1.7]
    x = torch.tensor(values, dtype=DT[dtype], device="cuda")[:, None].expand(-1, d).contiguous()
    w, b = rand((d,), DT[dtype], 1), rand((d,), DT[dtype], 2)
    y, mean, rstd = dense.layer_norm_forward(x, w, b)
    assert torch.equal(mean, x[:, 0].float())
    assert torch.equal(y, b.expand_as(y))
    assert ((rstd - 1000.0).abs() <= 1e-3).all()
    y, mean, _ = dense.layer_norm_modulate_forward(x[:, None], b, w)
    assert torch.equal(mean, x[:, 0].float()) and torch.equal(y[:, 0], b.expand_as(x))
    for value in (float("inf"), float("-inf")):  # an infinite mean stays what it is
        _, mean, _ = dense.layer_norm_forward(torch.full((2, d), value, dtype=DT[dtype], device="cuda"))
        assert (mean == value).all()
