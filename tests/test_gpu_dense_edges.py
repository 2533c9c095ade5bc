"""The dense linear and the layer norm at the ends of their range: row scales far
from one, guarded buffers, far strides, threads and saved-tensor hooks."""

from __future__ import annotations

import pytest
import torch

from qwen_image_shardedit_mlx_b200 import dense, ops
from test_gpu_dense import DT, check_norm, rand

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
