"""LayerNorm for training where values or sizes reach the edge of what its kernels are built for."""
from __future__ import annotations

import pytest
import training_reference as reference
from test_gpu_layernorm_train import _backward, _normal
from training_reference import within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hidden", [24, 77, 300, 1000, 1001, 4000, 5001])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("residual", [False, True])
def test_gradient_of_a_constant_row_whose_mean_times_rstd_overflows(hidden, dtype, residual):
    """Rows of one value 2^121 have no variance: mean 2^121, rstd = 1 / sqrt(1e-5) = 316, and mean * rstd is past f32's range
    although every normalised element is 0.  Widths that leave some of a thread's columns past the row's end."""
    import torch

    rows = 40
    x, d, w = _normal((rows, hidden), dtype, 1), _normal((rows, hidden), dtype, 2), _normal((hidden,), dtype, 3, 0.1, 1.0)
    r = _normal((rows, hidden), dtype, 4) if residual else None
    x[::3] = 2.0 ** 121
    _, _, mean, rstd = reference.layernorm_forward(x, None, w, None, 1e-5)
    mean, rstd = mean.float(), rstd.float()
    assert bool((mean[::3] == 2.0 ** 121).all()) and bool((mean[::3] * rstd[::3]).isinf().all())
    grad_x, grad_w, grad_b = torch.empty_like(x), torch.empty_like(w), torch.empty_like(w)
    _backward(d, x, mean, rstd, w, grad_x, grad_w, grad_b, r)()
    expected = reference.layernorm_backward(d, x, mean, rstd, w, r)
    errors = reference.layernorm_backward_errors(d, x, mean, rstd, w, r)
    for got, value, error in zip((grad_x, grad_w, grad_b), expected, errors):
        within(got, value, dtype, error)
