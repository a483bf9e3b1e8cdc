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


def _guarded(shape, dtype, fill=7.0, behind=64):
    """A 16-byte aligned tensor with elements behind it that nobody may touch."""
    import torch

    count = 1
    for extent in shape:
        count *= extent
    flat = torch.full((count + behind,), fill, device="cuda", dtype=dtype)
    return flat[:count].view(shape), flat[count:]


#: widths that are no whole vectors, more than 2^24 elements: the persistent form.  Both ends of every number of threads a row:
#: 32 (16 bits only), 64, 128, 256, 512 threads of 16 columns, 64 to 512 of 8 columns in f32
RAGGED = [(65537, 257), (33000, 511), (32705, 513), (17000, 1001), (16500, 1023), (16400, 1025), (9000, 2047), (8200, 2049), (4200, 4095)]
RAGGED_16 = [(4100, 4097), (2100, 8191)]


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("dtype,weight_dtype,shape", [("f32", "f32", s) for s in RAGGED] + [("bf16", "f32", s) for s in RAGGED + RAGGED_16]
                         + [("f16", "f16", s) for s in RAGGED + RAGGED_16] + [("bf16", "bf16", (64600, 260))])
def test_forward_of_many_ragged_rows(dtype, weight_dtype, shape, residual):
    import torch
    from test_gpu_layernorm_train import _forward

    rows, hidden = shape
    assert rows * hidden > 1 << 24
    x, w, b = _normal(shape, dtype, 1, 1.5, 0.5), _normal((hidden,), weight_dtype, 2, 0.1, 1.0), _normal((hidden,), weight_dtype, 3, 0.1)
    r = _normal(shape, dtype, 4) if residual else None
    (out, after_out), (resid, after_resid) = _guarded(shape, x.dtype), _guarded(shape, x.dtype)
    (mean, after_mean), (rstd, after_rstd) = _guarded((rows,), torch.float32), _guarded((rows,), torch.float32)
    _forward(x, out, mean, rstd, w, b, r, resid if residual else None)()
    expected, s, e_mean, e_rstd = reference.layernorm_forward(x, r, w, b, 1e-5)
    off_out, off_mean, off_rstd = reference.layernorm_forward_errors(x, r, w, b, 1e-5)
    within(out, expected, dtype, off_out)
    within(mean, e_mean, "f32", off_mean)
    within(rstd, e_rstd, "f32", off_rstd)
    if residual:
        within(resid, s, dtype, reference.U * s.abs())
    for behind in (after_out, after_resid, after_mean, after_rstd):
        assert bool((behind == 7).all())
    if not residual:
        return
    for own in ("residual", "x"):  # the sum over its own input, while neighbouring rows are being copied ahead
        stream = (r if own == "residual" else x).clone()
        out.fill_(float("nan"))
        _forward(x if own == "residual" else stream, out, mean, rstd, w, b, stream if own == "residual" else r, stream)()
        within(out, expected, dtype, off_out)
        within(stream, s, dtype, reference.U * s.abs())


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("dtype,shape", [("f32", s) for s in RAGGED] + [("bf16", s) for s in RAGGED + RAGGED_16 + [(70000, 33), (50000, 130)]] + [("f16", (17000, 1001))])
def test_gradient_of_many_ragged_rows(dtype, shape, residual):
    import torch

    rows, hidden = shape
    x, d, w = _normal(shape, dtype, 5, 1.5, 0.5), _normal(shape, dtype, 6), _normal((hidden,), "f32", 7, 0.1, 1.0)
    r = _normal(shape, dtype, 8) if residual else None
    _, _, mean, rstd = reference.layernorm_forward(x, None, w, None, 1e-5)
    mean, rstd = mean.float(), rstd.float()
    (grad_x, after_x), (grad_w, after_w), (grad_b, after_b) = _guarded(shape, x.dtype), _guarded((hidden,), w.dtype), _guarded((hidden,), w.dtype)
    _backward(d, x, mean, rstd, w, grad_x, grad_w, grad_b, r)()
    expected, errors = reference.layernorm_backward(d, x, mean, rstd, w, r), reference.layernorm_backward_errors(d, x, mean, rstd, w, r)
    for got, value, error, kind in zip((grad_x, grad_w, grad_b), expected, errors, (dtype, "f32", "f32")):
        within(got, value, kind, error)
    for behind in (after_x, after_w, after_b):
        assert bool((behind == 7).all())
    assert torch.isfinite(grad_x).all()
