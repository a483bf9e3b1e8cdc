"""64-bit references of the training operators, and the error that 32-bit arithmetic may add to them.

Every bound counts roundings: u = 2^-24 is half a step of f32 relative to the value, a stored result adds half a step of
its own dtype, and a sum whose additions are at most `depth` deep is off by at most ``depth * u`` times the sum of the
magnitudes."""
from __future__ import annotations

import math

U = 2.0 ** -24
#: numbers this small are stored with an absolute error (f16 is subnormal below 2^-14, steps of 2^-24)
FLOOR = {"f32": 2.0 ** -140, "bf16": 2.0 ** -130, "f16": 2.0 ** -25}


def half_step(dtype: str) -> float:
    return {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}[dtype]


def within(actual, expected, dtype: str, arithmetic) -> None:
    """|actual - expected| <= arithmetic + one rounding to ``dtype`` of a value that is off by ``arithmetic``."""
    actual, error = actual.double(), arithmetic
    allowed = error + half_step(dtype) * (expected.abs() + error) + FLOOR[dtype]
    off = (actual - expected).abs()
    assert bool(actual.isfinite().all()), "not finite"
    worst = float((off - allowed).max())
    assert worst <= 0, f"off by up to {float((off / allowed.clamp_min(1e-300)).max()):.3g} of what is allowed"


def layernorm_forward(x, residual, weight, bias, epsilon: float):
    """out, s, mean, rstd in f64."""
    s = x.double() + (residual.double() if residual is not None else 0.0)
    mean = s.mean(-1, keepdim=True)
    rstd = ((s - mean).square().mean(-1, keepdim=True) + epsilon).rsqrt()
    out = (s - mean) * rstd * weight.double() + (bias.double() if bias is not None else 0.0)
    return out, s, mean[..., 0], rstd[..., 0]


def norm_depth(hidden: int) -> int:
    """Additions one after another in a row's sum: a thread adds up at most 32 elements of a row kept in registers, or
    hidden / 256 element by element; shuffles and warps add ten levels."""
    return max(32, -(-hidden // 256)) + 12


def layernorm_forward_errors(x, residual, weight, bias, epsilon: float):
    """Error bounds of out, mean, rstd.

    mean: the sum's depth.  Variance: its terms are (s - mean)^2 with s - mean off by u |s - mean| and the mean's error, so
    it is off by (depth + 4) u variance + 2 e |.| + e^2 for the mean's error e; rstd is off by half that, relative, and the
    roundings of +, sqrt and the division."""
    hidden = x.shape[-1]
    depth = norm_depth(hidden)
    out, s, mean, rstd = layernorm_forward(x, residual, weight, bias, epsilon)
    mean, rstd = mean[..., None], rstd[..., None]
    e_mean = (depth + 2) * U * s.abs().mean(-1, keepdim=True) + U * s.abs().max(-1, keepdim=True).values
    variance = (s - mean).square().mean(-1, keepdim=True)
    e_variance = (depth + 6) * U * variance + 2 * e_mean * variance.sqrt() + e_mean.square()
    relative = 0.5 * e_variance / (variance + epsilon) * 1.5 + 4 * U
    normal = (s - mean) * rstd
    e_normal = normal.abs() * (relative + 4 * U) + (e_mean + U * s.abs()) * rstd
    e_out = e_normal * weight.double().abs() + 3 * U * ((normal * weight.double()).abs() + (bias.double().abs() if bias is not None else 0.0))
    return e_out, e_mean[..., 0], (relative * rstd)[..., 0]


def layernorm_backward(grad_out, x, mean, rstd, weight, grad_resid):
    """grad_x, grad_weight, grad_bias in f64, from the statistics as stored, and the normalised rows."""
    d, r = grad_out.double(), rstd.double()[..., None]
    n = (x.double() - mean.double()[..., None]) * r
    g = d * weight.double()
    grad_x = r * (g - g.mean(-1, keepdim=True) - n * (g * n).mean(-1, keepdim=True))
    if grad_resid is not None:
        grad_x = grad_x + grad_resid.double()
    rows = tuple(range(x.dim() - 1))
    return grad_x, (d * n).sum(rows), d.sum(rows), n


def layernorm_backward_errors(grad_out, x, mean, rstd, weight, grad_resid):
    """Error bounds of grad_x, grad_weight, grad_bias: products of a few roundings each; row sums of the depth above;
    column sums of any order over R rows, at most R deep."""
    depth = norm_depth(x.shape[-1])
    grad_x, _, _, n = layernorm_backward(grad_out, x, mean, rstd, weight, grad_resid)
    d, r = grad_out.double(), rstd.double()[..., None].abs()
    g = d * weight.double()
    e_n = 2 * U * (n.abs())  # the difference and the product
    mean_g, mean_gn = g.abs().mean(-1, keepdim=True), (g * n).abs().mean(-1, keepdim=True)
    e_inner = 4 * U * (g.abs() + mean_g + n.abs() * mean_gn) + (depth + 4) * U * mean_g + n.abs() * (depth + 6) * U * mean_gn + e_n * mean_gn
    e_x = r * e_inner + 2 * U * (grad_x.abs() + (grad_resid.double().abs() if grad_resid is not None else 0.0))
    rows = tuple(range(x.dim() - 1))
    count = math.prod(x.shape[:-1])
    e_weight = (count + 4) * U * (d * n).abs().sum(rows)
    e_bias = (count + 1) * U * d.abs().sum(rows)
    return e_x, e_weight, e_bias


def adamw(param, grad, exp_avg, exp_avg_sq, rate, step, factor, beta1, beta2, epsilon, decay):
    """The step in f64, and the error bounds of its three results.

    Four roundings for each moment (the products with constants that are themselves rounded).  The corrections
    1 - beta^step come from expm1 of a product that is off by 3 u: relative error below 6 u; quotient and root add as many
    again, and the moments' own errors pass through."""
    g = grad.double() * factor
    m, v = beta1 * exp_avg.double() + (1 - beta1) * g, beta2 * exp_avg_sq.double() + (1 - beta2) * g * g
    e_m = 4 * U * ((beta1 * exp_avg.double()).abs() + ((1 - beta1) * g).abs())
    e_v = 6 * U * (beta2 * exp_avg_sq.double() + (1 - beta2) * g * g)
    first, second = -math.expm1(step * math.log(beta1)) if beta1 else 1.0, -math.expm1(step * math.log(beta2)) if beta2 else 1.0
    denominator = (v / second).sqrt() + epsilon
    change = rate * (m / first) / denominator
    p = param.double() * (1 - rate * decay) - change
    e_p = 4 * U * param.double().abs() + 24 * U * change.abs() + rate / first * e_m / denominator
    return p, m, v, e_p, e_m, e_v
