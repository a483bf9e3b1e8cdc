"""Sums over rows and tokens of whole numbers, which 32 bits hold exactly in any order: a lost or doubled row shows.

The products are multiples of 1/2 and no sum of magnitudes reaches 2^23, so every addition is exact; the one rounding is the
result's, to its own type."""
from __future__ import annotations

import pytest
from gpu_util import TORCH_DTYPE
from test_gpu_embedding import GRADIENT_SHAPES, _gradient, _tokens
from test_gpu_layernorm_train import _backward

pytestmark = pytest.mark.gpu


def _whole(shape, dtype, most, seed):
    import torch

    generator = torch.Generator("cuda").manual_seed(seed)
    return torch.randint(-most, most + 1, shape, device="cuda", generator=generator).to(getattr(torch, TORCH_DTYPE[dtype]))


NORMS = [  # dtype, weight dtype, rows, hidden, offset of the tensors in elements
    ("bf16", "f32", 40000, 24, 0), ("f32", "f32", 40000, 8, 0), ("bf16", "f32", 65536, 64, 0), ("f16", "f16", 30011, 16, 0), ("bf16", "f32", 30000, 128, 0),
    ("bf16", "f32", 9001, 1024, 0), ("f32", "f32", 5003, 512, 0), ("bf16", "bf16", 7001, 2048, 0), ("f32", "f32", 3001, 4096, 0), ("bf16", "f32", 1501, 8192, 0),
    ("f32", "f32", 1203, 8192, 0), ("f32", "f32", 1203, 8188, 0), ("bf16", "f32", 2003, 4088, 0),
    ("f32", "f32", 64, 1024, 0), ("bf16", "f32", 300, 24, 0), ("bf16", "f32", 17, 8192, 0), ("f16", "f32", 1, 512, 0), ("f32", "f32", 31, 4096, 0),  # one cluster
    ("f16", "f32", 8191, 1001, 0), ("bf16", "f32", 70000, 33, 0), ("f32", "f32", 50000, 130, 0), ("bf16", "f32", 50000, 250, 0), ("bf16", "f32", 30000, 300, 0),
    ("f32", "f32", 9000, 2047, 0), ("bf16", "bf16", 5000, 4095, 0), ("bf16", "f32", 2000, 8191, 0), ("f32", "f32", 2500, 4095, 0), ("f16", "f32", 5, 77, 0),
    ("bf16", "f32", 700, 9001, 0), ("f32", "f32", 900, 5001, 0), ("bf16", "f32", 3001, 1024, 1), ("f32", "f32", 40000, 24, 1), ("f16", "f16", 3, 333, 3),
]


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("dtype,weight_dtype,rows,hidden,offset", NORMS)
def test_column_sums_of_the_norms_gradient(dtype, weight_dtype, rows, hidden, offset, residual):
    import torch

    def placed(value):
        flat = torch.empty(value.numel() + 16, device="cuda", dtype=value.dtype)
        view = flat[offset:offset + value.numel()].view(value.shape)
        view.copy_(value)
        return view

    x, d, w = placed(_whole((rows, hidden), dtype, 8, 1)), placed(_whole((rows, hidden), dtype, 4, 2)), _whole((hidden,), weight_dtype, 3, 3)
    r = placed(_whole((rows, hidden), dtype, 4, 4)) if residual else None
    mean, rstd = _whole((rows,), "f32", 2, 5), 2.0 ** -torch.randint(0, 2, (rows,), device="cuda", generator=torch.Generator("cuda").manual_seed(6)).float()
    n = (x.double() - mean.double()[:, None]) * rstd.double()[:, None]
    sums = (d.double() * n).sum(0), d.double().sum(0)
    assert float((d.double() * n).abs().sum(0).max()) < 2 ** 23
    grad_x, grad_w, grad_b = placed(torch.zeros_like(x)), torch.full_like(w, float("nan")), torch.full_like(w, float("nan"))
    for bias in (grad_b, None):
        grad_w.fill_(float("nan"))
        _backward(d, x, mean, rstd, w, grad_x, grad_w, bias, r)()
        assert torch.equal(grad_w, sums[0].to(w.dtype))
    assert torch.equal(grad_b, sums[1].to(w.dtype))


@pytest.mark.parametrize("grad_dtype,table_dtype", [("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16")])
@pytest.mark.parametrize("count,vocabulary,hidden,kind", GRADIENT_SHAPES + [(8192, 100, 40, "same"), (65536, 9, 24, "same"), (70000, 9, 24, "same"), (4096, 3, 1032, "even"),
                                                                           (16384, 2000, 40, "even"), (32768, 50257, 24, "zipf")])
def test_sums_over_tokens(count, vocabulary, hidden, kind, grad_dtype, table_dtype):
    import torch

    tokens, grad = _tokens(count, vocabulary, "i64" if count % 2 else "i32", 11, kind), _whole((count, hidden), grad_dtype, 8, 12)
    sums = torch.zeros(vocabulary, hidden, device="cuda", dtype=torch.float64).index_add_(0, tokens.long(), grad.double())
    table = _whole((vocabulary, hidden), table_dtype, 8, 13)
    added = (sums * 0.5 + table.double()).to(table.dtype)
    named = torch.zeros(vocabulary, device="cuda", dtype=torch.bool).index_fill_(0, tokens.long(), True)
    written = torch.full_like(table, float("nan"))
    _gradient(grad, tokens, written, scale=0.5)(grad, tokens, written)
    assert torch.equal(written, (sums * 0.5).to(table.dtype))
    before = table.clone()
    _gradient(grad, tokens, table, scale=0.5, accumulate=True)(grad, tokens, table)
    assert torch.equal(table[named], added[named]) and torch.equal(table[~named], before[~named])
