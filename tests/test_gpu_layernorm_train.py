"""LayerNorm forward with statistics and its backward pass on the GPU against 64 bits."""
from __future__ import annotations

import pytest
import training_reference as reference
from gpu_util import TORCH_DTYPE, current_stream, void_p
from training_reference import U, within

pytestmark = pytest.mark.gpu


def _torch():
    import torch

    return torch


def _dtype(name):
    return getattr(_torch(), TORCH_DTYPE[name])


def _normal(shape, dtype, seed, scale=1.0, shift=0.0):
    torch = _torch()
    return (torch.randn(shape, device="cuda", generator=torch.Generator("cuda").manual_seed(seed)) * scale + shift).to(_dtype(dtype))


def _forward(x, out, mean, rstd, weight, bias=None, residual=None, out_resid=None, *, epsilon=1e-5, backend="b200"):
    import baybridge_b200 as cute

    @cute.kernel
    def forward(x, out, mean, rstd, weight, bias, residual, out_resid):
        cute.layernorm_forward(x, out, mean, rstd, weight, bias, residual=residual, out_resid=out_resid, epsilon=epsilon)

    arguments = (x, out, mean, rstd, weight, bias, residual, out_resid)
    artifact = cute.compile(forward, *arguments, backend=backend)
    return lambda stream=None: artifact(*arguments, stream=stream)


def _backward(grad_out, x, mean, rstd, weight, grad_x, grad_weight, grad_bias=None, grad_resid=None, *, backend="b200"):
    import baybridge_b200 as cute

    @cute.kernel
    def backward(grad_out, x, mean, rstd, weight, grad_x, grad_weight, grad_bias, grad_resid):
        cute.layernorm_backward(grad_out, x, mean, rstd, weight, grad_x, grad_weight, grad_bias, grad_resid=grad_resid)

    arguments = (grad_out, x, mean, rstd, weight, grad_x, grad_weight, grad_bias, grad_resid)
    artifact = cute.compile(backward, *arguments, backend=backend)
    return lambda stream=None: artifact(*arguments, stream=stream)


SHAPES = [  # dtype, weight dtype, shape, residual, bias
    ("f32", "f32", (1,), False, True), ("bf16", "bf16", (7,), True, True), ("f32", "f32", (1, 1), False, False), ("bf16", "f32", (3, 2), True, True),
    ("f16", "f16", (5, 8), False, True), ("bf16", "bf16", (9, 64), True, False), ("bf16", "f32", (2, 3, 256), False, True),
    ("f32", "f32", (33, 128), True, True), ("f16", "f32", (70, 255), True, True), ("bf16", "bf16", (17, 512), False, False),
    ("bf16", "bf16", (4, 5, 520), True, True), ("f32", "f32", (6, 1000), False, True), ("f16", "f16", (300, 1001), False, True),
    ("bf16", "f32", (19, 1024), True, True), ("bf16", "bf16", (1000, 2048), False, True), ("f32", "f32", (11, 2052), True, True),
    ("bf16", "f32", (13, 4096), True, True), ("f32", "f32", (9, 4096), False, True), ("bf16", "bf16", (700, 8192), True, True),
    ("f32", "f32", (5, 8192), True, False), ("f16", "f16", (3, 8200), False, True), ("bf16", "f32", (4, 16384), False, True),
    ("f32", "f32", (3, 16384), True, True), ("f16", "f32", (2, 32768), True, True), ("bf16", "bf16", (2, 32767), False, True),
    ("f32", "f32", (2, 16383), True, True), ("bf16", "f32", (40000, 24), False, True), ("bf16", "f32", (701, 4000), False, True),
]


@pytest.mark.parametrize("dtype,weight_dtype,shape,residual,bias", SHAPES)
def test_forward(dtype, weight_dtype, shape, residual, bias):
    torch = _torch()
    hidden, rows = shape[-1], shape[:-1] or (1,)
    x, w = _normal(shape, dtype, 1, 1.5, 0.5), _normal((hidden,), weight_dtype, 2, 0.1, 1.0)
    b, r = _normal((hidden,), weight_dtype, 3, 0.1) if bias else None, _normal(shape, dtype, 4) if residual else None
    out, mean, rstd = torch.full_like(x, float("nan")), torch.full(rows, float("nan"), device="cuda"), torch.full(rows, float("nan"), device="cuda")
    resid = torch.full_like(x, float("nan")) if residual else None
    _forward(x, out, mean, rstd, w, b, r, resid)()
    expected, s, e_mean, e_rstd = reference.layernorm_forward(x, r, w, b, 1e-5)
    off_out, off_mean, off_rstd = reference.layernorm_forward_errors(x, r, w, b, 1e-5)
    within(out, expected, dtype, off_out)
    within(mean, e_mean.reshape(rows), "f32", off_mean.reshape(rows))
    within(rstd, e_rstd.reshape(rows), "f32", off_rstd.reshape(rows))
    if residual:
        within(resid, s, dtype, U * s.abs())


@pytest.mark.parametrize("dtype,weight_dtype,shape,residual,bias", SHAPES)
def test_backward(dtype, weight_dtype, shape, residual, bias):
    torch = _torch()
    hidden = shape[-1]
    x, w = _normal(shape, dtype, 5, 1.5, 0.5), _normal((hidden,), weight_dtype, 6, 0.1, 1.0)
    d, r = _normal(shape, dtype, 7), _normal(shape, dtype, 8) if residual else None
    _, _, mean, rstd = reference.layernorm_forward(x, None, w, None, 1e-5)
    mean, rstd = mean.float().reshape(shape[:-1] or (1,)), rstd.float().reshape(shape[:-1] or (1,))
    grad_x = torch.full_like(x, float("nan"))
    grad_w, grad_b = torch.full_like(w, float("nan")), torch.full_like(w, float("nan")) if bias else None
    run = _backward(d, x, mean, rstd, w, grad_x, grad_w, grad_b, r)
    run()
    flat = (lambda t: t.reshape(-1, hidden) if t is not None else None)
    arguments = (flat(d), flat(x), mean.reshape(-1), rstd.reshape(-1), w, flat(r))
    e_x, e_w, e_b, _ = reference.layernorm_backward(*arguments)
    off_x, off_w, off_b = reference.layernorm_backward_errors(*arguments)
    within(flat(grad_x), e_x, dtype, off_x)
    within(grad_w, e_w, weight_dtype, off_w)
    if bias:
        within(grad_b, e_b, weight_dtype, off_b)
    first = grad_x.clone(), grad_w.clone(), grad_b.clone() if bias else None
    for _ in range(3):  # the same call gives the same bits
        grad_x.fill_(0), grad_w.fill_(0)
        run()
        assert torch.equal(grad_x, first[0]) and torch.equal(grad_w, first[1]) and (not bias or torch.equal(grad_b, first[2]))


@pytest.mark.parametrize("rows,hidden,offset", [(6, 64, 1), (5, 96, 3), (4, 33, 1), (3, 1024, 5)])
def test_unaligned_tensors_and_their_neighbours(rows, hidden, offset):
    torch = _torch()

    def view(fill=None, seed=0):
        flat = torch.full((rows * hidden + 16,), 7.0, device="cuda", dtype=torch.bfloat16)
        inner = flat[offset:offset + rows * hidden].view(rows, hidden)
        if fill is None:
            inner.copy_(_normal((rows, hidden), "bf16", seed))
        return flat, inner

    (_, x), (_, d), (out_flat, out), (grad_flat, grad_x) = view(seed=1), view(seed=2), view(7.0), view(7.0)
    w, b = _normal((hidden,), "bf16", 3, 0.1, 1.0), _normal((hidden,), "bf16", 4)
    mean, rstd = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    _forward(x, out, mean, rstd, w, b)()
    within(out, reference.layernorm_forward(x, None, w, b, 1e-5)[0], "bf16", reference.layernorm_forward_errors(x, None, w, b, 1e-5)[0])
    grad_w, grad_b = torch.empty_like(w), torch.empty_like(b)
    _backward(d, x, mean, rstd, w, grad_x, grad_w, grad_b)()
    expected, errors = reference.layernorm_backward(d, x, mean, rstd, w, None), reference.layernorm_backward_errors(d, x, mean, rstd, w, None)
    within(grad_x, expected[0], "bf16", errors[0])
    within(grad_w, expected[1], "bf16", errors[1])
    within(grad_b, expected[2], "bf16", errors[2])
    for flat in (out_flat, grad_flat):
        assert bool((flat[:offset] == 7).all()) and bool((flat[offset + rows * hidden:] == 7).all())


def test_residual_stream_updated_in_place():
    torch = _torch()
    for hidden in (512, 77, 8192):
        x, stream = _normal((6, hidden), "bf16", 9), _normal((6, hidden), "bf16", 10)
        w = _normal((hidden,), "bf16", 11)
        out, mean, rstd = torch.empty_like(x), torch.empty(6, device="cuda"), torch.empty(6, device="cuda")
        expected, s, _, _ = reference.layernorm_forward(x, stream, w, None, 1e-5)
        errors = reference.layernorm_forward_errors(x, stream, w, None, 1e-5)
        _forward(x, out, mean, rstd, w, None, stream, stream)()
        within(out, expected, "bf16", errors[0])
        within(stream, s, "bf16", U * s.abs())


def test_a_large_mean_and_a_constant_row():
    """Statistics of rows around 1000, of a row without any variance, and of one with an infinity."""
    torch = _torch()
    x = _normal((4, 1024), "f32", 12, 1e-2, 1000.0)
    x[1] = 3.0
    x[2, 5] = float("inf")
    w = torch.ones(1024, device="cuda")
    out, mean, rstd = torch.empty_like(x), torch.empty(4, device="cuda"), torch.empty(4, device="cuda")
    _forward(x, out, mean, rstd, w)()
    rows = [0, 1, 3]
    expected, _, e_mean, e_rstd = reference.layernorm_forward(x[rows], None, w, None, 1e-5)
    errors = reference.layernorm_forward_errors(x[rows], None, w, None, 1e-5)
    within(out[rows], expected, "f32", errors[0])
    within(mean[rows], e_mean, "f32", errors[1])
    within(rstd[rows], e_rstd, "f32", errors[2])
    assert bool(out[1].eq(0).all()) and abs(float(rstd[1]) - 1e-5 ** -0.5) <= 1e-4
    assert bool(mean[2].isinf()) and bool(out[2].isnan().all())


@pytest.mark.parametrize("hidden", [48, 51])
def test_gradients_agree_with_differences_of_the_forward_pass(hidden):
    """Central differences of sum(out * d) in f64 from f32 outputs: the outputs' rounding, 2 u |out| each, divided by the
    step, and the step's cube times the third derivative bound how far they may be off."""
    torch = _torch()
    rows, step = 3, 2.0 ** -6
    x, w, b, d = (_normal(s, "f32", 20 + i) for i, s in enumerate([(rows, hidden), (hidden,), (hidden,), (rows, hidden)]))
    out, mean, rstd = torch.empty_like(x), torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")

    def loss(x, w, b):
        _forward(x, out, mean, rstd, w, b)()
        return float((out.double() * d.double()).sum())

    loss(x, w, b)
    grad_x, grad_w, grad_b = torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
    _backward(d, x, mean, rstd, w, grad_x, grad_w, grad_b)()
    noise = 64 * U * float((out.double() * d.double()).abs().sum()) / step
    for at in ((0, 0), (1, hidden - 1), (2, 17)):
        up, down = x.clone(), x.clone()
        up[at] += step
        down[at] -= step
        width = float(up[at].double() - down[at].double())
        assert abs((loss(up, w, b) - loss(down, w, b)) / width - float(grad_x[at])) <= noise + 64 * step * step
    for column in (0, hidden - 1):
        for tensor, grad, place in ((w, grad_w, 1), (b, grad_b, 2)):
            arguments = [[x, w, b], [x, w, b]]
            for sign, which in ((1, 0), (-1, 1)):
                moved = tensor.clone()
                moved[column] += sign * step
                arguments[which][place] = moved
            width = float(arguments[0][place][column].double() - arguments[1][place][column].double())
            assert abs((loss(*arguments[0]) - loss(*arguments[1])) / width - float(grad[column])) <= noise


def test_streams_and_recorded_launches():
    torch = _torch()
    import baybridge_b200 as cute
    from baybridge_b200.launch_graph import LaunchGraph

    backend = cute.B200Backend(synchronize=False)
    calls = []
    for index, (rows, hidden) in enumerate([(700, 1024), (65, 77), (300, 8192)]):
        x, d, w = _normal((rows, hidden), "bf16", 30 + index), _normal((rows, hidden), "bf16", 40 + index), _normal((hidden,), "f32", 50 + index)
        _, _, mean, rstd = reference.layernorm_forward(x, None, w, None, 1e-5)
        mean, rstd = mean.float(), rstd.float()
        outputs = torch.empty_like(x), torch.empty_like(w), torch.empty_like(w)
        handles = [cute.from_dlpack(t) for t in (d, x, mean, rstd, w, *outputs)]
        calls.append((_backward(*handles, backend=backend), (d, x, mean, rstd, w, None), outputs))

    def check():
        for _, arguments, outputs in calls:
            for got, expected, error, kind in zip(outputs, reference.layernorm_backward(*arguments), reference.layernorm_backward_errors(*arguments),
                                                  ("bf16", "f32", "f32")):
                within(got, expected, kind, error)
                got.fill_(float("nan"))

    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    for _ in range(10):
        for (run, _, _), stream in zip(calls, streams):
            run(stream)
    torch.cuda.synchronize()
    check()
    graph = LaunchGraph()
    with graph.record() as stream:
        for run, _, _ in calls:
            run(stream)
    for _, arguments, _ in calls:
        arguments[0].mul_(-0.5)
    torch.cuda.synchronize()
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    check()
    graph.close()


def test_c_abi_refusals():
    torch = _torch()
    from baybridge_b200 import CudaDriverError
    from baybridge_b200.backend import native

    x, w, stat = _normal((4, 64), "f32", 60), _normal((64,), "f32", 61), torch.empty(4, device="cuda")
    other, third = torch.empty_like(x), torch.empty(4, device="cuda")

    def forward(out=other, mean=stat, rstd=third, residual=None, out_resid=None, rows=4, hidden=64, weight_dtype=0):
        native.call("bb200_layernorm_forward", 0, weight_dtype, void_p(x), residual and void_p(residual), void_p(w), None, void_p(out),
                    out_resid and void_p(out_resid), void_p(mean), void_p(rstd), rows, hidden, 1e-5, current_stream())

    for arguments, status in (({"out": x}, -1), ({"rstd": stat}, -1), ({"rows": 0}, -1), ({"hidden": 16388}, -2), ({"weight_dtype": 1}, -1)):
        with pytest.raises(CudaDriverError) as info:
            forward(**arguments)
        assert info.value.status == status
    with pytest.raises(CudaDriverError, match="go together"):
        native.call("bb200_layernorm_forward", 0, 0, void_p(x), void_p(x), void_p(w), None, void_p(other), None, void_p(stat), void_p(third), 4, 64,
                    1e-5, current_stream())
    with pytest.raises(CudaDriverError, match="shares memory"):
        native.call("bb200_layernorm_backward", 0, 0, void_p(x), void_p(other), void_p(stat), void_p(third), void_p(w), None, void_p(x), void_p(w),
                    None, 4, 64, current_stream())
