"""Embedding lookup and its gradient on the GPU, through compile(..., backend="b200") and the C ABI, against 64 bits."""
from __future__ import annotations

import pytest
from gpu_util import TORCH_DTYPE, current_stream, void_p
from training_reference import U, within

pytestmark = pytest.mark.gpu


def _torch():
    import torch

    return torch


def _dtype(name):
    return getattr(_torch(), TORCH_DTYPE[name])


def _rows(shape, dtype, seed):
    torch = _torch()
    return torch.randn(shape, device="cuda", generator=torch.Generator("cuda").manual_seed(seed)).to(_dtype(dtype))


def _tokens(count, vocabulary, dtype, seed, kind="zipf"):
    torch = _torch()
    generator = torch.Generator("cuda").manual_seed(seed)
    u = torch.rand(count, device="cuda", dtype=torch.float64, generator=generator)
    if kind == "zipf":
        ids = ((vocabulary + 1) ** u).long() - 1
    elif kind == "same":
        ids = torch.full((count,), vocabulary // 2, device="cuda")
    elif kind == "distinct":
        ids = torch.randperm(max(count, vocabulary), device="cuda", generator=generator)[:count] % vocabulary
    else:
        ids = (u * vocabulary).long()
    return ids.clamp(0, vocabulary - 1).to(_dtype(dtype))


def _lookup(tokens, table, out, **options):
    import baybridge_b200 as cute

    @cute.kernel
    def lookup(tokens: cute.Tensor, table: cute.Tensor, out: cute.Tensor):
        cute.embedding(tokens, table, out, **options)

    return cute.compile(lookup, tokens, table, out, backend="b200")


def _gradient(grad_out, tokens, grad_table, **options):
    import baybridge_b200 as cute

    @cute.kernel
    def gradient(grad_out: cute.Tensor, tokens: cute.Tensor, grad_table: cute.Tensor):
        cute.embedding_backward(grad_out, tokens, grad_table, **options)

    return cute.compile(gradient, grad_out, tokens, grad_table, backend="b200")


def _expected_gradient(grad_out, tokens, grad_table, scale, padding, accumulate):
    """The sums in f64 and the error bound: a run of n rows is at most n deep, the product and the addition two more."""
    torch = _torch()
    vocabulary, hidden = grad_table.shape
    ids, rows = tokens.reshape(-1).long(), grad_out.reshape(-1, hidden).double()
    keep = (ids >= 0) & (ids < vocabulary)
    if padding is not None:
        keep &= ids != padding
    ids, rows = ids[keep], rows[keep]
    total = torch.zeros(vocabulary, hidden, device="cuda", dtype=torch.float64).index_add_(0, ids, rows)
    sizes = torch.zeros_like(total).index_add_(0, ids, rows.abs())
    runs = torch.bincount(ids, minlength=vocabulary).double()[:, None]
    error = (runs + 2) * U * sizes * abs(scale)
    if accumulate:
        old = grad_table.double()
        return total * scale + old, error + 2 * U * old.abs() * (runs > 0), runs[:, 0] > 0
    return total * scale, error, runs[:, 0] > 0


@pytest.mark.parametrize("table_dtype,out_dtype,token_dtype", [("bf16", "bf16", "i32"), ("f32", "f32", "i64"), ("f32", "bf16", "i32"),
                                                              ("f16", "f32", "i64"), ("f16", "f16", "i32"), ("bf16", "f16", "i64")])
@pytest.mark.parametrize("shape,vocabulary,hidden", [((1,), 1, 1), ((5,), 7, 8), ((3, 17), 50, 129), ((257,), 1000, 512), ((2, 2, 33), 300, 4104),
                                                    ((1000,), 31, 64), ((4,), 9, 8192)])
def test_lookup(table_dtype, out_dtype, token_dtype, shape, vocabulary, hidden):
    torch = _torch()
    table = _rows((vocabulary, hidden), table_dtype, 1)
    tokens = _tokens(int(torch.tensor(shape).prod()), vocabulary, token_dtype, 2).reshape(shape)
    out = torch.full((*shape, hidden), float("nan"), device="cuda", dtype=_dtype(out_dtype))
    _lookup(tokens, table, out, scale=2.5)(tokens, table, out)
    expected = table.double()[tokens.long()] * 2.5
    within(out, expected, out_dtype, U * expected.abs())


def test_lookup_without_scale_is_a_copy():
    torch = _torch()
    table, tokens = _rows((100, 96), "bf16", 3), _tokens(77, 100, "i32", 4)
    out = torch.empty(77, 96, device="cuda", dtype=torch.bfloat16)
    _lookup(tokens, table, out)(tokens, table, out)
    assert torch.equal(out, table[tokens.long()])


@pytest.mark.parametrize("offset", [1, 3])
def test_lookup_of_unaligned_tensors_leaves_their_neighbours_alone(offset):
    torch = _torch()
    storage = _rows((40 * 64 + 16,), "bf16", 5)
    table = storage[offset:offset + 40 * 64].view(40, 64)
    kept = torch.full((20 * 64 + 16,), 7.0, device="cuda", dtype=torch.bfloat16)
    out = kept[offset:offset + 20 * 64].view(20, 64)
    tokens = _tokens(20, 40, "i64", 6)
    _lookup(tokens, table, out)(tokens, table, out)
    assert torch.equal(out, table[tokens.long()])
    assert bool((kept[:offset] == 7).all()) and bool((kept[offset + 20 * 64:] == 7).all())


def test_rows_past_32_bits_of_offset():
    """The last rows of a table of more than 2^32 elements."""
    torch = _torch()
    vocabulary, hidden = 1 << 20, 4104
    table = torch.zeros(vocabulary, hidden, device="cuda", dtype=torch.bfloat16)
    table[-2:] = torch.arange(2, device="cuda", dtype=torch.bfloat16)[:, None] + 1
    tokens = torch.tensor([vocabulary - 1, 0, vocabulary - 2], device="cuda")
    out = torch.empty(3, hidden, device="cuda", dtype=torch.bfloat16)
    _lookup(tokens, table, out)(tokens, table, out)
    assert torch.equal(out[:, 0].float().cpu(), torch.tensor([2.0, 0.0, 1.0]))
    grad = torch.ones(3, hidden, device="cuda", dtype=torch.bfloat16)
    _gradient(grad, tokens, table, accumulate=True)(grad, tokens, table)
    assert torch.equal(table[[0, 1, vocabulary - 2, vocabulary - 1], -1].float().cpu(), torch.tensor([1.0, 0.0, 2.0, 3.0]))


@pytest.mark.parametrize("bad", [-1, 50, 2 ** 31 - 1, 2 ** 40])
def test_a_token_outside_the_table_reads_as_zeros_and_raises(bad):
    torch = _torch()
    table, tokens = _rows((50, 64), "f32", 7), _tokens(9, 50, "i64", 8)
    tokens[4] = bad
    out, grad = torch.full((9, 64), 3.0, device="cuda"), _rows((9, 64), "f32", 9)
    grad_table = torch.full((50, 64), 3.0, device="cuda")
    with pytest.raises(RuntimeError, match="311.*outside the table"):
        _lookup(tokens, table, out)(tokens, table, out)
    assert not out[4].any()
    good = [i for i in range(9) if i != 4]
    assert torch.equal(out[good], table[tokens[good]])
    expected, error, _ = _expected_gradient(grad, tokens, grad_table, 1.0, None, False)
    with pytest.raises(RuntimeError, match="311.*outside the table"):
        _gradient(grad, tokens, grad_table)(grad, tokens, grad_table)
    within(grad_table, expected, "f32", error)
    tokens[4] = 0
    _lookup(tokens, table, out)(tokens, table, out)  # the status word was cleared


GRADIENT_SHAPES = [
    # count, vocabulary, hidden, kind
    (1, 1, 1, "even"), (1, 1000, 8, "even"), (3, 2, 7, "even"), (31, 5, 64, "zipf"), (32, 40, 129, "zipf"), (33, 1, 520, "same"),
    (257, 300, 8, "zipf"), (1000, 2000, 96, "distinct"), (4096, 512, 64, "zipf"), (4097, 513, 40, "zipf"), (5000, 131072, 16, "even"),
    (8192, 100, 33, "same"), (16384, 700, 12, "zipf"), (20000, 50257, 24, "zipf"), (32769, 131072, 16, "zipf"), (65536, 999, 8, "even"),
    (65537, 999, 8, "zipf"), (3000, 40, 1032, "zipf"), (50000, 17, 264, "zipf"), (70000, 1 << 20, 8, "zipf"), (70000, 3, 17, "even"), (600000, 1000, 8, "zipf"),
    # up to 1024 tokens: runs of one token on both sides of 16, rows of several column tiles, many rows that no token names
    (1024, 3, 520, "even"), (1023, 1, 1032, "same"), (1024, 64, 264, "even"), (300, 3, 261, "even"), (1024, 1024, 136, "distinct"),
    (16, 1, 40, "same"), (17, 1, 40, "same"), (1025, 7, 40, "even"), (9, 70001, 36, "even"), (1000, 300000, 3, "zipf"),
    # as few tokens, of many columns: sorted all the same
    (900, 50, 1061, "zipf"), (30, 4, 40000, "even"), (1, 3, 80000, "even"),
]


@pytest.mark.parametrize("count,vocabulary,hidden,kind", GRADIENT_SHAPES)
@pytest.mark.parametrize("accumulate", [False, True])
def test_gradient(count, vocabulary, hidden, kind, accumulate):
    torch = _torch()
    tokens = _tokens(count, vocabulary, "i32" if count % 2 else "i64", 11, kind)
    grad = _rows((count, hidden), "f32", 12)
    guarded = torch.full((vocabulary * hidden + 64,), 5.0, device="cuda")
    grad_table = guarded[:vocabulary * hidden].view(vocabulary, hidden)
    if accumulate:
        grad_table.copy_(_rows((vocabulary, hidden), "f32", 13))
    before = grad_table.clone()
    expected, error, named = _expected_gradient(grad, tokens, before, 0.5, None, accumulate)
    artifact = _gradient(grad, tokens, grad_table, scale=0.5, accumulate=accumulate)
    artifact(grad, tokens, grad_table)
    within(grad_table, expected, "f32", error)
    assert torch.equal(grad_table[~named], before[~named] if accumulate else torch.zeros_like(before[~named]))
    assert bool((guarded[vocabulary * hidden:] == 5).all())
    first = grad_table.clone()
    for _ in range(3):  # the same call gives the same bits
        grad_table.copy_(before)
        artifact(grad, tokens, grad_table)
        assert torch.equal(grad_table, first)


@pytest.mark.parametrize("grad_dtype,table_dtype", [("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f32", "bf16"), ("f16", "f32"), ("bf16", "f16")])
@pytest.mark.parametrize("hidden", [72, 75])
def test_gradient_dtypes_padding_and_token_shape(grad_dtype, table_dtype, hidden):
    torch = _torch()
    tokens = _tokens(6 * 50, 97, "i64", 14).reshape(6, 50)
    tokens[:, 40:] = 3
    grad, table = _rows((6, 50, hidden), grad_dtype, 15), _rows((97, hidden), table_dtype, 16)
    for accumulate in (False, True):
        target = table.clone()
        expected, error, named = _expected_gradient(grad, tokens, target, 1.5, 3, accumulate)
        _gradient(grad, tokens, target, scale=1.5, padding_token=3, accumulate=accumulate)(grad, tokens, target)
        within(target, expected, table_dtype, error)
        assert not bool(named[3])
        assert torch.equal(target[3], table[3] if accumulate else torch.zeros_like(table[3]))


def test_gradient_when_every_token_is_padding():
    torch = _torch()
    for count in (5, 9000):
        tokens = torch.full((count,), 2, device="cuda", dtype=torch.int32)
        grad, table = _rows((count, 16), "f32", 17), _rows((4, 16), "f32", 18)
        kept = table.clone()
        _gradient(grad, tokens, table, padding_token=2, accumulate=True)(grad, tokens, table)
        assert torch.equal(table, kept)
        _gradient(grad, tokens, table, padding_token=2)(grad, tokens, table)
        assert not table.any()


def test_infinite_and_nan_gradients_stay_in_their_rows():
    torch = _torch()
    tokens = torch.tensor([1, 2, 3, 1, 2, 3] * 20, device="cuda")
    grad = _rows((120, 32), "bf16", 19)
    grad[0, 5], grad[1, 6] = float("inf"), float("nan")
    table = torch.zeros(5, 32, device="cuda")
    _gradient(grad, tokens, table)(grad, tokens, table)
    assert bool(table[1, 5].isinf()) and bool(table[2, 6].isnan())
    table[1, 5] = table[2, 6] = 0
    assert bool(table.isfinite().all())


@pytest.mark.parametrize("offset", [4, 8])
@pytest.mark.parametrize("grad_dtype,table_dtype", [("f32", "f32"), ("bf16", "f32"), ("f32", "bf16")])
def test_tensors_aligned_to_16_bytes_but_not_to_32(offset, grad_dtype, table_dtype):
    torch = _torch()
    count, vocabulary, hidden = 700, 60, 48
    tokens = _tokens(count, vocabulary, "i32", 90)

    def shifted(shape, dtype, seed):
        flat = torch.full((shape[0] * shape[1] + 32,), 9.0, device="cuda", dtype=_dtype(dtype))
        start = offset if dtype == "f32" else 2 * offset
        view = flat[start:start + shape[0] * shape[1]].view(shape)
        view.copy_(_rows(shape, dtype, seed))
        return flat, start, view

    _, _, grad = shifted((count, hidden), grad_dtype, 91)
    flat, start, table = shifted((vocabulary, hidden), table_dtype, 92)
    for accumulate in (True, False):
        expected, error, _ = _expected_gradient(grad, tokens, table, 1.0, None, accumulate)
        _gradient(grad, tokens, table, accumulate=accumulate)(grad, tokens, table)
        within(table, expected, table_dtype, error)
    out_flat, out_start, out = shifted((count, hidden), grad_dtype, 93)
    _lookup(tokens, table, out)(tokens, table, out)
    within(out, table.double()[tokens.long()], grad_dtype, 0 * table.double()[tokens.long()])
    for storage, first, view in ((flat, start, table), (out_flat, out_start, out)):
        assert bool((storage[:first] == 9).all()) and bool((storage[first + view.numel():] == 9).all())


def test_a_single_token_without_an_axis():
    torch = _torch()
    table, token = _rows((30, 40), "f32", 95), torch.tensor(7, device="cuda")
    out, grad_table = torch.empty(40, device="cuda"), torch.empty(30, 40, device="cuda")
    _lookup(token, table, out, scale=2.0)(token, table, out)
    assert torch.equal(out, table[7] * 2)
    _gradient(out, token, grad_table)(out, token, grad_table)
    assert torch.equal(grad_table[7], out) and not grad_table[:7].any() and not grad_table[8:].any()


def test_gradient_inside_a_torch_graph():
    """Captured by another program's graph: the workspace becomes the graph's own."""
    torch = _torch()
    import baybridge_b200 as cute

    tokens, grad, table = _tokens(3000, 400, "i32", 96), _rows((3000, 24), "f32", 97), torch.zeros(400, 24, device="cuda")

    @cute.kernel
    def gradient(grad_out: cute.Tensor, tokens: cute.Tensor, grad_table: cute.Tensor):
        cute.embedding_backward(grad_out, tokens, grad_table)

    handles = [cute.from_dlpack(t) for t in (grad, tokens, table)]
    artifact = cute.compile(gradient, *handles, backend=cute.B200Backend(synchronize=False))
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        artifact(*handles, stream=side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        artifact(*handles, stream=side)
    for seed in (98, 99):
        grad.copy_(_rows((3000, 24), "f32", seed))
        graph.replay()
        graph.replay()
        torch.cuda.synchronize()
        expected, error, _ = _expected_gradient(grad, tokens, table, 1.0, None, False)
        within(table, expected, "f32", error)


def test_calls_on_two_streams_do_not_share_a_workspace():
    torch = _torch()
    import baybridge_b200 as cute

    @cute.kernel
    def gradient(grad_out: cute.Tensor, tokens: cute.Tensor, grad_table: cute.Tensor):
        cute.embedding_backward(grad_out, tokens, grad_table)

    cases, streams = [], [torch.cuda.Stream() for _ in range(3)]
    for index in range(3):
        tokens, grad = _tokens(30000, 777, "i32", 20 + index), _rows((30000, 64), "bf16", 30 + index)
        table = torch.empty(777, 64, device="cuda")
        cases.append((grad, tokens, table, _expected_gradient(grad, tokens, table, 1.0, None, False)))
    artifact = cute.compile(gradient, *cases[0][:3], backend=cute.B200Backend(synchronize=False))
    torch.cuda.synchronize()
    for _ in range(20):
        for (grad, tokens, table, _), stream in zip(cases, streams):
            artifact(grad, tokens, table, stream=stream)
    torch.cuda.synchronize()
    for _, _, table, (expected, error, _) in cases:
        within(table, expected, "f32", error)


def test_recorded_gradients_replay_with_the_buffers_contents():
    torch = _torch()
    import baybridge_b200 as cute
    from baybridge_b200.launch_graph import LaunchGraph

    cases = []
    for count in (300, 9000):
        tokens, grad, table = _tokens(count, 500, "i32", 41), _rows((count, 40), "f32", 42), torch.empty(500, 40, device="cuda")
        cases.append((_gradient(grad, tokens, table), grad, tokens, table))
    graphs = [LaunchGraph(), LaunchGraph()]
    for graph in graphs:  # two graphs of the same launches: each has its own workspace
        with graph.record() as stream:
            for artifact, grad, tokens, table in cases:
                artifact(cute.from_dlpack(grad), cute.from_dlpack(tokens), cute.from_dlpack(table), stream=stream)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for round_ in range(3):
        for _, grad, tokens, _ in cases:
            grad.copy_(_rows(tuple(grad.shape), "f32", 50 + round_))
            tokens.copy_(_tokens(tokens.numel(), 500, "i32", 60 + round_))
        torch.cuda.synchronize()
        graphs[round_ % 2].replay(stream=streams[round_ % 2])
        torch.cuda.synchronize()
        for _, grad, tokens, table in cases:
            expected, error, _ = _expected_gradient(grad, tokens, table, 1.0, None, False)
            within(table, expected, "f32", error)
    for graph in graphs:
        graph.close()


def test_gradient_agrees_with_differences_of_the_lookup():
    """sum(lookup(table) * w) is linear in the table: its difference quotient is the gradient of w, whatever the step."""
    torch = _torch()
    tokens, table = _tokens(60, 12, "i32", 70), _rows((12, 20), "f32", 71)
    w = _rows((60, 20), "f32", 72)
    grad_table = torch.empty_like(table)
    _gradient(w, tokens, grad_table, scale=3.0)(w, tokens, grad_table)
    out = torch.empty(60, 20, device="cuda")
    artifact = _lookup(tokens, table, out, scale=3.0)

    def loss(t):
        artifact(tokens, t, out)
        return float((out.double() * w.double()).sum())

    base = loss(table)
    for row, column in ((0, 0), (3, 19), (11, 7)):
        moved = table.clone()
        moved[row, column] = 0.0
        step = float(table[row, column])
        size = float((table.double().abs()[tokens.long()] * 3 * w.double().abs()).sum())
        # both losses are exact sums of products rounded once each: off by at most u times their magnitudes
        assert abs((base - loss(moved)) - step * float(grad_table[row, column])) <= 4 * U * size


def test_c_abi_refuses_shared_memory_and_misaligned_tensors():
    torch = _torch()
    from baybridge_b200 import CudaDriverError
    from baybridge_b200.backend import native

    table, tokens = _rows((16, 32), "f32", 80), _tokens(4, 16, "i32", 81)
    for call in (
        lambda: native.call("bb200_embedding", 0, 0, 3, void_p(tokens), void_p(table), void_p(table), 4, 16, 32, 1.0, current_stream()),
        lambda: native.call("bb200_embedding_backward", 0, 0, 3, void_p(table), void_p(tokens), void_p(table), 4, 16, 32, 1.0, -1, 0, current_stream()),
    ):
        with pytest.raises(CudaDriverError, match="shares memory") as info:
            call()
        assert info.value.status == -1
    out = torch.empty(4 * 32 + 4, device="cuda")
    with pytest.raises(CudaDriverError) as info:
        import ctypes

        native.call("bb200_embedding", 0, 0, 3, void_p(tokens), void_p(table), ctypes.c_void_p(out.data_ptr() + 2), 4, 16, 32, 1.0, current_stream())
    assert info.value.status == -3
