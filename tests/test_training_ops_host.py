"""The training operators without a GPU: what the DSL traces and refuses, the plans, argument checks of the C ABI."""
from __future__ import annotations

import ctypes

import pytest
from test_fake_driver import ELEMENTWISE_CHILD, calls, fake_driver, run_child  # noqa: F401 - a fixture among them
from test_host_surface import FakeCudaTensor

import baybridge_b200 as cute
from baybridge_b200.backend import native
from baybridge_b200.backend.matcher import match


def tensor(shape, dtype="float32", ptr=4096, **options):
    return FakeCudaTensor(shape, dtype, ptr, **options)


def ir_of(body, *arguments, tmp_path):
    return cute.compile(cute.kernel(body), *arguments, backend="portable", cache_dir=tmp_path).ir


def test_embedding_plans(tmp_path, zoo):
    tokens, table, out = tensor((2, 5), "int64"), tensor((11, 24), "float32"), tensor((2, 5, 24), "bfloat16")
    ir = cute.compile(zoo.make_embedding(3.0), tokens, table, out, backend="portable", cache_dir=tmp_path).ir
    plan = match(ir)
    assert (plan.kind, plan.count, plan.vocabulary, plan.hidden, plan.scale) == ("embedding", 10, 11, 24, 3.0)
    assert (plan.token_dtype, plan.table_dtype, plan.out_dtype) == ("i64", "f32", "bf16")
    ir = cute.compile(zoo.make_embedding_backward(2.0, 7, True), out, tokens, table, backend="portable", cache_dir=tmp_path).ir
    plan = match(ir)
    assert (plan.kind, plan.padding_token, plan.accumulate, plan.scale) == ("embedding_backward", 7, True, 2.0)
    assert match(cute.compile(zoo.make_embedding_backward(), out, tokens, table, backend="portable", cache_dir=tmp_path).ir).padding_token == -1


def test_plans_survive_serialisation(tmp_path, zoo):
    x, stat, w = tensor((4, 16), "float16"), tensor((4,)), tensor((16,))
    for kernel, arguments in ((zoo.layernorm_forward, (x, x, stat, stat, w, w)), (zoo.layernorm_backward, (x, x, stat, stat, w, x, w, w))):
        ir = cute.compile(kernel, *arguments, backend="portable", cache_dir=tmp_path).ir
        assert match(cute.PortableKernelIR.from_dict(ir.to_dict())) == match(ir)


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("residual", [False, True])
def test_norm_plans_find_their_optional_operands(bias, residual, tmp_path):
    x, stat, w = (lambda: tensor((3, 4, 40), "bfloat16")), (lambda: tensor((3, 4))), (lambda: tensor((40,)))

    def forward(x, out, mean, rstd, weight, bias, residual, out_resid):
        cute.layernorm_forward(x, out, mean, rstd, weight, bias, residual=residual, out_resid=out_resid, epsilon=1e-6)

    plan = match(ir_of(forward, x(), x(), stat(), stat(), w(), w() if bias else None, *((x(), x()) if residual else (None, None)), tmp_path=tmp_path))
    rest = 5 + bias
    assert (plan.x, plan.out, plan.mean, plan.rstd, plan.weight) == (0, 1, 2, 3, 4)
    assert plan.bias == (5 if bias else None) and (plan.residual, plan.out_resid) == ((rest, rest + 1) if residual else (None, None))
    assert (plan.rows, plan.hidden, plan.dtype, plan.weight_dtype, plan.epsilon) == (12, 40, "bf16", "f32", 1e-6)

    def backward(grad_out, x, mean, rstd, weight, grad_x, grad_weight, grad_bias, grad_resid):
        cute.layernorm_backward(grad_out, x, mean, rstd, weight, grad_x, grad_weight, grad_bias, grad_resid=grad_resid)

    plan = match(ir_of(backward, x(), x(), stat(), stat(), w(), x(), w(), w() if bias else None, x() if residual else None, tmp_path=tmp_path))
    assert (plan.grad_out, plan.x, plan.mean, plan.rstd, plan.weight, plan.grad_x, plan.grad_weight) == tuple(range(7))
    assert plan.grad_bias == (7 if bias else None) and plan.grad_resid == (7 + bias if residual else None)


def test_adamw_plan(tmp_path):
    shapes = [(3, 5), (7,), (1,)]
    lists = [[tensor(s, dtype) for s in shapes] for dtype in ("bfloat16", "float32", "float32", "float32", "float32")]

    def step(params, grads, exp_avgs, exp_avg_sqs, masters, schedule):
        cute.adamw(params, grads, exp_avgs, exp_avg_sqs, schedule, masters=masters, weight_decay=[0.1, 0.0, 0.2], betas=(0.8, 0.95), epsilon=1e-6)

    plan = match(ir_of(step, *lists, tensor((3,)), tmp_path=tmp_path))
    assert (plan.params, plan.grads, plan.exp_avgs, plan.exp_avg_sqs, plan.masters) == ((0, 1, 2), (3, 4, 5), (6, 7, 8), (9, 10, 11), (12, 13, 14))
    assert plan.schedule == 15 and plan.numels == (15, 7, 1) and plan.weight_decay == (0.1, 0.0, 0.2)
    assert plan.param_dtypes == ("bf16",) * 3 and plan.grad_dtypes == ("f32",) * 3 and (plan.beta1, plan.beta2, plan.epsilon) == (0.8, 0.95, 1e-6)


def test_the_dsl_refuses_what_the_operators_do_not_take(tmp_path):
    ids, table, rows, stat, w = tensor((4,), "int32"), tensor((9, 16)), tensor((4, 16)), tensor((4,)), tensor((16,))

    def refused(body, *arguments, match, error=ValueError):
        with pytest.raises(error, match=match):
            ir_of(body, *arguments, tmp_path=tmp_path)

    refused(lambda t, e, o: cute.embedding(t, e, o), tensor((4,), "float32"), table, rows, match="tokens of dtype i32 or i64")
    refused(lambda t, e, o: cute.embedding(t, e, o), ids, tensor((9, 2, 8)), rows, match="rank-2 table")
    refused(lambda t, e, o: cute.embedding(t, e, o), ids, table, tensor((4, 17)), match="out shape")
    refused(lambda t, e, o: cute.embedding(t, e, o), ids, tensor((9, 16), "int32"), rows, match="dtype f32, bf16 or f16")
    refused(lambda g, t, e: cute.embedding_backward(g, t, e, padding_token=9), rows, ids, table, match=r"padding_token in \[0, 9\)")
    refused(lambda g, t, e: cute.embedding_backward(g, t, e), tensor((5, 16)), ids, table, match="grad_out shape")
    refused(lambda x, o, m, r, w: cute.layernorm_forward(x, o, m, r, w, residual=x), rows, rows, stat, stat, w, match="together or not at all")
    refused(lambda x, o, m, r, w: cute.layernorm_forward(x, o, m, r, w), rows, tensor((4, 16), "bfloat16"), stat, stat, w, match="out like x")
    refused(lambda x, o, m, r, w: cute.layernorm_forward(x, o, m, r, w), rows, rows, tensor((5,)), stat, w, match="mean f32")
    refused(lambda x, o, m, r, w: cute.layernorm_forward(x, o, m, r, w), rows, rows, stat, stat, tensor((16,), "float16"), match="of one dtype, x's or f32")
    refused(lambda x, o, m, r, w: cute.layernorm_forward(x, o, m, r, w), rows, rows, stat, stat, tensor((4, 16)), match="weight shape")
    refused(lambda d, x, m, r, w, g, v: cute.layernorm_backward(d, x, m, r, w, g, v), rows, rows, stat, stat, w, rows, tensor((15,)), match="grad_weight shape")
    refused(lambda p, g, m, v, s: cute.adamw(p, g, m, v, s), [table, w], [table], [table, w], [table, w], tensor((3,)), match="lists of one length")
    refused(lambda p, g, m, v, s: cute.adamw(p, g, m, v, s), [w], [table], [w], [w], tensor((3,)), match=r"grads\[0\]")
    refused(lambda p, g, m, v, s: cute.adamw(p, g, m, v, s), [w], [w], [tensor((16,), "bfloat16")], [w], tensor((3,)), match=r"exp_avgs\[0\]")
    refused(lambda p, g, m, v, s: cute.adamw(p, g, m, v, s), [w], [w], [w], [w], tensor((2,)), match="schedule f32")
    refused(lambda p, g, m, v, s: cute.adamw(p, g, m, v, s, betas=(0.9, 1.0)), [w], [w], [w], [w], tensor((3,)), match="betas")
    refused(lambda p, g, m, v, s: cute.adamw(p, g, m, v, s, weight_decay=[0.1, 0.2]), [w], [w], [w], [w], tensor((3,)), match="one weight_decay or 1")
    refused(lambda p, g, m, v, s: cute.adamw(p, g, m, v, s, epsilon=float("nan")), [w], [w], [w], [w], tensor((3,)), match="epsilon")
    refused(lambda t, e, o: cute.embedding(t, e, o), tensor((0,), "int32"), table, tensor((0, 16)), match="must be > 0")
    with pytest.raises(cute.BackendNotImplementedError, match="no CPU runtime"):
        cute.embedding(cute.tensor([0]), cute.tensor([[1.0]]), cute.tensor([[1.0]]))


def test_the_matcher_refuses_too_wide_rows_and_repeated_tensors(tmp_path, zoo):
    x, stat, w = tensor((1, 32769), "bfloat16"), tensor((1,)), tensor((32769,))
    ir = cute.compile(zoo.layernorm_forward, x, x, stat, stat, w, w, backend="portable", cache_dir=tmp_path).ir
    with pytest.raises(cute.BackendNotImplementedError, match="at most 32768"):
        match(ir)
    w, schedule = tensor((16,)), tensor((3,))

    def twice(p, g, m, v, s):
        cute.adamw([p, p], [g, g], [m, m], [v, v], s)

    with pytest.raises(cute.BackendNotImplementedError, match="same tensor argument twice"):
        match(ir_of(twice, w, w, w, w, schedule, tmp_path=tmp_path))


def test_tensor_groups():
    members = [tensor((4, 4), "bfloat16", 4096), tensor((7,), "bfloat16", 4096 + 32), tensor((1,), "float32", 8192)]
    group = cute.tensor_group(members)
    assert len(group) == 3 and [tuple(handle.shape) for handle in group] == [(4, 4), (7,), (1,)] and group[1].data_ptr() == 4128
    assert list(group.addresses) == [4096, 4128, 8192] and group.signature == "bf16(4, 4);bf16(7,);f32(1,)" and group.device_id == 0
    with pytest.raises(ValueError, match="members 0 and 1 share memory"):
        cute.tensor_group([members[0], tensor((7,), "bfloat16", 4096 + 30)])
    with pytest.raises(ValueError, match="at least one"):
        cute.tensor_group([])
    with pytest.raises(cute.BackendNotImplementedError, match="not a CUDA tensor"):
        cute.tensor_group([tensor((4,), device=(1, 0))])
    with pytest.raises(cute.BackendNotImplementedError, match="different devices"):
        cute.tensor_group([tensor((4,)), tensor((4,), ptr=1 << 20, device=(2, 1))])
    with pytest.raises(cute.BackendNotImplementedError, match="not contiguous"):
        cute.tensor_group([tensor((4, 4), stride=(1, 4))])


def _p(address):
    return ctypes.c_void_p(address)


def test_c_abi_checks_its_arguments_before_any_device_work():
    K = 1 << 20

    def status(name, *arguments):
        with pytest.raises(cute.CudaDriverError) as info:
            native.call(name, *arguments)
        return info.value.status

    lookup = lambda tokens=_p(K), table=_p(2 * K), out=_p(3 * K), types=(0, 0, 3), extents=(4, 9, 16): status(  # noqa: E731
        "bb200_embedding", *types, tokens, table, out, *extents, 1.0, None)
    assert lookup(tokens=None) == -1 and lookup(types=(0, 0, 0)) == -1 and lookup(types=(3, 0, 3)) == -1 and lookup(extents=(0, 9, 16)) == -1
    assert lookup(extents=(4, 1 << 31, 16)) == -2 and lookup(out=_p(3 * K + 2)) == -3 and lookup(out=_p(2 * K + 64)) == -1
    gradient = lambda grad=_p(K), tokens=_p(2 * K), table=_p(3 * K), extents=(4, 9, 16): status(  # noqa: E731
        "bb200_embedding_backward", 1, 0, 4, grad, tokens, table, *extents, 1.0, -1, 0, None)
    assert gradient(grad=None) == -1 and gradient(extents=(1 << 31, 9, 16)) == -2 and gradient(tokens=_p(2 * K + 4)) == -3 and gradient(table=_p(2 * K)) == -1
    places = [_p((i + 1) * K) for i in range(8)]
    forward = lambda order, extents=(4, 16), types=(1, 0): status("bb200_layernorm_forward", *types, *order, *extents, 1e-5, None)  # noqa: E731
    assert forward([None, *places[1:]]) == -1 and forward([places[0], None, *places[2:]]) == -1 and forward(places, (4, 0)) == -1
    assert forward(places, (4, 32769)) == -2 and forward(places, types=(1, 2)) == -1 and forward([_p(K + 1), *places[1:]]) == -3
    assert forward([*places[:4], places[0], *places[5:]]) == -1 and forward([*places[:7], places[6]]) == -1
    places = [_p((i + 1) * K) for i in range(9)]
    backward = lambda order, extents=(4, 16): status("bb200_layernorm_backward", 0, 0, *order, *extents, None)  # noqa: E731
    assert backward([*places[:6], None, *places[7:]]) == -1 and backward(places, (1 << 31, 16)) == -2 and backward(places, (4, 16385)) == -2
    assert backward([*places[:6], places[0], *places[7:]]) == -1 and backward([*places[:8], places[7]]) == -1 and backward([*places[:6], _p(7 * K + 2), *places[7:]]) == -3

    def adamw(numel=64, kinds=(1, 1), addresses=(K, 2 * K, 3 * K, 4 * K, 5 * K), beta1=0.9, epsilon=1e-8, count=1):
        one = lambda kind, value: (kind * 1)(value)  # noqa: E731
        lists = [one(ctypes.c_void_p, address) for address in addresses]
        return status("bb200_adamw", count, one(ctypes.c_size_t, numel), one(ctypes.c_int, kinds[0]), one(ctypes.c_int, kinds[1]),
                      one(ctypes.c_float, 0.0), *lists, _p(6 * K), beta1, 0.999, epsilon, None)

    assert adamw(count=0) == -1 and adamw(numel=0) == -1 and adamw(kinds=(3, 3)) == -1 and adamw(kinds=(0, 1)) == -1 and adamw(beta1=1.0) == -1
    assert adamw(epsilon=float("nan")) == -1 and adamw(addresses=(K, 2 * K, 3 * K, 4 * K, 0)) == -1 and adamw(addresses=(K + 1, 2 * K, 3 * K, 4 * K, 5 * K)) == -3
    assert adamw(addresses=(K, K, 3 * K, 4 * K, 5 * K)) == -1 and adamw(addresses=(K, 2 * K, 3 * K, 3 * K + 128, 5 * K)) == -1


@pytest.mark.parametrize("order", [(0, 1, 2), (2, 0, 1)])
@pytest.mark.parametrize("which", [(0, 0, 0, 1), (0, 0, 1, 2), (1, 2, 3, 0), (2, 1, 4, 1), (4, 0, 4, 2), (0, 1, 5, 0)])
def test_adamw_refuses_tensors_that_share_memory_across_indices_and_lists(which, order):
    """Three tensors of 64 f32 in each of five lists, in rising or mixed order of address; one of them moved onto the last
    element of another (list 5: the schedule)."""
    K = 1 << 20
    schedule = 64 * K
    lists = [[K * (1 + 3 * role + place) for place in order] for role in range(5)]
    from_list, from_index, to_list, to_index = which
    lists[from_list][from_index] = schedule if to_list == 5 else lists[to_list][to_index] + 252
    arrays = [(ctypes.c_void_p * 3)(*addresses) for addresses in lists]
    f32 = (ctypes.c_int * 3)(0, 0, 0)
    status = native.library().bb200_adamw(3, (ctypes.c_size_t * 3)(64, 64, 64), f32, f32, (ctypes.c_float * 3)(0, 0, 0), *arrays, _p(schedule),
                                          0.9, 0.999, 1e-8, None)
    assert status == -1 and b"share memory" in native.library().bb200_last_error()
    aligned = [(ctypes.c_void_p * 3)(*[K * (1 + 3 * role + place) for place in order]) for role in range(5)]
    status = native.library().bb200_adamw(3, (ctypes.c_size_t * 3)(64, 64, 64), f32, f32, (ctypes.c_float * 3)(0, 0, 0), *aligned, _p(schedule + 2),
                                          0.9, 0.999, 1e-8, None)
    assert status == -3


def test_lookups_and_norms_shard_by_rows_and_what_sums_over_them_does_not(tmp_path, zoo):
    from baybridge_b200.sharding import shard_spec

    x, stat, w = tensor((6, 4, 16), "bfloat16"), tensor((6, 4)), tensor((16,))
    tokens, table = tensor((6, 4), "int32"), tensor((9, 16), "bfloat16")

    def spec_of(kernel, *arguments):
        ir = cute.compile(kernel, *arguments, backend="portable", cache_dir=tmp_path).ir
        return shard_spec(match(ir), ir)

    lookup = spec_of(zoo.make_embedding(), tokens, table, x)
    assert (lookup.extent, lookup.sharded, lookup.replicated, lookup.outputs, lookup.reads) == (6, ((0, 0), (2, 0)), (1,), (2,), (0, 1))
    norm = spec_of(zoo.layernorm_forward, x, x, stat, stat, w, w)
    assert (norm.extent, norm.sharded, norm.replicated, norm.outputs) == (6, ((0, 0), (1, 0), (2, 0), (3, 0)), (4, 5), (1, 2, 3))
    for kernel, arguments in ((zoo.make_embedding_backward(), (x, tokens, table)), (zoo.layernorm_backward, (x, x, stat, stat, w, x, w, w)),
                              (zoo.make_adamw(), ([w], [w], [w], [w], tensor((3,))))):
        with pytest.raises(ValueError, match="does not shard"):
            spec_of(kernel, *arguments)


def test_a_launch_binds_its_tensors_device_again_where_another_was_made_current(fake_driver, tmp_path):  # noqa: F811
    """Two devices: between two launches on device 0 the program makes device 1 current; the second launch has to make
    device 0 current again.  With one device nothing is bound twice."""
    body = ELEMENTWISE_CHILD + """
    tensors = [FakeCudaTensor((n,), "float32", 0x10000 * (i + 1), 0) for i in range(3)]
    artifact = cute.compile(zoo.make_indexed_binary("add", n), *tensors, backend="b200", cache_dir=%r)
    artifact(*tensors)
    if %d > 1:
        native.call("bb200_init", 1)
    artifact(*tensors)
    result = {}
    """
    _, log = run_child(fake_driver, tmp_path, body % (str(tmp_path / "cache"), 2), devices=2)
    launches = [i for i, line in enumerate(log) if line.startswith("cuLaunchKernelEx")]
    for launch in launches:
        assert [line for line in log[:launch] if line.startswith("cuCtxSetCurrent")][-1] == "cuCtxSetCurrent context=0xc0de0000"
    (tmp_path / "driver_calls.log").unlink()
    _, log = run_child(fake_driver, tmp_path, body % (str(tmp_path / "cache"), 1), devices=1)
    assert len(calls(log, "cuCtxSetCurrent")) == 1


def test_launchers_take_the_short_path_only_for_what_they_were_compiled_for(tmp_path, zoo, monkeypatch):
    """Handles of the expected shapes go straight to the entry point; a wrong shape, dtype, device or number of arguments
    raises as on the long path."""
    seen = []

    class Entry:
        def __call__(self, *arguments):
            seen.append(arguments)
            return 0

    monkeypatch.setattr(native, "entry_point", lambda name: Entry())
    monkeypatch.setattr(native, "require_device", lambda: None)
    monkeypatch.setattr("baybridge_b200.backend.b200._bind_device", lambda device: None)
    tokens, table, out = (cute.from_dlpack(t) for t in (tensor((4,), "int32", 1 << 20), tensor((9, 16), ptr=2 << 20), tensor((4, 16), ptr=3 << 20)))
    artifact = cute.compile(zoo.make_embedding(2.0), tokens, table, out, backend=cute.B200Backend(synchronize=False), cache_dir=tmp_path)
    artifact(tokens, table, out)
    artifact(tokens, table, out, stream=77)
    artifact(tensor((4,), "int32", 1 << 20), tensor((9, 16), ptr=2 << 20), tensor((4, 16), ptr=3 << 20))  # exporters, not handles
    assert [a[3:6] for a in seen] == [(1 << 20, 2 << 20, 3 << 20)] * 3 and seen[0][-1] is None and seen[1][-1].value == 77
    with pytest.raises(TypeError, match="expects f32"):
        artifact(tokens, cute.from_dlpack(tensor((9, 17), ptr=2 << 20)), out)
    with pytest.raises(TypeError, match="expects f32"):
        artifact(tokens, cute.from_dlpack(tensor((9, 16), "bfloat16", 2 << 20)), out)
    with pytest.raises(cute.BackendNotImplementedError, match="different devices"):
        artifact(tokens, cute.from_dlpack(tensor((9, 16), ptr=2 << 20, device=(2, 1))), out)
    with pytest.raises(cute.BackendNotImplementedError, match="contiguous"):
        artifact(tokens, cute.from_dlpack(tensor((9, 16), ptr=2 << 20, stride=(1, 9))), out)
    with pytest.raises((TypeError, KeyError)):
        artifact(tokens, table)
    assert len(seen) == 3


def test_groups_of_adamw_reach_the_entry_point_whole_and_are_compared(tmp_path, zoo, monkeypatch):
    seen = []
    monkeypatch.setattr(native, "entry_point", lambda name: lambda *arguments: seen.append(arguments) or 0)
    monkeypatch.setattr(native, "require_device", lambda: None)
    monkeypatch.setattr("baybridge_b200.backend.b200._bind_device", lambda device: None)
    place = iter(range(1 << 20, 1 << 30, 1 << 16))
    lists = [cute.tensor_group([tensor(s, ptr=next(place)) for s in ((3, 5), (7,))]) for _ in range(4)]
    schedule = cute.from_dlpack(tensor((3,), ptr=next(place)))
    artifact = cute.compile(zoo.make_adamw(), *lists, schedule, backend=cute.B200Backend(synchronize=False), cache_dir=tmp_path)
    artifact(*lists, schedule)
    artifact(*[list(group) for group in lists], schedule)
    for arguments in seen:
        assert arguments[0] == 2 and [list(array) for array in arguments[5:9]] == [list(group.addresses) for group in lists] and arguments[9] is None
    short = cute.tensor_group([lists[0][0]])
    with pytest.raises(TypeError, match="the params of adamw_kernel differ"):
        artifact(short, *lists[1:], schedule)
    other = cute.tensor_group([tensor(s, ptr=next(place), device=(2, 1)) for s in ((3, 5), (7,))])
    with pytest.raises(cute.BackendNotImplementedError, match="different devices"):
        artifact(other, *lists[1:], schedule)
    assert len(seen) == 2
