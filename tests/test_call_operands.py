"""Calls of a compiled artifact that differ from what it was compiled for, without a GPU: nothing is left out silently."""
from __future__ import annotations

import pytest
from test_host_surface import FakeCudaTensor

import baybridge_b200 as cute
from baybridge_b200.backend import native


@pytest.fixture
def launches(monkeypatch):
    """Entry points that only record their arguments."""
    seen = []
    monkeypatch.setattr(native, "entry_point", lambda name: lambda *arguments: seen.append((name, arguments)) or 0)
    monkeypatch.setattr(native, "call", lambda *arguments: None)
    monkeypatch.setattr(native, "take_device_status", lambda stream: 0)
    monkeypatch.setattr(native, "require_device", lambda: None)
    monkeypatch.setattr("baybridge_b200.backend.b200._bind_device", lambda device: None)
    return seen


class Tensors:
    """Distinct stand-ins for device tensors, as exporters or as handles."""

    def __init__(self, handles: bool):
        self.place, self.handles = iter(range(1 << 20, 1 << 30, 1 << 16)), handles

    def __call__(self, shape, dtype="float32"):
        value = FakeCudaTensor(shape, dtype, next(self.place))
        return cute.from_dlpack(value) if self.handles else value

    def list(self, count, shape=(8,)):
        return [self(shape) for _ in range(count)]

    def group(self, count, shape=(8,)):
        return cute.tensor_group(self.list(count, shape))


def _norm(x, out, mean, rstd, weight, bias=None, residual=None, out_resid=None):
    cute.layernorm_forward(x, out, mean, rstd, weight, bias, residual=residual, out_resid=out_resid)


def _step(params, grads, exp_avgs, exp_avg_sqs, schedule, masters):
    cute.adamw(params, grads, exp_avgs, exp_avg_sqs, schedule, masters=masters)


@pytest.mark.parametrize("handles", [False, True])
@pytest.mark.parametrize("synchronize", [False, True])
def test_operands_left_out_at_compile_time_are_refused_at_the_call(handles, synchronize, launches, tmp_path):
    t = Tensors(handles)
    backend = cute.B200Backend(synchronize=synchronize)
    required = [t((4, 16)), t((4, 16)), t((4,)), t((4,)), t((16,))]
    given_none = cute.compile(cute.kernel(_norm), *required, None, None, None, backend=backend, cache_dir=tmp_path)
    defaulted = cute.compile(cute.kernel(_norm), *required, backend=backend, cache_dir=tmp_path)
    bias, residual, out_resid = t((16,)), t((4, 16)), t((4, 16))
    for artifact in (given_none, defaulted):
        artifact(*required, None, None, None)
        artifact(*required, None, None, None, stream=7)
        assert len(launches) == 2
        with pytest.raises(TypeError, match="'bias' is not an operand"):
            artifact(*required, bias, residual, out_resid)
        with pytest.raises(TypeError, match="'residual' is not an operand"):
            artifact(*required, None, residual, out_resid, stream=7)
        with pytest.raises(TypeError, match="'out_resid' is not an operand"):
            artifact(*required, out_resid=out_resid)
        assert len(launches) == 2
        launches.clear()
    defaulted(*required)
    whole = cute.compile(cute.kernel(_norm), *required, bias, residual, out_resid, backend=backend, cache_dir=tmp_path)
    whole(*required, bias, residual, out_resid)
    assert len(launches) == 2
    with pytest.raises((TypeError, KeyError)):  # the opposite mistake
        whole(*required, None, None, None)
    assert len(launches) == 2


@pytest.mark.parametrize("synchronize", [False, True])
def test_masters_left_out_at_compile_time_are_refused_at_the_call(synchronize, launches, tmp_path):
    t = Tensors(True)
    lists, schedule = [t.list(2) for _ in range(4)], t((3,))
    artifact = cute.compile(cute.kernel(_step), *lists, schedule, None, backend=cute.B200Backend(synchronize=synchronize), cache_dir=tmp_path)
    groups = [cute.tensor_group(members) for members in lists]
    for masters in (t.group(2), t.list(2), tuple(t.list(2)), {"a": t((8,))}):
        for arguments in (groups, lists, [groups[0], *lists[1:]]):
            with pytest.raises(TypeError, match="'masters' is not an operand"):
                artifact(*arguments, schedule, masters)
    assert not launches
    artifact(*groups, schedule, None)
    artifact(*lists, schedule, None)
    artifact(*groups, schedule, [])  # holds nothing that could be left out
    assert len(launches) == 3


def test_constants_of_a_kernel_keep_working_and_changed_numbers_are_refused(launches, tmp_path):
    def scaled(tokens, table, out, options, factor=2.0):
        cute.embedding(tokens, table, out, scale=factor if options["twice"] is None else 1.0)

    t = Tensors(True)
    arguments = t((4,), "int32"), t((9, 16)), t((4, 16))
    artifact = cute.compile(cute.kernel(scaled), *arguments, {"twice": None, "name": "a"}, backend=cute.B200Backend(synchronize=False), cache_dir=tmp_path)
    artifact(*arguments, {"twice": None, "name": "b"})
    artifact(*arguments, {"twice": None, "name": "a"}, 2.0)
    assert len(launches) == 2
    with pytest.raises(TypeError, match=r"'options\['twice'\]' is not an operand"):
        artifact(*arguments, {"twice": t((1,)), "name": "a"})
    with pytest.raises(TypeError, match="'factor' is not an operand of this artifact: it was 2.0"):
        artifact(*arguments, {"twice": None, "name": "a"}, 3.0)
    assert len(launches) == 2


@pytest.mark.parametrize("synchronize", [False, True])
@pytest.mark.parametrize("count", [1, 3])
def test_lists_of_another_length_are_refused(count, synchronize, launches, tmp_path):
    t = Tensors(True)
    schedule = t((3,))
    artifact = cute.compile(cute.kernel(_step), *[t.list(2) for _ in range(4)], schedule, t.list(2),
                            backend=cute.B200Backend(synchronize=synchronize), cache_dir=tmp_path)
    lists, groups = (lambda n: [t.list(n) for _ in range(4)]), (lambda n: [t.group(n) for _ in range(4)])
    artifact(*lists(2), schedule, t.list(2))
    artifact(*groups(2), schedule, t.group(2))
    artifact(t.group(2), *lists(2)[1:], schedule, tuple(t.list(2)))
    assert len(launches) == 3
    for arguments in (lists(count), groups(count), [t.group(count), *lists(count)[1:]], [t.list(2), *lists(count)[1:]], [*lists(2)[1:], t.list(count)]):
        for masters in (t.list(2), t.group(2), t.list(count)):
            with pytest.raises((TypeError, IndexError)):
                artifact(*arguments, schedule, masters)
    with pytest.raises(TypeError, match=f"'masters' has {count} members, but the kernel was compiled for 2"):
        artifact(*lists(2), schedule, t.list(count))
    assert len(launches) == 3


def test_parts_of_a_dict_that_were_not_there_at_compile_time_are_refused(launches, tmp_path):
    def lookup(operands):
        cute.embedding(operands["tokens"], operands["table"], operands["out"])

    t = Tensors(False)
    operands = {"tokens": t((4,), "int32"), "table": t((9, 16)), "out": t((4, 16))}
    artifact = cute.compile(cute.kernel(lookup), operands, backend=cute.B200Backend(synchronize=False), cache_dir=tmp_path)
    artifact(operands)
    artifact({**operands, "note": "not an operand"})

    class Record:
        tokens, table, out, more = (*operands.values(), t((1,)))

    artifact(Record)  # an object with these attributes, and others of its own
    assert len(launches) == 3
    with pytest.raises(TypeError, match="'operands' holds 'more'"):
        artifact({**operands, "more": t((1,))})
    assert len(launches) == 3


def test_a_kernel_that_steps_some_members_of_its_lists_takes_groups_as_well(launches, tmp_path):
    def step(params, grads, exp_avgs, exp_avg_sqs, schedule):
        cute.adamw(params[:2], grads[:2], exp_avgs[:2], exp_avg_sqs[:2], schedule)

    t = Tensors(True)
    lists, schedule = [t.list(3) for _ in range(4)], t((3,))
    artifact = cute.compile(cute.kernel(step), *lists, schedule, backend=cute.B200Backend(synchronize=False), cache_dir=tmp_path)
    artifact(*lists, schedule)
    artifact(*[cute.tensor_group(members) for members in lists], schedule)
    for _, arguments in launches:
        assert arguments[0] == 2 and [list(array) for array in arguments[5:9]] == [[m.data_ptr() for m in members[:2]] for members in lists]
    assert len(launches) == 2


def test_eager_launches_compile_again_for_other_lists(launches, tmp_path, monkeypatch):
    monkeypatch.setenv("BAYBRIDGE_CACHE_DIR", str(tmp_path))

    @cute.kernel
    def step(params, grads, exp_avgs, exp_avg_sqs, schedule, mode=None):
        cute.adamw(params, grads, exp_avgs, exp_avg_sqs, schedule, weight_decay=0.5 if mode == "decay" else 0.0)

    t = Tensors(True)
    schedule = t((3,))

    def launch(lists, *mode):
        step(*lists, schedule, *mode).launch(grid=(1, 1, 1), block=(1, 1, 1))
        name, arguments = launches[-1]
        return arguments[0], list(arguments[1]), list(arguments[5]), list(arguments[4])

    for count, shape in ((2, (8,)), (3, (8,)), (2, (5,)), (2, (8,)), (1, (2, 2))):
        lists = [t.list(count, shape) for _ in range(4)]
        numel = shape[0] * (shape[1] if len(shape) > 1 else 1)
        expected = count, [numel] * count, [member.data_ptr() for member in lists[0]], [0.0] * count
        assert launch(lists) == expected
        assert launch([cute.tensor_group(members) for members in lists]) == expected
        assert launch(lists, "decay") == expected[:3] + ([0.5] * count,)
        assert launch(lists, "none") == expected


def test_a_bad_token_found_by_a_later_launch_is_not_called_that_launchs_own(launches, tmp_path, zoo, monkeypatch):
    t = Tensors(True)
    a, b, c = t((256, 256), "bfloat16"), t((256, 256), "bfloat16"), t((256, 256), "bfloat16")
    tokens, table, out = t((4,), "int32"), t((9, 16)), t((4, 16))
    product = cute.compile(zoo.gemm_abt, a, b, c, backend="b200", cache_dir=tmp_path)
    lookup = cute.compile(zoo.make_embedding(), tokens, table, out, backend="b200", cache_dir=tmp_path)
    monkeypatch.setattr(native, "call_resolved", lambda *arguments: None)
    monkeypatch.setattr(native, "take_device_status", lambda stream: native.TOKEN_OUT_OF_RANGE)
    with pytest.raises(RuntimeError, match="device status 311: a token of a lookup before this launch, which was not waited for, lies outside the table"):
        product(a, b, c)
    with pytest.raises(RuntimeError, match="device status 311: a token of this lookup, or of one before that was not waited for, lies outside the table"):
        lookup(tokens, table, out)


@pytest.mark.parametrize("synchronize", [False, True])
def test_calls_on_handles_are_not_looked_over_twice(synchronize, launches, tmp_path, zoo, monkeypatch):
    """Device tensor handles need no normalisation, whether the launcher synchronises or not, and a launcher that waits for its
    kernel, which the short path cannot do, is not asked for the short path."""
    t = Tensors(True)
    handles = t((4,), "int32"), t((9, 16)), t((4, 16))
    artifact = cute.compile(zoo.make_embedding(), *handles, backend=cute.B200Backend(synchronize=synchronize), cache_dir=tmp_path)
    normalised = []
    monkeypatch.setattr("baybridge_b200.driver.normalize_runtime_argument", lambda value, stream=None: normalised.append(value) or value)
    artifact(*handles)
    artifact(*handles, stream=3)
    assert len(launches) == 2 and not normalised
    assert hasattr(artifact.runtime_callable, "quick") is not synchronize
