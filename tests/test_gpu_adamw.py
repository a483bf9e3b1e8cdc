"""The AdamW step over many tensors on the GPU against 64 bits."""
from __future__ import annotations

import pytest
import training_reference as reference
from gpu_util import TORCH_DTYPE
from training_reference import within

pytestmark = pytest.mark.gpu
BETAS, EPSILON = (0.9, 0.999), 1e-8


def _torch():
    import torch

    return torch


def _dtype(name):
    return getattr(_torch(), TORCH_DTYPE[name])


def _normal(shape, dtype, seed, scale=1.0):
    torch = _torch()
    return (torch.randn(shape, device="cuda", generator=torch.Generator("cuda").manual_seed(seed)) * scale).to(_dtype(dtype))


class Lists:
    """Parameters, gradients, moments and masters of given shapes and dtypes."""

    def __init__(self, members, masters=False, seed=0, decay=0.1):
        torch = _torch()
        self.kinds = [(p, g) for _, p, g in members]
        self.decay = decay if isinstance(decay, list) else [decay] * len(members)
        self.params = [_normal(shape, p, seed + 7 * i) for i, (shape, p, _) in enumerate(members)]
        self.grads = [_normal(shape, g, seed + 7 * i + 1, 0.5) for i, (shape, _, g) in enumerate(members)]
        self.exp_avgs = [_normal(shape, "f32", seed + 7 * i + 2, 0.1) for i, (shape, _, _) in enumerate(members)]
        self.exp_avg_sqs = [_normal(shape, "f32", seed + 7 * i + 3, 0.1).square() for i, (shape, _, _) in enumerate(members)]
        self.masters = [_normal(shape, "f32", seed + 7 * i + 4) for i, (shape, _, _) in enumerate(members)] if masters else None
        self.schedule = torch.tensor([1e-2, 3.0, 0.25], device="cuda")

    def arguments(self, wrap=list):
        return (wrap(self.params), wrap(self.grads), wrap(self.exp_avgs), wrap(self.exp_avg_sqs), self.schedule, wrap(self.masters) if self.masters else None)

    def compile(self, wrap=list, backend="b200", **options):
        import baybridge_b200 as cute

        options = {"betas": BETAS, "epsilon": EPSILON, "weight_decay": self.decay, **options}

        @cute.kernel
        def step(params, grads, exp_avgs, exp_avg_sqs, schedule, masters):
            cute.adamw(params, grads, exp_avgs, exp_avg_sqs, schedule, masters=masters, **options)

        return cute.compile(step, *self.arguments(wrap), backend=backend)

    def expect(self, betas=BETAS, epsilon=EPSILON):
        """What one step gives from the lists as they are: a function that checks the lists against it."""
        rate, step, factor = (float(value) for value in self.schedule)
        results = [reference.adamw((self.masters or self.params)[i], self.grads[i], self.exp_avgs[i], self.exp_avg_sqs[i], rate, step, factor, *betas,
                                   epsilon, self.decay[i]) for i in range(len(self.params))]
        grads = [g.clone() for g in self.grads]

        def check():
            torch = _torch()
            for i, (p, m, v, e_p, e_m, e_v) in enumerate(results):
                within(self.params[i], p, self.kinds[i][0], e_p)
                within(self.exp_avgs[i], m, "f32", e_m)
                within(self.exp_avg_sqs[i], v, "f32", e_v)
                if self.masters:
                    within(self.masters[i], p, "f32", e_p)
                    assert torch.equal(self.params[i], self.masters[i].to(self.params[i].dtype))
                assert torch.equal(self.grads[i], grads[i])

        return check


SIZES = [(1,), (7,), (8,), (9, 3), (2047,), (2048,), (2049,), (4, 5, 6), (100003,), (300, 1000)]


@pytest.mark.parametrize("param,grad,masters", [("f32", "f32", False), ("f32", "f32", True), ("bf16", "bf16", False), ("bf16", "f32", True),
                                                ("bf16", "bf16", True), ("f16", "f16", False), ("f16", "f32", True), ("bf16", "f32", False)])
def test_sizes_and_dtypes(param, grad, masters):
    import baybridge_b200 as cute

    for wrap in (list, cute.tensor_group):
        lists = Lists([(shape, param, grad) for shape in SIZES], masters, seed=1)
        artifact = lists.compile(wrap)
        for _ in range(2):
            check = lists.expect()
            artifact(*lists.arguments(wrap))
            check()


@pytest.mark.parametrize("count", [1, 32, 33, 513, 1100])
def test_many_tensors_of_mixed_dtypes_and_decays(count):
    import baybridge_b200 as cute

    kinds = [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16")] if count != 1100 else [("f32", "f32")]
    members = [((1 + (i * 37) % 300,), *kinds[i % len(kinds)]) for i in range(count)]
    lists = Lists(members, seed=2, decay=[0.0 if i % 3 else 0.2 for i in range(count)])
    check = lists.expect()
    lists.compile(cute.tensor_group)(*lists.arguments(cute.tensor_group))
    check()


def test_unaligned_tensors_and_their_neighbours():
    torch = _torch()
    storage, lists = {}, Lists([((1000 + i,), "bf16", "bf16") for i in range(4)], True, seed=3)
    for name in ("params", "grads", "exp_avgs", "exp_avg_sqs", "masters"):
        values = getattr(lists, name)
        flat = torch.full((6000,), 7.0, device="cuda", dtype=values[0].dtype)
        views, at = [], 0
        for i, value in enumerate(values):
            at += 1 + i  # odd starts, and gaps
            views.append(flat[at:at + value.numel()])
            views[-1].copy_(value)
            at += value.numel()
        mask = torch.ones(6000, dtype=torch.bool, device="cuda")
        for view in views:
            start = view.storage_offset()
            mask[start:start + view.numel()] = False
        storage[name] = flat, mask
        setattr(lists, name, views)
    check = lists.expect()
    lists.compile()(*lists.arguments())
    check()
    for flat, mask in storage.values():
        assert bool((flat[mask] == 7).all())


@pytest.mark.parametrize("offset", [4, 8])
def test_tensors_aligned_to_16_bytes_but_not_to_32(offset):
    torch = _torch()
    for param, grad, masters in (("f32", "f32", False), ("bf16", "f32", True)):
        lists = Lists([((5000,), param, grad), ((4097,), param, grad)], masters, seed=8)
        for name in ("params", "grads", "exp_avgs", "exp_avg_sqs", "masters"):
            values = getattr(lists, name)
            if values is None:
                continue
            views = []
            for value in values:
                start = offset if value.dtype == torch.float32 else 2 * offset
                views.append(torch.zeros(value.numel() + 64, device="cuda", dtype=value.dtype)[start:start + value.numel()])
                views[-1].copy_(value)
            setattr(lists, name, views)
        check = lists.expect()
        lists.compile()(*lists.arguments())
        check()


def test_a_parameter_without_an_axis():
    lists = Lists([((), "f32", "f32"), ((2,), "f32", "f32")], seed=9)
    check = lists.expect()
    lists.compile()(*lists.arguments())
    check()


@pytest.mark.parametrize("betas,epsilon,step", [((0.0, 0.0), 1e-6, 1.0), ((0.9, 0.999), 1e-8, 1.0), ((0.95, 0.99), 1e-8, 100000.0), ((0.5, 0.9999), 0.1, 7.0)])
def test_schedule_and_constants(betas, epsilon, step):
    lists = Lists([((500,), "f32", "f32")], seed=4, decay=0.0)
    lists.schedule[1] = step
    check = lists.expect(betas, epsilon)
    lists.compile(betas=betas, epsilon=epsilon)(*lists.arguments())
    check()


def test_zero_gradients_and_moments_and_values_that_are_not_finite():
    torch = _torch()
    lists = Lists([((64,), "f32", "f32")], seed=5, decay=0.0)
    lists.grads[0].zero_(), lists.exp_avgs[0].zero_(), lists.exp_avg_sqs[0].zero_()
    before = lists.params[0].clone()
    artifact = lists.compile()
    artifact(*lists.arguments())
    assert torch.equal(lists.params[0], before) and not lists.exp_avgs[0].any()
    lists.grads[0][3], lists.grads[0][9] = float("nan"), float("inf")
    artifact(*lists.arguments())
    bad = ~lists.params[0].isfinite()
    assert torch.equal(bad.nonzero().flatten().cpu(), torch.tensor([3, 9]))


def test_a_recorded_step_reads_the_schedule_when_it_replays():
    torch = _torch()
    import baybridge_b200 as cute
    from baybridge_b200.launch_graph import LaunchGraph

    lists = Lists([((700,), "bf16", "bf16")] * 40, True, seed=6)
    groups = [cute.tensor_group(value) for value in (lists.params, lists.grads, lists.exp_avgs, lists.exp_avg_sqs, lists.masters)]
    artifact, schedule = lists.compile(cute.tensor_group), cute.from_dlpack(lists.schedule)
    before = lists.masters[0].clone()
    graph = LaunchGraph()
    with graph.record() as stream:
        artifact(*groups[:4], schedule, groups[4], stream=stream)
    torch.cuda.synchronize()
    assert torch.equal(lists.masters[0], before)
    for step in (4.0, 5.0, 6.0):
        lists.schedule.copy_(torch.tensor([0.1 / step, step, 1.0], device="cuda"))
        check = lists.expect()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        check()
    graph.close()


def test_refusals():
    torch = _torch()
    import baybridge_b200 as cute

    lists = Lists([((50,), "f32", "f32")] * 3, seed=7)
    with pytest.raises(ValueError, match="share memory"):
        cute.tensor_group([lists.params[0], lists.params[1], lists.params[0][10:]])
    with pytest.raises(cute.BackendNotImplementedError, match="not a CUDA tensor"):
        cute.tensor_group([torch.zeros(3)])
    with pytest.raises(cute.BackendNotImplementedError, match="not contiguous"):
        cute.tensor_group([torch.zeros(4, 4, device="cuda").t()])
    artifact = lists.compile()
    params, grads, m, v, schedule, _ = lists.arguments()
    with pytest.raises(cute.CudaDriverError, match="share memory"):
        artifact(params, params, m, v, schedule, None)
    group = cute.tensor_group
    with pytest.raises(TypeError, match="differ in number"):
        artifact(group(params[:2]), group(grads), group(m), group(v), schedule, None)
    with pytest.raises(TypeError, match="expects f32"):
        artifact(params, grads, m, [t.half() for t in v], schedule, None)
    with pytest.raises(cute.CudaDriverError, match="share memory"):
        artifact(group(params), group(grads), group(m), group(m), schedule, None)
