"""The training operators together: tokens to embedding, norm, gradients and an AdamW step, several steps long, against the
same steps in 64 bits with torch's autograd.

The distance allowed, 2e-5 of a tensor's norm, counts 32-bit roundings: a norm's row sums are at most 44 additions deep and
its column sums 75 (u = 2^-24 each: 4.5e-6 of the magnitudes), the products around them a dozen more; five steps of 1 % move
the parameters by little more than the gradients' own distance."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hidden", [64, 77])
def test_steps_follow_the_same_steps_in_64_bits(hidden, zoo):
    import torch

    import baybridge_b200 as cute

    generator = torch.Generator("cuda").manual_seed(5)
    vocabulary, batch, length, scale, padding = 40, 3, 25, 2.0, 0
    tokens = torch.randint(0, vocabulary, (batch, length), device="cuda", generator=generator)
    tokens[:, 20:] = padding
    target = torch.randn(batch, length, hidden, device="cuda", generator=generator)
    names = ("table", "weight", "bias")
    shapes = ((vocabulary, hidden), (hidden,), (hidden,))
    params = [torch.randn(s, device="cuda", generator=generator) for s in shapes]
    grads, first, second = ([torch.zeros_like(p) for p in params] for _ in range(3))
    rows, stats = (batch, length, hidden), (batch, length)
    embedded, out, grad_x = (torch.empty(rows, device="cuda") for _ in range(3))
    mean, rstd = torch.empty(stats, device="cuda"), torch.empty(stats, device="cuda")
    schedule = torch.zeros(3, device="cuda")

    compiled = {}

    def launch(kernel, *arguments):
        if kernel not in compiled:
            compiled[kernel] = cute.compile(kernel, *arguments, backend="b200")
        compiled[kernel](*arguments)

    lookup, lookup_grad = zoo.make_embedding(scale), zoo.make_embedding_backward(scale, padding)
    optimizer = zoo.make_adamw(weight_decay=[0.1, 0.0, 0.0])
    wide = [p.double().requires_grad_() for p in params]
    reference = torch.optim.AdamW([{"params": wide[:1], "weight_decay": 0.1}, {"params": wide[1:], "weight_decay": 0.0}], lr=0.01)
    keep = (tokens != padding).double()[..., None]
    for step in range(1, 6):
        launch(lookup, tokens, params[0], embedded)
        launch(zoo.layernorm_forward, embedded, out, mean, rstd, params[1], params[2])
        grad_out = (out - target) * keep.float()  # of half the squared distance, over tokens that are no padding
        launch(zoo.layernorm_backward, grad_out, embedded, mean, rstd, params[1], grad_x, grads[1], grads[2])
        launch(lookup_grad, grad_x, tokens, grads[0])
        schedule.copy_(torch.tensor([0.01, float(step), 1.0]))
        launch(optimizer, params, grads, first, second, schedule)

        reference.zero_grad()
        x = torch.nn.functional.layer_norm(wide[0][tokens] * scale, (hidden,), wide[1], wide[2], 1e-5)
        (0.5 * ((x - target.double()).square() * keep).sum()).backward()
        for name, got, expected in zip(names, grads, wide):
            distance = float((got.double() - expected.grad).norm() / expected.grad.norm())
            assert distance <= 2e-5, f"step {step}: gradient of {name} is {distance:.2g} off"
        reference.step()
    for name, got, expected in zip(names, params, wide):
        distance = float((got.double() - expected.detach()).norm() / expected.detach().norm())
        assert distance <= 2e-5, f"{name} is {distance:.2g} off after the steps"


FIRST_CALL_RECORDED = '''
import sys
sys.path.insert(0, %r)
import torch
import baybridge_b200 as cute
from baybridge_b200.launch_graph import LaunchGraph
from baybridge_b200.samples import build_zoo

zoo = build_zoo(cute)
tokens = torch.randint(0, 50, (40000,), device="cuda", dtype=torch.int32)
grad, table = torch.randn(40000, 24, device="cuda"), torch.full((50, 24), 7.0, device="cuda")
rows, hidden = 3000, 512
x, d, w = torch.randn(rows, hidden, device="cuda"), torch.randn(rows, hidden, device="cuda"), torch.ones(hidden, device="cuda")
mean, rstd = x.mean(-1), (x.var(-1, correction=0) + 1e-5).rsqrt()
grad_x, grad_w, grad_b = torch.empty_like(x), torch.empty_like(w), torch.empty_like(w)
torch.cuda.synchronize()
lookup, norm = (grad, tokens, table), (d, x, mean, rstd, w, grad_x, grad_w, grad_b)
first = cute.compile(zoo.make_embedding_backward(), *lookup, backend="b200")
second = cute.compile(zoo.layernorm_backward, *norm, backend="b200")
graph = LaunchGraph()
with graph.record() as stream:  # nothing of the library has run before: pool, attributes and modules are made in here
    first(*(cute.from_dlpack(t) for t in lookup), stream=stream)
    second(*(cute.from_dlpack(t) for t in norm), stream=stream)
assert bool((table == 7).all())
for _ in range(2):
    graph.replay()
torch.cuda.synchronize()
expected = torch.zeros(50, 24, device="cuda", dtype=torch.float64).index_add_(0, tokens.long(), grad.double())
assert float((table.double() - expected).norm() / expected.norm()) < 1e-5
assert float((grad_b.double() - d.double().sum(0)).norm() / d.double().sum(0).norm()) < 1e-5
graph.close()
print("recorded")
'''


def test_the_first_calls_of_a_process_may_be_recorded(tmp_path):
    """Sums of 800 and 3000 f32 terms: their rounding (u = 2^-24 a step) is far below the 1e-5 of the norm allowed."""
    import subprocess
    import sys
    from pathlib import Path

    script = tmp_path / "first_call.py"
    script.write_text(FIRST_CALL_RECORDED % str(Path(__file__).resolve().parent.parent))
    done = subprocess.run([sys.executable, str(script)], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=300)
    assert done.returncode == 0 and "recorded" in done.stdout, done.stdout[-2000:]


def test_threads_may_call_one_artifact_at_once(zoo):
    """Four threads, four streams, one compiled kernel: launchers of these operators keep nothing between calls."""
    import threading

    import torch

    import baybridge_b200 as cute

    generator = torch.Generator("cuda").manual_seed(3)
    tokens = [torch.randint(0, 300, (9000,), device="cuda", dtype=torch.int32, generator=generator) for _ in range(4)]
    grads = [torch.randn(9000, 32, device="cuda", generator=generator) for _ in range(4)]
    tables = [torch.zeros(300, 32, device="cuda") for _ in range(4)]
    handles = [[cute.from_dlpack(t) for t in group] for group in zip(grads, tokens, tables)]
    artifact = cute.compile(zoo.make_embedding_backward(), *handles[0], backend=cute.B200Backend(synchronize=False))
    streams = [torch.cuda.Stream() for _ in range(4)]
    torch.cuda.synchronize()
    failures = []

    def work(index):
        try:
            for _ in range(50):
                artifact(*handles[index], stream=streams[index])
        except Exception as error:  # noqa: BLE001 - reported below
            failures.append(error)

    threads = [threading.Thread(target=work, args=(index,)) for index in range(4)]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    torch.cuda.synchronize()
    assert not failures
    for token, grad, table in zip(tokens, grads, tables):
        expected = torch.zeros(300, 32, device="cuda", dtype=torch.float64).index_add_(0, token.long(), grad.double())
        # runs of about thirty tokens: at most that many roundings of u = 2^-24 of the magnitudes' sum
        size = torch.zeros_like(expected).index_add_(0, token.long(), grad.double().abs())
        assert bool(((table.double() - expected).abs() <= 80 * 2.0 ** -24 * size).all())
