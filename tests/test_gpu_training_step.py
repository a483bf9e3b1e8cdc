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
