"""What the training operators record in the device status word, next to the pipelines that record theirs there."""
from __future__ import annotations

import pytest
from gpu_util import current_stream

pytestmark = pytest.mark.gpu

GIVE_UP, BAD_TOKEN = 99, 311


@pytest.mark.parametrize("count", [9, 3000, 70000])  # one launch, the sort in a cluster, the sort over the whole device
@pytest.mark.parametrize("gradient", [False, True])
def test_a_bad_token_does_not_replace_the_code_of_a_wait_that_gave_up(gradient, count):
    import torch

    import baybridge_b200 as cute
    from baybridge_b200.backend import native

    tokens = torch.arange(count, device="cuda", dtype=torch.int32) % 50
    tokens[count // 2] = 50
    table, rows = torch.zeros(50, 8, device="cuda"), torch.zeros(count, 8, device="cuda")

    @cute.kernel
    def lookup(tokens: cute.Tensor, table: cute.Tensor, out: cute.Tensor):
        cute.embedding(tokens, table, out)

    @cute.kernel
    def backward(grad_out: cute.Tensor, tokens: cute.Tensor, grad_table: cute.Tensor):
        cute.embedding_backward(grad_out, tokens, grad_table)

    body, arguments = (backward, (rows, tokens, table)) if gradient else (lookup, (tokens, table, rows))
    artifact = cute.compile(body, *arguments, backend=cute.B200Backend(synchronize=False))
    stream = current_stream()
    assert native.take_device_status(stream) == 0
    artifact(*arguments, stream=torch.cuda.current_stream())
    assert native.take_device_status(stream) == BAD_TOKEN
    native.call("bb200_selftest_bounded_wait", 1000, stream)  # a wait gives up; nobody has read its code yet
    artifact(*arguments, stream=torch.cuda.current_stream())
    assert native.take_device_status(stream) == GIVE_UP
    assert native.take_device_status(stream) == 0
