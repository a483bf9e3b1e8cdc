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


def test_a_call_that_finds_no_memory_for_its_workspace_leaves_the_next_one_alone():
    """The workspace's size follows from the extents alone: two rows of 2^22 f32 for each chunk of at most 512 of 2^24 tokens, 1.1
    TB, so the call ends on the host before any launch.  What it leaves must not be taken for a failure of the next one."""
    import torch
    from gpu_util import void_p

    from baybridge_b200 import CudaDriverError
    from baybridge_b200.backend import native

    rows, grad, table = torch.ones(4, 16, device="cuda"), torch.ones(4, 16, device="cuda"), torch.zeros(9, 16, device="cuda")
    tokens = torch.arange(4, device="cuda", dtype=torch.int32)
    count, hidden = 2 ** 24, 2 ** 22
    assert count // 512 * 2 * hidden * 4 > 4 * torch.cuda.get_device_properties(0).total_memory
    with pytest.raises(CudaDriverError, match="workspace.*cudaErrorMemoryAllocation"):
        native.call("bb200_embedding_backward", 0, 0, 3, 1 << 50, void_p(tokens), 1 << 52, count, 1, hidden, 1.0, -1, 1, current_stream())
    native.call("bb200_embedding", 0, 0, 3, void_p(tokens), void_p(table), void_p(rows), 4, 9, 16, 1.0, current_stream())
    assert not rows.any()
    native.call("bb200_embedding_backward", 0, 0, 3, void_p(grad), void_p(tokens), void_p(table), 4, 9, 16, 1.0, -1, 0, current_stream())
    assert bool((table[:4] == 1).all()) and not table[4:].any()
