"""The largest extents that the training operators take, without a GPU."""
from __future__ import annotations

import ctypes

import pytest
from test_host_surface import FakeCudaTensor

import baybridge_b200 as cute
from baybridge_b200.backend import native
from baybridge_b200.backend.matcher import match

#: the widest grid's stride over columns: gridDim.y, threads of a CTA (csrc/embedding.cu)
STRIDE = 65535 * 256


@pytest.mark.parametrize("hidden", [2**30 + 1, 2130706689, 2**31 - 2, 2**31])
def test_lookups_refuse_rows_whose_columns_an_int_cannot_count(hidden, tmp_path, zoo):
    """The last value of the kernels' column counter, which goes on past the row by a stride and a thread's four vectors."""
    reach = lambda width: width - 1 + STRIDE + 4 * 64  # noqa: E731
    assert reach(2**30) < 2**31
    p = ctypes.c_void_p
    for name, arguments in (("bb200_embedding", (1, 1, 3, p(1 << 20), p(1 << 40), p(1 << 50), 1, 1, hidden, 1.0, None)),
                            ("bb200_embedding_backward", (1, 1, 3, p(1 << 40), p(1 << 20), p(1 << 50), 1, 1, hidden, 1.0, -1, 0, None))):
        with pytest.raises(cute.CudaDriverError, match="at most 2") as info:
            native.call(name, *arguments)
        assert info.value.status == -2
    tokens, table, out = (FakeCudaTensor(shape, dtype, 4096) for shape, dtype in (((1,), "int32"), ((1, hidden), "bfloat16"), ((1, hidden), "bfloat16")))
    for kernel, order in ((zoo.make_embedding(), (tokens, table, out)), (zoo.make_embedding_backward(), (out, tokens, table))):
        with pytest.raises(cute.BackendNotImplementedError, match="at most 2"):
            match(cute.compile(kernel, *order, backend="portable", cache_dir=tmp_path).ir)


def test_the_widest_row_is_matched(tmp_path, zoo):
    tokens, table, out = (FakeCudaTensor(shape, dtype, 4096) for shape, dtype in (((1,), "int32"), ((1, 2**30), "bfloat16"), ((1, 2**30), "bfloat16")))
    assert match(cute.compile(zoo.make_embedding(), tokens, table, out, backend="portable", cache_dir=tmp_path).ir).hidden == 2**30
