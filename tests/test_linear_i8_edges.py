"""The 8-bit dense layers of the box head beyond the sizes and the values of tests/test_linear_i8.py: what 32 bits of an index
cannot hold, signs that hang on the last bit, gradients of very different sizes, modules as a user wires them up."""
import ctypes

import pytest
import torch

from .test_linear_i8 import BF16, F16, F32, dev, features, gpu, grad_bound, plain_codes, plain_grads, plain_product, same_bits  # noqa: F401,E501


# ------------------------------------------------------------------------------------------------ sizes past 32 bits
def test_rows_too_long_for_an_index_are_refused():
    """Column indices are 32-bit numbers: a row that they cannot step past is refused before any launch."""
    from objectdetection_amd import _lib, ops
    lib = _lib.load()
    p, null = ctypes.c_void_p(4096), ctypes.c_void_p(0)  # never dereferenced
    for k in ((1 << 30) + 1, (1 << 31) - 20000, (1 << 31) - 1):
        assert lib.frcnn_quantize_rows_i8(p, 1, k, 1, k, null, p, k + 1 | 1, p, null) == -1
        assert b"shape" in lib.frcnn_last_error_string()
    assert lib.frcnn_quantize_rows_i8(p, 1, 1 << 30, 0, 1 << 30, null, p, 1 << 30, p, null) == 0  # no rows: nothing to do
    for sizes in ((1 << 22, 1, 8), (1 << 32, 1, 8), (1, (1 << 32) + 3, 8), (1, 1, 1 << 17), (1, 1, (1 << 32) + 5)):
        with pytest.raises(ValueError):
            ops._i8_sizes("sizes", *sizes)
    ops._i8_sizes("sizes", ops.I8_MAX_ROWS, ops.I8_MAX_ROWS, ops.I8_MAX_K)


@gpu
def test_python_refuses_sizes_past_32_bits(dev):
    """Views of a few bytes with more rows or columns than a C int holds: refused, not cut to their low 32 bits."""
    from objectdetection_amd import ops
    x = torch.ones((1, 8), device=dev, dtype=BF16)
    codes, scale = ops.quantize_rows_i8(x)
    many, long = x.expand((1 << 32) + 1, 8), x[:, :1].expand(1, (1 << 32) + 5)
    many_codes, many_scale = codes.expand((1 << 32) + 1, 8), scale.expand((1 << 32) + 1)
    for bad in (lambda: ops.quantize_rows_i8(many), lambda: ops.quantize_rows_i8(long),
                lambda: ops.quantize_rows_i8(x.expand(1 << 22, 8)), lambda: ops.linear_i8(many, codes, scale),
                lambda: ops.linear_i8(x, many_codes, many_scale), lambda: ops.matmul_i8(many_codes, many_scale, codes, scale),
                lambda: ops.linear_i8(long, codes[:, :1].expand(1, (1 << 32) + 5), scale),
                lambda: ops.LinearI8.apply(many, x, None, False), lambda: ops.LinearI8.apply(x, many, None, False)):
        with pytest.raises(ValueError):
            bad()
