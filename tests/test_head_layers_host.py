"""The head's layers as a program uses them (data-parallel training, recomputation, ranks), with torch operations in place of the
kernels, and sizes that the library refuses."""
import ctypes

import pytest
import torch

from l_inf_dist_net_v2_b200._lib import lib

BAD = 1


# ---- sizes whose sums with a tile's or a grid's would pass 32 bits (none of these calls may launch anything) -----------------------------
MOST = (1 << 31) - 1


@pytest.mark.parametrize("C", [MOST, MOST - 255, MOST - (1 << 22) + 1])
def test_rows_that_are_too_long(C):
    here = ctypes.create_string_buffer(64)
    p = ctypes.cast(here, ctypes.c_void_p)
    assert lib.ldn_layer_norm(p, C, 2, C, 0, p, p, 0, 1e-5, p, p, p, None) == BAD
    assert lib.ldn_layer_norm_backward(p, p, C, 2, C, 0, p, p, p, 0, p, p, p, None) == BAD
    assert lib.ldn_dropout_add_layer_norm(p, C, p, C, 2, C, 0, p, p, 0, 1e-5, 0.5, 1, 0, None, p, p, p, p, None) == BAD
    assert lib.ldn_dropout_add_layer_norm_backward(p, p, p, 2, C, 0, p, p, p, 0, 0.5, 1, 0, None, p, p, p, p, None) == BAD
    assert lib.ldn_quantize_rows(p, C, 2, C, 0, p, C + 16, p, None) == BAD
    assert lib.ldn_layer_norm_quantized(p, C, 2, C, 0, p, p, 0, 1e-5, p, C + 16, p, None) == BAD


@pytest.mark.parametrize("N", [MOST, MOST - 127, MOST - (1 << 22) + 1])
def test_too_many_outputs(N):
    here = ctypes.create_string_buffer(64)
    p = ctypes.cast(here, ctypes.c_void_p)
    assert lib.ldn_int8_linear(p, 16, p, p, 16, p, None, 2, N, 4, 0, p, 0, None) == BAD
    assert lib.ldn_int8_linear_float(p, 16, 0, p, 16, p, None, 2, N, 4, 0, p, 0, None) == BAD
