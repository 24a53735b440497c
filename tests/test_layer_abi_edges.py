"""More answers of the layer operators' C entries, without a GPU."""
import ctypes

import pytest

from attnres_b200 import _native as N
from test_layer_cpu import INVALID, P, STRIDES, UNSUPPORTED, WORKSPACE, rope


@pytest.mark.parametrize("dtype", [N.DTYPE_F32, N.DTYPE_F16, N.DTYPE_BF16])
def test_rope_takes_float_weights_beside_any_type(dtype):
    assert rope(n=0, dtype=dtype | N.WEIGHTS_F32) == 0
    assert rope(dtype=dtype | N.WEIGHTS_F32, q=None) == INVALID  # past the type's check
    assert rope(dtype=9 | N.WEIGHTS_F32) == INVALID and rope(dtype=dtype | 0x200) == INVALID
    assert N.load().attnres_qk_norm_rope_backward(4, 2, 2, 1, 64, 64, dtype | N.WEIGHTS_F32, P, 256, P, P, 8, None, 0, P, None, 1,
                                                  1e-6, 1, P, P, P, STRIDES, P, P, None, ctypes.c_void_p(0), 0,
                                                  None) == WORKSPACE


def test_attention_workspace_of_sizes_that_the_call_refuses():
    need = N.load().attnres_kv4_attention_workspace_bytes
    big = (1 << 31) - 1
    assert need(2, 16, 64, 4096, 2, 1, 4) > 0
    for sizes in ((2, 16, 64, 4096, 2, big, 4096), (1, 16, 64, 4096, 1, 1 << 20, 1 << 11), (2, 16, 64, big, 2, 1, 4),
                  (2, 1 << 30, 64, big, 2, 1, 4), (2, 16, 64, 4096, 70000, 1, 4), (70000, 16, 64, 4096, 1, 1, 70000)):
        assert need(*sizes) == 0, sizes


def test_rope_refuses_more_rows_than_a_grid_holds():
    assert rope(n=1 << 31, T=1) == UNSUPPORTED  # 2^33 head rows, four a block: one block more than a grid has
