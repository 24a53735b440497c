"""More answers of the layer operators' C entries, without a GPU."""
import ctypes

import pytest

from attnres_b200 import _native as N
from test_layer_cpu import INVALID, P, STRIDES, WORKSPACE, rope


@pytest.mark.parametrize("dtype", [N.DTYPE_F32, N.DTYPE_F16, N.DTYPE_BF16])
def test_rope_takes_float_weights_beside_any_type(dtype):
    assert rope(n=0, dtype=dtype | N.WEIGHTS_F32) == 0
    assert rope(dtype=dtype | N.WEIGHTS_F32, q=None) == INVALID  # past the type's check
    assert rope(dtype=9 | N.WEIGHTS_F32) == INVALID and rope(dtype=dtype | 0x200) == INVALID
    assert N.load().attnres_qk_norm_rope_backward(4, 2, 2, 1, 64, 64, dtype | N.WEIGHTS_F32, P, 256, P, P, 8, None, 0, P, None, 1,
                                                  1e-6, 1, P, P, P, STRIDES, P, P, None, ctypes.c_void_p(0), 0,
                                                  None) == WORKSPACE
