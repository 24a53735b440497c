"""What kv4_append makes of finite values that float16 cannot scale: a group's step and low are float16, and a group for
which either overflows reads back as NaN, like one that holds an infinity."""
import pytest
import torch

import attnres_b200 as A
from test_gpu_kv4 import dirty, gen, ints, values

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_groups_beyond_float16(dtype):
    x = torch.randn(1, 6, 2, 64, device="cuda", generator=gen(1))
    x[0, 0, 1, 40] = -70000.0                                             # low
    x[0, 1, 1, 32:] = -1e5                                                # low, without a step
    x[0, 2, 1, 33], x[0, 2, 1, 50] = -6e4, 1.2e6                          # step
    x[0, 3, 1, 32:] = 1e5                                                 # low again, positive
    x[0, 4, 1, 35], x[0, 4, 1, 36] = -65504.0, 65504.0                    # both still fit; in bfloat16 they are +-65536: low
    x[0, 5, 1, 32:] = torch.linspace(0, 70000, 32, device="cuda")         # they fit, the largest value reads back beyond 65504
    x = x.to(dtype)
    cache, table = dirty(1, 16, 2, 64), ints(0)[None]
    A.kv4_append(cache, x, x, table, ints(0))
    want = values(x.float())
    for y in A.kv4_read(cache, table, ints(0), 6, dtype=torch.float32):
        fits = 4 if dtype == torch.float32 else 5
        assert bool(y[0, :fits, 1, 32:].isnan().all())
        assert torch.equal(y[0, :, 1, :32], want[0, :, 1, :32]) and torch.equal(y[0, :, 0], want[0, :, 0])
        assert torch.equal(y[0, fits:], want[0, fits:]) and bool(y[0, fits:].isfinite().all())


def test_such_values_turn_the_rows_that_see_them_into_nan():
    x = torch.randn(1, 9, 1, 64, device="cuda", generator=gen(1))
    v = x.clone()
    v[0, 8, 0, 40] = -70000.0
    cache, table = dirty(1, 16, 1, 64), ints(0)[None]
    A.kv4_append(cache, x, v, table, ints(0))
    out = A.kv4_attention(x[:, 7:].expand(1, 2, 1, 64).to(torch.bfloat16), cache, table, ints(9))
    assert bool(out[0, 0].isfinite().all()) and bool(out[0, 1, 0, 32:].isnan().all())
