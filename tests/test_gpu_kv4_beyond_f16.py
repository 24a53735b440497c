"""kv4_attention over values that read back beyond float16's 65504, which the cache can stand for: low + 15 step of a
group whose step and low are finite in float16. The kernel multiplies float16; such values must be neither infinite nor
reach a row that does not see them. Tolerances as in test_gpu_kv4."""
import pytest
import torch

import attnres_b200 as A
from attnres_b200 import _native
from test_gpu_kv4 import compare, definition, dirty, gen, ints, table_of, values

pytestmark = pytest.mark.gpu


def pool(places, D, big, dtype=torch.bfloat16, H=2):
    """Places of ordinary values except at `big`, whose second group runs to beyond 65504."""
    per = -(-places // 16)
    cache, table = dirty(per + 1, 16, H, D), table_of(1, per, per + 1)
    k = torch.randn(1, places, H, D, device="cuda", generator=gen(1)).to(dtype)
    v = torch.randn(1, places, H, D, device="cuda", generator=gen(2)).to(dtype)
    for at in big:
        if dtype == torch.float16:
            v[0, at, :, 32:64] = torch.linspace(-65504, 65504, 32, device="cuda").to(dtype)
        else:
            v[0, at, :, 32:64] = torch.linspace(0, 70000, 32, device="cuda").to(dtype)
    A.kv4_append(cache, k, v, table, ints(0))
    return cache, table, values(k.float()).double(), values(v.float()).double()


@pytest.mark.parametrize("source", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("heads", [4, 24])  # 8 or fewer query rows a key head, and more
@pytest.mark.parametrize("places,big", [(50, (49,)), (50, (10, 48)), (3000, (100, 2000, 2999)), (3000, (2998,))])
def test_large_values_are_finite_and_stay_with_the_rows_that_see_them(places, big, heads, D, dtype, source):
    cache, table, K, V = pool(places, D, big, source)
    assert float(V.abs().max()) > 65520
    T = 3
    q = torch.randn(1, T, heads, D, device="cuda", generator=gen(3)).to(dtype)
    out, lse = A.kv4_attention(q, cache, table, ints(places), return_lse=True)
    want = definition(q, K, V, [places], [T], D ** -0.5)
    assert bool((want[0].abs() < 65504).all())  # the outputs themselves fit
    compare(out, lse, want, dtype)
    assert _native.device_status() == 0
