"""A NaN value reaches every row that sees its place, whatever the row's weight for it."""
import pytest
import torch

import attnres_b200 as A
from test_gpu_kv4 import DTYPES, dirty, gen, ints, table_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("places", [20, 300])
def test_nan_value_under_a_weight_that_underflows(places, D, dtype):
    """Place 3's score lies 200 below the others: e^-200 is no fp32 number, and its product with NaN is NaN."""
    per = -(-places // 16)
    cache, table = dirty(per, 16, 1, D), table_of(1, per, per)
    k = torch.zeros(1, places, 1, D, device="cuda")
    k[:, 3, :, :32] = -200.0 * D ** 0.5 / 32
    v = torch.randn(1, places, 1, D, device="cuda", generator=gen(1))
    v[0, 3, 0, 0] = float("nan")
    A.kv4_append(cache, k, v, table, ints(0))
    q = torch.ones(1, 2, 1, D, device="cuda", dtype=dtype)
    out, lse = A.kv4_attention(q, cache, table, ints(places), return_lse=True)
    # NaN where the definition has it: the elements of the value's group, of the rows that see the place
    assert bool(out[..., :32].isnan().all()) and bool(out[..., 32:].isfinite().all()) and bool(lse.isfinite().all())
    assert bool(A.kv4_attention(q[:, :1], cache, table, ints(3)).isfinite().all())  # does not reach place 3
    two = A.kv4_attention(q, cache, table, ints(4))  # its first token stands before place 3, its second on it
    assert bool(two[0, 0].isfinite().all()) and bool(two[0, 1, 0, :32].isnan().all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads", [2, 24])
@pytest.mark.parametrize("places,at", [(40, 39), (40, 20), (3000, 5), (3000, 2990)])
def test_nan_value_reaches_its_group_only(at, places, heads, dtype):
    """Wherever the place lies: in the stage around the end, before it, or in another stretch."""
    per = -(-places // 16)
    cache, table = dirty(per, 16, 2, 128), table_of(1, per, per)
    k, v = (torch.randn(1, places, 2, 128, device="cuda", generator=gen(i)) for i in (1, 2))
    q = torch.randn(1, 2, heads, 128, device="cuda", generator=gen(3)).to(dtype)
    A.kv4_append(cache, k, v, table, ints(0))
    want, want_lse = A.kv4_attention(q, cache, table, ints(places), return_lse=True)
    v[0, at, 1, 70] = float("inf")
    A.kv4_append(cache, k, v, table, ints(0))
    out, lse = A.kv4_attention(q, cache, table, ints(places), return_lse=True)
    bad = torch.zeros_like(out, dtype=torch.bool)
    bad[0, :, heads // 2:, 64:96] = True
    if at == places - 1:
        bad[0, 0] = False  # the first token does not see the last place
    assert torch.equal(out.isnan(), bad) and bool(lse.isfinite().all())
    near = (out.float() - want.float()).abs() <= 2.0 ** -6 * (1 + want.float().abs())
    assert bool(near[~bad].all()) and bool(((lse - want_lse).abs() <= 2.0 ** -12).all())
