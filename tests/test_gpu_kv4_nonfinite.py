"""kv4_attention where queries or keys are not finite: such rows are NaN, as the softmax's definition has them, and only
a row that sees no place at all is zeros with an lse of -inf. Rows beside them keep their bits."""
import pytest
import torch

import attnres_b200 as A
from attnres_b200 import _native
from test_gpu_kv4 import DTYPES, filled, gen, ints, table_of, dirty

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("places", [1, 40, 3000])  # one stretch, and several with their join
@pytest.mark.parametrize("bad", [NAN, INF, -INF])
def test_query_that_is_not_finite(bad, places, D, dtype):
    cache, table, n, _, _ = filled([places, 0, 7], 2, D, 16, dtype)
    q = torch.randn(3, 2, 4, D, device="cuda", generator=gen(4)).to(dtype)
    want, want_lse = A.kv4_attention(q, cache, table, n, return_lse=True)
    q[0, 1, 2, 5] = bad
    q[1, 0, 1, 0] = bad  # of a sequence without keys
    out, lse = A.kv4_attention(q, cache, table, n, return_lse=True)
    assert bool(out[0, 1, 2].isnan().all()) and bool(lse[0, 1, 2].isnan())
    assert bool((out[1] == 0).all()) and bool((lse[1] == -INF).all())
    clean = torch.ones(3, 2, 4, dtype=torch.bool, device="cuda")
    clean[0, 1, 2] = False
    assert torch.equal(out[clean], want[clean]) and torch.equal(lse[clean], want_lse[clean])


@pytest.mark.parametrize("D", [64, 128])
def test_infinite_query_whose_scores_are_all_minus_infinity(D):
    """Positive keys and -inf in the query: every score is -inf, and exp(-inf - -inf) is NaN, not an empty row."""
    cache, table, n = dirty(3, 16, 1, D), table_of(1, 2, 3), ints(20)
    k = torch.rand(1, 20, 1, D, device="cuda", generator=gen(1)) + 0.5
    A.kv4_append(cache, k, k, table, ints(0))
    q = torch.zeros(1, 1, 2, D, device="cuda", dtype=torch.bfloat16)
    q[0, 0, 1, 3] = -INF
    out, lse = A.kv4_attention(q, cache, table, n, return_lse=True)
    assert bool(out[0, 0, 1].isnan().all()) and bool(lse[0, 0, 1].isnan())
    assert bool(out[0, 0, 0].isfinite().all()) and bool(lse[0, 0, 0].isfinite())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("places", [1, 5, 3000])
@pytest.mark.parametrize("bad", [NAN, INF])
def test_sequence_whose_keys_are_all_nan(bad, places, D, dtype):
    """A group that holds an infinity or a NaN is NaN in the cache; here every key of the first sequence has one."""
    cache, table, n, K, _ = filled([places, 30], 2, D, 16, dtype)
    q = torch.randn(2, 1, 4, D, device="cuda", generator=gen(4)).to(dtype)
    want, want_lse = A.kv4_attention(q, cache, table, n, return_lse=True)
    k = K[:1, :, :, :].float().clone()
    k[0, :, 0, D - 1] = bad
    v = torch.randn(1, K.shape[1], 2, D, device="cuda", generator=gen(5))
    A.kv4_append(cache, k, v, table[:1], ints(0), n[:1])
    out, lse = A.kv4_attention(q, cache, table, n, return_lse=True)
    assert bool(out[0, 0, :2].isnan().all()) and bool(lse[0, 0, :2].isnan().all())  # the query heads of key head 0
    assert bool(out[0, 0, 2:].isfinite().all()) and bool(lse[0, 0, 2:].isfinite().all())
    assert torch.equal(out[1], want[1]) and torch.equal(lse[1], want_lse[1])
    assert _native.device_status() == 0
