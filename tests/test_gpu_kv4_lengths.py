"""Lengths beyond what a sequence's page table has room for: its tokens keep their places, see what is there, and the
device status word tells that places without a page were asked for."""
import pytest
import torch

import attnres_b200 as A
from attnres_b200 import _native
from test_gpu_kv4 import compare, definition, filled, gen, ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("room,length", [(64, 66), (64, 100), (64, 65), (2048, 2050), (64, 2 ** 31 - 1)])
def test_tokens_past_the_table(room, length, D):
    dtype, T = torch.bfloat16, 3
    cache, table, n, K, V = filled([room], 2, D, 16, dtype)
    q = torch.randn(1, T, 4, D, device="cuda", generator=gen(3)).to(dtype)
    _native.device_status(reset=True)
    A.kv4_attention(q, cache, table, n)
    assert _native.device_status() == 0
    out, lse = A.kv4_attention(q, cache, table, ints(length), return_lse=True)
    assert _native.device_status(reset=True) == 8
    # token t stands at place length - T + t: it sees that and what comes before, as far as the table goes
    compare(out, lse, definition(q, K, V, [min(length, room + T)], [T], D ** -0.5), dtype)


def test_no_pages_at_all():
    cache, table, n, _, _ = filled([16], 1, 64, 16, torch.bfloat16)
    q = torch.randn(1, 2, 1, 64, device="cuda", generator=gen(3)).to(torch.bfloat16)
    _native.device_status(reset=True)
    out, lse = A.kv4_attention(q, cache, table[:, :0], n, return_lse=True)
    assert bool((out == 0).all()) and bool((lse == -float("inf")).all())
    assert _native.device_status(reset=True) == 8
    A.kv4_attention(q, cache, table[:, :0], ints(0))
    assert _native.device_status() == 0
