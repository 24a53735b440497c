"""The layer operators inside a CUDA graph, as a decoding loop captures them, and side by side on two streams."""
import pytest
import torch

import attnres_b200 as A
from attnres_b200 import _native

pytestmark = pytest.mark.gpu


class Step:
    """One layer's decoding step: projection output -> q, k, v -> cache -> attention, and the gated projection."""

    def __init__(self, B, H, D, tokens, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        new = lambda *s: torch.randn(*s, device="cuda", generator=g).to(torch.bfloat16)  # noqa: E731
        self.H, per = H, -(-tokens // 16)
        self.qkv, self.w = new(B, 1, 3 * H * D), new(2 * 96, H * D) / 16
        angle = torch.rand(tokens, D // 2, device="cuda", generator=g) * 6
        self.cos, self.sin = angle.cos(), angle.sin()
        self.cache = A.KV4Cache.empty(B * per, 16, H, D)
        for t in self.cache.tensors():
            t.zero_()
        self.table = torch.arange(B * per, device="cuda", dtype=torch.int32).view(B, per)
        self.n = torch.zeros(B, device="cuda", dtype=torch.int32)
        self.new = new

    def __call__(self):
        q, k, v = A.qk_norm_rope(self.qkv, self.H, self.H, self.cos, self.sin, positions=self.n[:, None])
        A.kv4_append(self.cache, k, v, self.table, self.n)
        out = A.kv4_attention(q, self.cache, self.table, self.n + 1)
        return out, A.swiglu_projection(out.flatten(2), self.w)


@pytest.mark.parametrize("tokens", [60, 400])  # one stretch, and several with their join
def test_decoding_loop_in_a_graph(tokens):
    a, b = Step(3, 2, 64, tokens, 1), Step(3, 2, 64, tokens, 1)
    inputs = [a.new(*a.qkv.shape) for _ in range(50)]
    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        b()
    torch.cuda.current_stream().wait_stream(warm)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = b()
        b.n.add_(1)
    b.n.zero_()
    for x in inputs:
        a.qkv.copy_(x)
        want = a()
        a.n.add_(1)
        b.qkv.copy_(x)
        graph.replay()
        for u, v in zip(got, want):
            assert torch.equal(u, v)
    assert _native.device_status() == 0


def test_two_streams_do_not_share_anything():
    steps = [Step(2, 4, 128, 200, s) for s in (1, 2)]
    alone = []
    for s in steps:
        for _ in range(20):
            out = s()
            s.n.add_(1)
        alone.append([t.clone() for t in out])
        s.n.zero_()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [None, None]
    for _ in range(20):
        for i, (s, st) in enumerate(zip(steps, streams)):
            with torch.cuda.stream(st):
                got[i] = s()
                s.n.add_(1)
    torch.cuda.synchronize()
    for x, y in zip(got, alone):
        for u, v in zip(x, y):
            assert torch.equal(u, v)


def test_training_step_in_a_graph():
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(300, 128, device="cuda", generator=g).to(torch.bfloat16).requires_grad_(True)
    w = (torch.randn(2 * 72, 128, device="cuda", generator=g) / 11).to(torch.bfloat16).requires_grad_(True)
    qkv = torch.randn(2, 40, 6 * 64, device="cuda", generator=g).to(torch.bfloat16).requires_grad_(True)
    qw = torch.ones(64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    cos = torch.rand(40, 32, device="cuda", generator=g)

    def step():
        h = A.swiglu_projection(x, w)
        q, k, v = A.qk_norm_rope(qkv, 2, 2, cos, cos, q_weight=qw)
        return torch.autograd.grad([h.float().square().sum(), (q * k).float().sum() + v.float().sum()], [x, w, qkv, qw])

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for t in got:
        t.zero_()
    graph.replay()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
