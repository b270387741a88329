"""Graphs captured on a handle and larger calls on it after them: replays use the workspace that they were captured with,
which the larger call has outgrown."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_replays_after_a_larger_call(hip):
    from tinygs_amd.network import LayerOps
    ops = LayerOps()
    g = torch.Generator().manual_seed(2)

    def inputs(rows, states):
        q, go = (torch.randn(rows, 128, generator=g).half().cuda() for _ in range(2))
        k, v = (torch.randn(states, 128, generator=g).half().cuda() for _ in range(2))
        return q, k, v, go

    def run(t):
        q, k, v, go = t
        out, lse = ops.attention(q, k, v, 2, keep_lse=True)
        return (out, lse) + ops.attention_backward(go, q, k, v, out, lse, 2)

    small, large = inputs(50, 600), inputs(900, 4000)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        want = [t.clone() for t in run(small)]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            got = run(small)
        first = [t.clone() for t in run(large)]   # grows the workspace: four times as many parts of longer rows
        for _ in range(3):
            for t in got:
                t.zero_()
            graph.replay()
            s.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(got, want))
            again = run(large)
            s.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(again, first))
