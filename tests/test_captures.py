"""Graphs captured on a stream that has run eager work, replayed beside each
other and beside that work (GPU)."""

import pytest
import torch

from turbopress_amd import hip_kernel as hk

pytestmark = pytest.mark.gpu


def test_graphs_captured_on_a_stream_with_eager_workspaces(cuda):
    """Split-K linears and attention run eagerly on a stream, then two graphs of
    both are captured there.  All three run at once, on three streams, and give
    what each gives alone."""
    from turbopress_amd import paged_attention
    from turbopress_amd.runtime import PackedTCQLinear
    from turbopress_amd.synthetic import make_activation, make_payload
    g = torch.Generator(device="cuda").manual_seed(1)
    lin = PackedTCQLinear(make_payload(9728, 2560, 3, 64, seed=1), mode="hip")
    xs = [make_activation(12, 2560, seed=i).to(cuda) for i in range(3)]
    qs = [torch.randn(2, 8, 64, generator=g, device="cuda").half() for _ in range(3)]
    k, v = (torch.randn(800, 16, 2, 64, generator=g, device="cuda").half() for _ in "kv")
    table = torch.randperm(800, generator=g, device="cuda").view(2, 400).int()
    lengths = torch.tensor([6400, 3001], dtype=torch.int32, device="cuda")

    def work(i):
        return paged_attention(qs[i], k, v, table, lengths), lin(xs[i])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = [[t.clone() for t in work(i)] for i in range(3)]
        eager = hk.shared_workspace(cuda, 1)
    torch.cuda.synchronize()
    graphs = []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs = work(i)
            mine = hk.shared_workspace(cuda, 1)
        assert mine.data_ptr() != eager.data_ptr()
        graphs.append((graph, outs, mine))
    assert graphs[0][2].data_ptr() != graphs[1][2].data_ptr()
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        for s, (graph, _, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        with torch.cuda.stream(side):
            got.append(work(2))
    torch.cuda.synchronize()
    # (the order of split-K sums may differ)
    for outs in ([graphs[0][1], want[0]], [graphs[1][1], want[1]], *([o, want[2]] for o in got)):
        (o, y), (o_want, y_want) = outs
        assert torch.equal(o, o_want)
        assert float((y.float() - y_want.float()).abs().max()) <= 2e-3 * float(y_want.float().abs().max())
