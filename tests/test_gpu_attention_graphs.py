"""Attention of few queries with a bias in recorded graphs: the splits of the keys, their join, and the bias as the kernels add it, whose workspaces are the
graph's own."""
import pytest
import torch

from gact import ops

pytestmark = pytest.mark.gpu


def normal(*shape, dtype=torch.float32, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed + 7919 * sum(shape))
    return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("batch,heads,kv_heads,queries,keys,width", [(1, 2, 2, 1, 3000, 64), (2, 8, 2, 3, 9001, 128), (5, 4, 4, 1, 517, 72)])
def test_few_queries_with_a_bias_that_changes(dtype, batch, heads, kv_heads, queries, keys, width):
    q, k, v = normal(batch, heads, queries, width, dtype=dtype), normal(batch, kv_heads, keys, width, dtype=dtype, seed=1), normal(batch, kv_heads, keys, width, dtype=dtype, seed=2)
    table = normal(32, heads, dtype=dtype, seed=3)
    bias = normal(heads, queries + keys - 1, seed=4)
    mask = torch.rand(batch, keys, generator=torch.Generator().manual_seed(5)).cuda() < 0.8

    def run():
        with torch.no_grad():
            return [ops.op_attention(q, k, v, bias, mask, True), ops.op_attention(q, k, v, ops.op_position_bias(table, queries, keys), mask)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run()
        graphs.append((graph, out))
    last = None
    for turn in range(4):
        for t in (q, k, v, table):
            t.mul_(0.9).add_(0.01 * turn)
        bias.copy_(normal(*bias.shape, seed=10 + turn))
        mask.logical_xor_(torch.rand(batch, keys, generator=torch.Generator().manual_seed(20 + turn)).cuda() < 0.1)
        for graph, out in graphs:
            graph.replay()
        want = run()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))
        # the bias is looked at: without it the result is another
        with torch.no_grad():
            assert not torch.equal(want[0], ops.op_attention(q, k, v, None, mask, True))
        assert last is None or not torch.equal(last, want[0])
        last = want[0]
