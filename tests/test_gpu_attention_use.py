"""Attention and the position bias as a program uses them: hooks for saved tensors, autocast, streams, graphs, layers together."""
import math

import pytest
import torch

import gact
from gact import ops
from gact.conf import config
from gact.controller import Controller
from attention_reference import attend
from layer_reference import close, half_step

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
ids = lambda v: str(v).replace("torch.", "") if isinstance(v, torch.dtype) else None  # noqa: E731


@pytest.fixture(autouse=True)
def _restore_config():
    saved = dict(config.__dict__)
    yield
    config.__dict__.clear()
    config.__dict__.update(saved)


def normal(*shape, dtype=torch.float32, seed=0):
    g = torch.Generator().manual_seed(seed + 7919 * sum(shape))
    return torch.randn(*shape, generator=g).to(dtype).cuda()


# ---- the position bias ----
def bucket_of(d, buckets, both, most):
    """In whole numbers."""
    if both and d > 0:
        return buckets // 2 + bucket_of(-d, buckets // 2, False, most)
    per, away = (buckets // 2, abs(d)) if both else (buckets, max(0, -d))
    near = per // 2
    if away < near:
        return away
    steps, k = per - near, 0
    while k + 1 < steps and away ** steps * near ** (k + 1) >= most ** (k + 1) * near ** steps:
        k += 1
    return near + k


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("buckets,heads,queries,keys,both,most", [(32, 4, 1, 1, True, 128), (32, 12, 197, 197, True, 128), (32, 1, 300, 300, False, 128), (4, 3, 5, 50, True, 20),
                                                                  (2, 2, 40, 30, False, 7), (64, 9, 1, 2000, False, 1000), (6, 17, 100, 3, True, 9),
                                                                  (512, 2, 700, 700, True, 129), (10, 5, 64, 64, False, 6)])
def test_position_bias(buckets, heads, queries, keys, both, most, dtype):
    table = normal(buckets, heads, dtype=dtype).requires_grad_()
    got = ops.op_position_bias(table, queries, keys, both, most)
    at = torch.tensor([bucket_of(t - (keys - 1), buckets, both, most) for t in range(queries + keys - 1)], device="cuda")
    assert got.dtype is torch.float32 and torch.equal(got, table.detach().float()[at].t())
    grad = normal(heads, queries + keys - 1, seed=1)
    d_table = torch.autograd.grad(got, table, grad)[0]
    want = torch.zeros(buckets, heads, dtype=torch.float64, device="cuda").index_add_(0, at, grad.t().double())
    size = torch.zeros_like(want).index_add_(0, at, grad.t().double().abs())
    assert d_table.dtype is dtype
    # sums of up to all distances in 32 bits, rounded once
    close(d_table, want, (queries + keys + 16) * 2.0 ** -24 * size + half_step(dtype) * want.abs() + torch.finfo(dtype).smallest_normal, "table")


def test_position_bias_of_large_sizes_and_strides():
    table = normal(32, 64, dtype=torch.bfloat16)
    long = ops.op_position_bias(table, 1, 1 << 20, False)
    assert long.shape == (64, 1 << 20) and torch.equal(long[:, 0], table[31].float()) and torch.equal(long[:, -1], table[0].float())
    assert torch.equal(ops.op_position_bias(table.t().contiguous().t(), 9, 9), ops.op_position_bias(table, 9, 9))
    leaf = table.clone().requires_grad_()
    y = ops.op_position_bias(leaf, 9, 9)
    assert torch.equal(torch.autograd.grad(y.sum(), leaf, retain_graph=True)[0], torch.autograd.grad(y, leaf, torch.ones_like(y))[0])
    with pytest.raises(RuntimeError, match="heads"):
        ops.op_position_bias(torch.zeros(32, 0, device="cuda"), 9, 9)


# ---- together ----
class Layer(torch.nn.Module):
    """One layer of an encoder on the package's operators, or in torch's own."""

    def __init__(self, width, heads, dtype):
        super().__init__()
        self.heads = heads
        self.norm, self.second = (torch.nn.LayerNorm(width) for _ in range(2))
        self.qkv, self.out = torch.nn.Linear(width, 3 * width), torch.nn.Linear(width, width)
        self.up, self.down = torch.nn.Linear(width, 4 * width), torch.nn.Linear(4 * width, width)
        self.table = torch.nn.Parameter(0.5 * torch.randn(32, heads))
        self.to(dtype).cuda()

    def forward(self, x, mask, own):
        b, n, w = x.shape
        if own:
            h = ops.op_linear(ops.op_layer_norm(x, self.norm.weight, self.norm.bias), self.qkv.weight, self.qkv.bias)
        else:
            h = self.qkv(self.norm(x))
        q, k, v = h.view(b, n, 3, self.heads, -1).permute(2, 0, 3, 1, 4)
        bias = ops.op_position_bias(self.table, n, n)
        if own:
            h = ops.op_attention(q, k, v, bias, mask).transpose(1, 2).reshape(b, n, w)
            x = ops.op_linear(h, self.out.weight, self.out.bias, residual=x)
            h = ops.op_linear(ops.op_layer_norm(x, self.second.weight, self.second.bias), self.up.weight, self.up.bias, "gelu")
            return ops.op_linear(h, self.down.weight, self.down.bias, residual=x)
        i = torch.arange(n, device="cuda")
        s = q @ k.mT / math.sqrt(w // self.heads) + bias[:, i[None, :] - i[:, None] + n - 1]
        p = torch.softmax(s.masked_fill(~mask[:, None, None, :], -math.inf), 3)
        x = x + self.out((p @ v).transpose(1, 2).reshape(b, n, w))
        return x + self.down(torch.nn.functional.gelu(self.up(self.second(x))))


def test_a_layer_of_an_encoder_trains_on_the_operators():
    torch.manual_seed(1)
    layer = Layer(128, 4, torch.float32)
    x, dy = normal(3, 50, 128), normal(3, 50, 128, seed=1)
    mask = torch.arange(50, device="cuda")[None] < torch.tensor([50, 20, 33], device="cuda")[:, None]
    grads = []
    for own in (True, False):
        layer.zero_grad(set_to_none=True)
        y = layer(x, mask, own)
        y.backward(dy)
        grads.append([y.detach()] + [p.grad for p in layer.parameters()])
    for a, b in zip(*grads):
        # the layers' 8-bit checkpoints are within half a 255th of a row's range: a few thousandths of the gradients
        assert (a - b).norm() <= 0.02 * b.norm()
    # and the optimizer's step of all of it
    optimizer = gact.optim.AdamW(layer.parameters(), lr=1e-3)
    before = [p.detach().clone() for p in layer.parameters()]
    optimizer.step()
    assert all(not torch.equal(a, b) and torch.isfinite(a).all() for a, b in zip(layer.parameters(), before))


# ---- hooks ----
def test_under_hooks_the_gradients_are_those_of_what_the_hooks_give_back():
    q, k, v = (normal(2, 4, 96, 64, dtype=torch.float16, seed=s).requires_grad_() for s in range(3))
    dy, bias = normal(2, 4, 96, 64, dtype=torch.float16, seed=3), normal(4, 191, seed=4)
    saved = []

    def pack(t):
        saved.append(t)
        return t

    def unpack(t):
        return (t * 1.0625).detach() if t.dtype is torch.float16 else t

    with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
        y = ops.op_attention(q, k, v, bias)
    assert [tuple(t.shape) for t in saved] == [(2, 4, 96, 64)] * 3        # neither the result nor sums, nor the bias
    got = torch.autograd.grad(y, [q, k, v], dy)
    moved = [(t.detach() * 1.0625).requires_grad_() for t in (q, k, v)]
    want = torch.autograd.grad(ops.op_attention(*moved, bias), moved, dy)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_hooks_that_give_back_something_else_are_refused():
    q = normal(1, 2, 40, 32).requires_grad_()
    for other in (lambda t: t[:, :1], lambda t: t.double(), lambda t: t.cpu()):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, other):
            y = ops.op_attention(q, q, q)
        with pytest.raises(RuntimeError, match="gave back another tensor"):
            y.sum().backward()


@pytest.mark.parametrize("bit", [2, 4, 8])
def test_under_the_controller(bit):
    """Codes of few bits: probabilities of other values, which still add up to one - the gradients are finite and of the size of the exact ones."""
    config.auto_prec, config.bit = False, bit
    torch.manual_seed(0)
    model = torch.nn.Linear(64, 192).cuda()
    controller = Controller(model)
    x, dy = normal(4, 60, 64), normal(4, 60, 64, seed=1)

    def run():
        q, k, v = model(x).view(4, 60, 3, 4, 16).permute(2, 0, 3, 1, 4)
        model.zero_grad()
        (ops.op_attention(2 * q, k, v).transpose(1, 2).reshape(4, 60, 64) * dy).sum().backward()
        return model.weight.grad.clone()

    want = run()
    controller.install_hook()
    got = run()
    controller.uninstall_hook()
    assert torch.isfinite(got).all() and 0.2 * want.norm() <= got.norm() <= 5 * want.norm()
    if bit == 8:
        assert (got - want).norm() <= 0.05 * want.norm()


@pytest.mark.parametrize("hidden", [-math.inf, torch.finfo(torch.float32).min, -1e30])
def test_under_the_controller_a_bias_hides_what_it_hid(hidden):
    config.auto_prec, config.bit, config.compress_bool_masks = False, 8, True
    torch.manual_seed(0)
    model = torch.nn.Linear(64, 192).cuda()
    bias = normal(4, 119, seed=2)
    bias[:, 70:] = hidden        # keys more than ten behind the query
    bias.requires_grad_()
    mask = torch.rand(4, 60, generator=torch.Generator().manual_seed(3)).cuda() < 0.8
    controller = Controller(model)
    x, dy = normal(4, 60, 64), normal(4, 60, 64, seed=1)

    def run():
        q, k, v = model(x).view(4, 60, 3, 4, 16).permute(2, 0, 3, 1, 4)
        y = ops.op_attention(2 * q, k, v, bias, mask).transpose(1, 2).reshape(4, 60, 64)
        return torch.autograd.grad((y * dy).sum(), [model.weight, bias])

    want = run()
    controller.install_hook()
    got = run()
    controller.uninstall_hook()
    # codes of 8 bits: steps of 1/255 of a group's range, which is some six deviations, of three factors
    for a, b in zip(got, want):
        assert (a - b).norm() <= 0.05 * b.norm()
    assert (got[1][:, 70:] == 0).all()


def test_a_bias_that_changes_before_the_backward_pass_is_refused():
    q, k, v = (normal(1, 2, 40, 32, seed=s).requires_grad_() for s in range(3))
    bias = normal(2, 79, seed=3)
    for hooks in (torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t), torch.enable_grad()):
        with hooks:
            y = ops.op_attention(q, k, v, bias)
        bias.add_(1.0)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()


def test_memory_that_is_kept():
    """A float32 training pass keeps q, k, v, the result and one float per query: nothing of queries x keys."""
    q, k, v = (normal(1, 4, 1024, 32, seed=s).requires_grad_() for s in range(3))
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    y = ops.op_attention(q, k, v)
    kept = torch.cuda.memory_allocated() - before
    assert kept <= y.numel() * 4 + 4 * 1024 * 4 + 4096
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    torch.autograd.grad(y.sum(), [q, k, v])
    # three gradients, that of the sum as a dense tensor, one float per query; floats of dk and dv from the 8 splits (two tiles of 64 queries each) of the
    # 32 tiles of 128 keys, which are fewer than the compute units
    assert torch.cuda.max_memory_allocated() - before <= (6 + 2 * 8) * y.numel() * 4 + (1 << 20)


# ---- autocast, modes, captures ----
def test_autocast():
    q, k, v = (normal(2, 4, 70, 64, seed=s).requires_grad_() for s in range(3))
    bias = normal(4, 139, seed=3).requires_grad_()
    for dtype in (torch.bfloat16, torch.float16):
        with torch.autocast("cuda", dtype):
            y = ops.op_attention(q, k, v, bias)
        assert y.dtype is dtype
        grads = torch.autograd.grad(y, [q, k, v, bias], torch.ones_like(y))
        low = [t.detach().to(dtype).requires_grad_() for t in (q, k, v)] + [bias]
        same = ops.op_attention(*low)
        assert torch.equal(same, y)
        for a, b in zip(grads, torch.autograd.grad(same, low, torch.ones_like(same))):
            assert a.dtype is torch.float32 and torch.equal(a, b.float())
    with torch.autocast("cuda", torch.bfloat16):
        half_bias = ops.op_attention(q, k, v, bias.half())
    assert half_bias.dtype is torch.bfloat16


def test_another_stream():
    q, k, v, dy = (normal(4, 8, 256, 64, dtype=torch.bfloat16, seed=s) for s in range(4))
    want = [t.detach() for t in train(q, k, v, dy)]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = train(q * 1, k * 1, v * 1, dy * 1)
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def train(q, k, v, dy, bias=None):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    y = ops.op_attention(*leaves, bias)
    return [y] + list(torch.autograd.grad(y, leaves, dy))


def test_graphs_are_captured_and_replayed():
    shapes = [(2, 4, 100, 64), (1, 2, 1, 64)]
    static = [[normal(*s, dtype=torch.float16, seed=n) for n in range(4)] for s in shapes]
    # one token behind a longer cache: splits and their join
    static[1][1:3] = [normal(1, 2, 3000, 64, dtype=torch.float16, seed=9 + n) for n in range(2)]
    bias = normal(2, 3000, seed=8)

    def run():
        first = train(*static[0])
        with torch.no_grad():
            return [t.detach() for t in first] + [ops.op_attention(*static[1][:3], bias)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):      # two graphs, each with workspaces of its own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run()
        graphs.append((graph, out))
    for turn in range(4):
        with torch.no_grad():
            for group in static:
                for t in group:
                    t.mul_(0.9).add_(0.01 * turn)
            bias.mul_(0.5)
        for graph, out in graphs:
            graph.replay()
        want = [t.detach() for t in run()]
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_a_bias_and_short_sequences_train_in_graphs():
    """The table's gradient from a backward pass in splits, and sequences that one kernel takes, replayed with other values and the eager pass in between."""
    q, k, v, dy = (normal(1, 2, 700, 64, dtype=torch.float16, seed=n) for n in range(4))
    table = normal(32, 2, dtype=torch.float16, seed=4)
    short = [normal(40, 3, 49, 32, seed=n) for n in range(4)]

    def run():
        leaves = [t.detach().requires_grad_() for t in (q, k, v, table)]
        y = ops.op_attention(*leaves[:3], ops.op_position_bias(leaves[3], 700, 700), None, True)
        return [t.detach() for t in [y] + list(torch.autograd.grad(y, leaves, dy)) + train(*short)]

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
    for turn in range(4):
        for t in [q, k, v, dy, table] + short:
            t.mul_(0.9).add_(0.01 * turn)
        for graph, out in graphs:
            graph.replay()
        want = run()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_a_capture_beside_an_eager_graph_of_the_same_leaves_is_refused():
    q = normal(1, 2, 40, 32).requires_grad_()
    alive = ops.op_attention(q, q, q)
    table = normal(32, 2).requires_grad_()
    bias = ops.op_position_bias(table, 40, 40)
    # the accumulators exist once a graph is alive
    alive.sum().backward(retain_graph=True)
    bias.sum().backward(retain_graph=True)
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        graph.capture_begin()
        try:
            for call in (lambda: ops.op_attention(q, q, q), lambda: ops.op_position_bias(table, 40, 40)):
                with pytest.raises(RuntimeError, match="eager graph"):
                    call()
        finally:
            graph.capture_end()
    torch.cuda.synchronize()


def test_refusals_on_the_gpu():
    q, k = normal(2, 4, 8, 32), normal(2, 2, 9, 32)
    for call, text in ((lambda: ops.op_attention(q, k, k[:, :, :8]), "key's shape"), (lambda: ops.op_attention(q, k.half(), k), "type of key"),
                       (lambda: ops.op_attention(q[0], k, k), "batch, heads"), (lambda: ops.op_attention(q[:1], k, k), "batch and width"),
                       (lambda: ops.op_attention(q[:, :3], k, k), "multiple"), (lambda: ops.op_attention(q[:, :0], k, k), "multiple"),
                       (lambda: ops.op_attention(q, k, k, torch.zeros(4, 15, device="cuda")), "bias must be"),
                       (lambda: ops.op_attention(q, k, k, torch.zeros(4, 16, device="cuda").half()), "type of bias"),
                       (lambda: ops.op_attention(q, k, k, None, torch.ones(2, 8, dtype=torch.bool, device="cuda")), "mask must be"),
                       (lambda: ops.op_attention(q, k, k, None, torch.ones(2, 9, device="cuda")), "type of mask"),
                       (lambda: ops.op_attention(q, k, k, scale=0.0), "positive"), (lambda: ops.op_attention(q, k, k, scale=-1.0), "positive"),
                       (lambda: ops.op_attention(q, k, k, scale=math.inf), "positive"), (lambda: ops.op_attention(q, k, k, scale=math.nan), "positive"),
                       (lambda: ops.op_attention(*[torch.zeros(1, 1, 4, 129, device="cuda")] * 3), "1 to 128"),
                       (lambda: ops.op_position_bias(torch.zeros(7, 2, device="cuda"), 4, 4), "even number"),
                       (lambda: ops.op_position_bias(torch.zeros(32, 2, device="cuda"), 0, 4), "queries and keys"),
                       (lambda: ops.op_position_bias(torch.zeros(32, 2, device="cuda"), 4, 4, True, 8), "max_distance"),
                       (lambda: ops.op_position_bias(torch.zeros(514, 2, device="cuda"), 4, 4), "buckets"),
                       (lambda: ops.op_position_bias(torch.zeros(32, 2, device="cuda").int(), 4, 4), "type of table")):
        with pytest.raises(RuntimeError, match=text):
            call()
    leaf = q.clone().requires_grad_()
    y = ops.op_attention(leaf, k, k)
    grad = torch.autograd.grad(y.sum(), leaf, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="differentiate twice"):
        grad.sum().backward()
    y = ops.op_attention(leaf, k, k)
    y.sum().backward()
    with pytest.raises(RuntimeError, match="second time"):
        y.sum().backward()
    y = ops.op_attention(leaf, k, k)
    with torch.no_grad():
        y.add_(1)       # what the backward pass would read
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()
    with pytest.raises(RuntimeError, match="forward-mode"):
        with torch.autograd.forward_ad.dual_level():
            ops.op_attention(torch.autograd.forward_ad.make_dual(q, q), k, k)
    with pytest.raises(RuntimeError, match="plain"):
        torch.func.vmap(lambda t: ops.op_attention(t, t, t))(normal(3, 1, 2, 8, 32))


def test_inference_mode_and_a_result_that_is_written_over():
    q = normal(1, 2, 40, 32, dtype=torch.bfloat16)
    with torch.inference_mode():
        y = ops.op_attention(q, q, q)
    assert torch.equal(y, ops.op_attention(q, q, q))
    close(y, *attend(q, q, q)["y"], "y")
