"""The layers on 8-bit checkpoints as programs use them: together, under the Controller, in captured graphs, on other streams, under
autocast, with memory that is not theirs beside them, and beyond 2^31 elements."""
import copy

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

import gact
from gact import layers, ops
from gact.conf import config
from gact.controller import Controller
from gact.cpp_extension import _abi
from layer_reference import gamma, half_step

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _restore_config():
    saved = copy.copy(config.__dict__)
    yield
    config.__dict__.update(saved)


def normal(*shape, dtype=torch.float32, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed + 31 * len(shape))
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def block_parameters(width, hidden, dtype):
    return [p.requires_grad_() for p in (1 + normal(width, dtype=dtype, seed=1, scale=0.1), normal(width, dtype=dtype, seed=2, scale=0.1),
                                         normal(hidden, width, dtype=dtype, seed=3, scale=width ** -0.5), normal(hidden, dtype=dtype, seed=4, scale=0.1),
                                         normal(width, hidden, dtype=dtype, seed=5, scale=hidden ** -0.5), normal(width, dtype=dtype, seed=6, scale=0.1))]


def block(x, nw, nb, w1, b1, w2, b2):
    """A transformer's feed-forward block: x + W2 gelu(W1 norm(x) + b1) + b2."""
    return ops.op_linear(ops.op_linear(ops.op_layer_norm(x, nw, nb), w1, b1, "gelu"), w2, b2, None, x)


def exact_block(x, nw, nb, w1, b1, w2, b2):
    return x + F.linear(F.gelu(F.linear(F.layer_norm(x, (x.shape[-1],), nw, nb), w1, b1)), w2, b2)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape,hidden", [((2, 37, 96), 384), ((300, 771), 1285), ((4, 256, 256), 1024)])
def test_block_is_the_chain_of_its_operators(shape, hidden, dtype):
    x, p = normal(*shape, dtype=dtype).requires_grad_(), block_parameters(shape[-1], hidden, dtype)
    dy = normal(*shape, dtype=dtype, seed=9)
    y = block(x, *p)
    grads = torch.autograd.grad(y, [x] + p, dy)
    again = torch.autograd.grad(block(x, *p), [x] + p, dy)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))          # nothing is drawn, no sum depends on timing
    # each operator by itself, its gradients handed on by hand
    leaf = lambda t: t.detach().requires_grad_()  # noqa: E731
    n = ops.op_layer_norm(x, p[0], p[1])
    n1 = leaf(n)
    h = ops.op_linear(n1, p[2], p[3], "gelu")
    h1, x1 = leaf(h), leaf(x)
    out = ops.op_linear(h1, p[4], p[5], None, x1)
    assert torch.equal(out, y)
    dh, dw2, db2, dres = torch.autograd.grad(out, [h1, p[4], p[5], x1], dy)
    dn, dw1, db1 = torch.autograd.grad(h, [n1, p[2], p[3]], dh)
    dx, dnw, dnb = torch.autograd.grad(n, [x, p[0], p[1]], dn)
    for got, want in zip(grads, (dx + dres, dnw, dnb, dw1, db1, dw2, db2)):
        assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_block_gradients_are_near_the_uncompressed_ones(dtype):
    """256 normal values span about 5.6 deviations, so a code's error, uniform over a 255th of that, is 0.0063 deviations; a product
    of a thousand independent terms keeps that as its relative error.  The norm's, the first layer's (input and pre-activation) and the
    second layer's checkpoints add up to at most twice that, and the type's own rounding at a few places to a few half steps."""
    x, p = normal(1024, 256, dtype=dtype).requires_grad_(), block_parameters(256, 1024, dtype)
    dy = normal(1024, 256, dtype=dtype, seed=9)
    grads = torch.autograd.grad(block(x, *p), [x] + p, dy)
    X, P = x.detach().double().requires_grad_(), [t.detach().double().requires_grad_() for t in p]
    y = exact_block(X, *P)
    wants = torch.autograd.grad(y, [X] + P, dy.double())
    out = block(x, *p)
    assert (out.double() - y).norm() <= 4 * half_step(dtype) * y.norm() + 1e-5 * y.norm()
    for name, got, want in zip(("x", "nw", "nb", "w1", "b1", "w2", "b2"), grads, wants):
        assert (got.double() - want).norm() <= (2 * 0.0063 + 6 * half_step(dtype)) * want.norm(), name


def test_checkpoints_take_the_memory_they_are_said_to():
    """Rows of 1024 halves: a byte for each and eight for 256 of them, where torch keeps two for each."""
    x, w = normal(4096, 1024, dtype=torch.bfloat16), normal(1024, 1024, dtype=torch.bfloat16).requires_grad_()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    y = ops.op_linear(x, w)
    kept = torch.cuda.memory_allocated() - before - y.numel() * 2
    assert kept <= 4096 * 1024 + 4096 * 4 * 8 + 4096        # (blocks of the allocator are whole 512 bytes)
    del y


class FeedForward(nn.Module):
    def __init__(self, width, hidden):
        super().__init__()
        self.norm, self.up, self.act, self.down = nn.LayerNorm(width), nn.Linear(width, hidden), nn.GELU(), nn.Linear(hidden, width)

    def forward(self, x):
        return x + self.down(self.act(self.up(self.norm(x))))


@pytest.mark.parametrize("level", ["L1", "L2"])
def test_controller_runs_a_models_layers_on_checkpoints(level, monkeypatch):
    torch.manual_seed(0)
    model = nn.Sequential(*[FeedForward(256, 512) for _ in range(2)], nn.Linear(256, 10)).cuda()
    x, target = torch.randn(64, 12, 256, device="cuda"), torch.randint(0, 10, (64 * 12,), device="cuda")

    def backprop():
        model.zero_grad(set_to_none=True)
        loss = F.cross_entropy(model(x).view(-1, 10), target)
        loss.backward()
        return loss.detach()

    exact_loss = backprop()
    exact = [p.grad.clone() for p in model.parameters()]
    gact.set_optimization_level(level)
    config.checkpoint_layers = True
    calls = []
    monkeypatch.setattr(layers, "op_linear", lambda *a: calls.append("linear") or ops.op_linear(*a))
    monkeypatch.setattr(layers, "op_layer_norm", lambda *a: calls.append("norm") or ops.op_layer_norm(*a))
    controller = Controller(model)
    controller.install_hook()
    try:
        loss = backprop()
        assert sorted(calls) == ["linear"] * 5 + ["norm"] * 2
        tensors = controller.quantizer.tid
        for p, want in zip(model.parameters(), exact):
            # the hooked GELU input at 4 bits (a 15th of the range in place of a 255th) is the coarsest part: 17 times 0.0063
            assert (p.grad - want).norm() <= 0.2 * want.norm() + 1e-7
        assert abs(loss - exact_loss) <= 1e-5 * abs(exact_loss)
        for _ in range(2):
            controller.iterate(backprop)
            backprop()
    finally:
        controller.uninstall_hook()
    assert type(model[2]) is nn.Linear
    # the linear layers' and norms' inputs never reach the hooks: without the swap the same pass saves more
    config.checkpoint_layers = False
    plain = Controller(model)
    with plain:
        backprop()
    assert 0 < tensors < plain.quantizer.tid


def test_autocast_is_torchs():
    x, w, b = normal(100, 64).requires_grad_(), normal(48, 64, seed=1).requires_grad_(), normal(48, seed=2).requires_grad_()
    nw = torch.ones(64, device="cuda", requires_grad=True)
    for dtype in (torch.bfloat16, torch.float16):
        with torch.autocast("cuda", dtype=dtype):
            y, n = ops.op_linear(x, w, b, "gelu"), ops.op_layer_norm(x.to(dtype), nw, None)
            m = layers.CheckpointedLinear(64, 48).cuda()(x)
        assert y.dtype is dtype and m.dtype is dtype and n.dtype is torch.float32
        grads = torch.autograd.grad(y.float().sum() + n.sum(), [x, w, b, nw])
        assert all(g.dtype is torch.float32 for g in grads)
        want = F.gelu(F.linear(x, w, b))
        # both operands, the result and the bias rounded to the type: each by half a step of its size
        size = F.linear(x.abs(), w.abs(), b.abs())
        assert ((y.float() - want).abs() <= 1.13 * 3.1 * half_step(dtype) * size + half_step(dtype) * want.abs() + 1e-5).all()


def test_only_what_is_asked_for():
    x, w, b, r = normal(80, 40), normal(24, 40, seed=1), normal(24, seed=2), normal(80, 24, seed=3)
    dy = normal(80, 24, seed=4)
    full = [t.clone().requires_grad_() for t in (x, w, b, r)]
    want = torch.autograd.grad(ops.op_linear(full[0], full[1], full[2], "silu", full[3]), full, dy)
    for n in range(4):
        args = [t.clone().requires_grad_(k == n) for k, t in enumerate((x, w, b, r))]
        got, = torch.autograd.grad(ops.op_linear(args[0], args[1], args[2], "silu", args[3]), [args[n]], dy)
        assert torch.equal(got, want[n])
    y = ops.op_linear(*full[:3], "silu", full[3])
    with pytest.raises(RuntimeError, match="backward through the graph a second time|Trying to backward"):
        torch.autograd.grad(y, full, dy)
        torch.autograd.grad(y, full, dy)
    y = ops.op_linear(*full[:3], "silu", full[3])
    g, = torch.autograd.grad(y, [full[0]], dy, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()
    changed = normal(24, 40, seed=5).requires_grad_()
    y = ops.op_linear(full[0], changed)
    with torch.no_grad():
        changed.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_gradients_that_are_broadcast_or_strided():
    x, w, b = normal(70, 48).requires_grad_(), normal(40, 48, seed=1).requires_grad_(), normal(40, seed=2).requires_grad_()
    nw = normal(48, seed=3).requires_grad_()
    for dy in (torch.ones((), device="cuda").expand(70, 40), normal(1, 40, seed=4).expand(70, 40), normal(40, 70, seed=5).t(),
               normal(70, 80, seed=6)[:, ::2], normal(70, 55, seed=7)[:, 3:43]):
        for act in (None, "gelu"):
            got = torch.autograd.grad(ops.op_linear(x, w, b, act), [x, w, b], dy)
            want = torch.autograd.grad(ops.op_linear(x, w, b, act), [x, w, b], dy.contiguous().clone())
            assert all(torch.equal(g, v) for g, v in zip(got, want))
    for dy in (torch.ones((), device="cuda").expand(70, 48), normal(48, 70, seed=8).t()):
        got = torch.autograd.grad(ops.op_layer_norm(x, nw), [x, nw], dy)
        want = torch.autograd.grad(ops.op_layer_norm(x, nw), [x, nw], dy.contiguous().clone())
        assert all(torch.equal(g, v) for g, v in zip(got, want))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_captured_training_steps_replay_like_eager_ones(dtype):
    """Two graphs of forward and backward pass, replayed in turn with eager passes and new data between."""
    sizes = [((600, 264), 520), ((70, 1000), 136)]
    made = []
    for shape, hidden in sizes:
        x, p = normal(*shape, dtype=dtype), [t.detach() for t in block_parameters(shape[-1], hidden, dtype)]
        dy = normal(*shape, dtype=dtype, seed=9)

        def step(x=x, p=p, dy=dy):      # leaves of its own: a graph's backward pass belongs to the stream of its forward pass
            leaves = [t.detach().requires_grad_() for t in [x] + p]
            y = block(*leaves)
            return [y.detach()] + list(torch.autograd.grad(y, leaves, dy))

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        made.append((x, dy, step, graph, outs))
    for rep in range(4):
        for n, (x, dy, _, graph, _) in enumerate(made):
            x.copy_(normal(*x.shape, dtype=dtype, seed=50 + 2 * rep + n))
            dy.copy_(normal(*x.shape, dtype=dtype, seed=70 + 2 * rep + n))
            graph.replay()
        for x, dy, step, _, outs in made:
            for got, want in zip(outs, step()):
                assert torch.equal(got, want), rep
        torch.cuda.synchronize()


def test_a_capture_beside_an_eager_graph_of_its_leaves_is_refused():
    """By the operator, before anything of autograd's is captured; without the eager graph the same capture goes through."""
    x, w = normal(40, 32).requires_grad_(), normal(24, 32, seed=1).requires_grad_()
    nw = torch.ones(32, device="cuda", requires_grad=True)
    eager = ops.op_linear(ops.op_layer_norm(x, nw), w)
    for call in (lambda: ops.op_linear(x, w), lambda: ops.op_layer_norm(x, nw)):
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="eager graph of one of its leaves"):
            with torch.cuda.graph(graph):
                call()
        with torch.no_grad():
            call()
    want = torch.autograd.grad(eager, [x, w, nw], torch.ones_like(eager))
    del eager
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.op_linear(ops.op_layer_norm(x, nw), w)
        got = torch.autograd.grad(y, [x, w, nw], torch.ones_like(y))
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_saved_tensors_go_through_hooks_and_come_back_as_they_were():
    x, w, b = normal(70, 48).requires_grad_(), normal(40, 48, seed=1).requires_grad_(), normal(40, seed=2).requires_grad_()
    nw = normal(48, seed=3).requires_grad_()
    dy, dn = normal(70, 40, seed=4), normal(70, 48, seed=5)
    calls = (lambda: (ops.op_linear(x, w, b, "gelu"), [x, w, b], dy), lambda: (ops.op_layer_norm(x, nw), [x, nw], dn))
    for call in calls:
        y, leaves, g = call()
        want = torch.autograd.grad(y, leaves, g)
        with torch.autograd.graph.save_on_cpu():
            y, leaves, g = call()
        assert all(torch.equal(a, c) for a, c in zip(torch.autograd.grad(y, leaves, g), want))
        for change in (lambda t: t.double(), lambda t: t[:1], lambda t: t.cpu(), lambda t: t.reshape(1, -1)):
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change):
                y, leaves, g = call()
            with pytest.raises(RuntimeError, match="gave back another tensor"):
                torch.autograd.grad(y, leaves, g)


def test_inference_mode_gives_the_same_results():
    x, w, b, nw = normal(70, 48), normal(40, 48, seed=1).requires_grad_(), normal(40, seed=2).requires_grad_(), normal(48, seed=3).requires_grad_()

    def step():
        h = ops.op_layer_norm(x, nw)
        c = ops.op_checkpoint(h.detach())
        return [h, ops.op_linear(h, w, b, "gelu"), ops.op_linear(h[:1], w, b), ops.op_restore(c), ops.op_checkpoint_product(normal(70, 24, seed=4), c)]

    want = step()
    with torch.inference_mode():
        got = step()
    assert all(t.is_inference() and not t.requires_grad for t in got)
    with torch.no_grad():
        plain = step()
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(got, want, plain))


def test_a_batch_of_gradients_is_refused():
    x, w, nw = normal(6, 16).requires_grad_(), normal(8, 16, seed=1).requires_grad_(), normal(16, seed=2).requires_grad_()
    for y, leaf in ((ops.op_linear(x, w), w), (ops.op_linear(x, w, None, "silu"), x), (ops.op_layer_norm(x, nw), nw)):
        with pytest.raises(RuntimeError):
            torch.autograd.grad(y, leaf, torch.ones(3, *y.shape, device="cuda"), is_grads_batched=True)


def test_two_streams_at_once():
    x, p = normal(2048, 256, dtype=torch.bfloat16), [t.detach() for t in block_parameters(256, 1024, torch.bfloat16)]
    dy = normal(2048, 256, dtype=torch.bfloat16, seed=9)

    def step():
        leaves = [t.detach().requires_grad_() for t in [x] + p]
        y = block(*leaves)
        return [y.detach()] + list(torch.autograd.grad(y, leaves, dy))

    want = step()
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for rep in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(step())
    torch.cuda.synchronize()
    for outs in got:
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_nothing_is_written_beside_the_results():
    """Results in the middle of larger memory, through the library's own entry points."""
    L = _abi.lib()
    stream = torch.cuda.current_stream().cuda_stream
    for dtype in (torch.float32, torch.bfloat16):
        code, esz = _abi.dtype_code(dtype), torch.empty((), dtype=dtype).element_size()
        for rows, inner, outer in ((3, 16, 9), (70, 24, 33), (130, 264, 257), (300, 72, 520), (24, 2056, 33), (100, 2104, 133)):
            guard = 4096
            held = []

            def room(nbytes):
                t = torch.full((nbytes + 2 * guard,), 0xA5, dtype=torch.uint8, device="cuda")
                held.append((t, nbytes))
                return t.data_ptr() + guard

            x, w = normal(rows, inner, dtype=dtype), normal(outer, inner, dtype=dtype, seed=1)
            g = F.pad(normal(rows, outer, dtype=dtype, seed=2), (0, -outer % 8)).contiguous()
            ldg = g.shape[1]
            ldz, gz = (outer + 15) // 16 * 16, (outer + 255) // 256
            ldc, gx = (inner + 15) // 16 * 16, (inner + 255) // 256
            z = [room(rows * ldz), room(rows * gz * 4), room(rows * gz * 4)]
            c = [room(rows * ldc), room(rows * gx * 4), room(rows * gx * 4)]
            for act, codes in ((0, None), (1, z[0])):
                assert L.gact_linear(x.data_ptr(), inner, w.data_ptr(), inner, None, None, 0, act, code, rows, inner, outer, room(rows * outer * esz),
                                     codes, ldz, z[1], z[2], room(L.gact_linear_workspace_bytes(code, rows, inner, outer, codes is not None)),
                                     stream) == 0
            assert L.gact_checkpoint(x.data_ptr(), code, rows, inner, inner, c[0], ldc, c[1], c[2], stream) == 0
            assert L.gact_restore(c[0], ldc, c[1], c[2], code, rows, inner, room(rows * inner * esz), stream) == 0
            assert L.gact_activation_backward(g.data_ptr(), ldg, z[0], ldz, z[1], z[2], 1, code, rows, outer, room(rows * ldg * esz), ldg,
                                              room(outer * esz), room(L.gact_activation_workspace_bytes(rows, outer)), stream) == 0
            wt = F.pad(w, (0, -inner % 8)).contiguous()
            assert L.gact_product(g.data_ptr(), ldg, wt.data_ptr(), wt.shape[1], code, rows, outer, inner, room(rows * inner * esz),
                                  room(L.gact_product_workspace_bytes(code, rows, inner, outer)), stream) == 0
            assert L.gact_checkpoint_product(g.data_ptr(), ldg, c[0], ldc, c[1], c[2], code, rows, outer, inner, room(outer * inner * esz),
                                             room(L.gact_product_workspace_bytes(code, outer, inner, rows)), stream) == 0
            st = room(rows * 8)
            assert L.gact_norm_forward(x.data_ptr(), inner, None, None, code, rows, inner, 1e-5, room(rows * inner * esz), c[0], ldc, c[1], c[2], st,
                                       stream) == 0
            assert L.gact_norm_backward(x.data_ptr(), inner, None, c[0], ldc, c[1], c[2], st, code, rows, inner, room(rows * inner * esz),
                                        room(inner * esz), room(inner * esz), room(L.gact_norm_workspace_bytes(rows, inner)), stream) == 0
            torch.cuda.synchronize()
            for t, n in held:
                assert (t[:guard] == 0xA5).all() and (t[guard + n:] == 0xA5).all(), (dtype, rows, inner, outer, n)


def test_beyond_32_bits_of_elements():
    """Offsets of rows past 2^31 elements: the last rows' results are those of the last rows alone, and sums see them."""
    rows, cols = 540000, 4096          # 2.2e9 elements
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
    tail = slice(rows - 300, rows)
    x[tail] = normal(300, cols, dtype=torch.bfloat16)
    x[:300] = normal(300, cols, dtype=torch.bfloat16, seed=1)
    w, b = normal(cols, dtype=torch.bfloat16, seed=2).requires_grad_(), normal(cols, dtype=torch.bfloat16, seed=3).requires_grad_()
    x.requires_grad_()
    y = ops.op_layer_norm(x, w, b)
    assert torch.equal(y[tail].detach(), ops.op_layer_norm(x[tail].detach(), w, b).detach())
    dy = torch.zeros_like(y)
    dy[tail] = normal(300, cols, dtype=torch.bfloat16, seed=4)
    dx, dw, db = torch.autograd.grad(y, [x, w, b], dy)
    xt = x[tail].detach().requires_grad_()
    want = torch.autograd.grad(ops.op_layer_norm(xt, w, b), [xt, w, b], dy[tail].contiguous())
    assert torch.equal(dx[tail], want[0]) and not dx[300:-300].any()
    for got, ref in ((dw, want[1]), (db, want[2])):      # 300 rows added up in another order
        assert ((got.float() - ref.float()).abs() <= 2 * half_step(torch.bfloat16) * ref.float().abs() + gamma(300) * 300).all()
    del y, dy, dx
    kept = ops.op_checkpoint(x)
    assert torch.equal(ops.op_restore(kept)[tail], ops.op_restore(ops.op_checkpoint(x[tail])))
    g = torch.zeros(rows, 8, dtype=torch.bfloat16, device="cuda")
    g[tail] = normal(300, 8, dtype=torch.bfloat16, seed=5)
    got = ops.op_checkpoint_product(g, kept)
    want = g[tail].double().t().contiguous() @ ops.op_restore(ops.op_checkpoint(x[tail])).double()
    size = g[tail].double().abs().t().contiguous() @ x[tail].detach().double().abs()
    assert ((got.double() - want).abs() <= gamma(rows) * size + half_step(torch.bfloat16) * want.abs()).all()
    del kept
    # y and dz of 2.2e9 elements
    xs, ws = torch.zeros(rows, 64, dtype=torch.bfloat16, device="cuda"), normal(cols, 64, dtype=torch.bfloat16, seed=6, scale=0.1)
    xs[tail] = normal(300, 64, dtype=torch.bfloat16, seed=7)
    xs.requires_grad_()
    y = ops.op_linear(xs, ws, None, "gelu")
    ref = F.gelu(xs[tail].double() @ ws.double().t().contiguous())
    assert ((y[tail].double() - ref).abs() <= half_step(torch.bfloat16) * ref.abs() + 1e-4).all() and not y[: rows - 300].any()
    dy = x.detach()
    dx, = torch.autograd.grad(y, [xs], dy)
    xt = xs[tail].detach().requires_grad_()
    want, = torch.autograd.grad(ops.op_linear(xt, ws, None, "gelu"), [xt], dy[tail].contiguous())
    scale = want.float().abs().max()
    assert ((dx[tail].float() - want.float()).abs() <= 4 * half_step(torch.bfloat16) * (want.float().abs() + 0.05 * scale)).all()
