"""The layers on 8-bit checkpoints where they are called in other ways than a plain training step: autocast, the Controller's and other hooks for
saved tensors, transforms, traces and modes, recomputation, several threads."""
import copy
import threading
import time

import pytest
import torch
import torch.nn as nn

from gact import layers
from gact.conf import config
from gact.controller import Controller

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _restore_config():
    saved = copy.copy(config.__dict__)
    yield
    config.__dict__.update(saved)


def normal(*shape, dtype=torch.float32, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed + 31 * len(shape))
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_autocast_under_the_hooks_keeps_the_weights_as_they_are(dtype):
    """The hooks compress what a layer saves, but for a model's parameters: none of these layers' tensors is theirs."""
    config.checkpoint_layers, config.auto_prec, config.bit = True, False, 2
    model = nn.Sequential(nn.Linear(64, 48), nn.LayerNorm(48), nn.Linear(48, 40)).cuda()
    x, dy = normal(130, 64).requires_grad_(), normal(130, 40, dtype=dtype, seed=1)
    leaves = [x] + list(model.parameters())

    def step():
        with torch.autocast("cuda", dtype=dtype):
            y = model(x)
        return [y.detach()] + list(torch.autograd.grad(y, leaves, dy))

    changed = layers.attach(model)
    want = step()
    layers.detach(changed)
    controller = Controller(model)
    with controller:
        got = step()
    assert controller.quantizer.tid == 0
    assert all(torch.equal(a, b) and a.dtype is b.dtype for a, b in zip(got, want))
    assert all(g.dtype is torch.float32 for g in got[1:])


def test_autocast_keeps_no_copy_of_the_weight():
    """And its gradients are those of the weight rounded beforehand."""
    x, w = normal(70, 264, dtype=torch.bfloat16).requires_grad_(), normal(520, 264, seed=1, scale=0.1).requires_grad_()
    dy, rounded = normal(70, 520, dtype=torch.bfloat16, seed=2), w.detach().bfloat16().requires_grad_()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = layers.op_linear(x, w, None, "gelu")
    codes = 70 * (272 + 528) + 70 * (2 + 3) * 8
    assert torch.cuda.memory_allocated() - before <= y.numel() * 2 + codes + 7 * 512 < y.numel() * 2 + w.numel() * 2
    z = layers.op_linear(x, rounded, None, "gelu")
    assert torch.equal(y, z)
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    want = torch.autograd.grad(z, [x, rounded], dy)
    assert torch.equal(dx, want[0]) and dw.dtype is torch.float32 and torch.equal(dw, want[1].float())
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = layers.op_linear(x, w)
    with torch.no_grad():
        w.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, [x], dy)
    empty = torch.empty(0, 264, device="cuda", requires_grad=True)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = layers.op_linear(empty, w)
    dw, = torch.autograd.grad(y, [w], torch.empty_like(y))
    assert dw.dtype is torch.float32 and not dw.any()


def test_a_capture_beside_an_eager_graph_is_refused_under_autocast():
    """Whichever argument is the leaf: what the operator runs on is a copy of it, and its backward pass ends in the leaf."""
    x, w, b, r = normal(40, 32), normal(24, 32, seed=1), normal(24, seed=2), normal(40, 24, seed=3)
    half = normal(40, 32, dtype=torch.bfloat16)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        for n in range(4):
            args = [t.clone().requires_grad_(k == n) for k, t in enumerate((x, w, b, r))]
            eager = layers.op_linear(args[0], args[1], args[2], None, args[3])
            with pytest.raises(RuntimeError, match="eager graph of one of its leaves"):
                with torch.cuda.graph(torch.cuda.CUDAGraph()):
                    layers.op_linear(args[0], args[1], args[2], None, args[3])
            torch.autograd.grad(eager, [args[n]], torch.ones_like(eager))
            del eager
        leaf = half.clone().requires_grad_()
        eager = layers.op_layer_norm(leaf)
        with pytest.raises(RuntimeError, match="eager graph of one of its leaves"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                layers.op_layer_norm(leaf)


def test_refusals_under_autocast():
    x, w = normal(8, 16), normal(4, 16, seed=1)
    with torch.autocast("cuda", dtype=torch.float16):
        for bad in (lambda: layers.op_linear(x, w.double()), lambda: layers.op_linear(x.double(), w), lambda: layers.op_linear(x, w, normal(4).int()),
                    lambda: layers.op_layer_norm(x.double())):
            with pytest.raises(RuntimeError, match="type of"):
                bad()
        with pytest.raises(RuntimeError, match="dimension of bias"):
            layers.op_linear(x, w, normal(5))
        with pytest.raises(RuntimeError, match="dimension of weight"):
            layers.op_layer_norm(x, normal(8))
        with pytest.raises(RuntimeError, match="residual"):
            layers.op_linear(x, w, None, None, normal(8, 5))
        with pytest.raises(RuntimeError, match="CUDA"):
            layers.op_linear(x, w.cpu())


class Wrapped(torch.Tensor):
    """A tensor around another, as a distributed tensor is: torch's functions go past it, the dispatcher's operators come to it."""
    __torch_function__ = torch._C._disabled_torch_function_impl

    @staticmethod
    def __new__(cls, inner):
        t = torch.Tensor._make_wrapper_subclass(cls, inner.shape, dtype=inner.dtype, device=inner.device)
        t.inner = inner
        return t

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        bare = lambda v: v.inner if isinstance(v, cls) else v  # noqa: E731
        return torch.utils._pytree.tree_map_only(torch.Tensor, cls, func(*[bare(a) for a in args], **(kwargs or {})))


def pair(kind, *args, **kwargs):
    """The layer on checkpoints and torch's own, of the same parameters."""
    torch.manual_seed(0)
    own = kind(*args, **kwargs).cuda()
    layer = copy.deepcopy(own)
    for p in own.parameters():
        torch.nn.init.normal_(p, 0, 0.3)
    layer.load_state_dict(own.state_dict())
    assert len(layers.attach(layer)) == 1
    return layer, own


PAIRS = [(nn.Linear, 16, 8), (nn.LayerNorm, 16)]


@pytest.mark.parametrize("kind", PAIRS, ids=lambda k: k[0].__name__)
def test_transforms_of_the_layers_are_torchs(kind):
    from torch.func import functional_call, grad, jvp, vmap
    layer, own = pair(*kind)
    x, p = normal(5, 16), {n: t.detach() for n, t in own.named_parameters()}
    got, want = (grad(lambda q: functional_call(m, q, (x,)).square().sum())(p) for m in (layer, own))
    assert all(torch.equal(got[n], want[n]) for n in p)
    many = {n: torch.stack([t, 2 * t, -t]) for n, t in p.items()}
    got, want = (vmap(lambda q: functional_call(m, q, (x,)))(many) for m in (layer, own))
    assert got.shape[0] == 3 and torch.equal(got, want)
    got, want = (vmap(m)(normal(4, 5, 16, seed=1)) for m in (layer, own))
    assert torch.equal(got, want)
    got, want = (jvp(m, (x,), (normal(5, 16, seed=2),)) for m in (layer, own))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    got, want = (jvp(lambda q: functional_call(m, q, (x,)), (p,), (p,)) for m in (layer, own))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("kind", PAIRS, ids=lambda k: k[0].__name__)
def test_forward_mode_traces_and_modes_see_torchs_layers(kind):
    import torch.autograd.forward_ad as forward
    from torch._subclasses import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    layer, own = pair(*kind)
    x, t = normal(5, 16), normal(5, 16, seed=1)
    with forward.dual_level():
        got, want = (forward.unpack_dual(m(forward.make_dual(x, t))) for m in (layer, own))
        assert torch.equal(got.primal, want.primal) and torch.equal(got.tangent, want.tangent)
    with FakeTensorMode(allow_non_fake_inputs=True) as mode:
        assert layer(mode.from_tensor(x)).shape == own(mode.from_tensor(x)).shape
    traced = torch.jit.trace(layer, x)
    assert torch.equal(traced(t), own(t))
    graph = make_fx(layer)(x)
    assert torch.equal(graph(t), own(t))
    assert torch.equal(layer(Wrapped(x)).inner, own(x).detach())
    w = layer.weight
    del layer.weight
    layer.weight = Wrapped(w.detach())
    assert torch.equal(layer(x).inner, own(x).detach())


def test_sizes_that_the_operators_do_not_have_are_torchs():
    layer, own = pair(nn.Linear, 16, 8)
    x = normal(5, 16)
    for m in (layer, own):
        m.weight, m.bias = nn.Parameter(m.weight[:0]), None
    assert layer(x).shape == own(x).shape == (5, 0)
    layer, own = pair(nn.Linear, 16, 8)
    for m in (layer, own):
        m.bias = nn.Parameter(m.bias[:1])         # for all columns
    assert torch.equal(layer(x), own(x))
    layer, own = pair(nn.LayerNorm, 16)
    with pytest.raises(RuntimeError) as got:
        layer(normal(5, 8))
    with pytest.raises(RuntimeError) as want:
        own(normal(5, 8))
    assert str(got.value) == str(want.value)


def test_plain_calls_are_the_operators(monkeypatch):
    """With a default device set, too, which is a mode of torch's functions; any other such mode sees torch's."""
    calls = []
    linear, norm = layers.op_linear, layers.op_layer_norm
    monkeypatch.setattr(layers, "op_linear", lambda *a: calls.append("linear") or linear(*a))
    monkeypatch.setattr(layers, "op_layer_norm", lambda *a: calls.append("norm") or norm(*a))
    model = nn.Sequential(*(pair(*kind)[0] for kind in ((nn.LayerNorm, 16), (nn.Linear, 16, 8), (nn.Linear, 8, 8, False)))).cuda()
    x = normal(5, 16)
    for around in (torch.enable_grad(), torch.no_grad(), torch.device("cuda"), torch.autocast("cuda", dtype=torch.bfloat16)):
        calls.clear()
        with around:
            model(x), model(x[0]), model(x.view(1, 5, 16))
        assert calls == ["norm", "linear", "linear"] * 3

    class Seen(torch.overrides.TorchFunctionMode):
        def __torch_function__(self, func, types, args=(), kwargs=None):
            seen.append(func)
            return func(*args, **(kwargs or {}))

    calls.clear()
    seen = []
    with torch.device("cuda"), Seen():
        model(x)
    assert not calls and nn.functional.linear in seen and nn.functional.layer_norm in seen


def test_the_operators_themselves_are_not_traced():
    x, w = normal(5, 16), normal(8, 16, seed=1)
    kept = layers.op_checkpoint(x)
    for call in (lambda t: layers.op_linear(t, w), lambda t: layers.op_layer_norm(t), lambda t: layers.op_checkpoint(t).scale,
                 lambda t: layers.op_restore(kept), lambda t: layers.op_checkpoint_product(t, kept)):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.jit.trace(call, x)
    assert torch.equal(layers.op_linear(x, w), layers.op_linear(x, w))          # and are none the worse for it


def test_one_graph_differentiated_by_several_threads():
    """Each of them gets the gradients; of those that let go of what was saved the first one does."""
    x, w, nw = normal(600, 264).requires_grad_(), normal(136, 264, seed=1).requires_grad_(), normal(264, seed=2).requires_grad_()
    dy = normal(600, 136, seed=3)
    for retain in (True, False):
        y = layers.op_linear(layers.op_layer_norm(x, nw), w, None, "silu")
        want = torch.autograd.grad(y, [x, w, nw], dy, retain_graph=True)
        got, errors = [], []

        def run():
            try:
                got.append(torch.autograd.grad(y, [x, w, nw], dy, retain_graph=retain))
            except RuntimeError as e:
                errors.append(str(e))

        threads = [threading.Thread(target=run) for _ in range(4)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        torch.cuda.synchronize()
        assert len(got) + len(errors) == 4 and (len(got) == 4 if retain else got)
        assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))
        assert all("second time" in e for e in errors), errors


def test_gradients_of_empty_batches_are_not_differentiated_either():
    x, w, nw = torch.empty(0, 16, device="cuda", requires_grad=True), normal(8, 16).requires_grad_(), normal(16, seed=1).requires_grad_()
    for y, leaf in ((layers.op_linear(x, w, None, "gelu"), w), (layers.op_linear(x, w), x), (layers.op_layer_norm(x, nw), nw)):
        g, = torch.autograd.grad(y, [leaf], torch.empty_like(y).requires_grad_(), create_graph=True)
        assert not g.any()
        with pytest.raises(RuntimeError, match="once_differentiable"):
            g.sum().backward()


def test_a_product_of_a_gradient_with_a_history_is_not_differentiated():
    """Where a custom function's backward pass uses it under create_graph, say."""
    import torch.autograd.forward_ad as forward
    kept, g = layers.op_checkpoint(normal(70, 24)), normal(70, 16, seed=1)
    want = layers.op_checkpoint_product(g, kept)
    assert not want.requires_grad
    g.requires_grad_()
    with torch.no_grad():
        assert not layers.op_checkpoint_product(g, kept).requires_grad
    for grad, rows in ((g, kept), (torch.empty(0, 16, device="cuda", requires_grad=True), layers.op_checkpoint(normal(0, 24)))):
        got = layers.op_checkpoint_product(grad, rows)
        assert torch.equal(got.detach(), want if rows is kept else torch.zeros_like(want))
        with pytest.raises(RuntimeError, match="once_differentiable"):
            got.sum().backward()
    with forward.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            layers.op_checkpoint_product(forward.make_dual(g.detach(), g.detach()), kept)


def test_other_threads_go_on_while_a_call_waits_for_room_to_launch():
    """Behind a kernel that takes long, enough calls to fill the queue to the GPU: the one that finds it full waits without the GIL."""
    x, w = normal(8, 64), normal(16, 64, seed=1)
    kept, g = layers.op_checkpoint(x), normal(8, 16, seed=2)
    for call in (lambda: layers.op_layer_norm(x), lambda: layers.op_linear(x, w), lambda: layers.op_checkpoint(x), lambda: layers.op_restore(kept),
                 lambda: layers.op_checkpoint_product(g, kept)):
        call()
        torch.cuda.synchronize()
        gaps, done = [], threading.Event()

        def tick():
            last = time.perf_counter()
            while not done.is_set():
                time.sleep(0.0005)
                now = time.perf_counter()
                gaps.append(now - last)
                last = now

        ticking = threading.Thread(target=tick)
        ticking.start()
        longest, start = 0, time.perf_counter()
        torch.cuda._sleep(2000000000)
        for _ in range(40000):
            before = time.perf_counter()
            call()
            longest = max(longest, time.perf_counter() - before)
            if longest > 0.1 or before - start > 5:
                break
        done.set()
        ticking.join()
        torch.cuda.synchronize()
        if longest <= 0.1:
            pytest.skip("the queue was not full before the GPU was done")
        assert max(gaps) < longest / 2


def test_hooks_for_saved_tensors_may_give_back_other_addresses():
    """Everything that a pass saves in one buffer, one behind the other."""
    x, w, b = normal(70, 48).requires_grad_(), normal(40, 48, seed=1).requires_grad_(), normal(40, seed=2).requires_grad_()
    nw = normal(48, seed=3).requires_grad_()
    buffer, used = torch.empty(1 << 20, dtype=torch.uint8, device="cuda"), []

    def pack(t):
        size, start = t.element_size(), sum(used)
        start += -start % size + size        # as the type's alignment allows
        used.append(start + t.numel() * size - sum(used))
        place = buffer[start:start + t.numel() * size].view(t.dtype).view(t.shape)
        with torch.no_grad():
            place.copy_(t)
        return place

    for call, dy in ((lambda: layers.op_linear(x, w, b, "gelu"), normal(70, 40, seed=4)), (lambda: layers.op_layer_norm(x, nw), normal(70, 48, seed=5))):
        want = torch.autograd.grad(call(), [x, w, b, nw], dy, allow_unused=True)
        with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
            y = call()
        got = torch.autograd.grad(y, [x, w, b, nw], dy, allow_unused=True)
        assert all((g is None and v is None) or torch.equal(g, v) for g, v in zip(got, want))


def test_an_error_of_a_hook_for_saved_tensors_is_raised():
    x, w = normal(8, 64), normal(16, 64, seed=1).requires_grad_()

    def refuse(t):
        raise KeyError("not here")

    for call in (lambda: layers.op_linear(x, w, None, "gelu"), lambda: layers.op_layer_norm(x, w[0])):
        with torch.autograd.graph.saved_tensors_hooks(refuse, lambda t: t), pytest.raises(KeyError, match="not here"):
            call()
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, refuse):
            y = call()
        with pytest.raises(KeyError, match="not here"):
            y.sum().backward()


@pytest.mark.parametrize("kind", PAIRS, ids=lambda k: k[0].__name__)
def test_a_weight_that_is_computed_is_computed_once_a_call(kind):
    calls = []

    class Doubled(nn.Module):
        def forward(self, weight):
            calls.append(weight)
            return 2 * weight

    layer, own = pair(*kind)
    x = normal(5, 16)
    torch.nn.utils.parametrize.register_parametrization(layer, "weight", Doubled())
    calls.clear()
    y = layer(x)
    assert len(calls) == 1
    assert torch.equal(y, (layers.op_linear if kind[0] is nn.Linear else layers.op_layer_norm)(x, 2 * own.weight, own.bias))


def test_a_step_captured_under_autocast_sees_the_weights_as_they_are_at_replay():
    x, dy = normal(300, 72), normal(300, 72, dtype=torch.bfloat16, seed=1)
    state = [1 + normal(72, scale=0.1), normal(72, seed=2), normal(200, 72, scale=0.1), normal(200, seed=3), normal(72, 200, seed=4, scale=0.1), normal(72, seed=5)]

    def step():
        leaves = [t.detach().requires_grad_() for t in [x] + state]
        with torch.autocast("cuda", dtype=torch.bfloat16):
            h = layers.op_layer_norm(*leaves[:3])
            y = layers.op_linear(layers.op_linear(h, *leaves[3:5], "gelu"), *leaves[5:])
        return [y.detach()] + list(torch.autograd.grad(y, leaves, dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for rep in range(4):
        for n, p in enumerate(state):
            p.add_(normal(*p.shape, seed=100 * rep + n, scale=0.05))
        x.copy_(normal(300, 72, seed=7 + rep))
        graph.replay()
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)), rep
        torch.cuda.synchronize()


@pytest.mark.parametrize("reentrant", [False, True])
def test_recomputed_layers_give_the_same_gradients(reentrant):
    """torch's recomputation in the backward pass, which saves through hooks of its own and stops the forward pass halfway, by an exception."""
    from torch.utils.checkpoint import checkpoint
    model = nn.Sequential(*(nn.Sequential(nn.LayerNorm(64), nn.Linear(64, 200), nn.Linear(200, 64)) for _ in range(3))).cuda()
    x, dy = normal(70, 64).requires_grad_(), normal(70, 64, seed=1)
    config.checkpoint_layers, config.auto_prec = True, False
    leaves, seen = [x] + list(model.parameters()), []

    def grads(run, hooked=False):
        for t in leaves:
            t.grad = None
        if hooked:
            with Controller(model) as controller:
                run(x).backward(dy)
            seen.append(controller.quantizer.tid)
        else:
            changed = layers.attach(model)
            run(x).backward(dy)
            layers.detach(changed)
        return [t.grad for t in leaves]

    def recomputed(h):
        for part in model:
            h = checkpoint(part, h, use_reentrant=reentrant)
        return h

    want = grads(model)
    assert all(torch.equal(a, b) for a, b in zip(grads(recomputed), want))
    # of what is saved only the parts' inputs, which recomputation keeps, are for the Controller's hooks to compress
    grads(recomputed, True)
    assert seen == [3]
