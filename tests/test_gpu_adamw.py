"""AdamW's step over many tensors on the GPU: states in 8 bits code for code, parameters within 32-bit arithmetic of the formula in 64 bits."""
import copy
import io
import math

import pytest
import torch

import gact
from gact import ops
from layer_reference import U, close, half_step, least

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
ids = lambda v: str(v).replace("torch.", "") if isinstance(v, torch.dtype) else None  # noqa: E731
UNITS = torch.tensor([127.0 ** 2, 4228250624.0], dtype=torch.float64)       # 255^4 as a float


def normal(*shape, dtype=torch.float32, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed + 7919 * sum(shape))
    return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda()


def groups_of(t):
    t = t.reshape(-1)
    return torch.cat([t, t.new_zeros(-t.numel() % 256)]).view(-1, 256)


def decode(m, v, scale):
    """float32 values of codes, by the format's roundings."""
    n, unit = m.numel(), (scale.double() / UNITS.cuda()).float()
    c, square = groups_of(m.float()), groups_of(v.float()).square()
    return (c * c.abs() * unit[:, :1]).view(-1)[:n], (square * square * unit[:, 1:]).view(-1)[:n]


def encode(m, v):
    n, gm, gv = m.numel(), groups_of(m), groups_of(v)
    scale = torch.stack([gm.abs().amax(1), gv.amax(1)], 1)
    scale = torch.where(scale < torch.tensor([1e-30, 1e-28], device="cuda"), torch.zeros_like(scale), scale)
    inverse = torch.where(scale > 0, (UNITS.cuda() / scale.double()).float(), torch.zeros_like(scale))
    # in 64 bits: how many borders (k - 1/2)^2, (k - 1/2)^4 there are up to the value
    c = torch.floor(torch.sqrt((gm.abs() * inverse[:, :1]).double()) + 0.5) * torch.sign(gm)
    d = torch.floor(torch.sqrt(torch.sqrt((gv * inverse[:, 1:]).double())) + 0.5)
    d = torch.where((gv > 0) & (scale[:, 1:] > 0), d.clamp(min=1), d)
    return c.view(-1)[:n].to(torch.int8), d.view(-1)[:n].to(torch.uint8), scale


def step32(m, v, g, betas):
    """The float moments after a step: each product is rounded together with the sum, of which 64 bits hold all but the last bits."""
    g = g.float()
    b = torch.tensor(betas, dtype=torch.float32).tolist()
    rest = torch.tensor([1 - x for x in betas], dtype=torch.float32).tolist()
    return (m.double() * b[0] + (g * rest[0]).double()).float(), (v.double() * b[1] + (g * g * rest[1]).double()).float()


def param(p, m, v, step, lr, betas, eps, decay):
    """The parameter in 64 bits from float32 moments, and how far 32 bits may be off: each operation half a step, the factors from the host as well."""
    p, m, v = p.double(), m.double(), v.double()
    root = (v / (1 - betas[1] ** step)).sqrt() + eps
    update = torch.where(m == 0, torch.zeros_like(m), lr / (1 - betas[0] ** step) * m / root)
    want = p * (1 - lr * decay) - update
    return want, 8 * U * (p.abs() + update.abs()) + least(torch.float32)


def run(shapes, dtype, bits, steps=3, lr=1e-2, betas=(0.9, 0.999), eps=1e-8, decay=0.1, scale=1e-3, first=1):
    params = [normal(*s, dtype=dtype, seed=n) for n, s in enumerate(shapes)]
    states = [ops.op_adamw_state(p, bits) for p in params]
    for t in range(first, first + steps):
        grads = [(normal(*p.shape, seed=100 * t + n) * scale * 10.0 ** (n % 4 - 2)).to(dtype) for n, p in enumerate(params)]
        before = [(p.clone(), [None if x is None else x.clone() for x in s]) for p, s in zip(params, states)]
        ops.op_adamw(params, grads, states, t, lr, betas, eps, decay)
        for p, g, s, (old, kept) in zip(params, grads, states, before):
            m, v = decode(*kept) if bits == 8 else (kept[0].view(-1), kept[1].view(-1))
            m, v = step32(m, v, g.view(-1), betas)
            if bits == 8:
                c, d, most = encode(m, v)
                assert torch.equal(s.exp_avg.view(-1), c) and torch.equal(s.exp_avg_sq.view(-1), d) and torch.equal(s.scale, most)
                x, y = ops.op_adamw_values([s])
                assert all(torch.equal(a, b) for a, b in zip((x, y), decode(c, d, most)))
            else:
                assert torch.equal(s.exp_avg.view(-1), m) and torch.equal(s.exp_avg_sq.view(-1), v)
            want, off = param(old.view(-1), m, v, t, lr, betas, eps, decay)
            close(p.view(-1), want, off + half_step(dtype) * (want.abs() + off) + least(dtype), "param")
    return params, states


SHAPES = [(1,), (8,), (255,), (256,), (257,), (5, 7, 3), (2048,), (2049,), (64, 771), (3, 1), (300, 41)]


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("bits", [8, 32])
def test_steps(bits, dtype):
    run(SHAPES, dtype, bits)
    run([(70,), (600,)], dtype, bits, 2, 1e-3, (0.5, 0.75), 0.1, 0.0, first=100000)
    run([(513,)], dtype, bits, 2, 0.0, (0.0, 0.0), 1e-8, 0.0)


@pytest.mark.parametrize("bits", [8, 32])
def test_more_tensors_than_a_launch_takes(bits):
    run([(n % 5 + 1, n * 3 % 401 + 1) for n in range(200)], torch.float32, bits, 2)


def test_codes_of_every_value():
    """Values along the whole range of either state, and next to every border between two codes."""
    k = torch.arange(1, 256, dtype=torch.float64, device="cuda") - 0.5
    around = torch.cat([(k[:127] / 127) ** 2, torch.logspace(-12, 0, 500, dtype=torch.float64, device="cuda")]).float()
    m = torch.cat([around, torch.nextafter(around, around + 1), torch.nextafter(around, around - 1)])
    fourth = torch.cat([(k / 255) ** 4, torch.logspace(-14, 0, 500, dtype=torch.float64, device="cuda")]).float()
    v = torch.cat([fourth, torch.nextafter(fourth, fourth + 1), torch.nextafter(fourth, fourth - 1)])
    n = 255 * (-(-max(m.numel(), v.numel()) // 255))
    # each group's largest is 1; beta 0 makes the moments g and g^2 themselves
    for values, power in ((m, 1), (v, 0.5)):
        g = torch.cat([values.double() ** power, torch.zeros(n - values.numel(), dtype=torch.float64, device="cuda")]).float().view(-1, 255)
        g = torch.cat([g, torch.ones_like(g[:, :1])], 1).reshape(-1)
        g[::2] *= -1
        p, state = torch.zeros_like(g), ops.op_adamw_state(g, 8)
        ops.op_adamw([p], [g], [state], 1, betas=(0.0, 0.0))
        for got, want in zip(state, encode(g, g * g)):
            assert torch.equal(got.view(-1), want.view(-1))


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_groups_of_nothing_and_of_next_to_nothing(dtype):
    p = normal(1024, dtype=dtype)
    g = torch.zeros(1024, device="cuda")
    g[256:512] = 1e-33 if dtype is torch.float32 else 0
    g[512] = 1e-3
    g[768:] = 1e-3
    g[800] = 0
    g, state, old = g.to(dtype), ops.op_adamw_state(p, 8), p.clone()
    ops.op_adamw([p], [g], [state], 1, weight_decay=0.0)
    assert torch.equal(p[:256], old[:256]) and not state.scale[:2].any() and not state.exp_avg[:512].any() and not state.exp_avg_sq[:512].any()
    assert state.exp_avg[512] == 127 and state.exp_avg_sq[512] == 255 and not state.exp_avg_sq[513:768].any()
    assert state.exp_avg_sq[768] == 255 and state.exp_avg_sq[800] == 0
    # a second moment far below its group's largest keeps the least code, and the step stays bounded
    g[:] = 0
    g[1], g[2] = 1.0, 1e-4
    ops.op_adamw([p], [g], [state], 2, weight_decay=0.0)
    assert state.exp_avg_sq[2] >= 1 and torch.isfinite(p).all()


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_nan_and_infinity(dtype):
    for bad in (math.nan, math.inf):
        for bits in (8, 32):
            p, g = normal(1000, dtype=dtype), normal(1000, dtype=dtype, seed=1)
            g[300] = bad
            state = ops.op_adamw_state(p, bits)
            ops.op_adamw([p], [g], [state], 1)
            finite = torch.isfinite(p)
            assert not finite[300] and int(finite.sum()) == 999
            g[300] = 0
            ops.op_adamw([p], [g], [state], 2)
            finite = torch.isfinite(p)
            if bits == 8:      # the group
                assert not finite[256:512].any() and finite[:256].all() and finite[512:].all()
            else:
                assert not finite[300] and int(finite.sum()) == 999


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("bits", [8, 32])
def test_layouts(bits, dtype):
    """Parameters in any dense order of dimensions, at any address; gradients of any layout."""
    flat, other = normal(4000, dtype=dtype), normal(4000, dtype=dtype, seed=1, scale=1e-2)
    cases = [(flat[1:1001], other[3:1003]), (flat[:1200].view(30, 40).t(), other[:1200].view(30, 40).t()), (flat[:1200].view(30, 40).t(), other[:1200].view(40, 30)),
             (flat[:960].view(2, 4, 10, 12).to(memory_format=torch.channels_last), other[:960].view(2, 4, 10, 12)),
             (flat[:40].view(1, 40), other[:1].expand(1, 40)), (flat[:40], other[:80:2]), (flat[:40], torch._neg_view(other[:40]))]
    for p, g in cases:
        p = p.clone(memory_format=torch.preserve_format) if p.storage_offset() == 0 else p
        plain, grad = p.detach().contiguous().clone(), g.resolve_neg().contiguous().clone()
        state, same = ops.op_adamw_state(p, bits), ops.op_adamw_state(plain, 32)
        ops.op_adamw([p], [g], [state], 1)
        ops.op_adamw([plain], [grad], [same], 1)
        assert torch.equal(p, plain)
        if bits == 32:
            assert torch.equal(state.exp_avg, same.exp_avg)
    buffer = normal(100, dtype=dtype)
    kept = buffer.clone()
    ops.op_adamw([buffer[7:50]], [normal(43, dtype=dtype)], [ops.op_adamw_state(buffer[7:50].clone(), bits)], 1)
    assert torch.equal(buffer[:7], kept[:7]) and torch.equal(buffer[50:], kept[50:]) and not torch.equal(buffer[7:50], kept[7:50])


def test_types_and_bits_mixed_in_a_list():
    params = [normal(50, 7, dtype=d, seed=n) for n, d in enumerate(TYPES * 2)]
    grads = [normal(50, 7, dtype=p.dtype, seed=9 + n) for n, p in enumerate(params)]
    bits = [8, 8, 8, 32, 32, 32]
    alone = [p.clone() for p in params]
    ops.op_adamw(params, grads, [ops.op_adamw_state(p, b) for p, b in zip(params, bits)], 1)
    for p, g, b, q in zip(params, grads, bits, alone):
        ops.op_adamw([q], [g], [ops.op_adamw_state(q, b)], 1)
        assert torch.equal(p, q)
    ops.op_adamw([], [], [], 1)
    empty = torch.zeros(0, 5, device="cuda")
    ops.op_adamw([empty, params[0]], [empty.clone(), grads[0]], [ops.op_adamw_state(empty, 8), ops.op_adamw_state(params[0], 8)], 1)
    m, v = ops.op_adamw_values([ops.op_adamw_state(t, 8) for t in (empty, params[0], empty)])
    assert m.shape == v.shape == (350,)


def test_values_of_several_states_one_behind_the_other():
    states = []
    for n, size in enumerate((3, 300, 1, 5000)):
        c = torch.randint(-127, 128, (size,), device="cuda", dtype=torch.int8)
        d = torch.randint(0, 256, (size,), device="cuda", dtype=torch.uint8)
        states.append(ops.AdamWState(c, d, torch.rand(-(-size // 256), 2, device="cuda") + 0.1))
    m, v = ops.op_adamw_values(states)
    for got, want in zip((m, v), zip(*(decode(*s) for s in states))):
        assert torch.equal(got, torch.cat(want))


def test_more_than_2_31_elements():
    n = (1 << 31) + 300
    p = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    g = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    g[-300:] = 1
    g[:10] = 1
    state = ops.op_adamw_state(p, 8)
    ops.op_adamw([p], [g], [state], 1, lr=0.5, weight_decay=0.0)
    assert (p[-300:] == 0.5).all() and (p[:10] == 0.5).all() and (p[10:-300] == 1).all()
    assert (state.exp_avg[-300:] == 127).all() and not state.exp_avg[10:-300].any() and (state.exp_avg_sq[-300:] == 255).all()


def test_captured_steps_count_and_read_the_rate_on_the_gpu():
    p, g = normal(3000, dtype=torch.bfloat16), normal(3000, dtype=torch.bfloat16, seed=1)
    step, lr = torch.zeros((), dtype=torch.int64, device="cuda"), torch.full((1,), 1e-2, device="cuda")
    state = ops.op_adamw_state(p, 8)
    q, same = p.clone(), ops.op_adamw_state(p, 8)

    def run():
        step.add_(1)
        ops.op_adamw([p], [g], [state], step, lr)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        run()
    torch.cuda.current_stream().wait_stream(stream)
    ops.op_adamw([q], [g], [same], 1, 1e-2)
    assert torch.equal(p, q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for t in range(2, 7):
        lr.fill_(1e-2 / t)
        g.copy_(normal(3000, dtype=torch.bfloat16, seed=t))
        graph.replay()
        # the rate as the float that the GPU holds
        ops.op_adamw([q], [g], [same], t, float(lr))
        torch.cuda.synchronize()
        # the corrections are of the GPU's power function there and of the host's here: within a unit of 64 bits, rounded to 32
        assert (p.double() - q.double()).abs().max() <= 2.0 ** -8 * q.double().abs().max() and (p != q).sum() <= 3
        assert torch.equal(state.exp_avg, same.exp_avg) and torch.equal(state.exp_avg_sq, same.exp_avg_sq)
        p.copy_(q)


def test_written_tensors_are_known_to_autograd():
    p = normal(100).requires_grad_()
    y = (p * p).sum()
    with torch.no_grad():
        g = torch.ones_like(p)
    state = ops.op_adamw_state(p, 8)
    versions = p._version, state.exp_avg._version
    ops.op_adamw([p], [g], [state], 1)
    assert p._version == versions[0] + 1 and state.exp_avg._version == versions[1] + 1
    with pytest.raises(RuntimeError, match="inplace"):
        y.backward()


def test_refusals_on_the_gpu():
    p, g = normal(64, 8), normal(64, 8, seed=1)
    s = ops.op_adamw_state(p, 8)
    f = ops.op_adamw_state(p, 32)
    step = lambda *a, **k: lambda: ops.op_adamw(*a, **k)  # noqa: E731
    for call, text in ((step([p], [g], [s], 0), "step counts"), (step([p], [g], [s, s], 1), "as many"), (step([p], [g[:32]], [s], 1), "gradient must have"),
                       (step([p], [g.half()], [s], 1), "gradient must have"), (step([p[:, :4]], [g[:, :4]], [s], 1), "dense"),
                       (step([p], [g], [ops.op_adamw_state(p[:32], 8)], 1), "state must have"), (step([p], [g], [ops.op_adamw_state(p.t().contiguous().t(), 8)], 1), "state must have"),
                       (step([p], [g], [(s.exp_avg, s.exp_avg_sq, None)], 1), "type of exp_avg"), (step([p], [g], [(f.exp_avg, s.exp_avg_sq, s.scale)], 1), "type of exp_avg"),
                       (step([p], [g], [(s.exp_avg, s.exp_avg_sq, s.scale[:1])], 1), "scale must be"), (step([p], [g], [s], 1, -1.0), "0 or more"),
                       (step([p], [g], [s], 1, math.nan), "0 or more"), (step([p], [g], [s], 1, betas=(1.0, 0.9)), "0 or more"), (step([p], [g], [s], 1, eps=-1.0), "0 or more"),
                       (step([p], [g], [s], 1, weight_decay=math.inf), "0 or more"), (step([p, p], [g, g], [s, ops.op_adamw_state(p, 8)], 1), "share memory"),
                       (step([p, g], [g, p], [s, ops.op_adamw_state(p, 8)], 1), "share memory"), (step([p, p.clone()], [g, g], [s, s], 1), "share memory"),
                       (step([p], [p], [s], 1), "share memory"), (step([p], [p.view(-1)[::1].view(64, 8)], [s], 1), "share memory"),
                       (step([p], [g], [s], torch.ones(2, dtype=torch.int64, device="cuda")), "one"), (step([p], [g], [s], torch.ones(1, device="cuda")), "one"),
                       (step([(p.clone().requires_grad_() * 1)], [g], [s], 1), "leaf"), (step([p.int()], [g], [s], 1), "type"),
                       (lambda: ops.op_adamw_values([f]), "8 bits"), (lambda: ops.op_adamw_values([]), "at least"), (lambda: ops.op_adamw_state(p, 4), "8 or 32")):
        with pytest.raises(RuntimeError, match=text):
            call()
    for call in (step(p, [g], [s], 1), step([p], [g], [3], 1), step([p], [None], [s], 1), step([None], [g], [s], 1)):
        with pytest.raises(TypeError):
            call()
    # two gradients may be the same tensor
    ops.op_adamw([p, p.clone()], [g, g], [s, ops.op_adamw_state(p, 8)], 1)


# ---- the optimizer ----
def a_model():
    torch.manual_seed(0)
    return torch.nn.Sequential(torch.nn.Conv2d(3, 8, 3), torch.nn.GELU(), torch.nn.Flatten(), torch.nn.Linear(8 * 36, 40), torch.nn.LayerNorm(40), torch.nn.Linear(40, 5)).cuda()


def losses(model, x):
    for p in model.parameters():
        p.grad = None
    model(x).square().mean().backward()


def test_optimizer_in_32_bits_is_torchs():
    x = normal(4, 3, 8, 8)
    mine, theirs = a_model(), a_model()
    ours = gact.optim.AdamW(mine.parameters(), lr=1e-2, weight_decay=0.1, bits=32)
    other = torch.optim.AdamW(theirs.parameters(), lr=1e-2, weight_decay=0.1)
    losses(mine, x)
    for a, b in zip(mine.parameters(), theirs.parameters()):
        b.grad = a.grad.clone()
    ours.step()
    other.step()
    # one step: both formulas are the same but for the order of a few roundings
    for a, b in zip(mine.parameters(), theirs.parameters()):
        assert (a - b).abs().max() <= 16 * U * (b.abs().max() + 1e-2)


def test_optimizer_trains_and_loads_its_state():
    x = normal(4, 3, 8, 8)
    model = a_model().to(memory_format=torch.channels_last)
    optimizer = gact.optim.AdamW([{"params": model[0].parameters(), "bits": 32}, {"params": [p for m in model[1:] for p in m.parameters()]}], lr=1e-2)
    for _ in range(3):
        losses(model, x)
        optimizer.step()
    kinds = {s["exp_avg"].dtype for s in optimizer.state.values()}
    assert kinds == {torch.int8, torch.float32} and all(s["step"] == 3 for s in optimizer.state.values())
    twin = copy.deepcopy(model)
    held = io.BytesIO()
    torch.save(optimizer.state_dict(), held)
    held.seek(0)
    other = gact.optim.AdamW([{"params": twin[0].parameters(), "bits": 32}, {"params": [p for m in twin[1:] for p in m.parameters()]}], lr=1e-2)
    other.load_state_dict(torch.load(held, weights_only=True))
    # the same gradients for both: the library's convolutions need not give them twice
    losses(model, x)
    for a, b in zip(model.parameters(), twin.parameters()):
        b.grad = a.grad.clone()
    optimizer.step()
    other.step()
    for a, b in zip(model.parameters(), twin.parameters()):
        assert torch.equal(a, b)
    for a, b in zip(model.parameters(), twin.parameters()):
        for name, t in optimizer.state[a].items():
            assert torch.equal(t, other.state[b][name]) if isinstance(t, torch.Tensor) else t == other.state[b][name]


def test_optimizer_of_parameters_without_gradients_and_late_ones():
    a, b = normal(100).requires_grad_(), normal(100, seed=1).requires_grad_()
    optimizer = gact.optim.AdamW([a, b])
    a.grad = torch.ones_like(a)
    kept = b.detach().clone()
    optimizer.step()
    assert torch.equal(b, kept) and b not in optimizer.state
    b.grad = torch.ones_like(b)
    optimizer.step()
    assert optimizer.state[a]["step"] == 2 and optimizer.state[b]["step"] == 1
    # b's first step is the rate, whatever a's count
    assert (b.detach() - (kept * (1 - 1e-5) - 1e-3)).abs().max() <= 1e-6
    with pytest.raises(ValueError, match="8 or 32"):
        optimizer.add_param_group({"params": [normal(3).requires_grad_()], "bits": 16})


def test_optimizer_in_a_graph():
    x = normal(4, 3, 8, 8)
    model, twin = a_model(), a_model()
    optimizer, other = (gact.optim.AdamW(m.parameters(), lr=1e-2, capturable=c) for m, c in ((model, True), (twin, False)))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        losses(model, x)
        fresh = gact.optim.AdamW([normal(5).requires_grad_()], capturable=True)
        optimizer.step()
    torch.cuda.current_stream().wait_stream(stream)
    losses(twin, x)
    other.step()
    graph = torch.cuda.CUDAGraph()
    for p in model.parameters():
        p.grad.zero_()
    with torch.cuda.graph(graph):
        optimizer.step()
    fresh.param_groups[0]["params"][0].grad = normal(5)
    empty = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        empty.capture_begin()
        try:
            with pytest.raises(RuntimeError, match="cannot be captured"):
                fresh.step()
        finally:
            empty.capture_end()
    for turn in range(3):
        grads = [normal(*p.shape, seed=turn) for p in model.parameters()]
        for p, q, g in zip(model.parameters(), twin.parameters(), grads):
            p.grad.copy_(g)
            q.grad = g
        graph.replay()
        other.step()
        for p, q in zip(model.parameters(), twin.parameters()):
            assert (p - q).abs().max() <= 1e-6
            assert torch.equal(optimizer.state[p]["exp_avg"], other.state[q]["exp_avg"])
    assert {int(s["step"]) for s in optimizer.state.values()} == {4}
