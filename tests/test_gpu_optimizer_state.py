"""gact.optim.AdamW on the GPU: parameters that miss gradients, and states that go from one optimizer to another."""
import pytest
import torch

import gact

pytestmark = pytest.mark.gpu


def normal(*shape, dtype=torch.float32, seed=0):
    g = torch.Generator().manual_seed(seed + 7919 * sum(shape))
    return torch.randn(*shape, generator=g).to(dtype).cuda()


def leaves(sizes, dtype=torch.float32):
    return [normal(*s, dtype=dtype, seed=n).requires_grad_() for n, s in enumerate(sizes)]


def test_counts_on_the_gpu_skip_parameters_without_gradients():
    sizes = [(300,), (7, 41), (1000,)]
    ours, theirs = leaves(sizes), leaves(sizes)
    opts = [gact.optim.AdamW(p, lr=1e-2, bits=32, capturable=c) for p, c in ((ours, True), (theirs, False))]
    for turn, some in enumerate([(0, 1, 2), (0,), (0,), (0, 2), (0, 1, 2), (1,), (0, 1, 2)]):
        for params in (ours, theirs):
            for n, p in enumerate(params):
                p.grad = normal(*sizes[n], seed=10 * turn + n) if n in some else None
        for opt in opts:
            opt.step()
        for p, q in zip(ours, theirs):
            # the corrections are of the GPU's power function there and of the host's here: a unit in the last place of the step, or of the parameter
            assert (p - q).abs().max() <= 2.0 ** -22 * (q.abs().max() + 1e-2 * 8)
            assert int(opts[0].state[p]["step"]) == opts[1].state[q]["step"]
    assert [opts[1].state[q]["step"] for q in theirs] == [6, 4, 4]


def test_a_recorded_step_counts_for_all_that_it_has():
    params, same = leaves([(300,), (50,)]), leaves([(300,), (50,)])
    opt, other = gact.optim.AdamW(params, capturable=True), gact.optim.AdamW(same)
    for p, q in zip(params, same):
        p.grad, q.grad = torch.ones_like(p), torch.ones_like(q)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        opt.step()
    torch.cuda.current_stream().wait_stream(stream)
    other.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for turn in range(3):
        graph.replay()
        other.step()
    kept, params[1].grad = params[1].grad, None
    with pytest.raises(RuntimeError, match="without a gradient"):
        opt.step()
    params[1].grad = kept
    opt.step()
    other.step()
    for p, q in zip(params, same):
        assert int(opt.state[p]["step"]) == other.state[q]["step"] == 5 and (p - q).abs().max() <= 2.0 ** -21


def test_a_rate_on_the_cpu_is_a_number():
    params, same = leaves([(300,), (50, 3)]), leaves([(300,), (50, 3)])
    opt, other = gact.optim.AdamW(params, lr=torch.tensor(0.01)), gact.optim.AdamW(same, lr=float(torch.tensor(0.01)))
    for p, q in zip(params, same):
        p.grad, q.grad = normal(*p.shape, seed=5), normal(*p.shape, seed=5)
    for turn in range(3):
        opt.step()
        other.step()
        assert all(torch.equal(p, q) for p, q in zip(params, same))
        opt.param_groups[0]["lr"].mul_(0.5)
        other.param_groups[0]["lr"] *= 0.5


def test_torchs_checkpoint_goes_on_as_torch_does():
    sizes = [(300,), (50, 3)]
    params, same = leaves(sizes), leaves(sizes)
    theirs = torch.optim.AdamW(params, lr=1e-2)
    for turn in range(2):
        for n, p in enumerate(params):
            p.grad = normal(*sizes[n], seed=turn)
        theirs.step()
    with torch.no_grad():
        for p, q in zip(params, same):
            q.copy_(p)
    opt = gact.optim.AdamW(same, bits=8)
    opt.load_state_dict(theirs.state_dict())
    for n, (p, q) in enumerate(zip(params, same)):
        p.grad = normal(*sizes[n], seed=9)
        q.grad = p.grad.clone()
    theirs.step()
    opt.step()
    # one step from the same state: a few roundings in another order
    for p, q in zip(params, same):
        assert (p - q).abs().max() <= 16 * 2.0 ** -24 * (p.abs().max() + 1e-2)


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="two devices")
def test_counts_on_another_device_are_refused_before_anything_runs():
    params = [torch.ones(300, device="cuda:%d" % n) for n in range(2)]
    step = torch.ones((), dtype=torch.int64, device="cuda:0")
    grads = [torch.ones_like(p) for p in params]
    with pytest.raises(RuntimeError, match="parameters' device"):
        gact.ops.op_adamw(params, grads, [gact.ops.op_adamw_state(p) for p in params], step)
    assert all((p == 1).all() for p in params)


def test_second_moments_next_to_nothing_are_kept():
    """Gradients whose squares are too small for a group's largest to be divided by, then none: with eps 0 a second moment lost would make the step infinite."""
    lr, betas = 1e-2, (0.9, 0.999)
    sizes = [10.0 ** -n for n in range(12, 18)]
    p = torch.zeros(256 * len(sizes), device="cuda")
    g = torch.tensor(sizes, device="cuda").repeat_interleave(256)
    for dtype in (torch.float32, torch.bfloat16):
        at, grad = p.to(dtype), g.to(dtype)
        state = gact.ops.op_adamw_state(at)
        m, v = torch.zeros_like(g).double(), torch.zeros_like(g).double()
        for step in range(1, 8):
            if step == 2:
                grad = torch.zeros_like(grad)
            before = at.clone()
            gact.ops.op_adamw([at], [grad], [state], step, lr, betas, 0.0, 0.0)
            m, v = betas[0] * m + (1 - betas[0]) * grad.double(), betas[1] * v + (1 - betas[1]) * grad.double() ** 2
            want = lr * (m / (1 - betas[0] ** step)) / (v / (1 - betas[1] ** step)).sqrt()
            moved = (before.double() - at.double()).abs()
            # a code c for a value between c - 1/2 and c + 1/2 is off by (1 + 1 / (2 c))^2 in the second moment's root; c is 1 or more.  The first moment's
            # one code is a group's largest, and exact
            assert torch.isfinite(at).all() and state.exp_avg_sq.min() >= 1
            close_to = 2.0 ** -8 * at.double().abs() if dtype is torch.bfloat16 else 1e-6
            assert (moved <= 2.25 * 1.01 * want + close_to).all() and (moved >= want / 2.25 / 1.01 - close_to).all()
