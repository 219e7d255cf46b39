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
