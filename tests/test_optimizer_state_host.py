"""What gact.optim.AdamW keeps of its parameters and loads, without a GPU: the step itself is replaced by one that notes the counts it is given."""
import copy
import pickle

import pytest
import torch

from gact import optim


@pytest.fixture
def counts(monkeypatch):
    """{parameter: the count of its last step}; a step on the CPU that changes nothing."""
    seen = {}

    def step(params, grads, states, count, *rest):
        for p in params:
            seen[p] = int(count)

    monkeypatch.setattr(optim, "op_adamw", step)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    return seen


def parameters(n):
    return [torch.nn.Parameter(torch.zeros(300)) for _ in range(n)]


def step_with(opt, params, some):
    for p in params:
        p.grad = torch.zeros(300) if p in some else None
    opt.step()


@pytest.mark.parametrize("loaded", [False, True], ids=["begun", "loaded"])
def test_a_parameter_without_a_gradient_is_not_counted(counts, loaded):
    """Whether counts are numbers or in device memory, where parameters that begin together, or are loaded with the same number, share one."""
    held = {}
    for capturable in (False, True):
        a, b, c = params = parameters(3)
        opt = optim.AdamW(params, capturable=capturable)
        step_with(opt, params, {a, b, c})
        if loaded:
            fresh = optim.AdamW(params, capturable=capturable)
            fresh.load_state_dict(copy.deepcopy(opt.state_dict()))
            opt = fresh
        order = [{a}, {a, c}, {a}, {a, b}, {b, c}, {a, b, c}, {a, b, c}, {c}, {a, b, c}]
        want = {p: 1 for p in params}
        for some in order:
            step_with(opt, params, some)
            for p in some:
                want[p] += 1
                assert counts[p] == want[p]
            assert [int(opt.state[p]["step"]) for p in params] == [want[p] for p in params]
        held[capturable] = [counts[p] for p in params]
        if capturable:      # those that go on together share a count as long as they do
            together = optim.AdamW(params, capturable=True)
            step_with(together, params, {a, b, c})
            step_with(together, params, {a, b})
            step_with(together, params, {a, b})
            assert together.state[a]["step"] is together.state[b]["step"] is not together.state[c]["step"]
    assert held[False] == held[True]


def test_a_count_that_a_graph_adds_to_is_not_divided(counts, monkeypatch):
    """A recorded step adds to the tensor that it was recorded with, for all parameters that it stepped."""
    a, b, c = params = parameters(3)
    opt = optim.AdamW([{"params": [a, b]}, {"params": [c]}], capturable=True)
    step_with(opt, params, {a, b, c})
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="without a gradient"):
        step_with(opt, params, {a})
    step_with(opt, params, {a, b})
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    with pytest.raises(RuntimeError, match="without a gradient"):
        step_with(opt, params, {b})
    assert [int(opt.state[p]["step"]) for p in params] == [2, 2, 1]
    step_with(opt, params, {c})
    step_with(opt, params, {a, b})
    assert [int(opt.state[p]["step"]) for p in params] == [3, 3, 2]
    # a loaded state has counts of its own, which no graph adds to
    opt.load_state_dict(copy.deepcopy(opt.state_dict()))
    step_with(opt, params, {b})
    assert [int(opt.state[p]["step"]) for p in params] == [3, 4, 2]


def a_state(p, bits, seed=0):
    """A parameter's state with something in it."""
    kept = {k: v for k, v in optim.op_adamw_state(p, bits)._asdict().items() if v is not None}
    g = torch.Generator().manual_seed(seed)
    for name, t in kept.items():
        t.copy_(torch.randint(0, 128, t.shape, generator=g))
    return {"step": 5, **kept}


def saved(opt, states):
    return {**opt.state_dict(), "state": dict(enumerate(states))}


def test_codes_in_another_order_of_memory_are_refused():
    """A group of codes is 256 neighbours in memory, and its scale theirs."""
    last = torch.zeros(8, 3, 5, 5).to(memory_format=torch.channels_last)
    first = torch.zeros(8, 3, 5, 5)
    for given, to in ((last, first), (first, last), (torch.zeros(40, 30).t(), torch.zeros(30, 40))):
        opt = optim.AdamW([torch.nn.Parameter(to)])
        with pytest.raises(ValueError, match="order of memory"):
            opt.load_state_dict(saved(opt, [a_state(given, 8)]))
        # floats stand for themselves
        opt = optim.AdamW([torch.nn.Parameter(to)], bits=32)
        state = a_state(given, 32)
        opt.load_state_dict(saved(opt, [state]))
        for name in ("exp_avg", "exp_avg_sq"):
            kept = opt.state[opt.param_groups[0]["params"][0]][name]
            assert torch.equal(kept, state[name]) and kept.stride() == to.stride()
    # the same order, whatever the strides of single rows are
    for given, to in ((last, last), (first, first), (torch.zeros(1, 5, 1).as_strided((1, 5, 1), (7, 1, 3)), torch.zeros(1, 5, 1))):
        opt = optim.AdamW([torch.nn.Parameter(to)])
        state = a_state(given, 8)
        opt.load_state_dict(saved(opt, [state]))
        kept = opt.state[opt.param_groups[0]["params"][0]]
        assert all(torch.equal(kept[name], state[name]) for name in ("exp_avg", "exp_avg_sq", "scale"))


def test_a_refused_load_leaves_everything_as_it_was(counts):
    params = parameters(2)
    opt = optim.AdamW(params, lr=0.5)
    step_with(opt, params, set(params))
    kept = {p: dict(opt.state[p]) for p in params}
    good = [a_state(p, 8) for p in params]
    short = {**good[1], "exp_avg": torch.zeros(299, dtype=torch.int8)}
    other = {**good[1], "exp_avg_sq": torch.zeros(300, dtype=torch.int8)}
    for states in ([good[0], short], [good[0], other], [good[0], {"step": 5, "momentum_buffer": torch.zeros(300)}], [good[0], {"exp_avg": good[1]["exp_avg"]}]):
        given = saved(opt, states)
        given["param_groups"] = [{**given["param_groups"][0], "lr": 0.25}]
        with pytest.raises(ValueError):
            opt.load_state_dict(given)
        assert opt.param_groups[0]["lr"] == 0.5 and list(opt.state) == params
        for p in params:
            assert all(opt.state[p][name] is t for name, t in kept[p].items()) and opt.state[p]["step"] == 1
    given = saved(opt, good)
    given["param_groups"] = given["param_groups"] * 2
    with pytest.raises(ValueError):
        opt.load_state_dict(given)
    assert list(opt.state) == params
    # of some of the parameters; an entry may be empty, as one whose first step was refused is
    for states in (good[:1], [good[0], {}]):
        opt.load_state_dict(saved(opt, states))
        assert opt.state[params[0]]["step"] == 5 and not opt.state[params[1]]


def test_a_checkpoint_of_torchs_adamw_is_loaded(counts):
    params = parameters(3)
    theirs = torch.optim.AdamW(params[:2], lr=0.125, betas=(0.5, 0.75), weight_decay=0.25)
    for p in params:
        p.grad = torch.ones(300)
    theirs.step()
    theirs.step()
    given = copy.deepcopy(theirs.state_dict())
    for bits in (8, 32):
        opt = optim.AdamW(params[:2], bits=bits)
        opt.load_state_dict(given)
        group = opt.param_groups[0]
        assert group["lr"] == 0.125 and group["betas"] == (0.5, 0.75) and group["weight_decay"] == 0.25 and group["bits"] == bits and not group["capturable"]
        assert opt.state[params[0]]["step"] == 2 and torch.equal(opt.state[params[1]]["exp_avg"], given["state"][1]["exp_avg"])
        # a parameter that comes later has the group's bits
        group["params"].append(params[2])
        opt.step()
        assert counts[params[0]] == 3 and counts[params[2]] == 1
        assert opt.state[params[2]]["exp_avg"].dtype is (torch.int8 if bits == 8 else torch.float32)
    # what was saved before an option existed
    given["param_groups"][0].pop("capturable")
    opt = optim.AdamW(params[:2])
    opt.load_state_dict({**given, "state": {}})
    assert opt.param_groups[0]["capturable"] is False
    step_with(opt, params, set(params))


@pytest.mark.parametrize("option", [dict(amsgrad=True), dict(maximize=True)], ids=lambda o: next(iter(o)))
def test_a_checkpoint_of_other_steps_is_refused(option):
    """Options that change what a step is, and that this optimizer does not have, are not passed over."""
    params = parameters(2)
    theirs = torch.optim.AdamW(params, **option)
    opt = optim.AdamW(params)
    with pytest.raises(ValueError, match=next(iter(option))):
        opt.load_state_dict(theirs.state_dict())
    other = torch.optim.Adam(params, weight_decay=0.1).state_dict()
    other["param_groups"][0]["decoupled_weight_decay"] = False
    with pytest.raises(ValueError, match="decay"):
        opt.load_state_dict(other)
    assert "amsgrad" not in opt.param_groups[0]


def test_a_rate_that_is_a_tensor_on_the_cpu(monkeypatch):
    """A number like any other; one on the GPU goes to the kernels as it is."""
    rates = []
    monkeypatch.setattr(optim, "op_adamw", lambda params, grads, states, count, lr, *rest: rates.append(lr))
    p = parameters(1)[0]
    p.grad = torch.zeros(300)
    opt = optim.AdamW([p], lr=torch.tensor(0.125))
    opt.step()
    opt.param_groups[0]["lr"].mul_(2)
    opt.step()
    opt.param_groups[0]["lr"] = 0.5
    opt.step()
    assert rates == [0.125, 0.25, 0.5] and not any(isinstance(r, torch.Tensor) for r in rates)
    with pytest.raises(ValueError):
        optim.AdamW([p], lr=torch.tensor(-1.0))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float64])
def test_a_checkpoint_with_moments_of_another_type_is_loaded(dtype):
    """torch's moments have their parameter's type; here they are float32, whatever that is."""
    p = torch.nn.Parameter(torch.zeros(300, dtype=dtype))
    theirs = torch.optim.AdamW([p])
    p.grad = torch.ones(300, dtype=dtype) * 0.3
    theirs.step()
    given = theirs.state_dict()
    opt = optim.AdamW([p], bits=32)
    opt.load_state_dict(given)
    for name in ("exp_avg", "exp_avg_sq"):
        kept = opt.state[p][name]
        assert kept.dtype is torch.float32 and torch.equal(kept, given["state"][0][name].float())
    # codes are not floats of another type
    state = a_state(torch.zeros(300), 32)
    state["exp_avg"] = state["exp_avg"].to(torch.int8)
    with pytest.raises(ValueError, match="exp_avg"):
        opt.load_state_dict(saved(opt, [state]))


def test_copies_of_an_optimizer_count_by_themselves(counts):
    params = parameters(2)
    opt = optim.AdamW(params, capturable=True)
    step_with(opt, params, set(params))
    for twin in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        held = twin.param_groups[0]["params"]
        assert twin.state[held[0]]["step"] is twin.state[held[1]]["step"] is not opt.state[params[0]]["step"]
        step_with(twin, held, {held[0]})
        assert [int(twin.state[p]["step"]) for p in held] == [2, 1]
    assert [int(opt.state[p]["step"]) for p in params] == [1, 1]
