"""Attention, the position bias and AdamW as far as they go without a GPU: what the library refuses before it touches the GPU, how its workspaces are
sized, what the operators refuse, and where the buckets of distances begin."""
import ctypes
import math

import pytest
import torch

from gact import ops, optim
from gact.cpp_extension import _abi

EINVAL, EALIGN, ELIMIT = -1, -2, -6


class Rows(ctypes.Structure):
    _fields_ = [("p", ctypes.c_void_p), ("batch", ctypes.c_int64), ("head", ctypes.c_int64), ("row", ctypes.c_int64)]


class Attention(ctypes.Structure):
    _fields_ = [("dtype", ctypes.c_int32), ("causal", ctypes.c_int32)] + [(n, ctypes.c_int64) for n in ("batch", "heads", "kv_heads", "queries", "keys", "width")] + [
        ("scale", ctypes.c_float), ("reserved", ctypes.c_float), ("bias", ctypes.c_void_p), ("mask", ctypes.c_void_p), ("mask_stride", ctypes.c_int64),
        ("q", Rows), ("k", Rows), ("v", Rows)]


class Tensor(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("p", "g", "m", "v", "scale")] + [("numel", ctypes.c_int64)]


class Options(ctypes.Structure):
    _fields_ = [(n, ctypes.c_double) for n in ("lr", "beta1", "beta2", "eps", "decay")] + [("step", ctypes.c_int64), ("lr_at", ctypes.c_void_p), ("step_at", ctypes.c_void_p)]


def call(dtype=2, batch=2, heads=4, kv_heads=2, queries=8, keys=9, width=64, scale=1.0, **other):
    a = Attention(dtype, 0, batch, heads, kv_heads, queries, keys, width, scale, 0.0, None, None, 0)
    a.q = Rows(16, heads * queries * width, queries * width, width)
    a.k = Rows(16, kv_heads * keys * width, keys * width, width)
    a.v = Rows(16, kv_heads * keys * width, keys * width, width)
    for name, value in other.items():
        setattr(a, name, value)
    return a


def test_attention_refuses_before_it_touches_the_gpu():
    L = _abi.lib()
    out = Rows(16, 4 * 8 * 64, 64, 4 * 64)
    forward = lambda a, o=out, ws=None, rest=None: L.gact_attention_forward(ctypes.byref(a), ctypes.byref(o), None, rest, ws, None)  # noqa: E731
    backward = lambda a, o=out, lse=16, ws=16, db=None, dq=None: L.gact_attention_backward(  # noqa: E731
        ctypes.byref(a), ctypes.byref(o), lse, None, ctypes.byref(o), ctypes.byref(dq) if dq else None, None, None, db, ws, None)
    for bad in (call(dtype=3), call(batch=-1), call(heads=0), call(kv_heads=0), call(heads=3), call(queries=-1), call(keys=(1 << 24) + 1), call(width=0),
                call(width=136), call(scale=0.0), call(scale=-1.0), call(scale=math.inf), call(scale=math.nan), call(q=Rows(None, 1, 1, 64)),
                call(q=Rows(16, 4096, 512, 56)), call(k=Rows(16, -8, 512, 64)), call(v=Rows(16, 4096, 512, 1 << 24)), call(mask=16, mask_stride=-1)):
        assert forward(bad) == EINVAL and backward(bad) == EINVAL
    for bad in (call(q=Rows(8, 2048, 512, 64)), call(width=60), call(k=Rows(16, 4096, 512, 68)), call(v=Rows(16, 4100, 512, 64)), call(k=Rows(16, 4096, 516, 64))):
        assert forward(bad) == EALIGN and backward(bad) == EALIGN
    assert forward(call(), Rows(8, 2048, 64, 256)) == EALIGN and forward(call(), Rows(None, 2048, 64, 256)) == EINVAL
    assert forward(call(), rest=4) == EALIGN
    assert forward(call(bias=16)) == EINVAL and forward(call(bias=16), ws=8) == EALIGN          # the bias needs room
    assert backward(call(), lse=None) == EINVAL and backward(call(), ws=None) == EINVAL and backward(call(), ws=8) == EALIGN
    assert backward(call(), db=16) == EINVAL                                                    # a gradient of no bias
    assert backward(call(), dq=Rows(8, 2048, 64, 256)) == EALIGN
    assert L.gact_attention_forward(None, ctypes.byref(out), None, None, None, None) == EINVAL
    assert L.gact_attention_forward(ctypes.byref(call()), None, None, None, None, None) == EINVAL
    # nothing to do
    assert forward(call(batch=0)) == 0 and forward(call(queries=0)) == 0 and forward(call(batch=0, q=Rows())) == 0


def test_attention_workspaces_are_sized():
    L = _abi.lib()
    forward = lambda **k: L.gact_attention_workspace_bytes(ctypes.byref(call(**k)))  # noqa: E731
    backward = lambda db=0, **k: L.gact_attention_backward_workspace_bytes(ctypes.byref(call(**k)), db)  # noqa: E731
    assert forward() == 0 and forward(queries=512, keys=512, batch=32, heads=16, kv_heads=16) == 0
    assert forward(dtype=3) == 0 and forward(batch=0) == 0 and forward(queries=0) == 0 and forward(queries=0, keys=0) == 0
    # one token behind many keys: splits of 32 rows, whole floats of the width rounded up and two numbers beside them
    size = forward(batch=1, heads=32, kv_heads=8, queries=1, keys=65537, width=72)
    assert size > 0 and size % (8 * 32 * (96 + 2) * 4) == 0 and size <= 1024 * 32 * 98 * 4
    for batch in (1, 3, 200):
        for queries in (1, 7, 100, 5000):
            for keys in (0, 1, 255, 256, 100000):
                for dtype in (0, 1):
                    kind = dict(dtype=dtype, batch=batch, queries=queries, keys=keys, bias=16)
                    bias = -(-4 * (queries + keys - 1) * 4 // 256) * 256
                    assert forward(**kind) >= bias and (forward(**kind) - bias) <= (1 << 31)
                    delta = -(-batch * 4 * queries * 4 // 256) * 256
                    # floats of few tiles' splits: for dq, or for dk and dv, at most three workgroups' rows to each of 256 compute units
                    parts = backward(**kind) - bias - delta
                    assert parts == 0 if batch == 200 and keys >= 255 else 0 <= parts <= 2 * 3 * 256 * 128 * 64 * 4
                    assert backward(1, **kind) >= bias + delta + parts + batch * 4 * (-(-queries // 32)) * (keys + 31) * 4


def test_position_bias_refuses_before_it_touches_the_gpu():
    L = _abi.lib()
    for f in (L.gact_position_bias, L.gact_position_bias_backward):
        one = lambda table=16, dtype=0, buckets=32, heads=4, queries=8, keys=8, both=1, most=128, out=16: f(table, dtype, buckets, heads, queries, keys, both, most, out, None)  # noqa: E731,B023
        for bad in (dict(table=None), dict(out=None), dict(dtype=3), dict(buckets=31), dict(buckets=2), dict(buckets=1, both=0), dict(buckets=514), dict(heads=0), dict(heads=65536),
                    dict(queries=0), dict(keys=0), dict(keys=(1 << 24) + 1), dict(most=8), dict(most=16, both=0), dict(most=(1 << 24) + 1)):
            assert one(**bad) == EINVAL, bad


def test_adamw_refuses_before_it_touches_the_gpu():
    L = _abi.lib()

    def step(tensor=(16, 16, 16, 16, 16, 8), dtype=0, bits=8, count=1, options=(1e-3, 0.9, 0.999, 1e-8, 0.01, 1, None, None)):
        return L.gact_adamw(ctypes.byref(Tensor(*tensor)), count, dtype, bits, ctypes.byref(Options(*options)), None)

    assert step(dtype=3) == EINVAL and step(bits=4) == EINVAL and step(count=-1) == EINVAL
    for n in range(4):
        assert step(tuple(None if i == n else 16 for i in range(5)) + (8,)) == EINVAL
    assert step((16, 16, 16, 16, None, 8)) == EINVAL and step((16, 16, 16, 16, 16, -1)) == EINVAL
    assert step((18, 16, 16, 16, 16, 8)) == EALIGN and step((16, 15, 16, 16, 16, 8), 1) == EALIGN
    assert step((16, 16, 24, 16, 16, 8)) == EALIGN and step((16, 16, 16, 24, 16, 8)) == EALIGN and step((16, 16, 16, 16, 20, 8)) == EALIGN
    for n, bad in ((0, -1.0), (0, math.nan), (1, 1.0), (1, -0.1), (2, 1.0), (2, math.nan), (3, -1.0), (4, -1.0), (5, 0)):
        options = [1e-3, 0.9, 0.999, 1e-8, 0.01, 1, None, None]
        options[n] = bad
        assert step(options=options) == EINVAL, (n, bad)
    assert L.gact_adamw(None, 1, 0, 8, ctypes.byref(Options()), None) == EINVAL and L.gact_adamw(None, 0, 0, 8, None, None) == EINVAL
    assert L.gact_adamw_values(ctypes.byref(Tensor(None, None, None, 16, 16, 8)), 1, 16, 16, None) == EINVAL
    # nothing to do
    assert step((None, None, None, None, None, 0)) == 0 and L.gact_adamw(None, 0, 0, 8, ctypes.byref(Options(1e-3, 0.9, 0.9, 0, 0, 1)), None) == 0
    assert L.gact_adamw_values(None, 0, 16, 16, None) == 0


def test_operators_refuse_what_is_not_on_the_gpu():
    x = torch.zeros(1, 2, 4, 8)
    for call_ in (lambda: ops.op_attention(x, x, x), lambda: ops.op_position_bias(x[0, 0], 4, 4), lambda: ops.op_adamw([x], [x], [ops.op_adamw_state(x, 8)], 1),
                  lambda: ops.op_adamw_values([ops.op_adamw_state(x, 8)])):
        with pytest.raises(RuntimeError, match="must be a CUDA tensor!"):
            call_()
    for call_ in (lambda: ops.op_attention(None, x, x), lambda: ops.op_position_bias([1.0], 4, 4), lambda: ops.op_adamw(x, x, x, 1), lambda: ops.op_adamw([1], [1], [1], 1),
                  lambda: ops.op_adamw_values([1])):
        with pytest.raises(TypeError):
            call_()
    with pytest.raises(RuntimeError, match="as many"):
        ops.op_adamw([x], [], [], 1)
    with pytest.raises(RuntimeError, match="step counts from 1"):
        ops.op_adamw([], [], [], 0)
    with pytest.raises(RuntimeError, match="betas"):
        ops.op_adamw([], [], [], 1, betas=(0.9, 1.0))


def test_states_have_their_parameters_shape_and_layout():
    p = torch.zeros(2, 4, 10, 12, dtype=torch.bfloat16).to(memory_format=torch.channels_last).requires_grad_()
    for bits, kinds in ((8, (torch.int8, torch.uint8)), (32, (torch.float32, torch.float32))):
        s = ops.op_adamw_state(p, bits)
        assert (s.exp_avg.dtype, s.exp_avg_sq.dtype) == kinds and s.exp_avg.shape == p.shape and s.exp_avg.stride() == p.stride()
        assert not s.exp_avg.requires_grad and not s.exp_avg.any()
        assert s.scale is None if bits == 32 else s.scale.shape == (4, 2)
    with pytest.raises(RuntimeError, match="8 or 32"):
        ops.op_adamw_state(p, 16)


def test_optimizer_checks_its_options():
    p = torch.zeros(3, requires_grad=True)
    for bad in (dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(eps=-1.0), dict(weight_decay=-1.0), dict(bits=4)):
        with pytest.raises(ValueError):
            optim.AdamW([p], **bad)
    optim.AdamW([p]).step()      # no gradient, nothing to do


def test_optimizer_groups_count_their_steps_by_themselves():
    """Counts in device memory are added to in place: two groups that were loaded with the same count must not share it."""
    params = [torch.nn.Parameter(torch.zeros(300)) for _ in range(4)]
    opt = optim.AdamW([{"params": params[:2]}, {"params": params[2:]}], capturable=True)
    state = opt.state_dict()
    moments = {n: {"step": torch.tensor(5), **ops.op_adamw_state(p)._asdict()} for n, p in enumerate(params)}
    opt.load_state_dict({**state, "state": moments})
    a, b, c, d = (opt.state[p]["step"] for p in params)
    assert a is b and c is d and a is not c and int(a) == int(c) == 5


def test_optimizer_does_not_count_a_step_that_was_refused():
    for capturable in (False, True):
        p = torch.nn.Parameter(torch.zeros(300))
        opt = optim.AdamW([p], capturable=capturable)
        p.grad = torch.zeros(300)
        with pytest.raises(RuntimeError):        # not on a GPU
            opt.step()
        assert int(opt.state[p].get("step", 0)) == 0
