"""AdamW over many tensors at once, with its states in 8 bits or in 32.

States in 8 bits take 2.06 bytes of an element where floats take 8: groups of 256 elements share the largest magnitude of either state, and a code is
the square root of the first moment or the fourth root of the second, rounded to nearest, so that both moments of a step have the same spacing: 0.8 %
of the largest next to it, finer below.  A second moment above zero is never rounded to zero, and a group's largest one is held as 1e-28 at least; a
group whose largest first moment is below 1e-30 has zeros.  Rounding is to nearest: steps are repeatable and need no seeds.

``op_adamw`` is one launch for every 72 tensors of a type; parameters and states are changed in place.  Whatever cannot be taken raises a RuntimeError (a
TypeError where no tensor was given), before anything is launched.
"""
import collections

import torch

from .cpp_extension import _abi

# bits 32: float32 moments, scale None; bits 8: int8 and uint8 codes, scale float32 [groups, 2]; the moments in their parameter's shape and layout
AdamWState = collections.namedtuple("AdamWState", "exp_avg exp_avg_sq scale")


def op_adamw_state(param, bits=8):
    """The state of a parameter before its first step."""
    if bits not in (8, 32):
        raise RuntimeError("states have 8 or 32 bits, got %r" % (bits,))
    kinds = (torch.int8, torch.uint8) if bits == 8 else (torch.float32, torch.float32)
    moments = [torch.zeros_like(param, dtype=kind, requires_grad=False) for kind in kinds]
    scale = torch.zeros(-(-param.numel() // 256), 2, dtype=torch.float32, device=param.device) if bits == 8 else None
    return AdamWState(*moments, scale)


def op_adamw(params, grads, states, step, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2):
    """One step, the step-th from 1 on, of all params: exp_avg = b1 exp_avg + (1 - b1) grad, exp_avg_sq = b2 exp_avg_sq + (1 - b2) grad^2, param =
    param (1 - lr weight_decay) - lr / (1 - b1^step) exp_avg / (sqrt(exp_avg_sq / (1 - b2^step)) + eps), computed in float32.

    params: leaves, float32, float16 or bfloat16, dense in memory in whatever order of dimensions; grads: of their shapes and types; states: an
    AdamWState each.  step and lr: numbers, or one int64 and one float32 on the GPU, which the kernels read (a step that is recorded in a graph).
    A group of 256 elements whose gradient has a NaN or an infinity is not finite any more where its state has 8 bits."""
    _abi.native().adamw(params, grads, states, step, lr, betas[0], betas[1], eps, weight_decay)


def op_adamw_values(states):
    """(exp_avg, exp_avg_sq): what the codes of states in 8 bits stand for, float32 [elements] each, one state behind the other in their order of
    memory."""
    return _abi.native().adamw_values(states)


def _order(t):
    """What the order of a dense tensor's elements in memory goes by."""
    return [stride for size, stride in zip(t.shape, t.stride()) if size > 1]


class AdamW(torch.optim.Optimizer):
    """torch.optim.AdamW's steps (decoupled weight decay) by op_adamw.  bits: 8 or 32, an option of every group of parameters.  lr: a number, a tensor on the
    CPU, which is read at every step, or one float32 on the GPU, which the kernels read.

    capturable: the count of steps is in device memory and every step adds one to it there, so that a step can be recorded in a graph; run one step
    before the capture, which makes the states.  Parameters that begin together, or are loaded with the same count, share it until a step finds only some
    of them with a gradient; those of a recorded step go on together, and a step of some of them is refused, as the graph would count for all."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, bits=8, capturable=False):
        if not 0.0 <= float(lr) or not 0.0 <= eps or not 0.0 <= weight_decay or not all(0.0 <= b < 1.0 for b in betas):
            raise ValueError("lr, eps and weight_decay must be 0 or more, and the betas from 0 to below 1")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, bits=bits, capturable=capturable))
        self._recorded = {}

    def __setstate__(self, state):
        super().__setstate__(state)
        self._recorded = {}      # a copy's counts are its own

    def add_param_group(self, param_group):
        if param_group.get("bits", self.defaults["bits"]) not in (8, 32):
            raise ValueError("states have 8 or 32 bits")
        super().add_param_group(param_group)

    def _begin(self, group, param, counts):
        """The state of a parameter that has its first step.  Counts on the GPU are shared by the parameters that begin together."""
        if group["capturable"]:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("a parameter's first step cannot be captured: run one step before the capture")
            if param.device not in counts:
                counts[param.device] = torch.zeros((), dtype=torch.int64, device=param.device)
        kept = op_adamw_state(param, group["bits"])
        self.state[param] = {"step": counts[param.device] if group["capturable"] else 0, "exp_avg": kept.exp_avg, "exp_avg_sq": kept.exp_avg_sq}
        if kept.scale is not None:
            self.state[param]["scale"] = kept.scale

    def _divide(self, work):
        """The counts of a step's work: one on the GPU that parameters without a gradient hold as well is divided.  -> whether the step is recorded"""
        if not any(isinstance(count, torch.Tensor) for _, count, _ in work):
            return False
        capturing = torch.cuda.is_current_stream_capturing()
        holders = collections.Counter(id(kept["step"]) for kept in self.state.values() if "step" in kept)
        for n, (group, count, params) in enumerate(work):
            if not isinstance(count, torch.Tensor) or holders[id(count)] == len(params):
                continue
            if capturing:
                raise RuntimeError("a parameter that is counted together with others is without a gradient: run a step of those that have one before "
                                   "the capture")
            if id(count) in self._recorded:
                raise RuntimeError("a parameter that is counted together with others in a recorded step is without a gradient: give all of them "
                                   "gradients, or load the state anew")
            work[n] = (group, count.clone(), params)
        return capturing

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        work = []
        for group in self.param_groups:
            # parameters whose counts are the same number, or the same tensor
            together, counts = {}, {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                if not self.state[p]:
                    self._begin(group, p, counts)
                count = self.state[p]["step"]
                key = id(count) if isinstance(count, torch.Tensor) else count
                together.setdefault(key, (group, count, []))[2].append(p)
            work.extend(together.values())
        capturing = self._divide(work)
        for group, count, params in work:
            states = [(kept["exp_avg"], kept["exp_avg_sq"], kept.get("scale")) for kept in map(self.state.__getitem__, params)]
            lr = group["lr"]
            if isinstance(lr, torch.Tensor) and lr.device.type == "cpu":
                lr = float(lr)
            count += 1      # in place where it is a tensor
            try:
                op_adamw(params, [p.grad for p in params], states, count, lr, group["betas"], group["eps"], group["weight_decay"])
            except Exception:
                count -= 1      # a step that was refused has not been made
                raise
            for p in params:
                self.state[p]["step"] = count
            if capturing and isinstance(count, torch.Tensor):
                self._recorded[id(count)] = count
        return loss

    def load_state_dict(self, state_dict):
        """torch's own would turn codes and scales into the parameters' type.  States in 8 bits belong to the layout that their parameter had; those in
        32 bits are loaded into any.  A checkpoint of torch.optim.AdamW's is one of states in 32 bits; options of its groups that make other steps
        (amsgrad, maximize) are refused, and those that it lacks stay as they are."""
        saved = state_dict["state"]
        for group in state_dict["param_groups"]:
            other = [name for name in ("amsgrad", "maximize") if group.get(name)]
            if group.get("weight_decay") and not group.get("decoupled_weight_decay", True):
                other.append("weight decay in the gradient")
            if other:
                raise ValueError("the saved optimizer's steps are other ones: %s" % ", ".join(other))
        numbers = [n for group in state_dict["param_groups"] for n in group["params"]]
        # everything that may be refused is looked at before anything is changed
        states = {p: self._loaded(p, saved[n]) for n, p in zip(numbers, (p for group in self.param_groups for p in group["params"])) if saved.get(n)}
        options = [{name: group[name] for name in self.defaults if name in group} for group in self.param_groups]
        super().load_state_dict({**state_dict, "state": {}})
        self._recorded = {}
        for group, had in zip(self.param_groups, options):      # torch's groups have no bits
            for name, value in had.items():
                group.setdefault(name, value)
        for group in self.param_groups:
            counts = {}      # a group's own: each adds to its counts by itself
            for p in group["params"]:
                if p not in states:
                    continue
                step = states[p]["step"]
                if group["capturable"]:
                    step = counts.setdefault((p.device, step), torch.full((), step, dtype=torch.int64, device=p.device))
                self.state[p] = {**states[p], "step": step}

    @staticmethod
    def _loaded(p, held):
        """A parameter's state as it was saved, on its device."""
        bits = 8 if "scale" in held else 32
        made = {name: t for name, t in op_adamw_state(p, bits)._asdict().items() if t is not None}
        for name, to in made.items():
            fits = name in held and (held[name].dtype is to.dtype or bits == 32 and held[name].is_floating_point()) and held[name].shape == to.shape
            if not fits:
                raise ValueError("the saved %s does not belong to its parameter" % name)
            if bits == 8 and _order(held[name]) != _order(to):
                raise ValueError("the saved %s is in another order of memory than its parameter, and its codes' scales go by that order: give the "
                                 "parameter the layout that it had" % name)
            to.copy_(held[name])
        if "step" not in held:
            raise ValueError("the saved state has no step")
        return {"step": int(held["step"]), **made}
