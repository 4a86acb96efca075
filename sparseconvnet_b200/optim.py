"""AdamW over all parameters of a network in one kernel, moments in 32 bits or in 8.

``adamw_step`` is the step on plain lists of tensors, ``AdamW`` the torch optimizer around it.  Stands beside the
data-parallel helpers of ``shard.py``: ``shard.sum_gradients(parameters)`` and then ``optimizer.step()``."""
import torch

from . import SCN

BLOCK = 256  # values of a block that shares a scale, in 8-bit moments


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, step, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2,
               exp_avg_scales=None, exp_avg_sq_scales=None, seed=0, copies=None):
    """One step, in place, over lists of contiguous CUDA tensors of one type each:

        m = b1 m + (1 - b1) g        v = b2 v + (1 - b2) g^2        t = step + 1
        p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v / (1 - b2^t)) + eps)

    params, grads: float32, bfloat16 or float16 (each list one type).  step: int64 CUDA tensor of one value, the steps done
    so far; it is advanced on the device, so a captured step counts on when it is replayed.  lr: a number, or a float32
    CUDA tensor of one value that is read when the step runs.

    exp_avgs, exp_avg_sqs: float32 m and v.  With the scales (float32, one per block of 256 values): float8_e4m3fn m and
    sqrt(v), which stand for value * scale of the block; they are rounded by chance in proportion to the distance of the two
    neighbours, with bits that depend on seed, step and place only, so a run can be repeated.  A gradient that is no
    number makes its value's moments NaN, in 8 bits those of its block.
    copies: bfloat16 or float16 tensors that receive the new parameters as well.

    All work is queued on the current stream.  The call refuses lists in which a tensor occurs twice; tensors that overlap in
    other ways must not be passed."""
    SCN._binding.adamw_step(params, grads, exp_avgs, exp_avg_sqs, exp_avg_scales, exp_avg_sq_scales, copies, step, lr,
                            betas[0], betas[1], eps, weight_decay, seed)


def _state_of(p, bits):
    if bits == 32:
        return {"exp_avg": torch.zeros(p.shape, dtype=torch.float32, device=p.device),
                "exp_avg_sq": torch.zeros(p.shape, dtype=torch.float32, device=p.device)}
    blocks = -(-p.numel() // BLOCK)
    made = {}
    for k in ("exp_avg", "exp_avg_sq"):
        made[k] = torch.zeros(p.shape, dtype=torch.uint8, device=p.device).view(torch.float8_e4m3fn)
        made[k + "_scale"] = torch.zeros(blocks, device=p.device)
    return made


def _check_group(group):
    if not isinstance(group["lr"], torch.Tensor) and not group["lr"] >= 0:
        raise ValueError("lr must not be negative")
    if not (0 <= group["betas"][0] < 1 and 0 <= group["betas"][1] < 1):
        raise ValueError("betas must lie in [0, 1)")
    if not group["eps"] >= 0 or not group["weight_decay"] >= 0:
        raise ValueError("eps and weight_decay must not be negative")
    if group["state_bits"] not in (8, 32):
        raise ValueError("state_bits must be 8 or 32")


def _captures(p):
    return p.is_cuda and torch.cuda.is_current_stream_capturing()


def _not_captured(p, what):
    if _captures(p):
        raise RuntimeError("AdamW cannot capture %s.  Take such a step before the capture." % what)


class AdamW(torch.optim.Optimizer):
    """torch.optim.AdamW's update on the GPU, one launch for all parameters of a group that have one type and as many steps.

    state_bits: 32, or 8 for moments of 8 bits with a scale per 256 values (2.03 bytes a value instead of 8).
    master_weights: for bfloat16 / float16 parameters, keep them in float32 as well and round the parameters from those;
    without it an update smaller than half a step of the parameter's type is lost.
    lr of a group may be a float32 CUDA tensor of one value.  Parameters without a gradient are left as they are, and their
    step is not counted.  A step can be captured into a graph after the same parameters have taken one outside.  There is no amsgrad, no maximize and no CPU path."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32, master_weights=False, seed=0):
        defaults = dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits, master_weights=master_weights, seed=seed)
        _check_group(defaults)
        super().__init__(params, defaults)

    def add_param_group(self, param_group):
        """As torch's; a group's own values are checked like the constructor's."""
        if isinstance(param_group, dict):
            _check_group({**self.defaults, **param_group})
        super().add_param_group(param_group)

    def _start(self, p, group):
        state = _state_of(p, group["state_bits"])
        if group["master_weights"] and p.dtype != torch.float32:
            state["master"] = p.detach().float()
        return state

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for number, group in enumerate(self.param_groups):
            fresh = {}     # device -> the counter of parameters that take their first step now
            keys = {}      # counter -> its count where the host knows it, and its device
            users = {}     # counter -> how many parameters have it
            together = {}  # parameters that step as one list: one count, one device, one type -> they and their states
            for p in group["params"]:
                grad = p.grad
                if grad is None:
                    state = self.state.get(p)
                    if state:
                        users[id(state["step"])] = users.get(id(state["step"]), 0) + 1
                    continue
                if grad.is_sparse:
                    raise RuntimeError("AdamW does not take sparse gradients")
                state = self.state[p]
                if not state:
                    _not_captured(p, "a parameter's first step: its moments would begin anew with every replay")
                    state.update(self._start(p, group))
                    if p.device not in fresh:
                        fresh[p.device] = self._note(torch.zeros(1, dtype=torch.int64, device=p.device), 0)
                    state["step"] = fresh[p.device]
                step = id(state["step"])
                users[step] = users.get(step, 0) + 1
                if step not in keys:
                    keys[step] = (self._count(state["step"]), p.device)
                    if keys[step][0] is None:
                        keys[step] = (None, step)
                ps, states = together.setdefault((keys[step], p.dtype, grad.dtype, "master" in state), ([], []))
                ps.append(p)
                states.append(state)
            for ((count, _), _, _, master), (ps, states) in together.items():
                step = self._one_counter(ps, states, users)
                column = lambda k: [s[k] for s in states] if k in states[0] else None  # noqa: E731
                adamw_step(column("master") if master else ps, [p.grad for p in ps], column("exp_avg"), column("exp_avg_sq"),
                           step, group["lr"], group["betas"], group["eps"], group["weight_decay"],
                           column("exp_avg_scale"), column("exp_avg_sq_scale"), group["seed"] + number, ps if master else None)
                self._note(step, None if count is None or _captures(ps[0]) else count + 1)
        return loss

    # What the host knows of the counters on the device, so that parameters whose counts have become equal step as one list
    # again: id -> (counter, its version then, count).  A captured step advances its counter without the host, so from
    # then on that one's count is not known; neither is it after someone else has written to it.
    def _note(self, step, count):
        known = self.__dict__.setdefault("_known", {})
        known.pop(id(step), None)
        if count is not None and not step.is_inference():
            if len(known) > 2 * len(self.state):
                used = {id(s["step"]) for s in self.state.values() if s}
                for k in [k for k in known if k not in used]:
                    del known[k]
            known[id(step)] = (step, step._version, count)
        return step

    def _count(self, step):
        held = self.__dict__.get("_known", {}).get(id(step))
        return held[2] if held is not None and held[0] is step and held[1] == step._version else None

    def _one_counter(self, ps, states, users):
        """The counter of a list that steps now.  The list alone advances it: parameters that had it too but step in another list, or
        not at all this time, keep the old count in the old one."""
        here = {}
        for state in states:
            here[id(state["step"])] = here.get(id(state["step"]), 0) + 1
        for state in states:
            if users[id(state["step"])] == here[id(state["step"])]:
                step = state["step"]
                break
        else:
            _not_captured(ps[0], "a step of some of the parameters that have stepped together: their count would begin anew with every replay")
            step = self._note(states[0]["step"].clone(), self._count(states[0]["step"]))
        if len(here) > 1 or id(step) not in here:
            for state in states:
                state["step"] = step
        return step

    def _check_checkpoint(self, state_dict):
        saved = state_dict["param_groups"]
        if [len(g["params"]) for g in saved] != [len(g["params"]) for g in self.param_groups]:
            return  # (torch refuses it)
        for s, group in zip(saved, self.param_groups):
            missing = sorted(set(self.defaults) - set(s))
            if missing:
                raise ValueError("the checkpoint is another optimizer's: a group of it has no %s" % ", ".join(missing))
            _check_group(s)
            for i, p in zip(s["params"], group["params"]):
                state = state_dict["state"].get(i)
                if not state:
                    continue
                n, master = p.numel(), s["master_weights"] and p.dtype != torch.float32
                moments = (torch.float32, n) if s["state_bits"] == 32 else (torch.float8_e4m3fn, n)
                want = dict(exp_avg=moments, exp_avg_sq=moments, step=(torch.int64, 1))
                if s["state_bits"] == 8:
                    want.update(exp_avg_scale=(torch.float32, -(-n // BLOCK)), exp_avg_sq_scale=(torch.float32, -(-n // BLOCK)))
                if master:
                    want["master"] = (torch.float32, n)
                have = {k: (v.dtype, v.numel()) if isinstance(v, torch.Tensor) else v for k, v in state.items()}
                if have != want:
                    raise ValueError("the checkpoint does not fit parameter %s: it holds %s, %s expected" % (i, have, want))

    def load_state_dict(self, state_dict):
        """As torch's, but states keep their types (torch casts them to the parameter's), and parameters with the same count
        share a counter again.  A checkpoint of another optimizer, or of parameters of other sizes, is refused."""
        self._check_checkpoint(state_dict)
        super().load_state_dict(state_dict)
        for saved, group in zip(state_dict["param_groups"], self.param_groups):
            counters = {}
            for i, p in zip(saved["params"], group["params"]):
                if state_dict["state"].get(i):
                    state = {k: v.to(p.device, copy=True) for k, v in state_dict["state"][i].items()}
                    count = int(state["step"])
                    state["step"] = counters.setdefault((count, p.device), state["step"])
                    self._note(state["step"], count)
                    self.state[p] = state
