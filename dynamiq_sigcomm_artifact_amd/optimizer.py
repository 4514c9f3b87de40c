"""What follows the all-reduce in a training step: the norm of the gradients with the factor that clips them, and the AdamW step,
its states in 32 bits or in 8.

``grad_norm`` and ``adamw_step`` are the operators, on lists of tensors of any sizes, a launch for every 192 and 112 of them (of one element
type at a time); ``AdamW`` keeps the states and the count of the steps for them.  ``include/dynamiq_eden.h`` (dq_grad_norm, dq_adamw_step) has the
formulas and the 8-bit format to the bit.  Everything runs on the current stream of the tensors' device and nothing is read back."""
import torch

from . import capi

_HALF = (torch.float16, torch.bfloat16)


def _tensors(of, what):
    """a list of tensors; one tensor would be taken apart into its rows"""
    if isinstance(of, torch.Tensor):
        raise RuntimeError("%s: a list of tensors is required" % what)
    return list(of)


def _contiguous(grad):
    return grad if grad is None or grad.is_contiguous() else grad.contiguous()


def norm_work(device):
    """the work buffer of grad_norm: kept from call to call, one for every stream (or recorded graph) whose calls may overlap"""
    return torch.empty(int(capi.lib().dq_grad_norm_work_doubles()), dtype=torch.float64, device=device)


def grad_norm(grads, max_norm=None, work=None, out=None):
    """float32 [2] on the device: the 2-norm of all tensors together, summed in 64 bits, and min(1, max_norm / (norm + 1e-6)), the
    ``grad_scale`` of a step that clips (1 without max_norm).  Where the norm is not finite the factor is NaN, and the step
    changes nothing.  grads: contiguous tensors; None among them takes no part (where all are, work or out names the device).
    work: from norm_work(); without it the call makes one."""
    listed = _tensors(grads, "grad_norm")
    grads = [g for g in listed if g is not None]
    beside = grads[0] if grads else out if work is None else work
    if not listed or beside is None:
        raise RuntimeError("grad_norm: no tensors")
    if work is None:
        work = norm_work(beside.device)
    if out is None:
        out = torch.empty(2, dtype=torch.float32, device=beside.device)
    capi.host().grad_norm(grads, float("inf") if max_norm is None else max_norm, work, out)
    return out


def padded_elements(params):
    """elements of the state arenas of a list of parameters: each padded to whole blocks of 32, one after the other"""
    return sum(-(-p.numel() // 32) * 32 for p in params)


def adamw_state(params, bits=32):
    """fresh states of a list of parameters for adamw_step: float32 [2, total] (the moments m and v), or for 8 bits (codes uint8
    [2, total], scales uint8 [2, total / 32]) of m and sqrt(v).  A parameter's states begin at a multiple of 32 (padded_elements)."""
    params = _tensors(params, "adamw_state")
    if not params:
        raise RuntimeError("adamw_state: no parameters")
    total, device = padded_elements(params), params[0].device
    if bits == 32:
        return torch.zeros((2, total), dtype=torch.float32, device=device)
    if bits != 8:
        raise RuntimeError("adamw_state: states are held in 32 or in 8 bits")
    return (torch.zeros((2, total), dtype=torch.uint8, device=device), torch.zeros((2, total // 32), dtype=torch.uint8, device=device))


def master_weights(params):
    """float32 copies of 16-bit parameters in one arena, laid out as their states are"""
    params = _tensors(params, "master_weights")
    if not params:
        raise RuntimeError("master_weights: no parameters")
    out = torch.zeros(padded_elements(params), dtype=torch.float32, device=params[0].device)
    at = 0
    for p in params:
        out[at:at + p.numel()].copy_(p.detach().reshape(-1))
        at += -(-p.numel() // 32) * 32
    return out


def adamw_step(params, grads, state, step, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, master=None, grad_scale=None, coefficients=None):
    """one AdamW step in place.  params, grads: lists of contiguous tensors of the same sizes (fp16, bf16 or fp32 each; a gradient None leaves
    its parameter as it is) that share no memory with the parameters; state: of adamw_state; step: the number of this step, from 1; master: of master_weights, for 16-bit
    parameters; grad_scale: float32 tensor [1] that multiplies the gradients (grad_norm's factor, a loss scale's inverse) -- where it is
    infinite or NaN the step changes nothing; coefficients: of adamw_coefficients, in place of step, lr and weight_decay."""
    if isinstance(params, torch.Tensor) or isinstance(grads, torch.Tensor):
        raise RuntimeError("adamw_step: lists of tensors are required")
    codes, scales = state if isinstance(state, (tuple, list)) else (state, None)
    capi.host().adamw_step(params, grads, codes, scales, master, grad_scale, coefficients, step, lr, betas[0], betas[1], eps, weight_decay)


def adamw_coefficients(steps, coefficients, lr=1e-3, betas=(0.9, 0.999), weight_decay=1e-2, grad_scale=None):
    """advances the count of the steps in device memory (int64 [1]) and writes what the next adamw_step takes from it (float32 [4]), unless
    grad_scale is infinite or NaN.  lr: a number or a float32 tensor [1].  For steps that are recorded into a graph."""
    capi.host().adamw_coefficients(steps, lr, betas[0], betas[1], weight_decay, grad_scale, coefficients)


class AdamW(object):
    """AdamW over parameters or groups of them (dicts with "params" and, where they differ, "lr", "betas", "eps", "weight_decay"):

        opt = AdamW(model.parameters(), lr=3e-4, bits=8)
        loss.backward()
        clip = grad_norm(opt.grads(), 1.0, work=opt.work)
        opt.step(grad_scale=clip[1:])

    bits: of the states.  master: float32 master weights beside 16-bit parameters.  ``param_groups`` may be changed between steps (a
    learning rate's schedule).  A parameter without a gradient is left as it is; the steps are counted for all parameters together, those that
    grad_scale makes do nothing excepted.  What grad_scale is the device alone knows: from the first step that is given one the count lives
    there, and advancing it is a launch more for each group.

    capturable: the count lives there from the beginning, and lr may be a float32
    tensor [1] that is read when a step runs: step() may then be recorded into a graph and replayed, with gradients at the addresses of the
    recording.  Replays and other steps of the object follow one another on one stream, or in an order that the caller sees to."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, bits=32, master=True, capturable=False):
        params = _tensors(params, "AdamW")
        if not params:
            raise RuntimeError("AdamW: no parameters")
        groups = params if isinstance(params[0], dict) else [{"params": params}]
        defaults = {"lr": lr, "betas": betas, "eps": eps, "weight_decay": weight_decay}
        self.bits, self.capturable = bits, bool(capturable)
        self.param_groups = [{**defaults, **g, "params": _tensors(g["params"], "AdamW")} for g in groups]
        every = self.params()
        if len({id(p) for p in every}) < len(every):
            raise RuntimeError("AdamW: a parameter appears twice")
        if not every:
            raise RuntimeError("AdamW: no parameters")
        self.device = every[0].device
        # parameters that share arenas: those of a group with master weights, and those without
        self._parts = []
        for g, group in enumerate(self.param_groups):
            for with_master in (False, True):
                chosen = [p for p in group["params"] if (bool(master) and p.dtype in _HALF) == with_master]
                if chosen:
                    self._parts.append({"group": g, "params": chosen, "state": adamw_state(chosen, bits),
                                        "master": master_weights(chosen) if with_master else None})
        # the steps done: a number, or None and a count per group on the device, all of them the same
        self._count = None if self.capturable else 0
        self._steps = torch.zeros(len(self.param_groups), dtype=torch.int64, device=self.device)
        self._coefficients = torch.zeros((len(self.param_groups), 4), dtype=torch.float32, device=self.device)
        self._work = None

    @property
    def work(self):
        """a work buffer for grad_norm"""
        if self._work is None:
            self._work = norm_work(self.device)
        return self._work

    @property
    def steps(self):
        """the steps done (waits for the device where it counts them)"""
        return int(self._steps[0]) if self._count is None else self._count

    @steps.setter
    def steps(self, done):
        self._steps.fill_(done)
        if self._count is not None:
            self._count = int(done)

    def params(self):
        return [p for group in self.param_groups for p in group["params"]]

    def grads(self):
        """the parameters' gradients as step() takes them: contiguous (copies of those that are not), None where there is none"""
        return [_contiguous(p.grad) for p in self.params()]

    def zero_grad(self, set_to_none=True):
        for p in self.params():
            if set_to_none:
                p.grad = None
            elif p.grad is not None:
                p.grad.detach_().zero_()

    @torch.no_grad()
    def step(self, grad_scale=None):
        if grad_scale is not None and self._count is not None and not torch.cuda.is_current_stream_capturing():
            self._steps.fill_(self._count)
            self._count = None
        counted = self._count is None
        if counted:
            for g, group in enumerate(self.param_groups):
                lr = group["lr"] if self.capturable else float(group["lr"])
                adamw_coefficients(self._steps[g:g + 1], self._coefficients[g], lr, group["betas"], group["weight_decay"], grad_scale)
        else:
            self._count += 1
        for part in self._parts:
            group = self.param_groups[part["group"]]
            grads = [_contiguous(p.grad) for p in part["params"]]
            if all(g is None for g in grads):
                continue
            adamw_step(part["params"], grads, part["state"], 1 if counted else self._count, 0.0 if counted else group["lr"], group["betas"], group["eps"],
                       group["weight_decay"], part["master"], grad_scale, self._coefficients[part["group"]] if counted else None)

    def state_dict(self):
        """copies of the states: a step after load_state_dict() is the step that would have followed"""
        def copy(x):
            return None if x is None else tuple(t.clone() for t in x) if isinstance(x, tuple) else x.clone()
        return {"bits": self.bits, "steps": self._steps.tolist() if self._count is None else [self._count] * len(self.param_groups),
                "groups": [{k: copy(v) if isinstance(v, torch.Tensor) else v for k, v in group.items() if k != "params"} for group in self.param_groups],
                "parts": [{"state": copy(part["state"]), "master": copy(part["master"])} for part in self._parts]}

    def load_state_dict(self, saved):
        def tensors(part):
            state = part["state"]
            return (list(state) if isinstance(state, (tuple, list)) else [state]) + ([] if part["master"] is None else [part["master"]])
        mine, theirs = [t for p in self._parts for t in tensors(p)], [t for p in saved["parts"] for t in tensors(p)]
        if saved["bits"] != self.bits or len(saved["groups"]) != len(self.param_groups) or [(t.shape, t.dtype) for t in mine] != [(t.shape, t.dtype) for t in theirs]:
            raise RuntimeError("AdamW: the saved states are of other parameters, or in another number of bits")
        for to, t in zip(mine, theirs):
            to.copy_(t)
        for group, was in zip(self.param_groups, saved["groups"]):
            for k, v in was.items():
                if isinstance(v, torch.Tensor) and isinstance(group.get(k), torch.Tensor):
                    group[k].copy_(v)
                elif isinstance(v, torch.Tensor): # (a step on the device reads it there)
                    group[k] = v.detach().to(self.device if self.capturable else v.device, copy=True)
                else:
                    group[k] = v
        if self._count is not None:
            self._count = saved["steps"][0]
        self._steps.copy_(torch.tensor(saved["steps"], dtype=torch.int64))
