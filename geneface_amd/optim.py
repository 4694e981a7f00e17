"""AdamW over many tensors in one launch, with moments in 32 or 8 bits, and the global norm of their gradients.

What the reference's tasks build around the model (tasks/radnerfs/radnerf.py:53-72: Adam over the networks and the grid tables, eps 1e-15) as
kernels of this library: `AdamW` is a torch optimizer (param groups, state dict, GradScaler), `adamw_step` and `grad_norm` are the two calls below
it.  With `weight_decay=0` it is Adam.

8-bit moments: e4m3 codes with one 32-bit scale for each 128 consecutive values of a tensor, max(largest magnitude, 2^-100) times 1 / 448.  The second
moment is held as its square root, which halves the range it needs.  Codes are rounded by a dither that depends on the step and on the value's
index only, so a step is reproducible and changes far below the format's spacing add up over the steps; a second moment above zero is never rounded
to zero.  Held as its root it does not overflow either: any finite gradient leaves a finite one (in 32 bits, as in torch.optim.AdamW, a gradient above
1.8e19 / sqrt(1 - beta2) leaves an infinite one, and its parameter stands still from then on).  A block that meets a gradient that is no finite number is none afterwards (all 128 values).

Everything is done on the current stream of the tensors' device and may be captured into a graph; a graph keeps the addresses, and numbers given
as Python numbers (`lr` as a one-element tensor on the device stays adjustable).  A step raises the version counters of what it writes; a replay does not:
whoever goes by them (the fused field's packed weights) needs `torch.autograd.graph.increment_version(params)` behind it.
"""
import ctypes as C
import math

import torch

from .lib import host

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
BLOCK = 128

_vp = C.c_void_p


class GfAdamw(C.Structure):
    """ctypes mirror of gf_adamw_t (include/geneface_train_hip.h)."""
    _fields_ = [("tensors_host", _vp), ("count", C.c_uint32), ("dtype", C.c_uint32), ("state_bits", C.c_uint32), ("_pad", C.c_uint32)] + \
               [(n, C.c_double) for n in ("lr", "beta1", "beta2", "eps", "weight_decay", "max_norm")] + \
               [(n, _vp) for n in ("lr_device", "grad_scale", "found_inf", "grad_norm", "grad_norm_wide")]


class GfGradNorm(C.Structure):
    """ctypes mirror of gf_grad_norm_t."""
    _fields_ = [("tensors_host", _vp), ("count", C.c_uint32), ("_pad", C.c_uint32)] + [(n, _vp) for n in ("grad_scale", "norm_out", "workspace", "norm_out_wide")]


def grad_norm(grads, grad_scale=None):
    """sqrt(sum of the squares of all `grads`) / grad_scale as a float32 tensor without dimensions, added up in 64 bits in a fixed order.

    grads: tensors of float32, bfloat16 or float16 on one device (None entries are left out).  grad_scale: one float32 on that device, the
    factor the gradients carry (GradScaler's scale).  Infinities and NaN among the gradients give an infinite norm or NaN.  The
    tensor's attribute `wide` holds the same in float64: `adamw_step` goes by it as long as it rounds to the tensor's own value."""
    norm, wide = host().grad_norm([g for g in grads if g is not None], grad_scale)
    norm.wide = wide
    return norm


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, steps, *, lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, exp_avg_scales=None,
               exp_avg_sq_scales=None, grad_scale=None, found_inf=None, grad_norm=None, max_norm=None):
    """One AdamW step over lists of tensors, in place, in one launch for every 56 tensors of a type.

    params, grads: float32, bfloat16 or float16, gradients of their parameter's type and size.  exp_avgs, exp_avg_sqs: float32 of the same sizes,
    or -- with exp_avg_scales and exp_avg_sq_scales, lists of float32 [ceil(numel / 128)] -- float8_e4m3fn.  steps: one float32 each, the number of
    steps taken so far.  Everything on one device; all but gradients must be contiguous.  What is written shares memory with
    nothing else that is given (a gradient may be its own parameter).

    lr: a number, or one float32 on the device.  grad_scale: the factor that the gradients carry.  found_inf: where it is not 0 nothing is
    changed, the step counts included.  grad_norm, max_norm: gradients are multiplied by min(1, max_norm / (grad_norm + 1e-6)); both or neither.
    grad_scale, found_inf, grad_norm: one float32 on the device each.  Gradients are only read: they keep their factor."""
    if (exp_avg_scales is None) != (exp_avg_sq_scales is None):
        raise RuntimeError("adamw_step: exp_avg_scales and exp_avg_sq_scales must both be given for 8-bit moments")
    beta1, beta2 = map(float, betas)
    if not (0 <= beta1 < 1 and 0 <= beta2 < 1):
        raise ValueError(f"adamw_step: betas must be in [0, 1), got {betas}")
    if (grad_norm is None) != (max_norm is None):
        raise RuntimeError("adamw_step: grad_norm and max_norm go together")
    lr_device = None
    if torch.is_tensor(lr) and lr.is_cuda:
        lr, lr_device = 0.0, lr
    host().adamw_step(params, grads, exp_avgs, exp_avg_sqs, steps, float(lr), lr_device, beta1, beta2, float(eps), float(weight_decay), exp_avg_scales,
                      exp_avg_sq_scales, grad_scale, found_inf, grad_norm, getattr(grad_norm, "wide", None), math.inf if max_norm is None else float(max_norm))


class AdamW(torch.optim.Optimizer):
    """torch.optim.AdamW's update (without amsgrad and maximize) in one launch for all tensors of a param group and type.

    state_bits: 32, or 8 for moments of one byte each and a scale per 128 values (16 bytes moved per float32 parameter instead of 28).
    max_grad_norm: clips the gradients of ALL groups to this norm inside the step; the norm of the last step stays in `last_grad_norm`.  The
    gradients themselves are not changed.  Under torch.amp.GradScaler unscaling and the skipped step after an overflow happen inside the kernel, without a
    host sync.  lr may be a one-element float32 tensor on the device, so that a captured step follows a schedule; a parameter's first step is not captured."""

    _step_supports_amp_scaling = True      # GradScaler.step hands its scale and found_inf over as attributes and calls step() itself

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, *, state_bits=32, max_grad_norm=None):
        if state_bits not in (32, 8):
            raise ValueError(f"state_bits must be 32 or 8, got {state_bits}")
        if not torch.is_tensor(lr) and not lr >= 0:
            raise ValueError(f"Invalid learning rate: {lr}")
        if not (0 <= betas[0] < 1 and 0 <= betas[1] < 1):
            raise ValueError(f"Invalid betas: {betas}")
        if not eps >= 0:
            raise ValueError(f"Invalid epsilon value: {eps}")
        if not weight_decay >= 0:
            raise ValueError(f"Invalid weight_decay value: {weight_decay}")
        if max_grad_norm is not None and not max_grad_norm > 0:
            raise ValueError(f"Invalid max_grad_norm: {max_grad_norm}")
        self.state_bits, self.max_grad_norm, self.last_grad_norm = state_bits, max_grad_norm, None
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay))

    def __getstate__(self):      # torch's keeps only state and groups: copies and pickles need these as well
        return {**super().__getstate__(), "state_bits": self.state_bits, "max_grad_norm": self.max_grad_norm, "last_grad_norm": None}

    def _keys(self):
        return ("exp_avg", "exp_avg_sq") + (("exp_avg_scale", "exp_avg_sq_scale") if self.state_bits == 8 else ())

    def _init_state(self, p):
        state = self.state[p]
        if not state:
            if p.dtype not in DTYPES or not p.is_cuda or not p.is_contiguous():
                raise RuntimeError("AdamW: parameters must be contiguous CUDA tensors of float32, bfloat16 or float16")
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("AdamW: a parameter's first step cannot be captured (every replay would start its state anew): take one before, or load a state")
            state["step"] = torch.zeros((), dtype=torch.float32, device=p.device)
            for k in self._keys():
                if k.endswith("scale"):
                    state[k] = torch.zeros(-(-p.numel() // BLOCK), dtype=torch.float32, device=p.device)
                elif self.state_bits == 8:
                    state[k] = torch.zeros(p.shape, dtype=torch.uint8, device=p.device).view(torch.float8_e4m3fn)
                else:
                    state[k] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
        return state

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        groups = [[p for p in g["params"] if p.grad is not None] for g in self.param_groups]
        used = [p for g in groups for p in g]
        if not used:
            return loss
        devices = {p.device for p in used}
        scale, found = getattr(self, "grad_scale", None), getattr(self, "found_inf", None)
        norm = None
        if self.max_grad_norm is not None:
            if len(devices) > 1:
                raise RuntimeError("AdamW: max_grad_norm needs all parameters on one device")
            norm = grad_norm([p.grad for p in used], grad_scale=None if scale is None else scale.to(used[0].device))
            self.last_grad_norm = norm
        for group, params in zip(self.param_groups, groups):
            for dev in sorted({p.device for p in params}, key=str):
                ps = [p for p in params if p.device == dev] if len(devices) > 1 else params
                states = [self._init_state(p) for p in ps]
                column = lambda k: [s[k] for s in states]      # noqa: E731
                there = lambda t: None if t is None else t.to(dev)      # noqa: E731
                eight = self.state_bits == 8
                adamw_step(ps, [p.grad for p in ps], column("exp_avg"), column("exp_avg_sq"), column("step"), lr=group["lr"], betas=group["betas"],
                           eps=group["eps"], weight_decay=group["weight_decay"], exp_avg_scales=column("exp_avg_scale") if eight else None,
                           exp_avg_sq_scales=column("exp_avg_sq_scale") if eight else None, grad_scale=there(scale), found_inf=there(found),
                           grad_norm=norm, max_norm=self.max_grad_norm if norm is not None else None)
        return loss

    def moments(self, p):
        """(first moment, second moment) of a parameter as new float32 tensors of its shape, whatever they are held in."""
        s = self.state[p]
        if self.state_bits == 32:
            return s["exp_avg"].clone(), s["exp_avg_sq"].clone()
        wide = lambda k: s[k].float().reshape(-1) * s[k + "_scale"].repeat_interleave(BLOCK)[:p.numel()]      # noqa: E731
        return wide("exp_avg").view(p.shape), wide("exp_avg_sq").square().view(p.shape)

    def load_state_dict(self, state_dict):
        """State of this class, or -- with 32-bit moments -- of torch.optim.Adam / AdamW.  Moments keep their own types (torch would cast them to the
        parameter's)."""
        want = {k: torch.float8_e4m3fn if self.state_bits == 8 and not k.endswith("scale") else torch.float32 for k in self._keys()}
        for s in state_dict["state"].values():
            missing = [k for k in ("step", *want) if k not in s]
            if missing or any(s[k].dtype != dt for k, dt in want.items()):
                raise RuntimeError(f"AdamW: the state does not hold {self.state_bits}-bit moments")
        for g in state_dict["param_groups"]:
            if g.get("amsgrad") or g.get("maximize") or (g.get("weight_decay") and not g.get("decoupled_weight_decay", True)):
                raise RuntimeError("AdamW: a state with amsgrad, maximize or Adam's own weight decay belongs to another update")
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        params = [p for g in self.param_groups for p in g["params"]]
        for i, p in zip(ids, params):
            for k in want if i in state_dict["state"] else ():
                held, shape = tuple(state_dict["state"][i][k].shape), (-(-p.numel() // BLOCK),) if k.endswith("scale") else tuple(p.shape)
                if held != shape:
                    raise RuntimeError(f"AdamW: {k} of shape {held} for a parameter of shape {tuple(p.shape)}")
        super().load_state_dict(state_dict)
        for i, p in zip(ids, params):
            s = state_dict["state"].get(i)
            if s is None:
                continue
            self.state[p] = {"step": torch.as_tensor(s["step"], dtype=torch.float32).detach().to(p.device, copy=True).reshape(()),
                             **{k: s[k].detach().to(p.device, copy=True).contiguous() for k in want}}
