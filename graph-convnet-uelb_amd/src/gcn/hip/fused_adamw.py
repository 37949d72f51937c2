"""Multi-tensor AdamW on the HIP library, with moments in fp32 or in 8 bits, and the global gradient norm it clips by.

``FusedAdamW`` is used like ``torch.optim.AdamW`` (the reference trains with ``torch.optim.Adam`` only,
``src/gcn/train/trainer.py:95``): the same constructor arguments but for amsgrad, maximize, foreach,
differentiable and fused, the same ``param_groups``, and with 32-bit states the same
``state_dict`` layout, so optimizer checkpoints move between the two.  ``adamw_step_`` and ``grad_norm`` are the same
operations on lists of tensors.  Formulas, formats and what the kernels do are described in ``include/gcn_uelb_hip.h``.

8-bit states hold one e4m3 code per element (uint8) and one exponent byte per ``STATE8_BLOCK`` elements, for the first moment
and for the square root of the second; ``state8_decode`` / ``state8_encode`` convert them.
"""
from __future__ import annotations

import ctypes
import itertools

import torch

from . import lib as L

STATE8_BLOCK = 128
_TYPES = (torch.float32, torch.bfloat16, torch.float16)

def _blocks_of(n):
    return -(-n // STATE8_BLOCK)


def adamw_step_(params, grads, exp_avgs, exp_avg_sqs, *, step, lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, masters=None,
                exp_avg_exps=None, exp_avg_sq_exps=None, grad_scale=None, clip_coef=None, seed=0, first_tensor=0, hyper=None):
    """One AdamW step on lists of tensors, in place (parameters, master copies and moments; gradients stay as they are).

    params, grads: float32, bfloat16 or float16, one type per call.  masters: float32 copies of 16-bit parameters (needed with
    them, not taken with float32).  exp_avgs, exp_avg_sqs: float32; or, with exp_avg_exps and exp_avg_sq_exps (uint8, one per
    STATE8_BLOCK elements), uint8 codes.  step: 1-based count of this update.  grad_scale, clip_coef: float32 scalars on the
    device that the gradients are multiplied by (``grad_norm`` returns the latter).  seed, first_tensor: enter the random
    bits of the 8-bit states' rounding, as does a tensor's place in the list.  hyper: what ``adamw_advance_`` filled, in place
    of step and of the numbers from lr on; a step that is captured into a graph needs it.  The tensors of a call must not
    overlap."""
    if hyper is None and (int(step) != step or step < 1):
        raise ValueError(f"step counts from 1, got {step}")
    L.binding().adamw_step(params, grads, exp_avgs, exp_avg_sqs, masters, exp_avg_exps, exp_avg_sq_exps, int(step), lr, betas[0], betas[1], eps,
                           weight_decay, seed, first_tensor, grad_scale, clip_coef, hyper)


def adamw_hyper(device):
    """Memory for ``adamw_advance_``."""
    return torch.zeros(L.load().gcn_adamw_hyper_bytes(), dtype=torch.uint8, device=device)


def _check_device_lr(lr, device):
    if lr.dtype != torch.float32 or lr.numel() != 1 or lr.device != device:
        raise TypeError("lr on the device is a float32 tensor of one element, where step is")


def adamw_advance_(step, hyper, *, lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, seed=0):
    """Adds 1 to ``step`` (an int64 scalar on the device) and puts what ``adamw_step_`` needs for that step into ``hyper``, both on
    the device, so that a captured graph counts on when it is replayed.  lr: a number, or a float32 scalar on the device."""
    if step.dtype != torch.int64 or step.numel() != 1:
        raise TypeError("step is an int64 tensor of one element")
    lib = L.load()
    L.require_cuda(step, "step")
    dev = step.device
    if hyper.device != dev or hyper.dtype != torch.uint8 or hyper.numel() < lib.gcn_adamw_hyper_bytes():
        raise ValueError("hyper is what adamw_hyper returned, on step's device")
    on_device = isinstance(lr, torch.Tensor)
    if on_device:
        _check_device_lr(lr, dev)
    desc = L.AdamWDesc(n=0, state_bits=32, lr=0.0 if on_device else lr, beta1=betas[0], beta2=betas[1], eps=eps,
                       weight_decay=weight_decay, seed=seed)
    with L.device_guard(dev):
        rc = lib.gcn_adamw_advance(ctypes.byref(desc), step.data_ptr(), lr.data_ptr() if on_device else None, hyper.data_ptr(), L.stream_ptr(dev))
    L.check(rc, "gcn_adamw_advance")


def grad_norm(grads, *, max_norm=None, grad_scale=None):
    """(norm, coefficient): the 2-norm of all gradients together, times grad_scale, and min(1, max_norm / (norm + 1e-6)) or None
    without max_norm, as scalars on the device.  The gradients are of one type and on one GPU and are not changed; autograd takes the
    results as constants."""
    return L.binding().grad_norm(grads, max_norm, grad_scale)


# ------------------------------------------------------------------------------------------------ 8-bit states
def state8_decode(codes, exps):
    """float32 values of the codes of one tensor (any shape) and its exponent bytes: the first moment, or the square root of the
    second."""
    n = codes.numel()
    scale = (exps.to(torch.int32) << 23).view(torch.float32).repeat_interleave(STATE8_BLOCK)[:n]
    return (codes.reshape(-1).view(torch.float8_e4m3fn).float() * scale).view(codes.shape)


def state8_encode(x, never_zero=False):
    """(codes, exponent bytes) of float32 values, rounded to the nearest code: how states in fp32 become 8-bit ones.
    never_zero: values above zero keep at least the smallest code (the square root of a second moment)."""
    n = x.numel()
    rows = torch.nn.functional.pad(x.detach().reshape(-1).float(), (0, -n % STATE8_BLOCK)).view(-1, STATE8_BLOCK)
    rows = torch.nan_to_num(rows, nan=0.0, posinf=0.0, neginf=0.0)
    exps = ((rows.abs().amax(1, keepdim=True).view(torch.int32) >> 23) - 7).clamp_(min=1)
    scaled = rows * ((254 - exps) << 23).view(torch.float32)
    if never_zero:
        scaled = torch.where(scaled > 0, scaled.clamp(min=2.0 ** -9), scaled)
    codes = scaled.to(torch.float8_e4m3fn).view(torch.uint8).view(-1)[:n].clone().view(x.shape)
    return codes, exps.view(-1).to(torch.uint8)


# ------------------------------------------------------------------------------------------------ optimizer
_KEPT = ("exp_avg", "exp_avg_sq", "exp_avg_exp", "exp_avg_sq_exp", "master")


class FusedAdamW(torch.optim.Optimizer):
    """AdamW over all parameters in a few launches.

    state_bits: 32, or 8 for parameters of at least ``min_8bit_numel`` elements (smaller ones keep fp32 moments: they are no
    memory, and biases and norms are the ones that suffer).  Parameters in bfloat16 or float16 get a float32 master copy
    (``state[p]["master"]``) that holds the exact weight: after writing to such a parameter from outside, call ``sync_masters``.
    max_grad_norm: clip all gradients together to this norm within the step (``.grad`` itself is not changed);
    ``grad_norm`` then holds the norm before clipping, a scalar on the device.  capturable: count the steps on the device, so
    that ``step`` can be captured into a graph; run one step before capturing, which makes the states.  seed: of the stochastic
    rounding of 8-bit states; leave it equal on all ranks of data-parallel training, so that they stay equal."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, state_bits=32, min_8bit_numel=4096,
                 max_grad_norm=None, capturable=False, seed=0):
        if not isinstance(lr, torch.Tensor) and not 0.0 <= lr:
            raise ValueError(f"Invalid learning rate: {lr}")
        if isinstance(lr, torch.Tensor) and not capturable:
            raise ValueError("lr as a tensor needs capturable=True")
        if not 0.0 <= eps:
            raise ValueError(f"Invalid epsilon value: {eps}")
        for k in range(2):
            if not 0.0 <= betas[k] < 1.0:
                raise ValueError(f"Invalid beta parameter at index {k}: {betas[k]}")
        if not 0.0 <= weight_decay:
            raise ValueError(f"Invalid weight_decay value: {weight_decay}")
        if state_bits not in (8, 32):
            raise ValueError(f"Invalid state_bits (8 or 32): {state_bits}")
        if max_grad_norm is not None and not max_grad_norm >= 0:
            raise ValueError(f"Invalid max_grad_norm: {max_grad_norm}")
        if not 0 <= seed < 1 << 64:
            raise ValueError(f"Invalid seed: {seed}")
        self.state_bits, self.min_8bit_numel, self.max_grad_norm = state_bits, min_8bit_numel, max_grad_norm
        self.capturable, self.seed = capturable, seed
        self.grad_norm = None
        self._hyper = {}
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))

    @staticmethod
    def _refuse_options(group):
        """Options of ``torch.optim.AdamW`` that change the update and that this optimizer does not have (foreach, fused and
        capturable change none)."""
        for name in ("amsgrad", "maximize", "differentiable"):
            if group.get(name):
                raise ValueError(f"FusedAdamW does not support {name}")

    def add_param_group(self, param_group):
        if isinstance(param_group, dict):
            self._refuse_options(param_group)
        super().add_param_group(param_group)

    # ------------------------------------------------------------------ states
    def _bits(self, p):
        return 8 if self.state_bits == 8 and p.numel() >= self.min_8bit_numel else 32

    def _zero_state(self, p):
        st = {}
        if self._bits(p) == 8:
            for key in ("exp_avg", "exp_avg_sq"):
                st[key] = torch.zeros(p.shape, dtype=torch.uint8, device=p.device)
                st[key + "_exp"] = torch.zeros(_blocks_of(p.numel()), dtype=torch.uint8, device=p.device)
        else:
            st["exp_avg"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
            st["exp_avg_sq"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
        if p.dtype != torch.float32:
            st["master"] = p.detach().to(torch.float32, copy=True)
        return st

    def _new_step(self, device, value=0):
        return torch.tensor(value, dtype=torch.int64, device=device) if self.capturable else torch.tensor(float(value))

    @torch.no_grad()
    def sync_masters(self):
        """Takes the master copies anew from the parameters: after parameters were written to from outside."""
        for p, st in self.state.items():
            if "master" in st:
                st["master"].copy_(p)

    @staticmethod
    def _check(p):
        L.require_cuda(p, "parameter")
        if p.grad.is_sparse:
            raise RuntimeError("FusedAdamW does not support sparse gradients")
        if p.dtype not in _TYPES:
            raise TypeError(f"FusedAdamW updates float32, bfloat16 and float16 parameters, got {p.dtype}")
        if not p.is_contiguous():
            raise RuntimeError("FusedAdamW needs contiguous parameters")

    def _collect(self):
        """(jobs, made, idle).  jobs: [[group, step tensor, number of the first tensor, parameters, gradients, states]]: what is
        updated together: one type, one device, one width of states, one step count.  made: [(parameter, state)] for new
        parameters, idle: states without a gradient that share a step tensor with updated ones; ``step`` adopts both once
        nothing can be refused any more."""
        jobs, made, idle, first = [], [], [], 0
        for group in self.param_groups:
            buckets, waiting, fresh = {}, [], {}
            for p in group["params"]:
                g, st = p.grad, self.state.get(p)
                if g is None:
                    if st:
                        waiting.append(st)
                    continue
                if not st:
                    self._check(p)
                    if torch.cuda.is_current_stream_capturing():
                        raise L.GcnHipError("FusedAdamW: run a step before capturing one (it makes the states)")
                    step = fresh.setdefault(p.device, None)
                    if step is None:
                        step = fresh[p.device] = self._new_step(p.device)
                    st = {"step": step, **self._zero_state(p)}
                    made.append((p, st))
                step = st["step"]
                bucket = buckets.get((id(step), p.dtype, p.device, "exp_avg_exp" in st))
                if bucket is None:
                    bucket = buckets[(id(step), p.dtype, p.device, "exp_avg_exp" in st)] = [group, step, first, [], [], []]
                bucket[3].append(p)
                bucket[4].append(g if g.is_contiguous() else g.contiguous())
                bucket[5].append(st)
            # parameters without a gradient keep their count: a step tensor that they share with updated ones is copied for them
            counted = {id(b[1]) for b in buckets.values()}
            idle += [st for st in waiting if id(st["step"]) in counted]
            if idle and torch.cuda.is_current_stream_capturing():
                raise L.GcnHipError("FusedAdamW: a parameter had a gradient before capture and has none now")
            # 8-bit tensors are numbered one after the other, also where a group falls into several lists: the numbers enter the
            # random bits of the rounding
            number = first
            for job in buckets.values():
                if "exp_avg_exp" in job[5][0]:
                    job[2] = number
                    number += len(job[3])
            jobs += buckets.values()
            first += len(group["params"])
        return jobs, made, idle

    def _prepare(self, group, step, first, params, grads, states, grad_scale):
        """The checked call of a job: what could be refused has been."""
        masters, eight = "master" in states[0], "exp_avg_exp" in states[0]
        call = L.binding().AdamwCall(params, grads, [s["exp_avg"] for s in states], [s["exp_avg_sq"] for s in states],
                                     [s["master"] for s in states] if masters else None, [s["exp_avg_exp"] for s in states] if eight else None,
                                     [s["exp_avg_sq_exp"] for s in states] if eight else None)
        lr = group["lr"]
        if self.capturable and isinstance(lr, torch.Tensor):
            _check_device_lr(lr, step.device)
            lr = 0.0
        call.check_numbers(lr, *group["betas"], group["eps"], group["weight_decay"], grad_scale)
        return call

    def _clip(self, jobs, max_norm, grad_scale):
        """The clip coefficient over all jobs; also sets ``grad_norm``."""
        by_type = {}
        for job in jobs:
            by_type.setdefault(job[4][0].dtype, []).extend(job[4])
        if len({g.device for gs in by_type.values() for g in gs[:1]}) > 1:
            raise ValueError("clipping to a global norm needs all parameters on one GPU")
        if len(by_type) == 1:
            self.grad_norm, coef = grad_norm(next(iter(by_type.values())), max_norm=max_norm, grad_scale=grad_scale)
            return coef
        norms = torch.stack([grad_norm(gs, grad_scale=grad_scale)[0] for gs in by_type.values()])
        self.grad_norm = norms.double().square().sum().sqrt().float()
        return (max_norm / (self.grad_norm + 1e-6)).clamp(max=1.0)

    @torch.no_grad()
    def step(self, closure=None, *, grad_scale=None, max_grad_norm=None):
        """One update, of all parameters or, where it is refused, of none: nothing is counted then.  grad_scale: float32 scalar on the device that the gradients are multiplied by (1 / loss scale).
        max_grad_norm: in place of the constructor's for this step."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        L.load()
        jobs, made, idle = self._collect()
        if jobs and not self.capturable and torch.cuda.is_current_stream_capturing():
            raise L.GcnHipError("FusedAdamW: a captured step would repeat its step count: pass capturable=True")
        # all of it is checked before anything is counted or updated: a step that is refused leaves everything as it was
        calls = [self._prepare(*job, grad_scale) for job in jobs]
        max_norm = self.max_grad_norm if max_grad_norm is None else max_grad_norm
        if max_norm is not None and not max_norm >= 0:
            raise ValueError(f"Invalid max_grad_norm: {max_norm}")
        coef = self._clip(jobs, max_norm, grad_scale) if max_norm is not None and jobs else None
        for p, st in made:
            self.state[p] = st
        copies = {}                 # those that shared a count go on sharing one, and will be one list again
        for st in idle:
            step = st["step"]
            if id(step) not in copies:
                copies[id(step)] = (step, step.clone())
            st["step"] = copies[id(step)][1]
        advanced = {}
        for (group, step, first, *_), call in zip(jobs, calls):
            options = dict(lr=group["lr"], betas=group["betas"], eps=group["eps"], weight_decay=group["weight_decay"], seed=self.seed)
            if id(step) not in advanced:
                if self.capturable:
                    hyper = self._hyper.get(step)
                    if hyper is None:
                        hyper = self._hyper[step] = adamw_hyper(step.device)
                    adamw_advance_(step, hyper, **options)
                    advanced[id(step)] = hyper
                else:
                    step += 1
                    advanced[id(step)] = int(step.item())
            now = advanced[id(step)]
            # capturable: step, lr and what depends on them are read from hyper
            call.run(0 if self.capturable else now, 0.0 if self.capturable else group["lr"], *group["betas"], group["eps"], group["weight_decay"],
                     self.seed, first, grad_scale, coef, now if self.capturable else None)
        return loss

    # ------------------------------------------------------------------ checkpoints
    def __getstate__(self):
        return {**super().__getstate__(), "state_bits": self.state_bits, "min_8bit_numel": self.min_8bit_numel,
                "max_grad_norm": self.max_grad_norm, "capturable": self.capturable, "seed": self.seed, "grad_norm": None, "_hyper": {}}

    def state_dict(self):
        """As ``torch.optim.AdamW`` saves it: every parameter with a step tensor of its own (here they share one, and an optimizer
        that counts per parameter would count a shared one several times)."""
        out = super().state_dict()
        out["state"] = {k: {**st, "step": st["step"].to(torch.float32, copy=True)} if "step" in st else st for k, st in out["state"].items()}
        return out

    @torch.no_grad()
    def load_state_dict(self, state_dict):
        """Takes states of this optimizer or of ``torch.optim.AdamW`` / ``Adam`` over the same parameters; moments are converted to
        this optimizer's width.  Refused are amsgrad, maximize, differentiable and a weight decay that is part of the gradient;
        nothing is loaded then."""
        groups = state_dict["param_groups"]
        for group in groups:
            self._refuse_options(group)
            if not group.get("decoupled_weight_decay", True) and group["weight_decay"] != 0:
                raise ValueError("the saved optimizer adds its weight decay to the gradient, which AdamW does not")
        # all states before anything is replaced; the base class refuses groups that do not match
        made, shared = [], {}
        if [len(g["params"]) for g in groups] == [len(g["params"]) for g in self.param_groups]:
            ids = itertools.chain.from_iterable(g["params"] for g in groups)
            for sid, (group_no, p) in zip(ids, ((k, p) for k, g in enumerate(self.param_groups) for p in g["params"])):
                saved = state_dict["state"].get(sid)
                if not saved:
                    continue
                st = self._from_saved(p, saved)
                key = (group_no, p.device, int(saved["step"]))
                if key not in shared:
                    shared[key] = self._new_step(p.device, int(saved["step"]))
                st["step"] = shared[key]
                made.append((p, st))
        super().load_state_dict(state_dict)
        # the base class casts every state to its parameter's type: take them as they were saved
        for p, st in made:
            self.state[p] = st
        for group in self.param_groups:
            if "decoupled_weight_decay" in group:
                group["decoupled_weight_decay"] = True
        self._hyper = {}

    def _from_saved(self, p, saved):
        if "max_exp_avg_sq" in saved:
            raise ValueError("FusedAdamW has no amsgrad: the saved state holds the largest second moments")
        if "step" not in saved:
            raise ValueError("the saved state holds no step count")
        st = {k: saved[k].to(p.device, copy=True).contiguous() for k in _KEPT if k in saved}
        for key in ("exp_avg", "exp_avg_sq"):
            if key not in st or st[key].numel() != p.numel():
                raise ValueError(f"{key} of a parameter of shape {tuple(p.shape)} is missing or of another size")
            have8, want8 = key + "_exp" in st, self._bits(p) == 8
            if have8 and (st[key].dtype != torch.uint8 or st[key + "_exp"].numel() != _blocks_of(p.numel())):
                raise ValueError(f"{key} is not a valid 8-bit state")
            st[key] = st[key].view(p.shape)
            if not have8:
                st[key] = st[key].float()
            if have8 and not want8:
                x = state8_decode(st[key], st.pop(key + "_exp"))
                st[key] = x if key == "exp_avg" else x.square()
            elif want8 and not have8:
                x = st[key] if key == "exp_avg" else st[key].sqrt()
                st[key], st[key + "_exp"] = state8_encode(x, never_zero=key == "exp_avg_sq")
        if p.dtype == torch.float32:
            st.pop("master", None)
        else:
            st["master"] = st["master"].float().view(p.shape) if "master" in st else p.detach().float()
        return st
