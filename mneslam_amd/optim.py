"""FusedAdam -- ``torch.optim.Adam``-compatible optimizer over the param groups of
MNESLAM.create_optimizer (mneslam_mp.py:459-469) whose ``step()`` is one HIP launch
(mne_adam_step: single pass over p, g, m, v for every tensor of every group).

Semantics are torch.optim.Adam's (amsgrad=False, maximize=False): L2 weight decay folded into the
gradient, bias correction by the per-parameter step count, dense update of every element (cells
with zero gradient still move while their first moment is non-zero -- required for parity,
SURVEY.md section 7).
"""
import ctypes as C

import torch

from . import _lib, plane_sums


def _dense_like(p, t):
    """``t`` as an fp32 tensor laid out exactly like ``p`` (same strides), copying only if needed."""
    if t.stride() == p.stride() and t.dtype == torch.float32:
        return t
    out = torch.empty_like(p, dtype=torch.float32)            # preserve_format
    out.copy_(t)
    return out


class FusedAdam(torch.optim.Optimizer):
    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0):
        defaults = dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay)
        super().__init__(params, defaults)

    def _state(self, p):
        st = self.state[p]
        if len(st) == 0:
            st["step"] = 0
            # preserve_format: same physical layout as p; the moments are fp32 also for half-precision planes
            st["exp_avg"] = torch.zeros_like(p, dtype=torch.float32)
            st["exp_avg_sq"] = torch.zeros_like(p, dtype=torch.float32)
        return st

    def segments(self, zero_grad_buffers=None, advance=True):
        """ctypes segment array for every parameter that has a gradient (advances the step counts unless
        ``advance`` is False: a recorded iteration reads its step from the device clock, ``step`` is then the base)."""
        segs = []
        keep = []
        for group in self.param_groups:
            b1, b2 = group["betas"]
            for p in group["params"]:
                if p.grad is None:
                    plane_sums.drop(p)           # .grad was dropped by someone else's zero_grad: the fp32 sum beside it is stale
                g = p.grad if zero_grad_buffers is None else zero_grad_buffers.get(p)   # explicit map: only those params
                if g is None:
                    continue
                if zero_grad_buffers is None and p.dtype == torch.float16:
                    # half-precision plane: autograd's .grad has the parameter's dtype, and a mean-reduced plane gradient
                    # sits below fp16's range (flushes to zero below ~3e-8; Adam is scale-free, so those would be lost
                    # updates).  The render node leaves the fp32 sum beside it (hip_path.RenderFunction.backward): that is
                    # what the update consumes.  Without it the step would silently run on the flushed fp16 gradient: refused.
                    if getattr(p, "grad32", None) is None:
                        raise RuntimeError("a half-precision plane has .grad but no fp32 gradient sum (grad32): its gradient did not "
                                           "come from this package's render node")
                    g = p.grad32 if p.grad32.device == p.device else p.grad32.to(p.device)
                if p.dtype not in (torch.float32, torch.float16):
                    raise TypeError("FusedAdam supports float32 parameters (and float16 planes: fp32 gradient and moments)")
                if not (p.is_contiguous() or p.is_contiguous(memory_format=torch.channels_last)):
                    raise ValueError("FusedAdam needs dense parameters")
                st = self._state(p)
                if advance:
                    st["step"] += 1
                g = _dense_like(p, g)
                keep.append(g)
                s = _lib.AdamSeg()
                s.p, s.g = p.data_ptr(), g.data_ptr()
                s.m, s.v = st["exp_avg"].data_ptr(), st["exp_avg_sq"].data_ptr()
                s.n = p.numel()
                s.lr, s.beta1, s.beta2 = float(group["lr"]), float(b1), float(b2)
                s.eps, s.weight_decay = float(group["eps"]), float(group["weight_decay"])
                s.step = st["step"] if advance else st["step"] + 1
                s.p_f16 = 1 if p.dtype == torch.float16 else 0
                segs.append((s, p))
        return segs, keep

    @torch.no_grad()
    def step(self, closure=None, zero_grad=False, grad_buffers=None, clock=None):
        """``clock`` (mneslam_amd._lib.Clock, graph recording only): the kernel adds the device step offset to the
        parameters' CURRENT step + 1 and the python step counts are left alone (the caller advances them per replay)."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        segs, keep = self.segments(grad_buffers, advance=clock is None)
        if not segs:
            return loss
        lib = _lib.load()
        for i in range(0, len(segs), 32):
            chunk = segs[i:i + 32]
            arr = (_lib.AdamSeg * len(chunk))(*[s for s, _ in chunk])
            _lib.check(lib.mne_adam_step(arr, len(chunk), 1 if zero_grad else 0,
                                         C.byref(clock) if clock is not None else None, _lib.stream_for(chunk[0][1])),
                       "mne_adam_step")
        if zero_grad and grad_buffers is None:
            # the kernel zeroed the buffers it was given: for a half-precision plane that is the fp32 side sum (or a temporary
            # fp32 copy of .grad), not autograd's fp16 .grad itself
            for _, p in segs:
                if p.dtype == torch.float16 and p.grad is not None:
                    p.grad.zero_()
        return loss

    def zero_grad(self, set_to_none=True):
        for group in self.param_groups:
            for p in group["params"]:
                plane_sums.drop(p)                       # the fp32 gradient sum of a half-precision plane (see ``segments``)
        return super().zero_grad(set_to_none=set_to_none)


# ---- AdamW -------------------------------------------------------------------------------------------------------------
MOMENT_BLOCK = 256             # consecutive elements of an 8-bit moment that share a scale


def _check_hyper(lr, betas, eps, weight_decay):
    if not 0.0 <= lr < float("inf"):
        raise ValueError(f"Invalid learning rate: {lr}")
    if not (len(betas) == 2 and 0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0):
        raise ValueError(f"Invalid betas: {betas}")
    if not 0.0 <= eps < float("inf"):
        raise ValueError(f"Invalid epsilon value: {eps}")
    if not 0.0 <= weight_decay < float("inf"):
        raise ValueError(f"Invalid weight_decay value: {weight_decay}")


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, scales=None, *, step, lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2,
               seed=0, ordinals=None, zero_grad=False, clock=None):
    """One AdamW step (decoupled decay, torch.optim.AdamW with amsgrad=False, maximize=False) over a list of tensors, in place and
    in as few launches as the list allows (80 tensors each, 64 with 8-bit moments): ``params``, ``grads``, ``exp_avgs`` and
    ``exp_avg_sqs`` are lists of one length.

    Parameters are float32, bfloat16 or float16; a gradient has its parameter's type or float32 (any of the three beside a float32
    parameter).  The arithmetic is fp32; a 16-bit parameter is rounded to nearest even.  Every tensor is dense (contiguous or
    channels_last); moments are laid out like their parameter, a gradient laid out otherwise (or negated lazily) is copied.  What the step
    writes does not overlap and is no negated view: parameters, moments, scales, gradients that it clears.  A gradient that it only reads
    may be another's too, but not a part of what is written.

    ``scales`` None: moments are float32.  Otherwise they are held in 8 bits: ``exp_avgs`` int8, ``exp_avg_sqs`` uint8, and
    ``scales`` the list of their float32 [ceil(n / 256), 2] scales, two for each 256 consecutive elements of the tensor's memory
    (all zero: all moments zero; ``adamw_moments`` gives the moments in fp32).  Their codes are rounded up or down with a dither that
    depends on ``seed``, the tensor's entry of ``ordinals`` (its place in the list by default; keep it the same at every step),
    ``step`` and the element alone.  A block that meets a gradient that is not finite, or one of 1.85e19 and more, whose square is not
    in fp32, holds NaN from then on: all its 256 elements (32-bit moments keep that to the one).

    ``step`` counts from 1 and is the list's; ``clock`` (mneslam_amd._lib.Clock, graph recording) adds the device's step offset.
    Without one a step is not recorded into a graph: every replay would be the same step."""
    params = list(params)
    args = _step_args(params, grads, exp_avgs, exp_avg_sqs, scales, ordinals, lr, betas, eps, weight_decay, step, seed, int(bool(zero_grad)), clock)
    if params:
        _lib.host_tensors().adamw_step(*args)


def _step_args(params, grads, exp_avgs, exp_avg_sqs, scales, ordinals, lr, betas, eps, weight_decay, step, seed, zero_grad, clock):
    lr, eps, weight_decay = float(lr), float(eps), float(weight_decay)
    _check_hyper(lr, betas, eps, weight_decay)
    if not 1 <= step < 1 << 31 or not 0 <= seed < 1 << 32:
        raise ValueError(f"adamw_step: step counts from 1 and seed is a number of 32 bits, got {step} and {seed}")
    if clock is None and params and params[0].is_cuda and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("adamw_step: recording a step needs a clock (the step count would be the same at every replay)")
    return (params, list(grads), list(exp_avgs), list(exp_avg_sqs), None if scales is None else list(scales),
            None if ordinals is None else list(ordinals), lr, float(betas[0]), float(betas[1]), eps, weight_decay, step, seed, zero_grad,
            0 if clock is None else C.addressof(clock))


def adamw_moments(exp_avg, exp_avg_sq, scales):
    """The fp32 moments (exp_avg, exp_avg_sq) that 8-bit codes and their ``scales`` stand for (see ``adamw_step``), in the codes'
    shape and layout."""
    return tuple(_lib.host_tensors().adamw_moments(exp_avg, exp_avg_sq, scales))


def _check_rule(group):
    """``group``: a saved group of FusedAdamW, or of an optimizer that goes on by the same rule."""
    for rule in ("amsgrad", "maximize"):
        if group.get(rule):
            raise ValueError(f"FusedAdamW has no {rule}: the loaded state would go on by another rule")
    if "state_bits" in group:
        return
    if any(key not in group for key in ("lr", "betas", "eps", "weight_decay")) or ("decoupled_weight_decay" in group and "amsgrad" not in group):
        raise ValueError("the saved state is none of AdamW: it would go on by another rule")
    # torch.optim.Adam says that its decay is folded into the gradient; FusedAdam's groups have the four entries above alone
    if group["weight_decay"] and not group.get("decoupled_weight_decay", "amsgrad" in group):
        raise ValueError("the saved state is Adam's, with a decay that is folded into the gradient: it would go on by another rule")


def _check_saved(p, st, bits):
    """``st``: a saved entry of FusedAdamW or torch.optim.AdamW for a parameter like ``p``, in a group with moments of ``bits`` bits."""
    if not st.keys() <= {"step", "exp_avg", "exp_avg_sq", "scales"}:
        raise ValueError(f"the saved state is none of AdamW: it has {sorted(st)}")
    if any(not torch.is_tensor(st.get(key)) or st[key].shape != p.shape for key in ("exp_avg", "exp_avg_sq")) or "step" not in st:
        raise ValueError(f"the saved state of a parameter of shape {tuple(p.shape)} is none, or has another shape")
    types = st["exp_avg"].dtype, st["exp_avg_sq"].dtype
    if all(t.is_floating_point for t in types) != (bits == 32):
        raise ValueError(f"a group with state_bits={bits} cannot go on from moments that are {types}")
    if bits == 32 and "scales" in st:
        raise ValueError("moments in 32 bits have no scales")
    if bits == 32:
        return
    if types != (torch.int8, torch.uint8):
        raise ValueError(f"moments are floating-point numbers, or int8 and uint8 codes, not {types}")
    scales = st.get("scales")
    if not torch.is_tensor(scales) or not scales.is_floating_point() or scales.shape != (-(-p.numel() // MOMENT_BLOCK), 2):
        raise ValueError("8-bit moments without scales for their blocks")
    if any(n > 1 and a != b for key in ("exp_avg", "exp_avg_sq") for n, a, b in zip(p.shape, p.stride(), st[key].stride())):
        raise ValueError("8-bit moments of a parameter that was laid out otherwise: its blocks are others")


class FusedAdamW(torch.optim.Optimizer):
    """torch.optim.AdamW (amsgrad=False, maximize=False) whose ``step()`` is ``adamw_step``: one launch for up to 80 tensors of a
    group that are at the same step count.  ``state_bits`` 8 (also per group) holds the moments in 8 bits with two scales for each 256
    elements -- 2.06 bytes an element instead of 8; ``moments(p)`` gives them in fp32.  ``seed`` is that of the codes' dither.

    The gradient is ``.grad``.  That of a half-precision plane is taken in fp32, before its rounding, wherever it is still what the render
    node's backward pass left; where it was changed since (clipped, unscaled, added to) it is taken as it is, in its own type."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32, seed=0):
        if not 0 <= int(seed) < 1 << 32:
            raise ValueError(f"Invalid seed: {seed}")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits, seed=int(seed)))

    def add_param_group(self, param_group):
        group = {**self.defaults, **param_group}
        _check_hyper(group["lr"], group["betas"], group["eps"], group["weight_decay"])
        if group["state_bits"] not in (8, 32):
            raise ValueError(f"Invalid state_bits: {group['state_bits']} (8 or 32)")
        super().add_param_group(param_group)

    def __setstate__(self, state):
        super().__setstate__(state)
        for group in self.param_groups:                 # (a state of torch.optim.AdamW has neither)
            group.setdefault("state_bits", 32)
            group.setdefault("seed", 0)

    def _state(self, p, bits):
        st = self.state[p]
        if len(st) == 0:
            if p.is_cuda and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("FusedAdamW: take a step before recording one (the moments would be cleared at every replay)")
            st["step"] = 0
            # preserve_format: the same physical layout as p
            st["exp_avg"] = torch.zeros_like(p, dtype=torch.int8 if bits == 8 else torch.float32)
            st["exp_avg_sq"] = torch.zeros_like(p, dtype=torch.uint8 if bits == 8 else torch.float32)
            if bits == 8:
                st["scales"] = torch.zeros(-(-p.numel() // MOMENT_BLOCK), 2, device=p.device)
        return st

    @torch.no_grad()
    def step(self, closure=None, zero_grad=False, clock=None):
        """All of it or, where something is refused, nothing.  ``zero_grad``: the gradients are zero behind the step (one pass less over
        them).  ``clock`` (graph recording): the kernels add the device step offset to the parameters' CURRENT step + 1, and the step counts
        here are left alone."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        ordinal, calls, counts, sums = 0, [], [], []
        for group in self.param_groups:
            batches = {}                                # tensors of one device at one step count
            for p in group["params"]:
                ordinal += 1
                if p.grad is None:
                    plane_sums.drop(p)                  # .grad was dropped by someone else: the fp32 sum beside it is stale
                    continue
                if p.grad.is_sparse:
                    raise RuntimeError("FusedAdamW does not support sparse gradients")
                g = plane_sums.gradient(p)              # (a half-precision plane: the fp32 sum that .grad is the rounding of)
                if getattr(p, "grad32", None) is not None:
                    sums.append(p)
                st = self._state(p, group["state_bits"])
                batches.setdefault((p.device, st["step"] + 1), []).append((p, g, st, ordinal - 1))
            for (_, step), batch in batches.items():
                ps, gs, sts, ords = zip(*batch)
                calls.append(_step_args(list(ps), gs, [s["exp_avg"] for s in sts], [s["exp_avg_sq"] for s in sts],
                                        [s["scales"] for s in sts] if group["state_bits"] == 8 else None, ords, group["lr"], group["betas"],
                                        group["eps"], group["weight_decay"], step, group["seed"], 2 if zero_grad else 0, clock))
                counts.append((step, sts))
        if not calls:
            return loss
        _lib.host_tensors().adamw_steps(calls)          # (all of them are checked before the first is launched)
        if clock is None:
            for step, sts in counts:
                for s in sts:
                    s["step"] = step
        if zero_grad:
            for p in sums:
                plane_sums.zero(p)
        return loss

    def moments(self, p):
        """(exp_avg, exp_avg_sq) of ``p`` in fp32 (zero before its first step)."""
        st = self.state.get(p)
        if not st:
            return torch.zeros_like(p, dtype=torch.float32), torch.zeros_like(p, dtype=torch.float32)
        return adamw_moments(st["exp_avg"], st["exp_avg_sq"], st["scales"]) if "scales" in st else (st["exp_avg"], st["exp_avg_sq"])

    def load_state_dict(self, state_dict):
        """Also of torch.optim.AdamW's states (not with amsgrad or maximize), and of Adam's without weight decay.  The base class casts floating-point state to its
        parameter's type: here moments and scales are float32 or the codes they were saved as, laid out like their parameter.  ``state_bits``
        and ``seed`` are the saved ones; where a state has none (torch's), they stay, and moments in 32 bits are refused by a group with
        8-bit ones.  A state that does not fit is refused before anything is loaded."""
        seen = []

        def check(_, state_dict):                        # (behind the hooks that may change it)
            groups = []
            for own, group in zip(self.param_groups, state_dict["param_groups"]):
                _check_rule(group)
                groups.append({"state_bits": own["state_bits"], "seed": own["seed"], **group})
            seen.append({**state_dict, "param_groups": groups + list(state_dict["param_groups"][len(groups):])})
            for group, p, st in self._saved_states(seen[0]):
                _check_saved(p, st, group["state_bits"])
            return seen[0]

        hook = self.register_load_state_dict_pre_hook(check)
        try:
            super().load_state_dict(state_dict)
        finally:
            hook.remove()
        for _, p, st in self._saved_states(seen[0]):
            for key, value in st.items():
                if key == "step":
                    self.state[p][key] = int(value)
                elif key in ("exp_avg", "exp_avg_sq", "scales"):
                    like = value if key == "scales" else p
                    dtype = torch.float32 if value.is_floating_point() else value.dtype
                    self.state[p][key] = torch.empty_like(like, dtype=dtype, device=p.device, requires_grad=False).copy_(value)

    def _saved_states(self, state_dict):
        """(saved group, parameter, its entry of ``state_dict``) of those that have one, as far as the groups are alike (the base class checks that)."""
        for group, saved in zip(self.param_groups, state_dict["param_groups"]):
            for p, i in zip(group["params"], saved["params"]):
                if state_dict["state"].get(i):
                    yield saved, p, state_dict["state"][i]

    def zero_grad(self, set_to_none=True):
        for group in self.param_groups:
            for p in group["params"]:
                plane_sums.drop(p)
        return super().zero_grad(set_to_none=set_to_none)
