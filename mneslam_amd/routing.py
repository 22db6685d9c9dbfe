"""Batches dealt to several experts and blended back: which rows go to which map, decoder or network.

    plan = expert_sort(ids, n_experts)              # ids [N, K]: the K experts of each token (point, sample), -1 for none
    xs = expert_dispatch(x, plan)                   # [N*K, D]: the tokens' rows in runs, expert e's from plan.offsets[e]
    ys = ...                                        # every expert on its own run
    out = expert_combine(ys, plan, weights)         # [N, D']: out[n] = sum_k weights[n, k] * ys[position[n, k]]

``expert_dispatch`` and ``expert_combine`` are differentiable (tokens, rows and weights; once).  Nothing waits for the GPU:
``plan.sizes()`` is the one call that does, for experts whose calls need their number of rows on the host.  The kernels are
csrc/routing.hip; there is no fallback."""
import torch
from torch.autograd.function import once_differentiable

from . import _lib


class ExpertPlan:
    """Where the rows are.  ``offsets`` [E + 1] int32: expert e has the rows offsets[e] .. offsets[e + 1] - 1, in the order of the slots
    n * K + k that name it.  ``order`` [N*K] int32: the slot of a row, -1 behind the last live row.  ``position`` [N, K] int32: the
    row of a slot, -1 where it names no expert."""

    __slots__ = ("order", "position", "offsets", "n_tokens", "top_k", "n_experts")

    def __init__(self, order, position, offsets):
        self.order, self.position, self.offsets = order, position, offsets
        (self.n_tokens, self.top_k), self.n_experts = position.shape, offsets.shape[0] - 1

    @property
    def live(self):
        """[1]: the number of rows that have a slot."""
        return self.offsets[-1:]

    def sizes(self):
        """Rows of every expert as a list (waits for the GPU)."""
        edges = self.offsets.tolist()
        return [b - a for a, b in zip(edges, edges[1:])]


def expert_sort(ids, n_experts):
    """The plan of ``ids`` [N, K] or [N] (int32 or int64) for experts 0 .. n_experts - 1 (at most 4096).  The sort is stable.  An id outside
    that range names no expert: its slot has no row, adds nothing to its token's output and gets no gradient."""
    if ids.dtype not in (torch.int32, torch.int64) or ids.dim() not in (1, 2):
        raise TypeError(f"expert_sort: ids must be int32 or int64 [N, K] or [N], got {ids.dtype} with {ids.dim()} dimensions")
    n_experts = int(n_experts)
    if not 1 <= n_experts <= 4096:
        raise ValueError(f"expert_sort: 1 to 4096 experts, got {n_experts}")
    n, k, m = ids.shape[0], ids.shape[1] if ids.dim() == 2 else 1, ids.numel()
    if k < 1:
        raise ValueError("expert_sort: ids without a choice")
    dev = _lib.one_device([ids], "expert_sort")
    lib, ids = _lib.load(), ids.contiguous()
    size = lib.mne_expert_sort_workspace_bytes(m, n_experts)
    # one allocation: order, position, offsets, workspace
    out = torch.empty(2 * m + n_experts + 1 + size // 4, dtype=torch.int32, device=dev)
    base = out.data_ptr()
    with _lib.device_guard(dev):
        _lib.check(lib.mne_expert_sort(ids.data_ptr(), ids.dtype == torch.int64, m, n_experts, base, base + 4 * m, base + 8 * m,
                                       base + 4 * (2 * m + n_experts + 1), size, _lib.raw_stream(dev)), "mne_expert_sort")
    return ExpertPlan(out[:m], out[m:2 * m].view(n, k), out[2 * m:2 * m + n_experts + 1])


def _rows(t, what):
    """``t`` with elements of a row next to each other (a copy where they are not)."""
    if t.dim() != 2:
        raise ValueError(f"{what}: rows must be [rows, width], got {tuple(t.shape)}")
    if t.dtype not in _lib.T_CODES:
        raise TypeError(f"{what}: {t.dtype} is not supported (float32, bfloat16, float16)")
    return t if (t.stride(1) == 1 or t.shape[1] <= 1) and t.stride(0) >= 0 else t.contiguous()


def _dispatch(x, position, offsets):
    x = _rows(x, "expert_dispatch")
    (n, k), width = position.shape, x.shape[1]
    dev = _lib.one_device([x, position, offsets], "expert_dispatch")
    out = torch.empty(n * k, width, dtype=x.dtype, device=dev)
    with _lib.device_guard(dev):
        _lib.check(_lib.load().mne_expert_dispatch(x.data_ptr(), x.stride(0), _lib.T_CODES[x.dtype], n, k, width, position.data_ptr(),
                                                   offsets.data_ptr() + 4 * (offsets.shape[0] - 1), out.data_ptr(), _lib.raw_stream(dev)),
                   "mne_expert_dispatch")
    return out


def _combine(y, position, weights):
    y = _rows(y, "expert_combine")
    (n, k), width = position.shape, y.shape[1]
    dev = _lib.one_device([y, position] + ([weights] if weights is not None else []), "expert_combine")
    out = torch.empty(n, width, dtype=y.dtype, device=dev)
    with _lib.device_guard(dev):
        _lib.check(_lib.load().mne_expert_combine(y.data_ptr(), y.stride(0), _lib.T_CODES[y.dtype], n, k, width, position.data_ptr(),
                                                  weights.data_ptr() if weights is not None else None, out.data_ptr(),
                                                  _lib.raw_stream(dev)), "mne_expert_combine")
    return out


def _combine_backward(dout, y, position, offsets, weights, want_dy, want_dw):
    dout, y = _rows(dout, "expert_combine"), _rows(y, "expert_combine")
    (n, k), width = position.shape, y.shape[1]
    dev = _lib.one_device([dout, y, position, offsets] + ([weights] if weights is not None else []), "expert_combine")
    dy = torch.empty(n * k, width, dtype=y.dtype, device=dev) if want_dy else None
    dw = (torch.empty if width else torch.zeros)(n, k, dtype=torch.float32, device=dev) if want_dw else None
    with _lib.device_guard(dev):
        _lib.check(_lib.load().mne_expert_combine_backward(
            dout.data_ptr(), dout.stride(0), y.data_ptr(), y.stride(0), _lib.T_CODES[y.dtype], n, k, width, position.data_ptr(),
            offsets.data_ptr() + 4 * (offsets.shape[0] - 1), weights.data_ptr() if weights is not None else None,
            dy.data_ptr() if want_dy else None, dw.data_ptr() if want_dw else None, _lib.raw_stream(dev)), "mne_expert_combine_backward")
    return dy, dw


class _DispatchFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, position, offsets):
        ctx.save_for_backward(position)
        return _dispatch(x.detach(), position, offsets)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        return _combine(dout, ctx.saved_tensors[0], None), None, None


class _CombineFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, position, offsets, weights):
        ctx.save_for_backward(y, position, offsets, weights)
        return _combine(y.detach(), position, None if weights is None else weights.detach().float().contiguous())

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        y, position, offsets, weights = ctx.saved_tensors
        want_dy, want_dw = ctx.needs_input_grad[0], ctx.needs_input_grad[3]
        w = None if weights is None else weights.float().contiguous()
        dy, dw = _combine_backward(dout, y, position, offsets, w, want_dy, want_dw)
        return dy, None, None, dw.to(weights.dtype) if want_dw else None


def expert_dispatch(x, plan):
    """``x`` [N, D] (float32, bfloat16 or float16) -> the rows [N*K, D] of its tokens, expert after expert.  Rows behind the last live one
    are zero.  d x[n] is the sum of the gradients of its rows, in fp32."""
    if x.dim() != 2 or x.shape[0] != plan.n_tokens:
        raise ValueError(f"expert_dispatch: {tuple(x.shape)} for a plan of {plan.n_tokens} tokens")
    if torch.is_grad_enabled() and x.requires_grad:
        return _DispatchFn.apply(x, plan.position, plan.offsets)
    return _dispatch(x.detach(), plan.position, plan.offsets)


def expert_combine(y, plan, weights=None):
    """``y`` [N*K, D] (float32, bfloat16 or float16), ``weights`` [N, K] (any of the three types, or None for 1) -> [N, D]:
    sum_k weights[n, k] * y[position[n, k]], added up in fp32 in the order of k and rounded once.  A slot without a row adds nothing,
    whatever its weight, and rows behind the last live one are not read.  Gradients: of y (zero behind the live rows) and of the weights
    (0 for a slot without a row)."""
    if y.dim() != 2 or y.shape[0] != plan.n_tokens * plan.top_k:
        raise ValueError(f"expert_combine: {tuple(y.shape)} for a plan of {plan.n_tokens} x {plan.top_k} slots")
    if weights is not None:
        if tuple(weights.shape) != (plan.n_tokens, plan.top_k):
            raise ValueError(f"expert_combine: weights {tuple(weights.shape)} for a plan of {plan.n_tokens} x {plan.top_k} slots")
        if weights.dtype not in _lib.T_CODES:
            raise TypeError(f"expert_combine: weights of {weights.dtype} (float32, bfloat16 or float16)")
    if torch.is_grad_enabled() and (y.requires_grad or (weights is not None and weights.requires_grad)):
        return _CombineFn.apply(y, plan.position, plan.offsets, weights)
    return _combine(y.detach(), plan.position, None if weights is None else weights.detach().float().contiguous())
