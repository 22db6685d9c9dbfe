"""Batches dealt to several experts and blended back: which rows go to which map, decoder or network.

    plan = expert_sort(ids, n_experts)              # ids [N, K]: the K experts of each token (point, sample), -1 for none
    xs = expert_dispatch(x, plan)                   # [N*K, D]: the tokens' rows in runs, expert e's from plan.offsets[e]
    ys = ...                                        # every expert on its own run
    out = expert_combine(ys, plan, weights)         # [N, D']: out[n] = sum_k weights[n, k] * ys[position[n, k]]

``expert_dispatch`` and ``expert_combine`` are differentiable (tokens, rows and weights; once).  Nothing waits for the GPU:
``plan.sizes()`` is the one call that does, for experts whose calls need their number of rows on the host.  All of it can be recorded into
a graph; a backward pass that is recorded while an eager graph of the same leaves lives on the default stream is refused.  Under a
tracer (torch.jit.trace, make_fx, torch.export) the calls are refused; torch.compile runs them between its graphs.  The kernels are
csrc/routing.hip; there is no fallback."""
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
    return ExpertPlan(*_lib.host_tensors().expert_sort(ids, n_experts))


def expert_dispatch(x, plan):
    """``x`` [N, D] (float32, bfloat16 or float16) -> the rows [N*K, D] of its tokens, expert after expert.  Rows behind the last live one
    are zero.  d x[n] is the sum of the gradients of its rows, in fp32."""
    return _lib.host_tensors().expert_dispatch(x, plan.position, plan.offsets)


def expert_combine(y, plan, weights=None):
    """``y`` [N*K, D] (float32, bfloat16 or float16), ``weights`` [N, K] (any of the three types, or None for 1) -> [N, D]:
    sum_k weights[n, k] * y[position[n, k]], added up in fp32 in the order of k and rounded once.  A slot without a row adds nothing,
    whatever its weight, and rows behind the last live one are not read.  Gradients: of y (zero behind the live rows) and of the weights
    (0 for a slot without a row)."""
    return _lib.host_tensors().expert_combine(y, plan.position, plan.offsets, weights)
