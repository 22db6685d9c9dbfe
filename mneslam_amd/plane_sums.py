"""The fp32 gradient sum (``grad32``) that the render node leaves beside a half-precision plane's ``.grad``, and whether it still stands
for it.

A mean-reduced plane gradient lies below fp16's range, so the optimizer should see the sum before autograd rounds it to the parameter's
type.  But ``.grad`` is what everybody else sees: it may be clipped or unscaled, another node may add to it, somebody may drop it and fill
it again.  The node notes its contributions here, a hook behind the accumulation notes what ``.grad`` was then (the object and its
version), and ``gradient`` uses the sum only where ``.grad`` is its rounding."""
import torch
from torch.utils.weak import WeakTensorKeyDictionary

_notes = WeakTensorKeyDictionary()


class _Note:
    __slots__ = ("task", "pending", "fresh", "whole", "grad", "version")

    def __init__(self):
        self.task, self.pending, self.fresh, self.whole, self.grad, self.version = -1, False, False, False, None, 0


def _accumulated(p):
    """Behind an accumulation into ``p.grad``: does the sum still cover it?"""
    note, g = _notes[p], p.grad
    continued = note.grad is g and g._version == note.version + 1                 # nobody touched it since the last one
    if note.pending and note.task == torch._C._current_graph_task_id():
        note.whole = note.fresh or (note.whole and continued)
    else:                                                                          # another node's backward pass
        note.whole = note.whole and continued and not note.pending
    note.pending, note.grad, note.version = False, g, g._version


def add(p, g):
    """The render node's fp32 gradient ``g`` of the half-precision ``p``, in a backward pass that goes on to round and accumulate it."""
    note = _notes.get(p)
    if note is None:
        note = _notes[p] = _Note()
        if p.is_leaf and p.requires_grad:
            p.register_post_accumulate_grad_hook(_accumulated)
    task, acc = torch._C._current_graph_task_id(), getattr(p, "grad32", None)
    same = note.pending and note.task == task                                      # the second node of this pass
    if note.pending and not same:
        note.whole = False                                                         # (what that pass added never arrived in .grad)
    if acc is None or acc.shape != g.shape or acc.device != g.device or (p.is_leaf and p.grad is None and not same):
        p.grad32, note.fresh = g.clone(), True
    else:
        acc.add_(g)
        note.fresh = note.fresh and same
    note.task, note.pending = task, True


def gradient(p):
    """The gradient an optimizer should take: ``p.grad``, in fp32 and unrounded wherever it is the rounding of the sum."""
    s = getattr(p, "grad32", None)
    note = None if s is None else _notes.get(p)
    if note is None or not note.whole or note.pending or note.grad is not p.grad or p.grad._version != note.version:
        return p.grad
    return torch.where(p.grad == s.to(p.grad), s.to(p.grad.device), p.grad.float())


def zero(p):
    """``p.grad`` and its sum become zero, and from here on the one stands for the other."""
    p.grad.zero_()
    if getattr(p, "grad32", None) is not None:
        p.grad32.zero_()
    note = _notes.get(p)
    if note is not None:
        note.pending, note.whole, note.grad, note.version = False, True, p.grad, p.grad._version


def drop(p):
    """``.grad`` is gone, or about to be cleared: so is its sum."""
    if getattr(p, "grad32", None) is None:
        return
    p.grad32 = None
    note = _notes.get(p)
    if note is not None:
        note.pending, note.whole, note.grad = False, False, None
