"""Activation checkpointing (recompute in backward).

Same API as the reference helper (``minispeed/activation_checkpointing.py:17-30``):
``checkpoint(fn, *args)`` and ``checkpoint_sequential(functions, segments,
input)``, non-reentrant by default.  The model blocks of
:mod:`minispeed_b200.models` call :func:`checkpoint` per block when built
with ``activation_checkpointing=True``; their fused kernels are simply run
again in the recompute.

``checkpoint(fn, *args, save_bits=8)`` keeps what it saves in 8 bits
(:func:`minispeed_b200.ops.nn.pack_activation`).  The reference has no
counterpart.
"""

from __future__ import annotations

import torch
from torch.utils.checkpoint import checkpoint as _checkpoint
from torch.utils.checkpoint import checkpoint_sequential as _checkpoint_sequential

from .ops.nn import PackedActivation, _check_save_bits, pack_activation


class _Saved8:
    """The arguments of a checkpointed call: as they were given for its
    forward, with the activations packed for its recompute.  An activation is a
    floating-point tensor that requires a gradient and is not a leaf; leaves
    (parameters), tables and integer tensors are held elsewhere anyway and are
    kept as they are."""

    def __init__(self, args):
        self.exact = args
        self.saved = [(pack_activation(a), self._layout(a)) if self._activation(a) else (a, None)
                      for a in args]

    @staticmethod
    def _activation(a) -> bool:
        return (isinstance(a, torch.Tensor) and a.requires_grad and not a.is_leaf
                and a.dtype in (torch.float32, torch.float16, torch.bfloat16) and a.dim() > 0)

    @staticmethod
    def _layout(a):
        """The strides of a dense tensor whose axes lie in the order of ``a``'s;
        None where that is contiguous."""
        return None if a.is_contiguous() else torch.empty_like(a, device="meta").stride()

    @staticmethod
    def _restore(packed, layout):
        x = packed.unpack()
        if layout is not None and layout != x.stride():
            x = torch.empty_strided(x.shape, layout, dtype=x.dtype, device=x.device).copy_(x)
        return x.requires_grad_()

    def take(self):
        if self.exact is not None:
            args, self.exact = self.exact, None
            return args
        return [self._restore(a, layout) if isinstance(a, PackedActivation) else a
                for a, layout in self.saved]


def checkpoint(function, *args, **kwargs):
    """``function(*args, **kwargs)`` without keeping its intermediate results:
    backward runs it again.

    ``save_bits=8`` also packs the activations among ``args`` (tensors that
    require a gradient and are not leaves) to 8 bits between the two runs.  The
    outputs are those of the exact arguments; the recompute, and so the
    gradients, start from the packed ones: dense tensors with the axes in the
    order of the arguments', each argument a tensor of its own.  Tensors inside
    containers and keyword arguments are kept as they are."""
    save_bits = kwargs.pop("save_bits", None)
    use_reentrant = kwargs.pop("use_reentrant", False)
    if not _check_save_bits(save_bits) or not torch.is_grad_enabled():
        return _checkpoint(function, *args, use_reentrant=use_reentrant, **kwargs)
    if use_reentrant:
        raise ValueError("checkpoint: save_bits=8 needs use_reentrant=False")
    saved = _Saved8(args)
    # empty tensors stand for the arguments' devices, whose random state
    # torch's checkpoint keeps for the recompute
    devices = {a.device: a for a in args if isinstance(a, torch.Tensor)}
    stand_ins = [a.new_empty(0) for a in devices.values()]

    def run(*ignored, **kw):
        return function(*saved.take(), **kw)

    return _checkpoint(run, *stand_ins, use_reentrant=False, **kwargs)


def checkpoint_sequential(functions, *args, **kwargs):
    use_reentrant = kwargs.pop("use_reentrant", False)
    return _checkpoint_sequential(functions, *args, use_reentrant=use_reentrant, **kwargs)


__all__ = ["checkpoint", "checkpoint_sequential"]

# keep torch importable name for type checkers
_ = torch
