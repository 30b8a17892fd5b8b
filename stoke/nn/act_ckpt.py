# -*- coding: utf-8 -*-
"""Activation checkpointing (recompute-in-backward).

The reference exposes activation checkpointing only as a DeepSpeed
pass-through (``DeepspeedActivationCheckpointingConfig``,
reference ``stoke/configs.py:222-249`` -> ``distributed.py:965-983``); the
work itself happened inside the DeepSpeed engine.  Here it is in-house:
eligible submodules get their forward routed through
``torch.utils.checkpoint`` (non-reentrant), trading one extra forward of the
wrapped block for not storing its activations — on MI355X the recompute is
usually HBM-resident and cheap relative to the 288 GB it frees for larger
batches/models.

``save_bits=8`` keeps the wrapped block's input in 8 bits (``stoke.nn.act8``):
half the bytes of a 16-bit checkpoint.  The forward runs on the exact input;
the recompute starts from the values held.  The input is the first argument
of the block's ``forward``; the others (masks, biases, tables, expressions of
parameters, an encoder's output) stay as they are: a mask's -inf or lowest
value would take the other values of its 32 along, and what several blocks
share would be held once for each.

Composes with the FSDP engine: the recompute re-fires the unit's
forward-pre hook, which re-gathers the flat-param shard it needs.
"""

import functools
import inspect
from typing import Callable, Optional

import torch
import torch.nn as nn
from torch.utils.checkpoint import checkpoint

from stoke.nn.act8 import (
    check_save_bits,
    compress_activation,
    restore_activation,
)

_MARK = "_stoke_act_ckpt"
_BITS = "_stoke_act_ckpt_bits"


class _Held:
    """An activation in 8 bits that comes back with its strides.

    The values are held in the order of memory, those of an expanded size
    once: a block may view its input in ways that its strides allow and
    others do not, and products pick their layout by them."""

    def __init__(self, x):
        strides = x.stride()
        self.shape = x.shape
        self.order = sorted(range(x.dim()), key=lambda d: -strides[d])
        for d in range(x.dim()):
            if strides[d] == 0 and x.shape[d] > 1:
                x = x.narrow(d, 0, 1)
        self.packed = compress_activation(x.permute(self.order))

    def restore(self):
        x = restore_activation(self.packed)
        back = [0] * x.dim()
        for i, d in enumerate(self.order):
            back[d] = i
        return x.permute(back).expand(self.shape)


class _StandIn(torch.autograd.Function):
    """A tensor of x's shape without its memory, through which the gradient
    for x flows; the checkpoint keeps it in x's place."""

    @staticmethod
    def forward(ctx, x):
        return x.new_zeros(()).expand(x.shape)

    @staticmethod
    def backward(ctx, grad):
        return grad


class _FillIn(torch.autograd.Function):
    """The block's input in place of its stand-in: the exact one in the
    forward pass, the one held in 8 bits in a recompute."""

    @staticmethod
    def forward(ctx, stand_in, held, exact):
        if exact:
            return exact.pop().detach()
        return held.restore()

    @staticmethod
    def backward(ctx, grad):
        return grad, None, None


def _holds(t) -> bool:
    # computed activations only: parameters and caller-held leaves stay alive
    # elsewhere, so compressing them would add memory
    return (isinstance(t, torch.Tensor) and t.grad_fn is not None
            and t.dtype in (torch.bfloat16, torch.float16, torch.float32))


def _first_parameter(forward) -> Optional[str]:
    """Name of the argument that holds a block's input, for calls that give it
    by name."""
    try:
        params = inspect.signature(forward).parameters.values()
    except (TypeError, ValueError):  # compiled code may have none
        return None
    for p in params:
        return p.name if p.kind is p.POSITIONAL_OR_KEYWORD else None
    return None


def _checkpoint8(fn, first, args, kwargs):
    """``checkpoint(fn, *args, **kwargs)`` with the activation in the first
    argument (by name, ``first``) held in 8 bits until the backward pass."""
    flat = list(args) + list(kwargs.values())
    x = args[0] if args else kwargs.get(first)
    held = {}
    if _holds(x):
        # also where it comes again: the exact one must not stay alive
        packed = _Held(x)
        held = {i: (packed, [t]) for i, t in enumerate(flat) if t is x}
    kept = [_StandIn.apply(t) if i in held else t for i, t in enumerate(flat)]
    n, names = len(args), list(kwargs)
    del x, flat, args, kwargs

    def run(*vals):
        vals = [_FillIn.apply(t, *held[i]) if i in held else t
                for i, t in enumerate(vals)]
        return fn(*vals[:n], **dict(zip(names, vals[n:])))

    return checkpoint(run, *kept, use_reentrant=False)


def _wrap_module(m: nn.Module, save_bits: int = 16) -> None:
    setattr(m, _BITS, save_bits)  # of the last call, also when wrapped
    if getattr(m, _MARK, False):
        return
    inner_forward = m.forward
    first = _first_parameter(inner_forward)

    @functools.wraps(inner_forward)
    def ckpt_forward(*args, **kwargs):
        if not torch.is_grad_enabled() or not m.training:
            return inner_forward(*args, **kwargs)
        if getattr(m, _BITS) == 8:
            return _checkpoint8(inner_forward, first, args, kwargs)
        return checkpoint(
            inner_forward, *args, use_reentrant=False, **kwargs
        )

    m.forward = ckpt_forward
    setattr(m, _MARK, True)


def apply_activation_checkpointing(
    model: nn.Module,
    predicate: Optional[Callable[[str, nn.Module], bool]] = None,
    min_params: int = 1_000_000,
    save_bits: int = 16,
) -> int:
    """Wrap eligible submodules with recompute-in-backward.

    Default eligibility: any non-container child subtree holding at least
    ``min_params`` parameters (the same granularity the FSDP engine uses for
    shard units).  A custom ``predicate(name, module)`` overrides it.
    ``save_bits=8`` holds the blocks' inputs, the first argument of their
    ``forward``, in 8 bits (see the module docstring); 16 keeps them as they
    are.
    Returns the number of modules wrapped.
    """
    check_save_bits(save_bits)
    wrapped = 0
    visited = set()

    def consider(name: str, m: nn.Module) -> bool:
        nonlocal wrapped
        if predicate is not None:
            if predicate(name, m):
                _wrap_module(m, save_bits)
                wrapped += 1
                return True
            return False
        if isinstance(m, (nn.ModuleList, nn.Sequential, nn.ModuleDict)):
            return False
        n = sum(p.numel() for p in m.parameters())
        if n >= min_params:
            _wrap_module(m, save_bits)
            wrapped += 1
            return True
        return False

    def recurse(root: nn.Module, prefix: str):
        for cname, child in root.named_children():
            path = f"{prefix}{cname}"
            if id(child) in visited:
                continue
            visited.add(id(child))
            if not consider(path, child):
                recurse(child, path + ".")

    recurse(model, "")
    return wrapped
