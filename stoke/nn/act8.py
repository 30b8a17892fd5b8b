# -*- coding: utf-8 -*-
"""Activations held in 8 bits between the forward and the backward pass.

32 consecutive values of the flattened tensor share a power of two (one byte
``E``) and keep a signed byte each, so that ``value = q * 2**(E - 127)``.  It
costs 1 1/32 bytes a value; a value is off by at most 1/127 of the largest of
its 32, or by 2^-127 where that one is below 2^-120.  A block with an infinity
or NaN (``E = 255``) reads back as NaN, so overflows still reach the gradients.
The published microscaling format of 8-bit integers looks alike, but its bytes
stand for ``q * 2**(E - 133)`` and its exponent is chosen by another rule: one
does not read the other.

``compress_activation`` / ``restore_activation`` are the format itself,
``apply_activation_checkpointing(..., save_bits=8)`` keeps a block's inputs
in it and ``swiglu(..., save_bits=8)`` the gate and up projections.  GPU
tensors (bf16, fp16, fp32) run csrc/act8.hip; CPU tensors take the same
steps in torch, bit for bit.
"""

from typing import NamedTuple

import torch

from stoke import ops

_BLOCK = 32
_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


class CompressedActivation(NamedTuple):
    """An activation in 8 bits; ``restore_activation`` brings it back."""

    values: torch.Tensor  # int8, the activation's shape
    scales: torch.Tensor  # uint8, one exponent for 32 values
    dtype: torch.dtype  # of the activation


def check_save_bits(save_bits: int) -> None:
    if save_bits not in (8, 16):
        raise ValueError(
            f"Stoke -- save_bits must be 16 (as they are) or 8, got "
            f"{save_bits!r}"
        )


def _pow2(e: torch.Tensor) -> torch.Tensor:
    """2**(e - 127) in fp32 for int32 e from 1 to 254."""
    return (e << 23).view(torch.float32)


def _eager_pack(x: torch.Tensor):
    n = x.numel()
    blk = x.new_zeros((n + _BLOCK - 1) // _BLOCK * _BLOCK, dtype=torch.float32)
    blk[:n] = x.detach().reshape(-1)
    blk = blk.view(-1, _BLOCK)
    # magnitudes order like the bits; NaN comes out above infinity
    top = (blk.view(torch.int32) & 0x7FFFFFFF).amax(-1, keepdim=True)
    be = top >> 23
    e = (be - 6 + ((top & 0x7FFFFF) >= 0x7F0000).to(torch.int32)).clamp_min(1)
    bad = be == 255
    q = (blk * _pow2(254 - e)).round().masked_fill(bad, 0)
    e = e.masked_fill(bad, 255)
    return (q.to(torch.int8).view(-1)[:n].view(x.shape),
            e.view(-1).to(torch.uint8))


def _eager_unpack(q: torch.Tensor, scale: torch.Tensor,
                  dtype: torch.dtype) -> torch.Tensor:
    e = scale.to(torch.int32).repeat_interleave(_BLOCK)[: q.numel()]
    most = torch.finfo(dtype).max
    v = (q.reshape(-1).float() * _pow2(e)).clamp(-most, most)
    return v.masked_fill(e == 255, float("nan")).to(dtype).view(q.shape)


def compress_activation(x: torch.Tensor) -> CompressedActivation:
    """``x`` (bf16, fp16 or fp32, any shape) in 8 bits, without gradient."""
    if x.is_cuda:
        # the extension checks its arguments in the same way
        return CompressedActivation(*ops._require_ext().act8_pack(x), x.dtype)
    if x.dtype not in _DTYPES:
        raise ValueError(
            f"Stoke -- compress_activation takes bf16, fp16 or fp32, got "
            f"{x.dtype}"
        )
    return CompressedActivation(*_eager_pack(x), x.dtype)


def restore_activation(held: CompressedActivation) -> torch.Tensor:
    """The values that ``held`` stands for, in the activation's dtype."""
    q, scale, dtype = held
    if q.is_cuda:
        return ops._require_ext().act8_unpack(q, scale, dtype)
    if dtype not in _DTYPES or q.dtype != torch.int8 \
            or scale.dtype != torch.uint8 or scale.is_cuda \
            or scale.numel() != (q.numel() + _BLOCK - 1) // _BLOCK:
        raise ValueError(
            "Stoke -- restore_activation takes what compress_activation "
            "returned: int8 values and one uint8 exponent for every 32"
        )
    return _eager_unpack(q, scale, dtype)


class _SwiGLU8Fn(torch.autograd.Function):
    """silu(gate) * up; gate and up wait for the backward in 8 bits."""

    @staticmethod
    def forward(ctx, g, u):
        ctx.save_for_backward(*_eager_pack(g), *_eager_pack(u))
        gf = g.float()
        return (gf * torch.sigmoid(gf) * u.float()).to(g.dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        qg, sg, qu, su = ctx.saved_tensors
        # in the inputs' dtype: its range bounds what is read back
        g = _eager_unpack(qg, sg, dy.dtype).float()
        u = _eager_unpack(qu, su, dy.dtype).float()
        s, d = torch.sigmoid(g), dy.float()
        return ((d * u * s * (1 + g * (1 - s))).to(dy.dtype),
                (d * g * s).to(dy.dtype))


def swiglu8(g: torch.Tensor, u: torch.Tensor) -> torch.Tensor:
    if g.is_cuda:
        # the extension checks its arguments in the same way
        return ops._require_ext().swiglu8(g, u)
    if g.shape != u.shape or g.dtype != u.dtype or g.device != u.device \
            or g.dtype not in _DTYPES:
        raise ValueError(
            "Stoke -- swiglu(save_bits=8) takes gate and up of one shape, "
            f"device and dtype (bf16, fp16, fp32), got {tuple(g.shape)} "
            f"{g.dtype} and {tuple(u.shape)} {u.dtype}"
        )
    return _SwiGLU8Fn.apply(g, u)
