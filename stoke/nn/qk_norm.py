# -*- coding: utf-8 -*-
"""Per-head RMS norm of queries and keys with the rotary rotation in the
same pass (csrc/qk_norm_rope.hip).

``qk_norm_rope`` stands where a block calls ``apply_rope`` on each of its
projections: it takes the ``[B, S, H, D]`` projections (also views of one
fused projection, without a copy), normalises each head over D, rotates, and
returns contiguous ``[B, S, H, D]``.  Positions may be given for each token
(decoding, packed sequences) and on several axes (time, height, width).

GPU tensors in bf16, fp16 and fp32 run the HIP kernels, one launch forward
and two backward for queries and keys together; CPU tensors and float64 take
the same formulas in torch.
"""

from typing import Optional, Sequence, Tuple

import torch
import torch.nn as nn

from stoke import ops

_MAX_AXES = 4
_MAX_DIM = 1024


def _check(q, k, qw, kw, cos, sin, positions, sections):
    if q.dim() != 4 or k.dim() != 4 or q.shape[:2] != k.shape[:2] \
            or q.shape[3] != k.shape[3] or q.dtype != k.dtype \
            or q.device != k.device or not q.is_floating_point() \
            or not 1 <= q.shape[3] <= _MAX_DIM:
        raise ValueError(
            "Stoke -- qk_norm_rope takes q [B, S, H, D] and k [B, S, Hk, D] "
            f"of one floating dtype and device, D up to {_MAX_DIM}, got "
            f"{tuple(q.shape)} {q.dtype} and {tuple(k.shape)} {k.dtype}"
        )
    for w in (qw, kw):
        if w is not None and (
                w.shape != q.shape[3:] or w.device != q.device
                or w.dtype not in (q.dtype, torch.float32)):
            raise ValueError(
                f"Stoke -- qk_norm_rope weights are [{q.shape[3]}] in fp32 "
                f"or {q.dtype}, got {tuple(w.shape)} {w.dtype}"
            )
    if qw is not None and kw is not None and qw.dtype != kw.dtype:
        raise ValueError("Stoke -- qk_norm_rope weights have one dtype")
    if cos.dim() != 2 or cos.shape != sin.shape or cos.device != q.device \
            or sin.device != q.device or not cos.is_floating_point() \
            or not sin.is_floating_point() \
            or 2 * cos.shape[1] > q.shape[3] or cos.requires_grad \
            or sin.requires_grad:
        raise ValueError(
            "Stoke -- qk_norm_rope takes constant tables cos, sin "
            f"[P, <= D / 2], got {tuple(cos.shape)} and {tuple(sin.shape)}"
        )
    axes = 1
    if sections is not None:
        axes = len(sections)
        if not 1 <= axes <= _MAX_AXES or min(sections) < 0 \
                or sum(sections) != cos.shape[1]:
            raise ValueError(
                f"Stoke -- sections are 1 to {_MAX_AXES} numbers of pairs "
                f"that add up to {cos.shape[1]}, got {tuple(sections)}"
            )
    if positions is None:
        if axes > 1 or cos.shape[0] < q.shape[1]:
            raise ValueError(
                "Stoke -- without positions there is one axis and the tables "
                f"cover the sequence ({cos.shape[0]} rows for {q.shape[1]})"
            )
        return
    want = tuple(q.shape[:2])
    if sections is not None:
        want = (axes,) + want
    got = tuple(positions.shape)
    if positions.dtype not in (torch.int64, torch.int32) \
            or positions.device != q.device or len(got) != len(want) \
            or any(a not in (1, b) for a, b in zip(got[-2:], want[-2:])) \
            or (sections is not None and got[0] != axes):
        raise ValueError(
            f"Stoke -- positions are whole numbers {want} (B and S of 1 "
            f"broadcast) on the heads' device, got {got} {positions.dtype}"
        )


def _eager(q, k, qw, kw, cos, sin, pos, sections, eps, interleaved):
    """The formulas in fp32 (float64 for float64), rounded once."""
    dt = torch.float64 if q.dtype == torch.float64 else torch.float32
    cos, sin = cos.to(dt), sin.to(dt)
    half = cos.shape[1]
    if pos is None:
        c, s = cos[None, : q.shape[1]], sin[None, : q.shape[1]]
    else:
        pos = pos if sections is not None else pos[None]
        bad = (pos < 0) | (pos >= cos.shape[0])
        at = pos.clamp(0, max(0, cos.shape[0] - 1))

        def rows(table):
            # a position outside the table gives NaN
            parts = table.split(list(sections or [half]), -1)
            return torch.cat(
                [(p[a] if len(p) else p.new_zeros(*a.shape, p.shape[1]))
                 .masked_fill(b[..., None], float("nan"))
                 for p, a, b in zip(parts, at, bad)], -1)

        c, s = rows(cos), rows(sin)
    c, s = c[:, :, None], s[:, :, None]

    def one(x, w):
        n = x.to(dt)
        n = n * torch.rsqrt(n.square().mean(-1, keepdim=True) + eps)
        if w is not None:
            n = n * w.to(dt)
        if interleaved:
            a, b = n[..., 0: 2 * half: 2], n[..., 1: 2 * half: 2]
        else:
            a, b = n[..., :half], n[..., half: 2 * half]
        ya, yb = a * c - b * s, b * c + a * s
        y = torch.stack((ya, yb), -1).flatten(-2) if interleaved \
            else torch.cat((ya, yb), -1)
        return torch.cat((y, n[..., 2 * half:]), -1).to(x.dtype)

    return one(q, qw), one(k, kw)


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor,
                 q_weight: Optional[torch.Tensor],
                 k_weight: Optional[torch.Tensor], cos: torch.Tensor,
                 sin: torch.Tensor,
                 positions: Optional[torch.Tensor] = None,
                 sections: Optional[Sequence[int]] = None,
                 eps: float = 1e-6, interleaved: bool = True,
                 ) -> Tuple[torch.Tensor, torch.Tensor]:
    """RMS-normalise every head of q [B, S, H, D] and k [B, S, Hk, D] and
    rotate its first ``2 * cos.shape[1]`` values.

    q_weight, k_weight: [D] in fp32 or the heads' dtype, or None for ones.
    cos, sin: [P, pairs] tables, used in fp32.  positions: [B, S] rows of
    the tables (None: 0, 1, ... along S); with ``sections`` [axes, B, S],
    where the first ``sections[0]`` pairs follow the first axis and so on.
    interleaved: pairs (2i, 2i + 1) as ``apply_rope`` has them, else
    (i, i + pairs).  A position outside the tables gives NaN.
    """
    if q.is_cuda and q.dtype != torch.float64:
        # the extension checks the arguments as _check does
        return tuple(ops._require_ext().qk_norm_rope(
            q, k, q_weight, k_weight, cos, sin, positions, sections, eps,
            interleaved))
    _check(q, k, q_weight, k_weight, cos, sin, positions, sections)
    if positions is not None:
        positions = positions.expand(*positions.shape[:-2], *q.shape[:2])
    return _eager(q, k, q_weight, k_weight, cos, sin, positions, sections,
                  eps, interleaved)


class StokeQKNorm(nn.Module):
    """The norm weights of a block's query and key heads with
    ``qk_norm_rope``; call it on the projections before the attention."""

    def __init__(self, head_dim: int, eps: float = 1e-6,
                 interleaved: bool = True):
        super().__init__()
        self.q_weight = nn.Parameter(torch.ones(head_dim))
        self.k_weight = nn.Parameter(torch.ones(head_dim))
        self.eps = eps
        self.interleaved = interleaved

    def forward(self, q, k, cos, sin, positions=None, sections=None):
        return qk_norm_rope(q, k, self.q_weight, self.k_weight, cos, sin,
                            positions=positions, sections=sections,
                            eps=self.eps, interleaved=self.interleaved)

    def extra_repr(self):
        return f"{self.q_weight.numel()}, eps={self.eps}"
