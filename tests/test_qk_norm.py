# -*- coding: utf-8 -*-
"""Norm and rotation of query and key heads against float64 (torch path
here, HIP kernels in the gpu tier)."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

from stoke import ops
from stoke.nn import StokeQKNorm, StokeRMSNorm, qk_norm_rope
from stoke.nn.rope import apply_rope

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
U = 2.0 ** -24  # half an fp32 step


def _skip(device):
    if device == "cuda" and not torch.cuda.is_available():
        pytest.skip("no GPU")


def _tables(n, pairs, base=500000.0):
    inv = base ** (-torch.arange(pairs).double() / max(1, pairs))
    ang = torch.arange(n).double()[:, None] * inv
    return ang.cos().float(), ang.sin().float()


def _case(b, s, hq, hk, d, rot, dtype, wtype, axes=1, table=300, seed=0,
          device="cpu"):
    g = torch.Generator().manual_seed(seed)
    size = torch.exp(torch.randn(d, generator=g))
    q = (torch.randn(b, s, hq, d, generator=g) * size).to(dtype)
    k = (torch.randn(b, s, hk, d, generator=g) * size.flip(0)).to(dtype)
    qw = (1 + 0.3 * torch.randn(d, generator=g)).to(wtype)
    kw = (1 + 0.3 * torch.randn(d, generator=g)).to(wtype)
    cos, sin = _tables(table, rot // 2)
    pos = torch.randint(0, table, (axes, b, s), generator=g)
    half = rot // 2
    sections = None
    if axes > 1:
        sections = [half - half // axes * (axes - 1)] + [half // axes] * (
            axes - 1)
    dq = torch.randn(b, s, hq, d, generator=g).to(dtype)
    dk = torch.randn(b, s, hk, d, generator=g).to(dtype)
    t = [v.to(device) for v in (q, k, qw, kw, cos, sin,
                                pos if axes > 1 else pos[0], dq, dk)]
    return t, sections


def _oracle(x, w, dy, cos, sin, pos, sections, eps, inter):
    """(y, dx, dw) in float64, and how far fp32 steps may move each."""
    x, dy = x.detach().cpu().double(), dy.detach().cpu().double()
    d, half = x.shape[-1], cos.shape[1]
    w = (torch.ones(d) if w is None else w.detach().cpu()).double()
    pos = pos.cpu() if sections else pos.cpu()[None]
    axis = torch.repeat_interleave(torch.arange(len(sections or [0])),
                                   torch.tensor(sections or [half]))
    row = pos.permute(1, 2, 0)[..., axis]
    col = torch.arange(half).expand_as(row)
    c = cos.cpu().double()[row, col][:, :, None]
    s = sin.cpu().double()[row, col][:, :, None]
    e = torch.arange(half)
    a, b = (2 * e, 2 * e + 1) if inter else (e, e + half)

    def turn(v, sn, absolute=False):
        out = v.clone().abs() if absolute else v.clone()
        if absolute:
            v, ca, sa = v.abs(), c.abs(), sn.abs()
            out[..., a] = v[..., a] * ca + v[..., b] * sa
            out[..., b] = v[..., b] * ca + v[..., a] * sa
        else:
            out[..., a] = v[..., a] * c - v[..., b] * sn
            out[..., b] = v[..., b] * c + v[..., a] * sn
        return out

    r = 1 / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    steps = (d / 16 + 24) * U  # additions of one lane, joins, root, quotient
    y, y_err = turn(x * r * w, s), turn(x * r * w, s, True) * steps
    dn, dn_err = turn(dy, -s), turn(dy, s, True) * 3 * U
    g = dn * w
    k = (g * x).mean(-1, keepdim=True) * r * r
    k_abs = (g * x).abs().mean(-1, keepdim=True) * r * r
    k_err = (dn_err * (w * x).abs()).mean(-1, keepdim=True) * r * r \
        + k_abs * 3 * steps
    dx = r * (g - x * k)
    dx_err = r * (dn_err * w.abs() + x.abs() * k_err) \
        + r * (g.abs() + (x * k).abs()) * steps
    term = dn * x * r
    depth = min(512, term[..., 0].numel()) + 60
    dw = term.sum((0, 1, 2))
    dw_err = (term.abs() * (depth * U + steps)
              + dn_err * (x * r).abs()).sum((0, 1, 2))
    return (y, y_err), (dx, dx_err), (dw, dw_err)


def _close(got, want, dtype, what):
    want, err = want
    fin = torch.finfo(dtype)
    tol = err + fin.eps / 2 * (want.abs() + err) + fin.tiny * fin.eps / 2
    off = (got.detach().cpu().double() - want).abs()
    assert got.dtype == dtype and got.shape == want.shape, what
    assert bool((off <= tol).all()), (
        what, float((off / tol).nan_to_num(posinf=9e9).max()))


CASES = [
    # b, s, hq, hk, d, rot, axes
    (1, 1, 1, 1, 2, 2, 1),
    (2, 3, 2, 1, 8, 8, 1),
    (1, 5, 3, 2, 7, 4, 1),
    (3, 1, 8, 2, 64, 64, 1),
    (2, 33, 4, 2, 80, 40, 2),
    (1, 17, 6, 3, 96, 96, 3),
    (2, 65, 5, 1, 128, 128, 3),
    (2, 9, 4, 4, 128, 64, 1),
    (2, 11, 4, 2, 128, 24, 1),
    (1, 6, 2, 2, 80, 72, 3),
    (1, 9, 2, 1, 512, 8, 1),
    (1, 31, 2, 2, 192, 96, 4),
    (1, 40, 4, 1, 256, 256, 2),
    (1, 3, 2, 1, 600, 200, 1),
    (1, 2, 2, 1, 1024, 1024, 2),
    (1, 4, 2, 2, 128, 0, 1),
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("inter", [True, False])
@pytest.mark.parametrize("w32", [True, False])
@pytest.mark.parametrize("case", CASES)
def test_against_float64(case, w32, inter, dtype, device):
    _skip(device)
    b, s, hq, hk, d, rot, axes = case
    wtype = torch.float32 if w32 else dtype
    (q, k, qw, kw, cos, sin, pos, dq, dk), sec = _case(
        b, s, hq, hk, d, rot, dtype, wtype, axes=axes, device=device)
    leaves = [v.requires_grad_(True) for v in (q, k, qw, kw)]
    yq, yk = qk_norm_rope(q, k, qw, kw, cos, sin, positions=pos,
                          sections=sec, eps=1e-5, interleaved=inter)
    grads = torch.autograd.grad((yq, yk), leaves, (dq, dk))
    for y, x, w, dy, dx, dw in ((yq, q, qw, dq, grads[0], grads[2]),
                                (yk, k, kw, dk, grads[1], grads[3])):
        oy, odx, odw = _oracle(x, w, dy, cos, sin, pos, sec, 1e-5, inter)
        assert y.is_contiguous()
        _close(y, oy, dtype, "y")
        _close(dx, odx, dtype, "dx")
        _close(dw, odw, wtype, "dw")


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,inter", [(128, False), (64, True), (80, False)])
def test_views_of_one_projection_and_other_layouts(d, inter, dtype, device):
    _skip(device)
    (q, k, qw, kw, cos, sin, pos, dq, dk), _ = _case(
        2, 7, 4, 2, d, d, dtype, torch.float32, device=device)

    def run(a, b):
        a, b = a.requires_grad_(True), b.requires_grad_(True)
        y = qk_norm_rope(a, b, qw, kw, cos, sin, positions=pos,
                         interleaved=inter)
        return (*y, *torch.autograd.grad(y, (a, b), (dq, dk)))

    want = run(q.clone(), k.clone())
    fused = torch.cat((q.flatten(2), k.flatten(2), k.flatten(2)), -1)
    odd = torch.cat((q.flatten(2)[..., :3], q.flatten(2), k.flatten(2)), -1)
    for a, b in (
        (fused[..., : 4 * d].view(2, 7, 4, d),
         fused[..., 4 * d: 6 * d].view(2, 7, 2, d)),
        (odd[..., 3: 3 + 4 * d].view(2, 7, 4, d),
         odd[..., 3 + 4 * d:].view(2, 7, 2, d)),
        (q.transpose(1, 2).contiguous().transpose(1, 2),
         k.transpose(0, 1).contiguous().transpose(0, 1)),
        (q.transpose(2, 3).contiguous().transpose(2, 3), k.clone()),
    ):
        got = run(a.detach(), b.detach())
        for x, y in zip(got, want):
            # another alignment may add a row's squares in another order
            off = (x.double() - y.double()).abs()
            tol = 4 * torch.finfo(dtype).eps * y.double().abs().amax()
            assert bool((off <= tol).all())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("d,inter", [(128, False), (64, True), (50, True)])
def test_gradients_in_other_layouts(d, inter, device):
    _skip(device)
    (q, k, qw, kw, cos, sin, pos, dq, dk), _ = _case(
        3, 7, 4, 2, d, d // 2 * 2, torch.bfloat16, torch.float32,
        device=device)
    leaves = [v.requires_grad_(True) for v in (q, k, qw, kw)]
    y = qk_norm_rope(q, k, qw, kw, cos, sin, positions=pos,
                     interleaved=inter)

    def run(a, b):
        return torch.autograd.grad(y, leaves, (a, b), retain_graph=True)

    want = run(dq, dk)
    turn = [v.transpose(1, 2).contiguous().transpose(1, 2) for v in (dq, dk)]
    last = [v.transpose(2, 3).contiguous().transpose(2, 3) for v in (dq, dk)]
    for got in (run(*turn), run(dq, turn[1]), run(*last)):
        assert all(torch.equal(p, r) for p, r in zip(got, want))
    # one value for all: strides of 0
    ones = [torch.ones((), dtype=v.dtype, device=device).expand(v.shape)
            for v in (dq, dk)]
    full = [v.contiguous() for v in ones]
    assert all(torch.equal(p, r) for p, r in zip(run(*ones), run(*full)))


@pytest.mark.parametrize("device", DEVICES)
def test_matches_the_norm_and_rope_it_replaces(device):
    _skip(device)
    (q, k, qw, kw, cos, sin, pos, dq, dk), _ = _case(
        2, 12, 4, 2, 64, 64, torch.float32, torch.float32, device=device)
    norms = []
    for w in (qw, kw):
        m = StokeRMSNorm(64, eps=1e-6).to(device)
        m.weight.data.copy_(w)
        norms.append(m)
    mod = StokeQKNorm(64).to(device)
    mod.q_weight.data.copy_(qw)
    mod.k_weight.data.copy_(kw)
    yq, yk = mod(q, k, cos, sin)
    assert torch.allclose(yq, apply_rope(norms[0](q), cos, sin), atol=2e-5)
    assert torch.allclose(yk, apply_rope(norms[1](k), cos, sin), atol=2e-5)
    at = torch.arange(12, device=device).expand(2, 12)
    for p in (at, at[:1], at.int()):
        zq, zk = mod(q, k, cos, sin, positions=p)
        assert torch.equal(zq, yq) and torch.equal(zk, yk)
    # weights that lie anywhere in a flat parameter
    flat = torch.cat((qw[:3], qw, kw)).requires_grad_(True)
    zq, zk = qk_norm_rope(q, k, flat[3:67], flat[67:], cos, sin)
    assert torch.equal(zq, yq) and torch.equal(zk, yk)
    gf, = torch.autograd.grad((zq, zk), flat, (dq, dk))
    gw = torch.autograd.grad((yq, yk), (mod.q_weight, mod.k_weight), (dq, dk))
    assert torch.equal(gf[3:67], gw[0]) and torch.equal(gf[67:], gw[1])
    # positions of several axes broadcast over the batch
    p3 = torch.stack((at[0], at[0].flip(0)))[:, None]
    za = mod(q, k, cos, sin, positions=p3, sections=[20, 12])
    zb = mod(q, k, cos, sin, positions=p3.expand(2, 2, 12).contiguous(),
             sections=(20, 12))
    assert torch.equal(za[0], zb[0]) and torch.equal(za[1], zb[1])
    # one section for all pairs is the single axis
    zq, _ = mod(q, k, cos, sin, positions=at[None], sections=[32])
    assert torch.equal(zq, yq)
    # decoding: token 7 alone at its position
    zq, zk = mod(q[:, 7:8], k[:, 7:8], cos, sin, positions=at[:, 7:8])
    assert torch.equal(zq, yq[:, 7:8]) and torch.equal(zk, yk[:, 7:8])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("inter", [True, False])
@pytest.mark.parametrize("d", [64, 50])
@pytest.mark.parametrize("sections", [
    [1, 1, -2], [0, 3, -3], [-2, 1, 1], [2, 0, 0, -2], [-0, 0], [5, 9, 1, -15]])
def test_short_and_empty_sections(sections, d, inter, device):
    _skip(device)
    half = d // 2
    # the negative entry takes the rest of the pairs
    rest = half - sum(n for n in sections if n > 0)
    sec = [n if n > 0 else 0 for n in sections]
    sec[min(range(len(sections)), key=lambda i: sections[i])] = rest
    (q, k, qw, kw, cos, sin, _, dq, dk), _ = _case(
        2, 5, 3, 1, d, d // 2 * 2, torch.bfloat16, torch.float32,
        device=device)
    g = torch.Generator().manual_seed(8)
    pos = torch.randint(0, 300, (len(sec), 2, 5), generator=g).to(device)
    pos[-1] = pos[0]  # first and last axis at the same position
    for v in (q, k, qw, kw):
        v.requires_grad_(True)
    y = qk_norm_rope(q, k, qw, kw, cos, sin, positions=pos, sections=sec,
                     interleaved=inter)
    grads = torch.autograd.grad(y, (q, k), (dq, dk))
    for out, x, w, dy, dx in ((y[0], q, qw, dq, grads[0]),
                              (y[1], k, kw, dk, grads[1])):
        oy, odx, _ = _oracle(x, w, dy, cos, sin, pos, sec, 1e-6, inter)
        _close(out, oy, torch.bfloat16, "y")
        _close(dx, odx, torch.bfloat16, "dx")


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("d", [64, 100])
def test_edges(d, device):
    _skip(device)
    (q, k, qw, kw, cos, sin, pos, dq, dk), _ = _case(
        2, 6, 3, 1, d, d, torch.bfloat16, torch.float32, device=device)
    # a row of zeros is finite in both directions
    q[0, 2, 1] = 0
    q.requires_grad_(True)
    yq, yk = qk_norm_rope(q, k, None, None, cos, sin, positions=pos)
    assert bool((yq[0, 2, 1] == 0).all())
    g, = torch.autograd.grad(yq, q, dq)
    assert torch.isfinite(g).all()
    q, yq = q.detach(), yq.detach()
    # a position outside the tables gives NaN there and nowhere else
    for bad in (-1, cos.shape[0], 1 << 40):
        p = pos.clone()
        p[1, 3] = bad
        zq, zk = qk_norm_rope(q, k, None, None, cos, sin, positions=p)
        assert torch.isnan(zq[1, 3]).all() and torch.isnan(zk[1, 3]).all()
        zq[1, 3], yq2 = 0, yq.clone()
        yq2[1, 3] = 0
        assert torch.equal(zq, yq2)
    # NaN in a row stays in that row
    q2 = q.clone()
    q2[1, 0, 2, 5] = float("nan")
    zq, _ = qk_norm_rope(q2, k, None, None, cos, sin, positions=pos)
    assert torch.isnan(zq[1, 0, 2]).all()
    zq[1, 0, 2] = yq[1, 0, 2]
    assert torch.equal(zq, yq)
    # nothing to do
    for b, s, h in ((0, 6, 3), (2, 0, 3), (2, 6, 0)):
        e = q[:b, :s, :h].requires_grad_(True)
        w = qw.clone().requires_grad_(True)
        y, z = qk_norm_rope(e, k[:b, :s], w, kw, cos, sin,
                            positions=pos[:b, :s])
        assert y.shape == e.shape
        ge, gw = torch.autograd.grad((y.sum() + z.sum()), (e, w))
        assert ge.shape == e.shape and bool((gw == 0).all())


@pytest.mark.parametrize("device", DEVICES)
def test_only_one_output_used_and_one_weight(device):
    _skip(device)
    (q, k, qw, kw, cos, sin, pos, dq, dk), _ = _case(
        2, 6, 3, 1, 64, 64, torch.float32, torch.float32, device=device)
    for v in (q, k, qw):
        v.requires_grad_(True)
    yq, yk = qk_norm_rope(q, k, qw, None, cos, sin, positions=pos)
    gq, gk, gw = torch.autograd.grad(yk, (q, k, qw), dk, allow_unused=True,
                                     materialize_grads=True)
    assert bool((gq == 0).all()) and bool((gw == 0).all())
    assert bool((gk != 0).any())


def test_gradients_against_differences():
    (q, k, qw, kw, cos, sin, pos, dq, dk), sec = _case(
        1, 3, 2, 1, 12, 8, torch.float32, torch.float32, axes=2)
    q, k, qw, kw = (v.double().requires_grad_(True) for v in (q, k, qw, kw))
    for inter in (True, False):
        assert torch.autograd.gradcheck(
            lambda a, b, c, d: qk_norm_rope(
                a, b, c, d, cos.double(), sin.double(), positions=pos,
                sections=sec, interleaved=inter), (q, k, qw, kw))


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    _skip(device)
    (q, k, qw, kw, cos, sin, pos, _, _), _ = _case(
        2, 6, 3, 1, 64, 64, torch.float32, torch.float32, device=device)
    ok = dict(positions=pos)
    pos3 = pos.expand(3, 2, 6)
    cases = [
        lambda: qk_norm_rope(q[0], k[0], qw, kw, cos, sin, **ok),
        lambda: qk_norm_rope(q, k[:, :5], qw, kw, cos, sin, **ok),
        lambda: qk_norm_rope(q, k[..., :32], qw, kw, cos, sin, **ok),
        lambda: qk_norm_rope(q, k.half(), qw, kw, cos, sin, **ok),
        lambda: qk_norm_rope(q.long(), k.long(), qw, kw, cos, sin, **ok),
        lambda: qk_norm_rope(q, k, qw[:32], kw, cos, sin, **ok),
        lambda: qk_norm_rope(q, k, qw.half(), kw, cos, sin, **ok),
        lambda: qk_norm_rope(q.half(), k.half(), qw, kw.half(), cos, sin,
                             **ok),
        lambda: qk_norm_rope(q, k, qw, kw, cos, sin[:5], **ok),
        lambda: qk_norm_rope(q, k, qw, kw, cos.repeat(1, 2),
                             sin.repeat(1, 2), **ok),
        lambda: qk_norm_rope(q, k, qw, kw, cos[:5], sin[:5]),
        lambda: qk_norm_rope(q, k, qw, kw, cos, sin, positions=pos[:, :5]),
        lambda: qk_norm_rope(q, k, qw, kw, cos, sin, positions=pos.float()),
        lambda: qk_norm_rope(q, k, qw, kw, cos, sin, positions=pos3),
        lambda: qk_norm_rope(q, k, qw, kw, cos, sin, positions=pos3,
                             sections=[16, 16]),
        lambda: qk_norm_rope(q, k, qw, kw, cos, sin, positions=pos3,
                             sections=[16, 8, 4]),
        lambda: qk_norm_rope(q, k, qw, kw, cos, sin, positions=pos3,
                             sections=[40, -16, 8]),
        lambda: qk_norm_rope(q, k, qw, kw, cos, sin, sections=[16, 16]),
        lambda: qk_norm_rope(q, k, qw, kw, cos, sin, positions=pos,
                             sections=[32]),
        lambda: qk_norm_rope(q.repeat(1, 1, 1, 20), k.repeat(1, 1, 1, 20),
                             None, None, cos, sin, **ok),
    ]
    for call in cases:
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("device", DEVICES)
def test_forward_mode_is_refused_by_the_kernels(device):
    """A tangent must not vanish; the extension sees it before the device."""
    _skip(device)
    if not ops.has_ext():
        pytest.skip("extension not built")
    (q, k, qw, kw, cos, sin, pos, _, _), _ = _case(
        2, 6, 3, 1, 64, 64, torch.float32, torch.float32, device=device)
    with fwd.dual_level():
        for i in range(6):
            args = [q, k, qw, kw, cos, sin]
            args[i] = fwd.make_dual(args[i], torch.ones_like(args[i]))
            for grad in (False, True):
                q.requires_grad_(grad)
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    ops._require_ext().qk_norm_rope(*args, pos, None, 1e-6,
                                                    True)
                if device == "cuda":
                    with pytest.raises(NotImplementedError):
                        qk_norm_rope(*args, positions=pos)
            q.requires_grad_(False)
            if device == "cpu":
                y, _ = qk_norm_rope(*args, positions=pos)
                z = qk_norm_rope(*args, positions=pos)[1]
                assert any(fwd.unpack_dual(o).tangent is not None
                           for o in (y, z))


@pytest.mark.gpu
def test_gpu_long_offsets():
    """Rows whose offset in the projection passes 2^31 elements."""
    _skip("cuda")
    d, stride = 64, (1 << 31) // 4 + 64
    store = torch.zeros(5 * stride, dtype=torch.bfloat16, device="cuda")
    (q, k, qw, kw, cos, sin, pos, dq, dk), _ = _case(
        5, 2, 2, 1, d, d, torch.bfloat16, torch.float32, device="cuda")
    view = store.as_strided(q.shape, (stride, 2 * d, d, 1))
    view.copy_(q)
    want = qk_norm_rope(q, k, qw, kw, cos, sin, positions=pos)
    got = qk_norm_rope(view, k, qw, kw, cos, sin, positions=pos)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.gpu
def test_gpu_repeats_and_replays_bit_for_bit():
    _skip("cuda")
    (q, k, qw, kw, cos, sin, pos, dq, dk), sec = _case(
        4, 300, 8, 2, 128, 128, torch.bfloat16, torch.float32, axes=3,
        device="cuda")
    leaves = [v.requires_grad_(True) for v in (q, k, qw, kw)]

    def step():
        y = qk_norm_rope(q, k, qw, kw, cos, sin, positions=pos, sections=sec)
        return (*(v.detach() for v in y),
                *torch.autograd.grad(y, leaves, (dq, dk)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, first))
    for i in range(1, 4):
        with torch.no_grad():
            q.mul_(1.0 + i)
            pos.add_(1).remainder_(cos.shape[0])
        graph.replay()
        torch.cuda.synchronize()
        got = [v.clone() for v in out]
        assert all(torch.equal(a, b) for a, b in zip(got, step())), i


@pytest.mark.gpu
def test_gpu_capture_over_a_live_graph_of_the_weights_is_refused():
    _skip("cuda")
    (q, k, qw, kw, cos, sin, pos, dq, dk), _ = _case(
        2, 6, 3, 1, 64, 64, torch.bfloat16, torch.float32, device="cuda")
    kw.requires_grad_(True)
    alive = qk_norm_rope(q, k, qw, kw, cos, sin, positions=pos)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="drop that graph"):
            qk_norm_rope(q, k, qw, kw, cos, sin, positions=pos)
        with torch.no_grad():
            out = qk_norm_rope(q, k, qw, kw, cos, sin, positions=pos)
    graph.replay()
    assert torch.equal(out[0], alive[0]) and torch.equal(out[1], alive[1])


@pytest.mark.gpu
@pytest.mark.parametrize("inter", [True, False])
def test_gpu_heads_past_the_cached_size(inter):
    """Large calls take other accesses: the same values."""
    _skip("cuda")
    b, s, hq, hk, d = 4, 4097, 32, 8, 128
    (q, k, qw, kw, cos, sin, pos, dq, dk), sec = _case(
        b, 1, hq, hk, d, d, torch.bfloat16, torch.float32, axes=3,
        device="cuda")
    gen = torch.Generator("cuda").manual_seed(0)
    q, k, dq, dk = (torch.randn(b, s, h, d, device="cuda", generator=gen,
                                dtype=torch.bfloat16)
                    for h in (hq, hk, hq, hk))
    pos = torch.randint(0, 300, (3, b, s), device="cuda", generator=gen)
    for w in (q, k, qw, kw):
        w.requires_grad_(True)
    y = qk_norm_rope(q, k, qw, kw, cos, sin, positions=pos, sections=sec,
                     interleaved=inter)
    g = torch.autograd.grad(y, (q, k, qw, kw), (dq, dk))
    dw = [torch.zeros(d, dtype=torch.float64, device="cuda")] * 2
    for i in range(b):
        x = [v.detach()[i:i + 1].requires_grad_(True) for v in (q, k)]
        yi = qk_norm_rope(*x, qw, kw, cos, sin, positions=pos[:, i:i + 1],
                          sections=sec, interleaved=inter)
        gi = torch.autograd.grad(yi, (*x, qw, kw),
                                 (dq[i:i + 1], dk[i:i + 1]))
        for whole, part in zip((*y, *g[:2]), (*yi, *gi[:2])):
            assert torch.equal(whole[i:i + 1], part)
        dw = [a + p.double() for a, p in zip(dw, gi[2:])]
    for a, p, x, dy in zip(g[2:], dw, (q, k), (dq, dk)):
        # both are sums of the same terms in another order: a wave adds up to
        # 64 rows by itself, the rest is fp64; terms are |dn x r| with
        # |dn| <= sqrt 2 max|dy| and |x r| <= |x| / rms
        size = (2 ** 0.5 * dy.float().abs() * x.detach().float().abs()).sum(
            (0, 1, 2)) * 2
        assert bool(((a.double() - p).abs() <= 64 * U * size + 1e-6).all())
