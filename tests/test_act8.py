# -*- coding: utf-8 -*-
"""Activations held in 8 bits: the format, SwiGLU and the checkpoints that
use it (CPU steps here, HIP kernels in the gpu tier) against float64."""

import gc
import math
import weakref

import pytest
import torch
import torch.autograd.forward_ad as fwd

from stoke import ops
from stoke.nn import (
    CompressedActivation,
    apply_activation_checkpointing,
    compress_activation,
    restore_activation,
    swiglu,
)

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
# around a block of 32, around 16-byte pieces, several blocks of threads
SIZES = [(1,), (31,), (32,), (33,), (5, 7), (3, 64), (2, 3, 100), (4, 4096),
         (257, 1367)]


@pytest.fixture(autouse=True)
def _collected(request):
    """A wrapped module refers to itself: what it holds on the GPU must not
    be freed in the middle of a test that counts memory."""
    yield
    if "checkpoint8" in request.node.name:
        gc.collect()


def _skip(device):
    if device == "cuda" and not torch.cuda.is_available():
        pytest.skip("no GPU")


def _act(shape, dtype, device, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g)
    x = x * torch.exp(2 * torch.randn(shape[-1], generator=g))
    return x.to(dtype).to(device)


def _blocks64(x):
    v = x.detach().cpu().double().flatten()
    return torch.nn.functional.pad(v, (0, -v.numel() % 32)).view(-1, 32)


def _held64(x):
    """(values, exponents) by the definition, in Python numbers."""
    blk = _blocks64(x)
    out, exps = torch.empty_like(blk), []
    for i, row in enumerate(blk.tolist()):
        top = max(abs(v) for v in row)
        e = max(math.frexp(top)[1] - 7, -126) if top else -126
        if round(math.ldexp(top, -e)) > 127:
            e += 1
        exps.append(e + 127)
        out[i] = torch.tensor(
            [math.ldexp(round(math.ldexp(v, -e)), e) for v in row],
            dtype=torch.float64)
    return out.view(-1)[: x.numel()].view(x.shape), exps


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SIZES)
def test_format_matches_definition(shape, dtype, device):
    _skip(device)
    x = _act(shape, dtype, device)
    held = compress_activation(x)
    want, exps = _held64(x)
    assert held.values.dtype == torch.int8 and held.values.shape == x.shape
    assert held.scales.tolist() == exps
    assert int(held.values.abs().max()) <= 127
    back = restore_activation(held)
    assert back.dtype == dtype and back.shape == x.shape
    # 7 bits fit into every dtype above its subnormals: equal, one rounding
    assert torch.equal(back.cpu().double(), want.to(dtype).double())
    # the bound the format promises: half a step, 1/127 of the block's top
    off = (_blocks64(back) - _blocks64(x)).abs()
    assert bool((off <= _blocks64(x).abs().amax(-1, keepdim=True) / 127).all())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_format_at_the_ends_of_the_range(dtype, device):
    _skip(device)
    fin = torch.finfo(dtype)
    x = torch.zeros(7, 32, dtype=dtype)
    x[0, 3] = fin.max
    x[1, 5], x[1, 6] = -fin.max, fin.max / 2
    x[2] = fin.tiny
    x[3, 0] = fin.tiny * 2.0 ** -(7 if dtype != torch.float16 else 10)
    x[4] = -0.0
    x[5] = torch.linspace(-1, 1, 32)
    x[6, :2] = torch.tensor([127.5, 1.5]).to(dtype)  # 127.5 rounds past 127
    x = x.to(device)
    held = compress_activation(x)
    want, exps = _held64(x)
    assert held.scales.tolist() == exps
    back = restore_activation(held)
    assert torch.isfinite(back).all()
    # the largest value rounds to a power of two out of range: it comes back
    want = want.clamp(-fin.max, fin.max)
    assert torch.equal(back.cpu().double(), want.to(dtype).double())
    assert float(back[0, 3]) == fin.max and float(back[1, 5]) == -fin.max


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("size", [1e-35, 1e-36, 1e-37, 1e-38, 1e-39])
def test_bound_of_tiny_blocks(size, dtype, device):
    _skip(device)
    g = torch.Generator().manual_seed(0)
    x = (size * torch.randn(40, 32, generator=g).double()).to(dtype)
    back = restore_activation(compress_activation(x.to(device))).cpu()
    off = (back.double() - x.double()).abs()
    top = x.double().abs().amax(-1, keepdim=True)
    bound = torch.where(top < 2.0 ** -120, torch.full_like(top, 2.0 ** -127),
                        top / 127)
    assert bool((off <= bound).all())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
def test_non_finite_blocks_read_back_as_nan(bad, dtype, device):
    _skip(device)
    x = torch.ones(100, dtype=dtype)
    x[40] = bad
    back = restore_activation(compress_activation(x.to(device))).cpu()
    assert torch.isnan(back[32:64]).all()
    assert torch.equal(back[:32], x[:32]) and torch.equal(back[64:], x[64:])


@pytest.mark.parametrize("device", DEVICES)
def test_empty_and_strided_and_offset_inputs(device):
    _skip(device)
    e = compress_activation(torch.empty(0, 5, device=device))
    assert restore_activation(e).shape == (0, 5)
    base = _act((40, 66), torch.bfloat16, device)
    for x in (base.t(), base[:, 1:], base[1:, ::2], base.flatten()[3:]):
        a, b = compress_activation(x), compress_activation(x.clone(
            memory_format=torch.contiguous_format))
        assert torch.equal(a.values, b.values)
        assert torch.equal(a.scales, b.scales)


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    _skip(device)
    def zeros(*shape, dtype=torch.float32):
        return torch.zeros(*shape, dtype=dtype, device=device)

    held = compress_activation(zeros(40))
    cases = [
        lambda: compress_activation(zeros(4, dtype=torch.float64)),
        lambda: restore_activation(CompressedActivation(
            held.values, held.scales[:1], held.dtype)),
        lambda: restore_activation(CompressedActivation(
            held.values.float(), held.scales, held.dtype)),
        lambda: restore_activation(CompressedActivation(
            held.values, held.scales, torch.int32)),
        lambda: swiglu(zeros(4), zeros(4), save_bits=4),
        lambda: swiglu(zeros(4, 4), zeros(4), save_bits=8),
        lambda: swiglu(zeros(4), zeros(4).half(), save_bits=8),
        lambda: swiglu(zeros(4).double(), zeros(4).double(), save_bits=8),
        lambda: apply_activation_checkpointing(
            torch.nn.Linear(2, 2), save_bits=12),
    ]
    for call in cases:
        with pytest.raises(ValueError):
            call()


# ------------------------------------------------------------------ SwiGLU
def _steps(g):
    # fp32 steps, in units of 2^-24: e^-g from exp2 is off by |g| (rounding
    # of g log2 e) + 0.25 |g| (log2 e itself) + 2; a sum, a quotient (2 ulp)
    # and up to 4 products follow.  1 - s loses up to |g| more in g (1 - s).
    return (24 + 4 * g.detach().abs()) * 2.0 ** -24


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SIZES)
def test_swiglu8_against_float64(shape, dtype, device):
    _skip(device)
    g = _act(shape, dtype, device, 1).clamp(-40, 40).requires_grad_(True)
    u = _act(shape, dtype, device, 2).clamp(-40, 40).requires_grad_(True)
    dy = _act(shape, dtype, device, 3).clamp(-4, 4)
    y = swiglu(g, u, save_bits=8)
    y.backward(dy)

    def f(a, b):
        return a * torch.sigmoid(a) * b

    tiny = torch.finfo(dtype).tiny
    tol = torch.finfo(dtype).eps / 2 + _steps(g.cpu().double())
    want = f(g.detach().cpu().double(), u.detach().cpu().double())
    off = (y.detach().cpu().double() - want).abs()
    # below the smallest normal number a rounding is absolute
    assert bool((off <= tol * want.abs() + tiny * tol).all())
    hg = _held64(g)[0].requires_grad_(True)
    hu = _held64(u)[0].requires_grad_(True)
    dg, du = torch.autograd.grad(f(hg, hu), (hg, hu), dy.cpu().double())
    # 1 + g (1 - s) cancels near its root at g = -1.28: its error is relative
    # to the terms, |dy u s| (1 + |g| (1 - s))
    s = torch.sigmoid(hg)
    size = (dy.cpu().double() * hu * s).abs() * (1 + hg.abs() * (1 - s))
    slack = _steps(hg) * size.detach()
    off = (g.grad.cpu().double() - dg).abs()
    assert bool((off <= tol * dg.abs() + slack + tiny * tol).all())
    off = (u.grad.cpu().double() - du).abs()
    assert bool((off <= tol * du.abs() + tiny * tol).all())


def test_swiglu8_gradient_against_differences():
    # whole multiples of 1/64 below 2 are held exactly
    g = torch.randint(-100, 101, (3, 40)).double() / 64
    u = torch.randint(-100, 101, (3, 40)).double() / 64
    g[:, 0] = u[:, 0] = g[:, 32] = u[:, 32] = 1.75
    gf, uf = g.float().requires_grad_(True), u.float().requires_grad_(True)
    swiglu(gf, uf, save_bits=8).sum().backward()
    h = 1e-5

    def f(a, b):
        return a * torch.sigmoid(a) * b

    dg = (f(g + h, u) - f(g - h, u)) / (2 * h)
    du = (f(g, u + h) - f(g, u - h)) / (2 * h)
    # differences: h^2 f'''/6 < 1e-10 and 2^-53 |f| / h < 1e-10; fp32: 24 ulp
    # of terms up to 2 * 1.75
    assert (gf.grad.double() - dg).abs().max() < 24 * 2.0 ** -24 * 4
    assert (uf.grad.double() - du).abs().max() < 24 * 2.0 ** -24 * 4


@pytest.mark.parametrize("device", DEVICES)
def test_swiglu8_strided_gradient_and_halves_of_one_projection(device):
    _skip(device)
    both = _act((6, 2 * 96), torch.bfloat16, device).requires_grad_(True)
    g, u = both.chunk(2, -1)
    y = swiglu(g, u, save_bits=8)
    dy = _act((96, 6), torch.bfloat16, device, 5).t()
    grad, = torch.autograd.grad(y, both, dy)
    gc = g.detach().contiguous().requires_grad_(True)
    uc = u.detach().contiguous().requires_grad_(True)
    yc = swiglu(gc, uc, save_bits=8)
    dg, du = torch.autograd.grad(yc, (gc, uc), dy.contiguous())
    assert torch.equal(y, yc)
    assert torch.equal(grad, torch.cat((dg, du), -1))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("shape", [(6, 96), (1, 8), (5, 1, 40), (3, 7, 24),
                                   (2, 3, 50), (4, 3), (9, 1), (300, 1000)])
def test_swiglu8_rows_at_any_distance(shape, device):
    _skip(device)
    f = shape[-1]
    wide = _act((*shape[:-1], 2 * f + 3), torch.bfloat16, device)
    dense = _act(shape, torch.bfloat16, device, 4)
    turned = dense.transpose(0, -1).contiguous().transpose(0, -1)
    wider = _act((*shape[:-2], 2 * shape[-2], f), torch.bfloat16, device, 6)
    pairs = [(wide[..., :f], wide[..., f:2 * f]),
             (wide[..., 3:3 + f], dense), (dense, wide[..., -f:]),
             (turned, dense), (dense, turned), (wider[..., ::2, :], dense),
             (dense[..., :1].expand(shape), dense),
             (dense[:1].expand(shape), dense),
             (dense.narrow(-2, 0, 1).expand(shape), dense)]
    for g, u in pairs:
        g, u = g.detach().requires_grad_(True), u.detach().requires_grad_(True)
        y = swiglu(g, u, save_bits=8)
        got = torch.autograd.grad(y, (g, u), dense)
        gc = g.detach().clone(memory_format=torch.contiguous_format)
        uc = u.detach().clone(memory_format=torch.contiguous_format)
        gc.requires_grad_(True), uc.requires_grad_(True)
        yc = swiglu(gc, uc, save_bits=8)
        want = torch.autograd.grad(yc, (gc, uc), dense)
        assert torch.equal(y, yc)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [40, 64])
def test_swiglu8_gradient_at_the_largest_value(n, dtype, device):
    """8 bits round it to a power of two out of range; it stays the largest."""
    _skip(device)
    top = torch.finfo(dtype).max
    g = torch.zeros(n, dtype=dtype)
    g[3] = g[-1] = top
    u = torch.zeros(n, dtype=dtype)
    g, u = (v.to(device).requires_grad_(True) for v in (g, u))
    y = swiglu(g, u, save_bits=8)
    dg, du = torch.autograd.grad(y, (g, u), torch.ones_like(y))
    want = torch.zeros(n, dtype=dtype)
    want[3] = want[-1] = top  # silu(top) = top
    assert torch.equal(du.cpu(), want)
    assert bool((dg == 0).all())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SIZES + [(0, 8)])
def test_swiglu8_without_gradient_is_the_same(shape, dtype, device):
    _skip(device)
    wide = _act((*shape[:-1], 2 * shape[-1]), dtype, device, 1)
    for g, u in (wide.chunk(2, -1),
                 [v.contiguous() for v in wide.chunk(2, -1)]):
        want = swiglu(g.detach().requires_grad_(True), u, save_bits=8)
        assert want.requires_grad
        plain = swiglu(g, u, save_bits=8)
        with torch.no_grad():
            scored = swiglu(g.detach().requires_grad_(True), u, save_bits=8)
        for y in (plain, scored):
            assert not y.requires_grad
            assert torch.equal(y, want)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1 << 20, (65 << 20) + 40])
def test_gpu_swiglu8_without_gradient_holds_nothing(n):
    _skip("cuda")
    g = torch.randn(n, device="cuda", dtype=torch.bfloat16,
                    generator=torch.Generator("cuda").manual_seed(0))
    want = swiglu(g.clone().requires_grad_(True), g, save_bits=8).detach()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    y = swiglu(g, g, save_bits=8)
    # the output alone, in the allocator's pieces of 2 MB at most
    assert torch.cuda.max_memory_allocated() - before <= 2 * n + (2 << 20)
    assert torch.equal(y, want)


def test_swiglu8_forward_mode_is_refused_by_the_kernel():
    if not ops.has_ext():
        pytest.skip("extension not built")
    x = torch.ones(40)
    with fwd.dual_level():
        d = fwd.make_dual(x, x)
        for args in ((d, x), (x, d)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                ops._require_ext().swiglu8(*args)


# -------------------------------------------------------------- checkpoints
class _Block(torch.nn.Module):
    def __init__(self, d):
        super().__init__()
        self.a = torch.nn.Linear(d, d)
        self.b = torch.nn.Linear(d, d)
        self.drop = torch.nn.Dropout(0.2)
        self.calls = []

    def forward(self, x, shift, scale=None, flag=True):
        self.calls.append(x.detach().clone())
        assert flag
        y = self.drop(torch.tanh(self.a(x))) + shift
        return x + self.b(y) * scale


class _Net(torch.nn.Module):
    def __init__(self, d=40, n=3):
        super().__init__()
        self.blocks = torch.nn.ModuleList([_Block(d) for _ in range(n)])

    def forward(self, x, shift, scale):
        for blk in self.blocks:
            x = blk(x, shift, scale=scale, flag=True)
        return x


def _run_net(device, bits, x, shift, scale):
    torch.manual_seed(3)
    net = _Net().to(device)
    if bits:
        apply_activation_checkpointing(
            net, predicate=lambda n, m: isinstance(m, _Block),
            save_bits=bits)
    out = net(x * 1.0, shift, scale)
    return net, out


@pytest.mark.parametrize("device", DEVICES)
def test_checkpoint8_runs_exact_forward_and_held_recompute(device):
    _skip(device)
    x = _act((5, 7, 40), torch.float32, device).clamp(-2, 2)
    shift = torch.randn(40, generator=torch.Generator().manual_seed(9)).to(
        device)
    x.requires_grad_(True)
    scale = torch.full((), 0.5, device=device, requires_grad=True)
    plain, out = _run_net(device, 0, x, shift, scale)
    want = torch.autograd.grad(out.square().sum(),
                               [x, scale, *plain.parameters()])
    net, got_out = _run_net(device, 8, x, shift, scale)
    assert torch.equal(out, got_out)  # the forward sees the exact inputs
    got = torch.autograd.grad(got_out.square().sum(),
                              [x, scale, *net.parameters()])
    for i, blk in enumerate(net.blocks):
        first, again = blk.calls
        assert torch.equal(
            again, restore_activation(compress_activation(first)))
        assert torch.equal(first, plain.blocks[i].calls[0])
    for a, b in zip(got, want):
        assert a.shape == b.shape
        assert not torch.isnan(a).any()
        # inputs are off by 1/127 of a block's largest: the gradients follow
        # them, they are not those of another function
        assert float((a - b).norm() / b.norm()) < 0.05


def test_checkpoint8_gradients_are_those_at_the_held_values():
    # inputs that 8 bits hold exactly: bit-equal gradients
    x = (torch.randint(-127, 128, (4, 40)) / 64).float()
    x[:, ::8] = 1.75
    w = torch.randn(40, 40)

    class Lin(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.w = torch.nn.Parameter(w.clone())

        def forward(self, x):
            return torch.tanh(x @ self.w)

    nets = [torch.nn.Sequential(Lin()) for _ in range(2)]
    apply_activation_checkpointing(nets[1], predicate=lambda n, m: True,
                                   save_bits=8)
    grads = []
    for net in nets:
        leaf = x.clone().requires_grad_(True)
        net(leaf * 1.0).sum().backward()
        grads.append((leaf.grad, net[0].w.grad))
    assert torch.equal(grads[0][0], grads[1][0])
    assert torch.equal(grads[0][1], grads[1][1])


def test_checkpoint8_keeps_no_other_copy_of_its_input():
    import gc
    import weakref

    seen = []

    class Ident(torch.nn.Module):
        def forward(self, x):
            return x.square()

    net = torch.nn.Sequential(Ident())
    apply_activation_checkpointing(net, predicate=lambda n, m: True,
                                   save_bits=8)
    leaf = torch.randn(64, requires_grad=True)
    x = leaf * 2.0
    seen.append(weakref.ref(x))
    y = net(x)
    del x
    gc.collect()
    assert seen[0]() is None
    y.sum().backward()
    assert leaf.grad is not None


def test_checkpoint8_eval_no_grad_and_change_of_bits():
    net = _Net().train()
    n = apply_activation_checkpointing(
        net, predicate=lambda n, m: isinstance(m, _Block), save_bits=8)
    assert n == 3
    apply_activation_checkpointing(
        net, predicate=lambda n, m: isinstance(m, _Block))
    x = torch.randn(2, 40, requires_grad=True)
    net(x * 1.0, torch.zeros(40), torch.ones(())).sum().backward()
    # back at 16 bits: the recompute sees the exact input
    first, again = net.blocks[0].calls
    assert torch.equal(first, again)
    net.eval()
    with torch.no_grad():
        net(x, torch.zeros(40), torch.ones(()))
    assert len(net.blocks[0].calls) == 3


@pytest.mark.gpu
def test_gpu_checkpoint8_saves_memory_under_autocast():
    _skip("cuda")
    d, n = 1024, 6

    class Mlp(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.a = torch.nn.Linear(d, d)

        def forward(self, x):
            return x + torch.tanh(self.a(x))

    held = {}
    for bits in (16, 8):
        torch.manual_seed(0)
        net = torch.nn.Sequential(*[Mlp() for _ in range(n)]).cuda().bfloat16()
        apply_activation_checkpointing(
            net, predicate=lambda n, m: isinstance(m, Mlp), save_bits=bits)
        leaf = torch.randn(8192, d, device="cuda", dtype=torch.bfloat16,
                           requires_grad=True)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        y = net(leaf * 1.0)
        held[bits] = torch.cuda.memory_allocated() - before
        y.float().square().mean().backward()
        assert torch.isfinite(leaf.grad).all()
    # n inputs of 2 bytes against 1 1/32, and the output of both
    per = 8192 * d
    assert held[16] >= (n + 1) * 2 * per
    assert held[8] <= n * per * 33 / 32 + 2 * per + (1 << 22)


class _Scores(torch.nn.Module):
    """Attention over rows of x with an additive bias."""

    def __init__(self, d):
        super().__init__()
        self.w = torch.nn.Parameter(torch.eye(d))

    def forward(self, x, bias, kv=None):
        kv = x if kv is None else kv
        return x + torch.softmax(x @ self.w @ kv.t() + bias, -1) @ kv


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("mask", ["-inf", "lowest", "-1e4"])
@pytest.mark.parametrize("by_name", [False, True])
def test_checkpoint8_leaves_biases_and_masks_exact(by_name, mask, device):
    """A learned bias with a causal mask has a grad_fn as activations do."""
    _skip(device)
    low = {"-inf": -float("inf"), "lowest": torch.finfo(torch.float32).min,
           "-1e4": -1e4}[mask]
    # inputs that 8 bits hold exactly: the gradients are bit-equal
    x = (torch.randint(-127, 128, (8, 32),
                       generator=torch.Generator().manual_seed(1)) / 64)
    x[:, 0] = 1.75
    rel = torch.randn(8, 8, generator=torch.Generator().manual_seed(2))
    far = torch.full((8, 8), low).triu(1)
    grads = []
    for bits in (16, 8):
        net = torch.nn.Sequential(_Scores(32)).to(device)
        apply_activation_checkpointing(net, predicate=lambda n, m: True,
                                       save_bits=bits)
        leaf = x.float().to(device).requires_grad_(True)
        bias = rel.clone().to(device).requires_grad_(True)
        seen = bias + far.to(device)
        args = dict(bias=seen, x=leaf * 1.0)
        y = net[0](**args) if by_name else net[0](args["x"], seen)
        y.square().sum().backward()
        grads.append((leaf.grad, bias.grad, net[0].w.grad))
    for a, b in zip(*grads):
        assert torch.isfinite(b).all() and bool((a != 0).any())
        assert torch.equal(a, b)


@pytest.mark.parametrize("bits", [16, 8])
def test_checkpoint8_of_a_forward_without_a_signature(bits):
    class Tanh(torch.nn.Module):
        forward = staticmethod(torch.tanh)

    net = torch.nn.Sequential(Tanh())
    apply_activation_checkpointing(net, predicate=lambda n, m: True,
                                   save_bits=bits)
    leaf = torch.linspace(-1, 1, 33).mul(64).round().div(64)
    leaf.requires_grad_(True)
    net(leaf * 1.0).sum().backward()
    want = 1 - leaf.detach().double().tanh().square()
    # tanh to 2 ulp, its square twice that, and three more roundings
    assert bool(((leaf.grad.double() - want).abs() <= 8 * 2.0 ** -24).all())


def test_checkpoint8_input_that_comes_twice():
    x = (torch.randint(-127, 128, (8, 32),
                       generator=torch.Generator().manual_seed(1)) / 64)
    x[:, 0] = 1.75
    bias = torch.zeros(8, 8)
    leaves = [x.clone().requires_grad_(True) for _ in range(3)]
    nets = [_Scores(32), torch.nn.Sequential(_Scores(32))]
    apply_activation_checkpointing(nets[1], predicate=lambda n, m: True,
                                   save_bits=8)
    y = nets[0](leaves[0], bias, kv=leaves[1])
    y.square().sum().backward()
    t = leaves[2] * 1.0
    alive = weakref.ref(t)
    z = nets[1][0](t, bias, kv=t)
    del t
    gc.collect()
    assert alive() is None
    assert torch.equal(z, y)
    z.square().sum().backward()
    assert torch.equal(nets[0].w.grad, nets[1][0].w.grad)
    # the same parts (of x: the residual's 2 y and the rest) in another order
    a, b = (v.grad.double() for v in leaves[:2])
    size = a.abs() + b.abs() + 4 * y.detach().double().abs()
    assert bool(((leaves[2].grad.double() - a - b).abs()
                 <= 4 * 2.0 ** -24 * size).all())


class _Strides(torch.nn.Module):
    def __init__(self, view):
        super().__init__()
        self.view, self.seen = view, []

    def forward(self, x):
        self.seen.append((x.shape, x.stride(), x.detach().clone()))
        return torch.tanh(self.view(x))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("name", [
    "contiguous", "channels_last", "channels_last_3d", "transposed", "slice",
    "expanded", "one", "scalar", "empty"])
def test_checkpoint8_recompute_sees_the_layout_of_the_forward(name, device):
    _skip(device)
    shape = {"channels_last_3d": (2, 8, 3, 4, 5), "scalar": (),
             "one": (3, 1, 5, 1), "empty": (0, 4, 5, 6)}.get(
                 name, (2, 8, 6, 5))
    g = torch.Generator().manual_seed(1)
    x = (torch.randint(-127, 128, shape, generator=g) / 64).to(device)
    n, c = shape[0] if shape else 1, shape[1] if shape else 1

    # each made from the leaf, with the view that these strides allow
    make, view = {
        "contiguous": (lambda t: t * 1.0, lambda t: t.view(n, -1)),
        "channels_last": (
            lambda t: (t * 1.0).contiguous(memory_format=torch.channels_last),
            lambda t: t.permute(0, 2, 3, 1).view(-1, c)),
        "channels_last_3d": (
            lambda t: (t * 1.0).contiguous(
                memory_format=torch.channels_last_3d),
            lambda t: t.permute(0, 2, 3, 4, 1).view(-1, c)),
        "transposed": (lambda t: (t.transpose(0, 3) * 1.0).contiguous()
                       .transpose(0, 3),
                       lambda t: t.transpose(0, 3).view(-1)),
        "slice": (lambda t: torch.cat((t, t), -1)[..., :shape[-1]],
                  lambda t: t.flatten(1, 2).view(n, -1, shape[-1])),
        "expanded": (lambda t: (t[:, :1, :, :1] * 1.0).expand(shape),
                     lambda t: t[:, :, :, 0]),
        "one": (lambda t: t * 1.0, lambda t: t.view(-1)),
        "scalar": (lambda t: t * 1.0, lambda t: t.view(1)),
        "empty": (lambda t: t * 1.0, lambda t: t.view(0, 5)),
    }[name]
    grads = []
    for bits in (16, 8):
        net = torch.nn.Sequential(_Strides(view))
        apply_activation_checkpointing(net, predicate=lambda n, m: True,
                                       save_bits=bits)
        leaf = x.clone().requires_grad_(True)
        inp = make(leaf)
        net[0](inp).square().sum().backward()
        (s0, t0, v0), (s1, t1, v1) = net[0].seen
        assert s0 == s1 == x.shape
        if name != "slice":  # gaps are not kept
            assert all(a == b for a, b, k in zip(t0, t1, x.shape) if k > 1)
        # 32 of these values share a step of at most 1/64
        assert torch.equal(v0, v1)
        grads.append(leaf.grad)
    assert torch.equal(*grads)


@pytest.mark.gpu
def test_gpu_replays_in_a_graph():
    _skip("cuda")
    x = _act((64, 1000), torch.bfloat16, "cuda", 1)
    u = _act((64, 1000), torch.bfloat16, "cuda", 2)
    dy = _act((64, 1000), torch.bfloat16, "cuda", 3)
    g = x.clone().requires_grad_(True)
    u.requires_grad_(True)

    def step():
        held = compress_activation(g)
        y = swiglu(g, u, save_bits=8)
        return (held.values, held.scales, restore_activation(held),
                y.detach(), *torch.autograd.grad(y, (g, u), dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        with torch.no_grad():
            g.copy_(x * (1 + 3 * i))
        graph.replay()
        torch.cuda.synchronize()
        got = [v.clone() for v in out]
        assert all(torch.equal(a, b) for a, b in zip(got, step())), i


@pytest.mark.gpu
def test_gpu_tensors_past_the_cached_size():
    """Large tensors take other accesses: the same values."""
    _skip("cuda")
    n = (65 << 20) + 40  # bf16: over 128 MB, an odd last block
    x = torch.randn(n, device="cuda", dtype=torch.bfloat16,
                    generator=torch.Generator("cuda").manual_seed(0))
    held = compress_activation(x)
    back = restore_activation(held)
    dy = x.flip(0)
    u = dy.clone()
    g, u = x.clone().requires_grad_(True), u.requires_grad_(True)
    y = swiglu(g, u, save_bits=8)
    dg, du = torch.autograd.grad(y, (g, u), dy)
    step = 32 << 20
    for a in range(0, n, step):
        b = min(n, a + step)
        part = compress_activation(x[a:b])
        assert torch.equal(part.values, held.values[a:b])
        assert torch.equal(part.scales, held.scales[a // 32:(b + 31) // 32])
        assert torch.equal(restore_activation(part), back[a:b])
        gp = x[a:b].clone().requires_grad_(True)
        up = u.detach()[a:b].clone().requires_grad_(True)
        yp = swiglu(gp, up, save_bits=8)
        assert torch.equal(yp, y[a:b])
        dgp, dup = torch.autograd.grad(yp, (gp, up), dy[a:b])
        assert torch.equal(dgp, dg[a:b]) and torch.equal(dup, du[a:b])
