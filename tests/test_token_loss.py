# -*- coding: utf-8 -*-
"""Token log-probabilities, policy and preference loss against float64
formulas (torch path here, HIP kernels in the gpu tier)."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

from stoke import ops
from stoke.nn import fused_policy_loss, fused_preference_loss, token_logprobs

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
U = 2.0 ** -24  # half an fp32 step
IGN = -100
# one logit, odd and even vocabularies, rows split over blocks and not
SHAPES = [(1, 1, 1), (1, 1, 2), (2, 3, 7), (2, 5, 255), (4, 3, 1000),
          (2, 2, 4097), (2, 1, 50257), (6, 200, 129)]


def _skip(device):
    if device == "cuda" and not torch.cuda.is_available():
        pytest.skip("no GPU")


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _inputs(shape, dtype, device, seed=0, keep=0.7):
    b, s, v = shape
    g = _gen(seed)
    x = 3 * torch.randn(b, s, v, generator=g)
    t = torch.randint(0, v, (b, s), generator=g)
    x.scatter_add_(-1, t[..., None], 12 * torch.rand(b, s, 1, generator=g))
    live = torch.rand(b, s, generator=g) < keep
    live[0, 0] = True
    if b > 1:
        live[1] = False  # a sequence without any token
    t = torch.where(live, t, torch.full_like(t, IGN))
    return x.to(dtype).to(device), t.to(device)


class Oracle:
    """float64 rows of softmax, lp and how far fp32 sums may be off."""

    def __init__(self, x, t):
        x, t = x.detach().cpu().double(), t.cpu()
        v = x.shape[-1]
        self.live = (t != IGN) & (t >= 0) & (t < v)
        at = torch.where(self.live, t, torch.zeros_like(t))[..., None]
        m = x.amax(-1, keepdim=True)
        d = x - m
        e = d.exp()
        z = e.sum(-1, keepdim=True)
        self.p = e / z
        lp = (d.gather(-1, at) - z.log())[..., 0]
        self.lp = torch.where(self.live, lp, torch.zeros_like(lp))
        self.hot = torch.zeros_like(x).scatter_(-1, at, 1.0)
        # a term exp(d) is off by 1.25 |d| U (argument of exp2, log2 e) and
        # 3 U; a thread adds up to v / 256 of them one after another, 80
        # counts the joins and their factors; with the same again for the
        # factors' own arguments
        self.d_u = 1.25 * d.abs().nan_to_num(posinf=0.0) * U
        far = (self.p * d.abs()).nan_to_num().sum(-1)
        self.tol_lp = (v / 256 + 80 + 2.5 * far) * U

    def grad(self, c, c_err, dtype, got):
        """Checks got = c (onehot - p) for row values c known to c_err."""
        got = got.detach().cpu().double()
        c_err = torch.where(self.live, c_err, torch.zeros_like(c_err))
        c = torch.where(self.live, c, torch.zeros_like(c))[..., None]
        side = self.hot - self.p
        want = torch.where(self.live[..., None], c * side,
                           torch.zeros_like(side))
        slack = (c_err[..., None] + 8 * U * c.abs()) * side.abs() \
            + c.abs() * self.p * (self.d_u + self.tol_lp[..., None] + 8 * U)
        fin = torch.finfo(dtype)
        tol = fin.eps / 2 * (want.abs() + slack) + slack \
            + fin.tiny * fin.eps / 2
        bad = (got - want).abs() > torch.where(self.live[..., None], tol,
                                               torch.zeros_like(tol))
        assert not bool(bad.any()), (
            (got - want)[bad][:5], want[bad][:5], int(bad.sum()))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_logprobs(shape, dtype, device):
    _skip(device)
    x, t = _inputs(shape, dtype, device)
    x.requires_grad_(True)
    lp = token_logprobs(x, t)
    o = Oracle(x, t)
    assert lp.dtype == torch.float32 and lp.shape == t.shape
    off = (lp.detach().cpu().double() - o.lp).abs()
    assert bool((off <= o.tol_lp + U * o.lp.abs()).all())
    assert bool((lp[~o.live.to(device)] == 0).all())
    up = torch.randn(t.shape, generator=_gen(5)).to(device)
    lp.backward(up)
    o.grad(up.cpu().double(), torch.zeros(t.shape).double(), dtype, x.grad)


def _policy_inputs(x, t, seed=1):
    g, o = _gen(seed), Oracle(x, t)
    shift = 0.3 * torch.randn(t.shape, generator=g).double()
    for edge in (0.7, 1.4):  # away from the steps of the gradient
        at = torch.tensor(edge).double().log()
        shift = torch.where((shift - at).abs() < 1e-3, shift + 5e-3, shift)
    old = (o.lp - shift).float()
    adv = torch.randn(t.shape, generator=g)
    ref = (o.lp + 0.4 * torch.randn(t.shape, generator=g)).float()
    return o, old, adv, ref


def _policy64(o, old, adv, ref, kl):
    rho = (o.lp - old.double()).exp()
    a = adv.double()
    held = rho.clamp(0.7, 1.4) * a
    tok = -torch.minimum(rho * a, held)
    coef = torch.where(rho * a <= held, -rho * a, torch.zeros_like(rho))
    steep = (rho * a).abs()
    if kl:
        d = ref.double() - o.lp
        tok = tok + kl * (d.exp() - d - 1)
        coef = coef + kl * (1 - d.exp())
        steep = steep + kl * (1 + d.exp())
    n = max(1, int(o.live.sum()))
    return tok[o.live].sum() / n, coef / n, steep / n, tok


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kl", [0.0, 0.3])
@pytest.mark.parametrize("shape", SHAPES)
def test_policy(shape, kl, dtype, device):
    _skip(device)
    x, t = _inputs(shape, dtype, device)
    o, old, adv, ref = _policy_inputs(x, t)
    x.requires_grad_(True)
    loss = fused_policy_loss(
        x, t, old.to(device), adv.to(device),
        ref_logprobs=ref.to(device) if kl else None, clip_low=0.3,
        clip_high=0.4, kl_coef=kl)
    want, coef, steep, tok = _policy64(o, old, adv, ref, kl)
    assert loss.dtype == torch.float32 and loss.dim() == 0
    tol = (steep * o.tol_lp)[o.live].sum() + 2 * U * want.abs()
    assert abs(float(loss.detach()) - float(want)) <= float(tol)
    loss.backward(torch.tensor(3.0, device=device))
    o.grad(3 * coef, 3 * steep * o.tol_lp, dtype, x.grad)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("smooth", [0.0, 0.2])
@pytest.mark.parametrize(
    "shape", [(2, 1, 1), (2, 3, 7), (4, 5, 255), (2, 2, 4097), (2, 1, 50257),
              (6, 200, 129), (4, 700, 40)])
def test_preference(shape, smooth, dtype, device):
    _skip(device)
    x, t = _inputs(shape, dtype, device)
    o = Oracle(x, t)
    ref = (o.lp + 0.5 * torch.randn(t.shape, generator=_gen(3))).float()
    x.requires_grad_(True)
    loss, rewards = fused_preference_loss(
        x, t, ref.to(device), beta=0.3, label_smoothing=smooth)
    assert rewards.shape == (shape[0],) and not rewards.requires_grad
    gap = torch.where(o.live, o.lp - ref.double(),
                      torch.zeros_like(o.lp)).sum(-1) * 0.3
    half = shape[0] // 2
    h = gap[:half] - gap[half:]
    down, upw = 1 / (1 + h.exp()), 1 / (1 + (-h).exp())
    want = (-(1 - smooth) * upw.log() - smooth * down.log()).mean()
    err = 0.3 * torch.where(o.live, o.tol_lp,
                            torch.zeros_like(o.lp)).sum(-1)
    off = (rewards.cpu().double() - gap).abs()
    assert bool((off <= err + 2 * U * gap.abs()).all())
    assert abs(float(loss.detach()) - float(want)) <= float(
        err.sum() / half + 2 * U * want.abs())
    loss.backward(torch.tensor(2.0, device=device))
    dh = 2 * 0.3 / half * (smooth - down)
    dh_err = 2 * 0.3 / half * 0.25 * (err[:half] + err[half:]) \
        + 4 * U * dh.abs()
    c = torch.cat((dh, -dh))[:, None].expand(t.shape)
    c_err = torch.cat((dh_err, dh_err))[:, None].expand(t.shape)
    o.grad(c, c_err, dtype, x.grad)


# ------------------------------------------------------------------- edges
@pytest.mark.parametrize("device", DEVICES)
def test_ignored_rows_are_left_out_whatever_they_hold(device):
    _skip(device)
    x, t = _inputs((4, 6, 300), torch.bfloat16, device, keep=1.0)
    t[0, 2], t[2, 3], t[3, 5] = IGN, 300, -7
    bad = torch.zeros(4, 6, dtype=torch.bool, device=device)
    bad[0, 2] = bad[2, 3] = bad[3, 5] = bad[1] = True
    x[bad] = float("nan")
    x[0, 2, 5] = float("inf")
    vals = torch.randn(4, 6, generator=_gen(0)).to(device)
    vals[bad] = float("nan")
    up = torch.ones(4, 6, device=device)
    for fn in (
        lambda y: (token_logprobs(y, t) * up).sum(),
        lambda y: fused_policy_loss(y, t, vals, vals, ref_logprobs=vals,
                                    kl_coef=0.1),
        lambda y: fused_preference_loss(y, t, vals)[0],
    ):
        y = x.clone().requires_grad_(True)
        loss = fn(y)
        loss.backward()
        assert torch.isfinite(loss)
        assert torch.isfinite(y.grad).all()
        assert bool((y.grad[bad] == 0).all())
        assert bool((y.grad[~bad] != 0).any())


@pytest.mark.parametrize("device", DEVICES)
def test_no_token_left(device):
    _skip(device)
    x = torch.randn(2, 3, 10, device=device, requires_grad=True)
    t = torch.full((2, 3), IGN, device=device)
    v = torch.zeros(2, 3, device=device)
    assert float(fused_policy_loss(x, t, v, v)) == 0.0
    loss, rewards = fused_preference_loss(x, t, v)
    assert abs(float(loss) - 0.6931471805599453) < 1e-7
    assert rewards.tolist() == [0.0, 0.0]
    (fused_policy_loss(x, t, v, v) + loss).backward()
    assert bool((x.grad == 0).all())
    e = torch.empty(2, 0, 10, device=device, requires_grad=True)
    te, ve = t[:, :0], v[:, :0]
    assert token_logprobs(e, te).shape == (2, 0)
    assert float(fused_policy_loss(e, te, ve, ve)) == 0.0
    fused_preference_loss(e, te, ve)[0].backward()
    assert e.grad.shape == e.shape


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_vocabulary_and_lowest_values(dtype, device):
    _skip(device)
    fin = torch.finfo(dtype)
    x = torch.randn(1, 5, 600, generator=_gen(4)).to(dtype)
    x[0, 0, 10:] = -float("inf")  # a constrained step
    x[0, 1, 1:] = fin.min  # masked by the type's lowest value
    x[0, 2] = -float("inf")
    x[0, 2, 7] = 3.0  # one token left
    x[0, 3] = fin.min  # all equal
    x[0, 4, :300] = fin.max
    t = torch.tensor([[3, 0, 7, 5, 1]])
    x, t = x.to(device).requires_grad_(True), t.to(device)
    lp = token_logprobs(x, t)
    o = Oracle(x, t)
    assert torch.isfinite(lp).all()
    off = (lp.detach().cpu().double() - o.lp).abs()
    assert bool((off <= o.tol_lp + U * o.lp.abs()).all())
    lp.sum().backward()
    assert torch.isfinite(x.grad).all()
    assert bool((x.grad[0, 0, 10:] == 0).all())
    assert bool((x.grad[0, 2] == 0).all())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("at", [
    -6e4, -8192.0, -8160.0, -300.0, 500.0, 4090.0, 8160.0, 8192.0, 3e4, 6e4,
    1e6, -2e6, 3e8, 6e8, -6e8, 1e20])
@pytest.mark.parametrize("v", [40, 9000])
def test_logits_far_from_zero(v, at, dtype, device):
    _skip(device)
    if abs(at) > torch.finfo(dtype).max:
        pytest.skip("out of the type's range")
    g = _gen(6)
    x = (at + 4 * torch.randn(2, 3, v, generator=g).double()).to(dtype)
    x[0, 0, ::7] = -1e4  # masks of a usual value
    x[0, 1, ::3] = torch.finfo(dtype).min
    x[0, 2] = x[0, 2, :1]  # all the same
    x[1, 0, : v // 2] = x[1, 0].amax()
    t = torch.tensor([[1, 2, 3], [v // 2 - 1, v - 1, 0]])
    o = Oracle(x, t)
    x, t = x.to(device).requires_grad_(True), t.to(device)
    lp = token_logprobs(x, t)
    off = (lp.detach().cpu().double() - o.lp).abs()
    assert bool((off <= o.tol_lp + U * o.lp.abs()).all()), off
    up = torch.randn(2, 3, generator=_gen(5)).to(device)
    lp.backward(up)
    o.grad(up.cpu().double(), torch.zeros(2, 3).double(), dtype, x.grad)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_gpu_logprobs_have_no_bias(dtype):
    _skip("cuda")
    rows, v = 20000, 4096
    gen = torch.Generator("cuda").manual_seed(0)
    x = (2.5 * torch.randn(rows, v, device="cuda", generator=gen)).to(dtype)
    t = torch.randint(0, v, (rows,), device="cuda", generator=gen)
    lp = token_logprobs(x, t).double()
    y = x.double()
    want = y.gather(1, t[:, None])[:, 0] - torch.logsumexp(y, -1)
    off = lp - want
    # fp32 lp of 4 to 16 are rounded to 2^-21 or 2^-20: 2.8e-7 in the mean
    # square at most, 2e-9 on the mean of 20000; exp2 is 3e-8 off for each
    # value, the few hundred of a bf16 row 3e-9 on their mean
    assert abs(float(off.mean())) < 1e-8
    assert float(off.std()) < 4e-7


def _lp_errors(x, t, per_call):
    """lp - float64 of single tokens, past the rounding to fp32: a sequence of
    one token has the reward lp - ref, and next to lp a reference leaves a
    reward of at most U |lp|, which fp32 holds to 1e-13."""
    off = []
    for i in range(0, len(x), per_call):
        y, at = x[i:i + per_call].double(), t[i:i + per_call, None]
        want = (y.gather(1, at) - torch.logsumexp(y, -1, True))[:, 0]
        ref = want.float()
        _, r = fused_preference_loss(x[i:i + per_call, None], at,
                                     ref[:, None], beta=1.0)
        off.append(r.double() + ref.double() - want)
    return torch.cat(off)


def _lp_model(x):
    """What the roundings of lp come to: the mean square over the rows, and
    the variance of the mean.

    Relative to a term p are off the argument a of exp2, by half an ulp of it
    at most, and exp2, by an ulp at most, both taken as even over their range
    (a third of the square), and 5 levels of fp32 sums of 32 values, U each,
    over groups that hold 32 / V of the row by their other values.  The
    largest term is exact, and so is the sum next to it.  In 16 bits the rows
    share their values, and a value is off the same way in each: it counts in
    the mean with its share of all rows."""
    v = x.shape[1]
    square, mass, worst = 0.0, {}, {}
    for i in range(0, len(x), 256):
        y = x[i:i + 256].double()
        p = torch.softmax(y, -1)
        top = p.argmax(-1, True)
        rest = 1 - p.gather(1, top)
        # a is relative to a whole number up to 1 above the maximum
        a = (y.gather(1, top) - y) * 1.4426950408889634 + 1
        ulp = 2.0 ** (torch.log2(a).floor() - 23)
        var = (0.6931 * ulp / 2) ** 2 / 3 + (2 * U) ** 2 / 3
        p = p.scatter(1, top, 0.0)
        square += float((p * p * (var + 5 * U * U / 3)).sum())
        square += float((rest ** 2).sum()) * 32 / v * 5 * U * U / 3
        if x.dtype == torch.float32:
            continue
        vals, inv = x[i:i + 256].float().unique(return_inverse=True)
        inv = inv.flatten()
        m = torch.zeros_like(vals, dtype=torch.float64)
        m = m.index_add(0, inv, p.flatten())
        w = torch.zeros_like(m).scatter_reduce(0, inv, var.flatten(), "amax")
        for u, b, c in zip(vals.tolist(), m.tolist(), w.tolist()):
            mass[u] = mass.get(u, 0.0) + b
            worst[u] = max(worst.get(u, 0.0), c)
    n = len(x)
    shared = sum(mass[u] ** 2 * worst[u] for u in mass) / n / n
    return square / n, square / n / n + shared


@pytest.mark.gpu
@pytest.mark.parametrize("peaked", [False, True])
@pytest.mark.parametrize("per_call", [1024, 32])  # rows whole and in 32 pieces
@pytest.mark.parametrize("dtype", DTYPES)
def test_gpu_rewards_have_no_bias_that_sequences_add_up(dtype, per_call,
                                                        peaked):
    _skip("cuda")
    rows, v = 1024, 128256
    gen = torch.Generator("cuda").manual_seed(0)
    x = torch.randn(rows, v, device="cuda", generator=gen)
    t = torch.randint(0, v, (rows,), device="cuda", generator=gen)
    if peaked:  # one token has half of the weight to almost all of it
        at = torch.randint(0, v, (rows, 1), device="cuda", generator=gen)
        lse = torch.logsumexp(x, -1, True)
        x.scatter_(1, at, lse + 4 * torch.rand(rows, 1, device="cuda",
                                               generator=gen))
    else:
        x *= 2.5
    x = x.to(dtype)
    off = _lp_errors(x, t, per_call)
    square, mean = _lp_model(x)
    assert float(off.std()) <= square ** 0.5
    # the bias of exp2, 3.2e-9, is given back to a third of it, 4 deviations
    assert abs(float(off.mean())) <= 1e-9 + 4 * mean ** 0.5


@pytest.mark.parametrize("device", DEVICES)
def test_rows_without_a_distribution_are_nan(device):
    _skip(device)
    x = torch.zeros(1, 4, 500)
    x[0, 0] = -float("inf")
    x[0, 1, 3] = float("inf")
    x[0, 2, 400] = float("nan")
    t = torch.tensor([[1, 3, 0, 0]], device=device)
    x = x.to(device).requires_grad_(True)
    lp = token_logprobs(x, t)
    assert torch.isnan(lp[0, :3]).all() and torch.isfinite(lp[0, 3])
    lp.sum().backward()
    assert torch.isnan(x.grad[0, 2]).any()
    assert torch.isfinite(x.grad[0, 3]).all()
    v = torch.zeros(1, 4, device=device)
    assert torch.isnan(fused_policy_loss(x, t, v, v + 1.0))


@pytest.mark.parametrize("device", DEVICES)
def test_policy_on_a_token_that_it_rules_out(device):
    _skip(device)
    x = torch.randn(1, 2, 5, generator=_gen(8))
    x[0, 0, 3] = -float("inf")
    t = torch.tensor([[3, 2]], device=device)
    x = x.to(device).requires_grad_(True)
    v = torch.full((1, 2), -1.0, device=device)
    # rho is 0: without the KL term only the other token counts
    a = fused_policy_loss(x, t, v, v + 2)
    ga, = torch.autograd.grad(a, x)
    b = fused_policy_loss(x[:, 1:], t[:, 1:], v[:, 1:], v[:, 1:] + 2)
    gb, = torch.autograd.grad(b, x)
    assert abs(float(a.detach()) - float(b.detach()) / 2) <= 4 * U * abs(
        float(b.detach()))
    assert bool((ga[0, 0] == 0).all())
    assert torch.allclose(ga[0, 1], gb[0, 1] / 2, rtol=8 * U, atol=0)
    # with it the loss is infinite, as e^d is
    loss = fused_policy_loss(x, t, v, v + 2, v, kl_coef=0.1)
    assert float(loss.detach()) == float("inf")
    # where the reference rules it out too there is no value
    ref = v.clone()
    ref[0, 0] = -float("inf")
    assert torch.isnan(fused_policy_loss(x, t, v, v + 2, ref, kl_coef=0.1))


@pytest.mark.parametrize("device", DEVICES)
def test_preference_at_an_infinite_margin(device):
    _skip(device)
    # one pair of two tokens, a constrained vocabulary: token 3 is at -inf
    x = torch.randn(2, 2, 5, generator=_gen(8))
    t = torch.full((2, 2), 2)
    ref = torch.zeros(2, 2)

    def call(side, smooth):
        y, u = x.clone(), t.clone()
        y[side, 0, 3] = -float("inf")
        u[side, 0] = 3
        y = y.to(device).requires_grad_(True)
        loss, rewards = fused_preference_loss(
            y, u.to(device), ref.to(device), beta=0.3, label_smoothing=smooth)
        g, = torch.autograd.grad(loss, y)
        assert float(rewards[side]) == -float("inf")
        assert torch.isfinite(rewards[1 - side])
        return float(loss.detach()), g.cpu().double(), y

    # the rejected one is impossible: -log sigmoid(+inf) = 0, and flat
    loss, g, _ = call(1, 0.0)
    assert loss == 0.0
    assert bool((g == 0).all())
    # with smoothing the second term is infinite, its slope is not: d / dh of
    # -eps log sigmoid(-h) is eps sigmoid(h) = eps
    for side, smooth, slope in ((1, 0.1, 0.1), (0, 0.0, -1.0), (0, 0.1, -0.9)):
        loss, g, y = call(side, smooth)
        assert loss == float("inf")
        p = torch.softmax(y.detach().cpu().double(), -1)
        hot = torch.zeros_like(p)
        hot[..., 2] = 1
        hot[side, 0] = torch.tensor([0.0, 0, 0, 1, 0])
        c = torch.tensor([1.0, -1.0]).double()[:, None, None]
        want = 0.3 * slope * c * (hot - p)
        # |d| < 6: terms are off by (1.25 * 6 + 3) U, twice, and 5 sums
        assert bool(((g - want).abs() <= 40 * U * 0.3).all())


@pytest.mark.parametrize("device", DEVICES)
def test_ratio_on_the_clip_and_beyond(device):
    _skip(device)
    # uniform over 4 tokens: lp = -log 4; rho = 1/2, 1, 2 with clip [1/2, 2]
    x = torch.zeros(1, 4, 4, device=device, requires_grad=True)
    t = torch.zeros(1, 4, dtype=torch.int64, device=device)
    lp = -torch.tensor(4.0).double().log()
    old = torch.stack((lp, lp, lp + 2, lp - 2)).float()[None].to(device)
    adv = torch.tensor([[1.0, -1.0, -1.0, 1.0]], device=device)
    loss = fused_policy_loss(x, t, old, adv, clip_low=0.5, clip_high=1.0)
    # rho = 1: -A each; rho = e^-2, A < 0: held at 0.5; rho = e^2, A > 0: at 2
    assert abs(float(loss) - (-1 + 1 + 0.5 - 2) / 4) < 1e-6
    loss.backward()
    g = x.grad[0]
    assert bool((g[2:] == 0).all())
    assert abs(float(g[0, 0]) + 0.75 / 4) < 1e-6
    assert abs(float(g[1, 0]) - 0.75 / 4) < 1e-6
    # no clip at all: rho stays on it, and the gradient flows
    x.grad = None
    old = torch.full((1, 4), float(x[0].log_softmax(-1)[0, 0]), device=device)
    fused_policy_loss(x, t, old, adv, clip_low=1.0, clip_high=0.0,
                      ).backward()
    assert bool((x.grad[0, 1] != 0).any())


@pytest.mark.parametrize("device", DEVICES)
def test_layouts_and_broadcast_values(device):
    _skip(device)
    x, t = _inputs((2, 9, 101), torch.bfloat16, device, keep=1.0)
    o, old, adv, ref = _policy_inputs(x, t)
    old, adv = old.to(device), adv[:, :1].contiguous().to(device)
    want = token_logprobs(x, t)
    wide = torch.zeros(2, 11, 130, dtype=x.dtype, device=device)
    wide[:, 1:10, 3:104] = x
    view = wide[:, 1:10, 3:104]  # rows at another alignment and stride
    turned = x.transpose(0, 1).contiguous().transpose(0, 1)
    last = x.transpose(1, 2).contiguous().transpose(1, 2)  # stride(-1) != 1
    loss64, coef, steep, _ = _policy64(o, old.cpu(), adv.cpu(), None, 0.0)
    tol = (steep * o.tol_lp)[o.live].sum() + 2 * U * loss64.abs()
    for y in (view, turned, last, x):
        # a row that starts elsewhere in its 16 bytes is added up in another
        # order: each within the same distance of float64
        y = y.detach().requires_grad_(True)
        lp = token_logprobs(y, t).detach().cpu().double()
        assert bool(((lp - o.lp).abs() <= o.tol_lp + U * o.lp.abs()).all())
        a = fused_policy_loss(y, t, old, adv, clip_low=0.3, clip_high=0.4)
        b = fused_policy_loss(y, t, old, adv.expand(2, 9).clone(),
                              clip_low=0.3, clip_high=0.4)
        assert torch.equal(a, b)
        assert abs(float(a.detach()) - float(loss64)) <= float(tol)
        ga, = torch.autograd.grad(a, y)
        o.grad(coef, steep * o.tol_lp, torch.bfloat16, ga)
    assert torch.equal(token_logprobs(x[0], t[0]), want[0])
    assert torch.equal(token_logprobs(x[None], t[None]), want[None])
    assert torch.equal(
        token_logprobs(x[:, :-1], t[:, 1:].contiguous() * 0), token_logprobs(
            x, torch.zeros_like(t))[:, :-1])
    flat = fused_policy_loss(x.flatten(0, 1), t.flatten(), old.flatten(),
                             adv.expand(2, 9).flatten())
    # another split of the same float64 sum over the tokens
    assert abs(float(flat) - float(fused_policy_loss(x, t, old, adv))) \
        <= 4 * U * abs(float(flat)) + 1e-12


def test_gradients_against_differences():
    x, t = _inputs((4, 3, 11), torch.float32, "cpu", keep=1.0)
    x = x.double()
    o, old, adv, ref = _policy_inputs(x, t)
    old, adv, ref = old.double(), adv.double(), ref.double()
    for fn in (
        lambda y: fused_policy_loss(y, t, old, adv, ref, 0.3, 0.4, 0.2),
        lambda y: fused_preference_loss(y, t, ref, 0.3, 0.1)[0],
        lambda y: (token_logprobs(y, t) * adv).sum(),
    ):
        assert torch.autograd.gradcheck(fn, (x.requires_grad_(True),))


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    _skip(device)
    x = torch.zeros(2, 3, 5, device=device)
    t = torch.zeros(2, 3, dtype=torch.int64, device=device)
    v = torch.zeros(2, 3, device=device)
    cases = [
        lambda: token_logprobs(x, t.int()),
        lambda: token_logprobs(x, t[:, :2]),
        lambda: token_logprobs(x[0, 0], t[0, 0]),
        lambda: token_logprobs(x.long(), t),
        lambda: token_logprobs(x[..., :0], t),
        lambda: fused_policy_loss(x, t, v[:, :2], v),
        lambda: fused_policy_loss(x, t, v, v[0]),
        lambda: fused_policy_loss(x, t, v.long(), v),
        lambda: fused_policy_loss(x, t, v.clone().requires_grad_(True), v),
        lambda: fused_policy_loss(x, t, v, v, kl_coef=0.1),
        lambda: fused_policy_loss(x, t, v, v, v, kl_coef=-0.1),
        lambda: fused_policy_loss(x, t, v, v, clip_low=1.5),
        lambda: fused_policy_loss(x, t, v, v, clip_high=-0.1),
        lambda: fused_preference_loss(x[:1], t[:1], v[:1]),
        lambda: fused_preference_loss(x[0], t[0], v[0]),
        lambda: fused_preference_loss(x[:0], t[:0], v[:0]),
        lambda: fused_preference_loss(x, t, v, beta=0.0),
        lambda: fused_preference_loss(x, t, v, label_smoothing=0.6),
        lambda: fused_preference_loss(x, t, v[:, :2]),
    ]
    for call in cases:
        with pytest.raises(ValueError):
            call()


def _tangent_calls(x, t, v, dx):
    """The losses with a forward-mode tangent in each of their inputs."""
    return [
        lambda: token_logprobs(dx(x), t),
        lambda: fused_policy_loss(dx(x), t, v, v + 1),
        lambda: fused_policy_loss(x, t, dx(v), v + 1),
        lambda: fused_policy_loss(x, t, v, dx(v + 1)),
        lambda: fused_policy_loss(x, t, v, v, dx(v), kl_coef=0.1),
        lambda: fused_preference_loss(dx(x), t, v)[0],
        lambda: fused_preference_loss(x, t, dx(v))[0],
    ]


def test_forward_mode_on_the_cpu():
    x, t = _inputs((2, 3, 11), torch.float32, "cpu", keep=1.0)
    x, v = x.double(), torch.zeros(2, 3).double()
    with fwd.dual_level():
        for call in _tangent_calls(
                x, t, v, lambda y: fwd.make_dual(y, torch.ones_like(y))):
            assert fwd.unpack_dual(call()).tangent is not None
    for fn in (lambda y: token_logprobs(y, t),
               lambda y: fused_policy_loss(y, t, v - 3, v + 1),
               lambda y: fused_preference_loss(y, t, v)[0]):
        assert torch.autograd.gradcheck(
            fn, (x.clone().requires_grad_(True),), check_forward_ad=True)


@pytest.mark.parametrize("device", DEVICES)
def test_forward_mode_is_refused_by_the_kernels(device):
    """A tangent must not vanish; the extension sees it before the device."""
    _skip(device)
    if not ops.has_ext():
        pytest.skip("extension not built")
    ext = ops._require_ext()
    x = torch.zeros(2, 3, 5, device=device)
    t = torch.zeros(2, 3, dtype=torch.int64, device=device)
    v = torch.zeros(2, 3, device=device)
    with fwd.dual_level():
        def dx(y):
            return fwd.make_dual(y, torch.ones_like(y))

        calls = [
            lambda: ext.token_logprobs(dx(x), t, IGN),
            lambda: ext.policy_loss(dx(x), t, v, v, None, .2, .2, 0., IGN),
            lambda: ext.policy_loss(x, t, dx(v), v, None, .2, .2, 0., IGN),
            lambda: ext.policy_loss(x, t, v, dx(v), None, .2, .2, 0., IGN),
            lambda: ext.policy_loss(x, t, v, v, dx(v), .2, .2, .1, IGN),
            lambda: ext.preference_loss(dx(x), t, v, .1, 0., IGN),
            lambda: ext.preference_loss(x, t, dx(v), .1, 0., IGN),
        ]
        if device == "cuda":
            calls += _tangent_calls(x, t, v, dx)
        for grad in (False, True):
            x.requires_grad_(grad)
            for call in calls:
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    call()


@pytest.mark.gpu
def test_gpu_results_repeat_bit_for_bit():
    _skip("cuda")
    x, t = _inputs((4, 300, 5000), torch.bfloat16, "cuda", keep=1.0)
    o, old, adv, ref = _policy_inputs(x, t)
    old, adv, ref = old.cuda(), adv.cuda(), ref.cuda()
    first = None
    for _ in range(3):
        y = x.clone().requires_grad_(True)
        a = fused_policy_loss(y, t, old, adv, ref, kl_coef=0.1)
        b, r = fused_preference_loss(y, t, ref)
        g, = torch.autograd.grad(a + b, y)
        now = (a.detach(), b.detach(), r, g)
        first = first or now
        assert all(torch.equal(p, q) for p, q in zip(first, now))


@pytest.mark.gpu
def test_gpu_losses_replay_in_a_graph():
    _skip("cuda")
    x, t = _inputs((4, 70, 777), torch.bfloat16, "cuda", keep=1.0)
    o, old, adv, ref = _policy_inputs(x, t)
    old, adv, ref = old.cuda(), adv.cuda(), ref.cuda()
    logits = x.clone().requires_grad_(True)

    def step():
        a = fused_policy_loss(logits, t, old, adv, ref, kl_coef=0.1)
        b, r = fused_preference_loss(logits, t, ref)
        return (a.detach(), b.detach(), r,
                *torch.autograd.grad((a, b), logits))

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
            logits.copy_(x * (1 + 0.1 * i))
        graph.replay()
        torch.cuda.synchronize()
        got = [v.clone() for v in out]
        want = step()
        assert all(torch.equal(p, q) for p, q in zip(got, want)), i


@pytest.mark.gpu
def test_gpu_on_another_stream():
    _skip("cuda")
    x, t = _inputs((2, 40, 3001), torch.bfloat16, "cuda", keep=1.0)
    want = token_logprobs(x, t)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = x.clone().requires_grad_(True)
        lp = token_logprobs(y, t)
        g, = torch.autograd.grad(lp.sum(), y)
    side.synchronize()
    assert torch.equal(lp, want)
    z = x.clone().requires_grad_(True)
    gz, = torch.autograd.grad(token_logprobs(z, t).sum(), z)
    assert torch.equal(g, gz)


@pytest.mark.gpu
def test_gpu_second_derivative_is_refused():
    _skip("cuda")
    x, t = _inputs((2, 3, 50), torch.float32, "cuda", keep=1.0)
    x.requires_grad_(True)
    v = torch.zeros(2, 3, device="cuda")
    for loss in (token_logprobs(x, t).sum(),
                 fused_policy_loss(x, t, v, v + 1),
                 fused_preference_loss(x, t, v)[0]):
        g, = torch.autograd.grad(loss, x, create_graph=True)
        with pytest.raises(RuntimeError):
            g.square().sum().backward()


@pytest.mark.gpu
def test_gpu_logits_of_more_than_2_31_elements():
    _skip("cuda")
    rows, v = 18000, 128256
    x = torch.empty(1, rows, v, dtype=torch.bfloat16, device="cuda")
    x[0, 0].normal_(generator=torch.Generator("cuda").manual_seed(0))
    x[:, 1:] = 0
    x[0, -1] = x[0, 0]
    x.requires_grad_(True)
    t = torch.full((1, rows), IGN, device="cuda")
    t[0, 0] = t[0, -1] = 77
    t[0, 17000] = 5
    lp = token_logprobs(x, t)
    # equal rows at both ends, a uniform row past 2^31 elements
    assert float(lp[0, 0].detach()) == float(lp[0, -1].detach())
    assert abs(float(lp[0, 17000].detach()) + 11.761783) < 1e-5
    lp.sum().backward()
    assert torch.equal(x.grad[0, 0], x.grad[0, -1])
    assert abs(float(x.grad[0, 17000].float().sum())) < 1e-2
    assert bool((x.grad[0, 17000] != 0).all())
    assert bool((x.grad[0, 1:17000:997] == 0).all())


@pytest.mark.gpu
def test_gpu_capture_over_a_live_graph_of_the_same_leaf_is_refused():
    _skip("cuda")
    x, t = _inputs((2, 3, 50), torch.float32, "cuda", keep=1.0)
    x.requires_grad_(True)
    alive = token_logprobs(x, t)  # a graph of the default stream
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="drop that graph"):
            token_logprobs(x, t)
        with torch.no_grad():
            out = token_logprobs(x, t)
    graph.replay()
    assert torch.equal(out, alive.detach())
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, = torch.autograd.grad(token_logprobs(x, t).sum(), x)
    graph.replay()
    want, = torch.autograd.grad(token_logprobs(x, t).sum(), x)
    assert torch.equal(out, want)


@pytest.mark.gpu
def test_gpu_capture_over_a_live_graph_of_a_transposed_leaf_is_refused():
    """Logits that are copied first: the leaf is behind the copy."""
    _skip("cuda")
    x, t = _inputs((2, 3, 50), torch.float32, "cuda", keep=1.0)
    x = x.transpose(1, 2).contiguous().transpose(1, 2).requires_grad_(True)
    assert x.is_leaf and x.stride(-1) != 1
    v = torch.zeros(2, 3, device="cuda")
    alive = token_logprobs(x, t)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        for call in (lambda: token_logprobs(x, t),
                     lambda: fused_policy_loss(x, t, v, v),
                     lambda: fused_preference_loss(x, t, v)):
            with pytest.raises(RuntimeError, match="drop that graph"):
                call()
        with torch.no_grad():
            out = token_logprobs(x, t)
    graph.replay()
    assert torch.equal(out, alive.detach())


@pytest.mark.gpu
@pytest.mark.parametrize("v", [50257, 131072])
def test_gpu_logits_past_the_cached_size(v):
    """Large calls take other accesses and blocks: the same values."""
    _skip("cuda")
    b, s = 2, (140 << 20) // (4 * v) + 1  # bf16: over 128 MB
    gen = torch.Generator("cuda").manual_seed(0)
    x = torch.randn(b, s, v, device="cuda", dtype=torch.bfloat16,
                    generator=gen)
    t = torch.randint(0, v, (b, s), device="cuda", generator=gen)
    t[:, ::3] = IGN
    up = torch.randn(b, s, device="cuda", generator=gen)
    x.requires_grad_(True)
    lp = token_logprobs(x, t)
    g, = torch.autograd.grad(lp, x, up)
    for i in (0, 1, s // 2, s - 1):
        o = Oracle(x[:, i:i + 1], t[:, i:i + 1])
        off = (lp[:, i:i + 1].detach().cpu().double() - o.lp).abs()
        assert bool((off <= o.tol_lp + U * o.lp.abs()).all())
        c = up[:, i:i + 1].cpu().double()
        o.grad(c, torch.zeros_like(c), torch.bfloat16, g[:, i:i + 1])


@pytest.mark.gpu
def test_gpu_two_streams_at_once():
    _skip("cuda")
    sets = []
    for seed in (0, 1):
        x, t = _inputs((4, 90, 3000), torch.bfloat16, "cuda", seed, keep=1.0)
        o, old, adv, ref = _policy_inputs(x, t, seed)
        sets.append([v.cuda() for v in (x, t, old, adv, ref)])

    def step(x, t, old, adv, ref):
        y = x.clone().requires_grad_(True)
        a = fused_policy_loss(y, t, old, adv, ref, kl_coef=0.1)
        b, r = fused_preference_loss(y, t, ref)
        return (a.detach(), b.detach(), r,
                *torch.autograd.grad((a, b), y))

    want = [step(*s) for s in sets]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(10):
        got = []
        for st, s in zip(streams, sets):
            with torch.cuda.stream(st):
                got.append(step(*s))
        torch.cuda.synchronize()
        for w, g in zip(want, got):
            assert all(torch.equal(p, q) for p, q in zip(w, g))
