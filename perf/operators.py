# -*- coding: utf-8 -*-
"""The fine-tuning operators of ``stoke.nn`` as measured calls.

Each case is one pass that a training or scoring program makes:

* ``qk``       -- per-head RMS norm of queries and keys with the rotary
                  rotation (forward only for decoding, with gradients for
                  training),
* ``logprobs`` -- log-probabilities of given tokens under logits,
* ``policy``   -- clipped policy loss with a KL term, and its gradient,
* ``prefer``   -- paired preference loss, and its gradient,
* ``act8``     -- an activation held in 8 bits (32 values share a power of
                  two) and brought back,
* ``swiglu8``  -- silu(gate) * up whose inputs wait for the backward in
                  8 bits.

``own`` picks the framework's calls; otherwise ``run`` computes the plain
form from elementary torch operations in 32 bits.
"""

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
_IGNORE = -100


# ------------------------------------------------------------------- cases
def listed():
    return [
        # one decoding step of 16 sequences far into their context; the
        # smallest call, heads as in the 8B decoder config
        dict(name="qk-decode", op="qk", b=16, s=1, hq=32, hk=8, d=128,
             rot=128, axes=1, table=32768, dtype="bf16", wtype="bf16",
             inter=False, grad=False),
        # training step of the 8B decoder's heads on image/video tokens:
        # time, height and width positions; q and k are views of one fused
        # projection; norm weights are fp32 masters as under autocast
        dict(name="qk-train-3axes", op="qk", b=4, s=4096, hq=32, hk=8, d=128,
             rot=128, axes=3, table=4096, dtype="bf16", wtype="fp32",
             inter=True, grad=True),
        # scoring the next token of 16 sequences: few rows, long vocabulary
        dict(name="logprobs-few", op="logprobs", b=16, s=1, v=128256,
             dtype="bf16", keep=1.0, grad=False),
        # a ragged batch with GPT-2's odd vocabulary in fp16 under a scaled
        # loss, with the gradient
        dict(name="logprobs-odd", op="logprobs", b=5, s=211, v=50257,
             dtype="fp16", keep=0.8, grad=True),
        # the CPU-test decoder's vocabulary in fp32
        dict(name="policy-tiny", op="policy", b=4, s=63, v=1024,
             dtype="fp32", keep=0.7, kl=0.05),
        # one policy step at the 8B vocabulary; prompts (40 %) are ignored
        dict(name="policy-large", op="policy", b=8, s=1024, v=128256,
             dtype="bf16", keep=0.6, kl=0.04),
        # two pairs of short ragged answers at GPT-2's odd vocabulary
        dict(name="prefer-odd", op="prefer", b=4, s=255, v=50257,
             dtype="bf16", keep=0.5, smooth=0.1),
        # four pairs at the 8B vocabulary
        dict(name="prefer-large", op="prefer", b=8, s=768, v=128256,
             dtype="bf16", keep=0.75, smooth=0.0),
        # the CPU-test decoder's block input
        dict(name="act8-tiny", op="act8", b=2, s=127, f=256, dtype="bf16"),
        # a block input of the 8B decoder, 32k tokens
        dict(name="act8-large", op="act8", b=8, s=4096, f=4096,
             dtype="bf16"),
        # an odd number of tokens of an odd width in fp16
        dict(name="swiglu8-odd", op="swiglu8", b=3, s=127, f=1367,
             dtype="fp16"),
        # the 8B decoder's MLP on 8k tokens
        dict(name="swiglu8-large", op="swiglu8", b=2, s=4096, f=14336,
             dtype="bf16"),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["qk", "logprobs", "policy", "prefer", "act8", "swiglu8"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    case = dict(op=op, dtype=dtype)
    if op == "qk":
        d = rng.choice([64, 80, 96, 128, 192, 256])
        hk = rng.choice([1, 2, 4, 8])
        hq = hk * rng.choice([1, 2, 4])
        grad = rng.random() < 0.6
        axes = rng.choice([1, 1, 2, 3])
        tokens = _spread(rng, 1, 32 * 1024 * 1024 // (d * (hq + hk)))
        b = min(tokens, _spread(rng, 1, 64))
        case.update(b=b, s=max(1, tokens // b), hq=hq, hk=hk, d=d,
                    rot=rng.choice([d, d, d // 2]), axes=axes,
                    table=_spread(rng, 256, 32768),
                    wtype=rng.choice([dtype, "fp32"]),
                    inter=rng.random() < 0.5, grad=grad)
    elif op in ("logprobs", "policy", "prefer"):
        v = rng.choice([1024, 32000, 50257, 50304, 128256,
                        _spread(rng, 1000, 200000)])
        most = (256 if dtype == "fp32" else 512) * 1024 * 1024 // v
        rows = _spread(rng, 4, min(most, 16384))
        b = 2 * rng.randint(1, 8)
        b = min(b, max(2, rows // 2 * 2))
        case.update(b=b, s=max(1, rows // b), v=v,
                    keep=rng.choice([1.0, 0.75, 0.5]))
        if op == "logprobs":
            case.update(grad=rng.random() < 0.5)
        elif op == "policy":
            case.update(kl=rng.choice([0.0, 0.04, 0.2]))
        else:
            case.update(smooth=rng.choice([0.0, 0.1]))
    else:
        f = rng.choice([256, 1024, 4096, 14336, _spread(rng, 1, 20000)])
        most = (16 if dtype == "fp32" else 64) * 1024 * 1024 // f
        rows = _spread(rng, 1, min(max(1, most), 32768))
        b = min(rows, rng.randint(1, 8))
        case.update(b=b, s=max(1, rows // b), f=f)
    return case


# ------------------------------------------------------------------ inputs
def _split(rot, axes):
    """Pairs of the rotation that each axis takes; the first takes the rest."""
    half = rot // 2
    each = half // axes
    return [half - each * (axes - 1)] + [each] * (axes - 1)


def _prepare_qk(c, gen):
    dev, dt = "cuda", _DTYPES[c["dtype"]]
    b, s, hq, hk, d = c["b"], c["s"], c["hq"], c["hk"], c["d"]
    # one fused projection: q, k and v are views of it with its row stride
    qkv = torch.randn(b, s, (hq + 2 * hk) * d, device=dev, generator=gen,
                      dtype=dt)
    # channels of real heads differ in size by an order of magnitude
    size = torch.exp(0.7 * torch.randn((hq + 2 * hk) * d, device=dev,
                                       generator=gen)).to(dt)
    qkv *= size
    q = qkv[..., : hq * d].view(b, s, hq, d)
    k = qkv[..., hq * d: (hq + hk) * d].view(b, s, hk, d)
    wt = _DTYPES[c["wtype"]]
    wq = (1 + 0.3 * torch.randn(d, device=dev, generator=gen)).to(wt)
    wk = (1 + 0.3 * torch.randn(d, device=dev, generator=gen)).to(wt)
    half = c["rot"] // 2
    inv = 500000.0 ** (-torch.arange(half, device=dev).double() / half)
    ang = torch.arange(c["table"], device=dev).double()[:, None] * inv
    pos = torch.randint(0, c["table"], (c["axes"], b, s), device=dev,
                        generator=gen)
    st = dict(q=q, k=k, wq=wq, wk=wk, cos=ang.cos().float(),
              sin=ang.sin().float(),
              pos=pos if c["axes"] > 1 else pos[0],
              sections=_split(c["rot"], c["axes"]) if c["axes"] > 1 else None)
    if c["grad"]:
        st["dq"] = torch.randn(b, s, hq, d, device=dev, generator=gen,
                               dtype=dt)
        st["dk"] = torch.randn(b, s, hk, d, device=dev, generator=gen,
                               dtype=dt)
        for n in ("q", "k", "wq", "wk"):
            st[n].requires_grad_(True)
    return st


def _prepare_logits(c, gen):
    dev, dt = "cuda", _DTYPES[c["dtype"]]
    b, s, v = c["b"], c["s"], c["v"]
    logits = torch.empty(b, s, v, device=dev, dtype=dt)
    logits.normal_(generator=gen)
    logits *= 2.5
    tgt = torch.randint(0, v, (b, s), device=dev, generator=gen)
    # a trained model gives the taken token a fair share
    up = 4 + 12 * torch.rand(b, s, 1, device=dev, generator=gen)
    at = tgt[..., None]
    logits.scatter_(-1, at, (logits.gather(-1, at).float() + up).to(dt))
    lp = torch.empty(b, s, device=dev, dtype=torch.float64)
    for i in range(b):
        x = logits[i].float()
        m = x.amax(-1, keepdim=True)
        z = (x - m).exp().sum(-1, dtype=torch.float64).log()
        lp[i] = (x.gather(-1, at[i]) - m)[:, 0].double() - z
    # a run of prompt tokens before, and padding behind, is ignored
    keep = torch.rand(b, 1, device=dev, generator=gen) * 0.4 + c["keep"] - 0.2
    first = torch.rand(b, 1, device=dev, generator=gen) * (1 - keep)
    where = (torch.arange(s, device=dev)[None] + 0.5) / s
    live = (where >= first) & (where < first + keep)
    if c["keep"] >= 1.0:
        live = torch.ones_like(live)
    tgt = torch.where(live, tgt, torch.full_like(tgt, _IGNORE))
    return logits, tgt, lp, live


def _prepare_losses(c, gen):
    dev = "cuda"
    logits, tgt, lp, live = _prepare_logits(c, gen)
    b, s = tgt.shape
    st = dict(logits=logits, targets=tgt)

    def noise(k):
        return k * torch.randn(b, s, device=dev, generator=gen,
                               dtype=torch.float64)

    # fp16 trains under a scaled loss, the others under 4 accumulated steps
    up = 1024.0 if c["dtype"] == "fp16" else 0.25
    if c["op"] == "logprobs":
        if c["grad"]:
            st["up"] = up * torch.randn(b, s, device=dev, generator=gen) / s
    else:
        st["up"] = torch.full((), up, device=dev)
    if c["op"] == "policy":
        shift = noise(0.15)
        # the clip has a step in its gradient at 0.8 and 1.2: no token sits
        # closer to it than the logits' own rounding moves it
        for edge in (math.log(0.8), math.log(1.2)):
            near = (shift - edge).abs() < 1e-3
            shift = torch.where(near, shift + 4e-3, shift)
        st.update(old=(lp - shift).float(),
                  adv=torch.randn(b, s, device=dev, generator=gen))
        st["ref"] = (lp + noise(0.3)).float() if c["kl"] > 0 else None
    if c["op"] == "prefer":
        st["ref"] = (lp + noise(0.2)).float()
    if st.get("up") is not None:
        logits.requires_grad_(True)
    return st


def _prepare_act8(c, gen):
    dev, dt = "cuda", _DTYPES[c["dtype"]]

    def act():
        x = torch.empty(c["b"], c["s"], c["f"], device=dev, dtype=dt)
        x.normal_(generator=gen)
        # a few channels are far larger than the others
        size = torch.exp(torch.randn(c["f"], device=dev, generator=gen))
        x *= size.to(dt)
        return x

    if c["op"] == "act8":
        return dict(x=act())
    st = dict(gate=act().requires_grad_(True), up=act().requires_grad_(True))
    st["dy"] = torch.empty_like(st["gate"]).normal_(generator=gen)
    return st


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    if case["op"] == "qk":
        st = _prepare_qk(case, gen)
    elif case["op"] in ("act8", "swiglu8"):
        st = _prepare_act8(case, gen)
    else:
        st = _prepare_losses(case, gen)
    st["case"] = case
    return st


# -------------------------------------------------------------- plain form
def _lookup(table, pos, sections):
    """Rows of a rotation table by position: [B, S, 1, pairs]."""
    if sections is None:
        return table[pos][:, :, None]
    parts = table.split(sections, -1)
    return torch.cat([p[i] for p, i in zip(parts, pos)], -1)[:, :, None]


def _turn(x, cos, sin, inter):
    half = cos.shape[-1]
    a, b = ((x[..., 0: 2 * half: 2], x[..., 1: 2 * half: 2]) if inter else
            (x[..., :half], x[..., half: 2 * half]))
    ra, rb = a * cos - b * sin, b * cos + a * sin
    r = torch.stack((ra, rb), -1).flatten(-2) if inter else torch.cat(
        (ra, rb), -1)
    return torch.cat((r, x[..., 2 * half:]), -1)


def _plain_qk(st):
    c = st["case"]
    cos = _lookup(st["cos"], st["pos"], st["sections"])
    sin = _lookup(st["sin"], st["pos"], st["sections"])

    def one(x, w, dy):
        xf, wf = x.detach().float(), w.detach().float()
        r = torch.rsqrt((xf * xf).mean(-1, keepdim=True) + 1e-6)
        y = _turn(xf * r * wf, cos, sin, c["inter"]).to(x.dtype)
        if dy is None:
            return y, None, None
        dn = _turn(dy.float(), cos, -sin, c["inter"])
        g = dn * wf
        dx = r * (g - xf * r * r * (g * xf).mean(-1, keepdim=True))
        dw = (dn * xf * r).sum((0, 1, 2))
        return y, dx.to(x.dtype), dw.to(w.dtype)

    yq, dq, dwq = one(st["q"], st["wq"], st.get("dq"))
    yk, dk, dwk = one(st["k"], st["wk"], st.get("dk"))
    if not c["grad"]:
        return dict(q=yq, k=yk)
    return dict(q=yq, k=yk, dq=dq, dk=dk, dwq=dwq, dwk=dwk)


def _plain_logprobs(logits, targets):
    """(lp, live, safe targets, shifted exponentials, their sums)."""
    x = logits.detach().float()
    live = targets != _IGNORE
    at = torch.where(live, targets, torch.zeros_like(targets))
    m = x.amax(-1, keepdim=True)
    picked = (x.gather(-1, at[..., None]) - m)[..., 0]
    e = (x - m).exp()
    z = e.sum(-1, dtype=torch.float64)
    # differences to old and reference values follow: 64 bits per token
    lp = torch.where(live, picked.double() - z.log(), 0.0)
    return lp, live, at, e, z.float()


def _plain_dlogits(coef, live, at, e, z, dtype):
    """coef * (onehot - softmax) of the live rows."""
    coef = torch.where(live, coef, 0.0).float()[..., None]
    d = e * (-coef / z[..., None])
    d.scatter_add_(-1, at[..., None], coef)
    return d.to(dtype)


def _plain_losses(st):
    c = st["case"]
    dt = st["logits"].dtype
    lp, live, at, e, z = _plain_logprobs(st["logits"], st["targets"])
    if c["op"] == "logprobs":
        if not c["grad"]:
            return lp.float()
        return dict(lp=lp.float(),
                    dlogits=_plain_dlogits(st["up"], live, at, e, z, dt))
    if c["op"] == "policy":
        n = live.sum().clamp_min(1)
        rho = (lp - st["old"]).exp()
        adv = st["adv"].double()
        free, held = rho * adv, rho.clamp(0.8, 1.2) * adv
        tok = -torch.minimum(free, held)
        coef = torch.where(free <= held, -free, 0.0)
        if st["ref"] is not None:
            gap = st["ref"].double() - lp
            tok = tok + c["kl"] * (gap.exp() - gap - 1)
            coef = coef + c["kl"] * (1 - gap.exp())
        loss = torch.where(live, tok, 0.0).sum() / n
        coef = coef * (st["up"] / n)
        return dict(loss=loss.float(),
                    dlogits=_plain_dlogits(coef, live, at, e, z, dt))
    half = lp.shape[0] // 2
    gain = 0.1 * torch.where(live, lp - st["ref"], 0.0).sum(-1)
    h = gain[:half] - gain[half:]
    soft = c["smooth"]
    # -log sigmoid(h) = max(-h, 0) + log(1 + exp(-|h|))
    tail = (1 + (-h.abs()).exp()).log()
    loss = ((1 - soft) * ((-h).clamp_min(0) + tail)
            + soft * (h.clamp_min(0) + tail)).mean()
    dh = (soft - (1 - soft) * (-h).exp()) / (1 + (-h).exp())
    dh = dh * (0.1 * st["up"] / half)
    coef = torch.cat((dh, -dh))[:, None].expand_as(lp)
    return dict(loss=loss.float(), rewards=gain.float(),
                dlogits=_plain_dlogits(coef, live, at, e, z, dt))


def _pow2(e):
    """2^e for int32 e from -126 to 127, put together from its bits."""
    return ((e + 127) << 23).view(torch.float32)


def _plain_hold(x):
    """(values the 8 bits stand for in fp32, exponent of each 32)."""
    flat = x.detach().float().reshape(-1)
    n = flat.numel()
    pad = torch.zeros((n + 31) // 32 * 32, device=x.device)
    pad[:n] = flat
    blk = pad.view(-1, 32)
    top = blk.abs().amax(-1, keepdim=True)
    # top = f * 2^e with f in [0.5, 1): 7 bits hold round(top * 2^(7-e))
    e = (torch.frexp(top).exponent - 7).clamp_min(-126)
    e = e + ((top * _pow2(-e)).round() > 127).to(e.dtype)
    e = torch.where(top > 0, e, torch.full_like(e, -126))
    held = (blk * _pow2(-e)).round() * _pow2(e)
    return held.view(-1)[:n].view(x.shape), (e + 127).view(-1).to(torch.uint8)


def _plain_act8(st):
    c = st["case"]
    if c["op"] == "act8":
        held, scale = _plain_hold(st["x"])
        return dict(x=held.to(st["x"].dtype), scale=scale)
    g, u, dt = st["gate"].detach().float(), st["up"].detach().float(), st[
        "gate"].dtype
    y = (g / (1 + (-g).exp()) * u).to(dt)
    g, u = _plain_hold(st["gate"])[0], _plain_hold(st["up"])[0]
    dy = st["dy"].float()
    sig = 1 / (1 + (-g).exp())
    dg = dy * u * sig * (1 + g * (1 - sig))
    return dict(y=y, dgate=dg.to(dt), dup=(dy * g * sig).to(dt))


# ------------------------------------------------------------------- calls
def _own(st):
    from stoke import nn

    c = st["case"]
    if c["op"] == "qk":
        q, k = nn.qk_norm_rope(
            st["q"], st["k"], st["wq"], st["wk"], st["cos"], st["sin"],
            positions=st["pos"], sections=st["sections"], eps=1e-6,
            interleaved=c["inter"])
        if not c["grad"]:
            return dict(q=q, k=k)
        dq, dk, dwq, dwk = torch.autograd.grad(
            (q, k), (st["q"], st["k"], st["wq"], st["wk"]),
            (st["dq"], st["dk"]))
        return dict(q=q, k=k, dq=dq, dk=dk, dwq=dwq, dwk=dwk)
    if c["op"] == "logprobs":
        lp = nn.token_logprobs(st["logits"], st["targets"])
        if not c["grad"]:
            return lp
        return dict(lp=lp, dlogits=torch.autograd.grad(
            lp, st["logits"], st["up"])[0])
    if c["op"] == "policy":
        loss = nn.fused_policy_loss(
            st["logits"], st["targets"], st["old"], st["adv"],
            ref_logprobs=st["ref"], clip_low=0.2, clip_high=0.2,
            kl_coef=c["kl"])
        return dict(loss=loss, dlogits=torch.autograd.grad(
            loss, st["logits"], st["up"])[0])
    if c["op"] == "prefer":
        loss, rewards = nn.fused_preference_loss(
            st["logits"], st["targets"], st["ref"], beta=0.1,
            label_smoothing=c["smooth"])
        return dict(loss=loss, rewards=rewards, dlogits=torch.autograd.grad(
            loss, st["logits"], st["up"])[0])
    if c["op"] == "act8":
        held = nn.compress_activation(st["x"])
        return dict(x=nn.restore_activation(held), scale=held.scales)
    y = nn.swiglu(st["gate"], st["up"], save_bits=8)
    dg, du = torch.autograd.grad(y, (st["gate"], st["up"]), st["dy"])
    return dict(y=y, dgate=dg, dup=du)


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "qk":
        return _plain_qk(state)
    if op in ("act8", "swiglu8"):
        return _plain_act8(state)
    return _plain_losses(state)


# -------------------------------------------------------------------- work
def work(case):
    c, n = case, case["b"] * case["s"]
    w = _BYTES[c["dtype"]]
    if c["op"] == "qk":
        x = n * (c["hq"] + c["hk"]) * c["d"]
        # positions, and the rows of cos and sin that the tokens use
        rows = min(n, c["table"]) * c["rot"] * 4 + n * c["axes"] * 8
        ends = 2 * c["d"] * _BYTES[c["wtype"]]
        if not c["grad"]:
            return dict(bytes=2 * x * w + rows + ends, flops=8 * x)
        return dict(bytes=5 * x * w + 2 * rows + 3 * ends, flops=28 * x)
    if c["op"] in ("logprobs", "policy", "prefer"):
        live = min(1.0, c["keep"])
        x = n * c["v"]
        per = n * {"logprobs": 12, "policy": 20, "prefer": 12}[c["op"]]
        if c["op"] == "logprobs" and not c["grad"]:
            return dict(bytes=int(live * x * w) + per, flops=int(live * 4 * x))
        # ignored rows are not read; their gradient is written all the same
        return dict(bytes=int((2 * live + 1) * x * w) + 2 * per,
                    flops=int(live * 8 * x))
    x = n * c["f"]
    held = x + (x + 31) // 32
    if c["op"] == "act8":
        return dict(bytes=2 * (x * w + held), flops=4 * x)
    # forward: gate, up -> y, held; backward: dy, held -> dgate, dup
    return dict(bytes=6 * x * w + 4 * held, flops=30 * x)


# ------------------------------------------------------------------- exact
def _exact_qk(st, c):
    f64 = torch.float64
    half = c["rot"] // 2
    sections = st["sections"] or [half]
    pos = st["pos"] if st["sections"] else st["pos"][None]
    axis = torch.repeat_interleave(
        torch.arange(len(sections), device=pos.device),
        torch.tensor(sections, device=pos.device))
    row = pos.permute(1, 2, 0)[..., axis]                  # [B, S, half]
    col = torch.arange(half, device=pos.device).expand_as(row)
    turn = torch.complex(st["cos"][row, col].double(),
                         st["sin"][row, col].double())[:, :, None]

    def one(x, w, dy):
        x = x.detach().to(f64).requires_grad_(True)
        w = w.detach().to(f64).requires_grad_(True)
        y = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w
        p = y[..., : 2 * half]
        p = (p.unflatten(-1, (half, 2)) if c["inter"] else
             p.unflatten(-1, (2, half)).transpose(-1, -2))
        z = torch.view_as_real(torch.view_as_complex(p.contiguous()) * turn)
        z = z.flatten(-2) if c["inter"] else z.transpose(-1, -2).flatten(-2)
        y = torch.cat((z, y[..., 2 * half:]), -1)
        if dy is None:
            return y.detach(), None, None
        dx, dw = torch.autograd.grad(y, (x, w), dy.to(f64))
        return y.detach(), dx, dw

    yq, dq, dwq = one(st["q"], st["wq"], st.get("dq"))
    yk, dk, dwk = one(st["k"], st["wk"], st.get("dk"))
    if not c["grad"]:
        return dict(q=yq, k=yk)
    return dict(q=yq, k=yk, dq=dq, dk=dk, dwq=dwq, dwk=dwk)


def _exact_losses(st, c):
    x = st["logits"].detach().double().requires_grad_(True)
    live = st["targets"].ne(_IGNORE)
    rows = torch.log_softmax(x, -1)
    lp = rows.gather(-1, st["targets"].clamp_min(0).unsqueeze(-1)).squeeze(-1)
    lp = lp.masked_fill(~live, 0.0)
    up = st.get("up")
    if c["op"] == "logprobs":
        if not c["grad"]:
            return lp.detach()
        d, = torch.autograd.grad(lp, x, up.double())
        return dict(lp=lp.detach(), dlogits=d)
    if c["op"] == "policy":
        a = st["adv"].double()
        ratio = torch.exp(lp - st["old"].double())
        tok = torch.max(-a * ratio, -a * torch.clip(ratio, 0.8, 1.2))
        if st["ref"] is not None:
            gap = st["ref"].double() - lp
            tok = tok + c["kl"] * (torch.expm1(gap) - gap)
        loss = tok[live].sum() / max(1, int(live.sum()))
        d, = torch.autograd.grad(loss, x, up.double())
        return dict(loss=loss.detach(), dlogits=d)
    gain = 0.1 * (lp - st["ref"].double().masked_fill(~live, 0.0)).sum(-1)
    good, bad = gain.chunk(2)
    h, s = good - bad, c["smooth"]
    ls = torch.nn.functional.logsigmoid
    loss = (-(1 - s) * ls(h) - s * ls(-h)).mean()
    d, = torch.autograd.grad(loss, x, up.double())
    return dict(loss=loss.detach(), rewards=gain.detach(), dlogits=d)


def _exact_hold(x):
    v = x.detach().double().flatten()
    n = v.numel()
    v = torch.nn.functional.pad(v, (0, -n % 32)).view(-1, 32)
    top = v.abs().max(-1, keepdim=True).values
    # the least exponent, from -126 up, at which 32 values fit into +-127
    e = torch.floor(torch.log2(top.clamp_min(2.0 ** -140))) - 6
    e = torch.where(torch.round(top / torch.exp2(e)) > 127, e + 1, e)
    e = e.clamp_min(-126)
    held = torch.round(v / torch.exp2(e)) * torch.exp2(e)
    return (held.flatten()[:n].view(x.shape),
            (e + 127).flatten().to(torch.uint8))


def _exact_act8(st, c):
    if c["op"] == "act8":
        held, scale = _exact_hold(st["x"])
        return dict(x=held, scale=scale)

    def f(g, u):
        return g * torch.sigmoid(g) * u

    y = f(st["gate"].detach().double(), st["up"].detach().double())
    g = _exact_hold(st["gate"])[0].requires_grad_(True)
    u = _exact_hold(st["up"])[0].requires_grad_(True)
    dg, du = torch.autograd.grad(f(g, u), (g, u), st["dy"].double())
    return dict(y=y, dgate=dg, dup=du)


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "qk":
        return _exact_qk(st, case)
    if case["op"] in ("act8", "swiglu8"):
        return _exact_act8(st, case)
    return _exact_losses(st, case)
