# -*- coding: utf-8 -*-
"""The fine-tuning operators together, as a step uses them: scoring, policy
and preference losses over a decoder with normalised heads, 8-bit SwiGLU
inputs and 8-bit checkpoints."""

import importlib.util
import os
import subprocess
import sys
from contextlib import nullcontext
from functools import partial

import pytest
import torch

from benchmarks.models import LlamaBlock, llama_tiny
from stoke import Stoke, StokeOptimizer
from stoke.nn import (
    apply_activation_checkpointing,
    fused_policy_loss,
    fused_preference_loss,
    qk_norm_rope,
    swiglu,
    token_logprobs,
)

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _skip(device):
    if device == "cuda" and not torch.cuda.is_available():
        pytest.skip("no GPU")


def _model(bits, device, dtype, ckpt=True):
    torch.manual_seed(0)
    m = llama_tiny(qk_norm=True, act_bits=bits).to(device=device, dtype=dtype)
    if ckpt:
        n = apply_activation_checkpointing(
            m, predicate=lambda _, x: isinstance(x, LlamaBlock),
            save_bits=bits)
        assert n == 2
    return m.train()


def _batch(device):
    g = torch.Generator().manual_seed(7)
    x = torch.randint(0, 1024, (4, 33), generator=g)
    y = x[:, 1:].clone()
    y[:, :5] = -100  # prompts
    y[2, 20:] = -100  # a padded answer
    return x[:, :-1].to(device), y.to(device)


def _step(m, x, y, amp=nullcontext):
    # a region for each forward, as the facade has it: autocast keeps its
    # weight casts until the region ends, and those made without gradient
    # must not serve a forward that needs one
    with torch.no_grad(), amp():
        old = token_logprobs(m(x), y)
    ref = old - 0.05
    adv = torch.tensor([[1.0], [-0.5], [0.3], [-1.0]], device=x.device)
    with amp():
        logits = m(x)
    a = fused_policy_loss(logits, y, old, adv, ref_logprobs=ref, kl_coef=0.1)
    b, rewards = fused_preference_loss(logits, y, ref, beta=0.2)
    params = dict(m.named_parameters())
    grads = torch.autograd.grad(a + b, list(params.values()))
    return a.detach(), b.detach(), rewards, dict(zip(params, grads))


def test_step_on_the_cpu():
    x, y = _batch("cpu")
    plain = _step(_model(16, "cpu", torch.float32, ckpt=False), x, y)
    ck16 = _step(_model(16, "cpu", torch.float32), x, y)
    held = _step(_model(8, "cpu", torch.float32), x, y)
    assert any("qk_norm.q_weight" in n for n in plain[3])
    # with the policy that sampled, rho is 1: loss = -mean(A over tokens)
    n = (y >= 0).sum(-1).double()
    adv = torch.tensor([1.0, -0.5, 0.3, -1.0]).double()
    kl = 0.1 * (torch.tensor(-0.05).double().exp() + 0.05 - 1)
    want = -(adv * n).sum() / n.sum() + kl
    for loss, pref, rewards, grads in (plain, ck16, held):
        # lp of the two passes agree to fp32; so does the ratio to 1
        assert abs(float(loss) - float(want)) < 1e-5
        assert torch.allclose(rewards.double(), 0.2 * 0.05 * n, atol=1e-4)
    for name, g in plain[3].items():
        assert torch.allclose(ck16[3][name], g, atol=1e-6, rtol=1e-4), name
        off = float((held[3][name] - g).norm() / g.norm())
        assert off < 0.1, (name, off)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 8])
def test_gpu_step_follows_the_cpu(bits):
    _skip("cuda")
    # fp32 runs the same kernels for norm, SwiGLU, checkpoints and losses;
    # only the products differ from the CPU's
    a = _step(_model(bits, "cpu", torch.float32), *_batch("cpu"))
    b = _step(_model(bits, "cuda", torch.float32), *_batch("cuda"))
    assert abs(float(a[0]) - float(b[0])) < 1e-4
    assert abs(float(a[1]) - float(b[1])) < 1e-4
    for name, g in a[3].items():
        off = float((b[3][name].cpu() - g).norm() / g.norm())
        # a value near the middle of two 8-bit steps may go to the other one
        assert off < (1e-3 if bits == 16 else 2e-2), (name, off)


@pytest.mark.gpu
def test_gpu_step_under_autocast_and_in_bf16():
    _skip("cuda")
    want = _step(_model(16, "cpu", torch.float32), *_batch("cpu"))
    x, y = _batch("cuda")
    m = _model(8, "cuda", torch.float32)
    auto = _step(m, x, y, lambda: torch.autocast("cuda", torch.bfloat16))
    half = _step(_model(8, "cuda", torch.bfloat16), x, y)
    for got in (auto, half):
        assert abs(float(got[0]) - float(want[0])) < 0.05
        for name, g in got[3].items():
            assert torch.isfinite(g).all(), name
            w = want[3][name]
            cos = torch.nn.functional.cosine_similarity(
                g.float().cpu().flatten(), w.flatten(), dim=0)
            assert float(cos) > 0.9, (name, float(cos))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("accum", [1, 2])
@pytest.mark.parametrize("kind", ["policy", "preference"])
def test_losses_under_the_facade(kind, accum, device):
    _skip(device)
    x, y = _batch(device)
    adv = torch.tensor([[1.0], [-0.5], [0.3], [-1.0]], device=device)
    m = _model(8, device, torch.float32)
    with torch.no_grad():
        old = token_logprobs(m(x), y)
    if kind == "policy":
        loss = partial(fused_policy_loss, kl_coef=0.1)
        args = (y, old, adv, old - 0.05)
    else:
        loss = partial(fused_preference_loss, beta=0.2, return_rewards=False)
        args = (y, old - 0.05)
    params = dict(m.named_parameters())
    want = {n: p.detach().clone() for n, p in params.items()}
    grads = torch.autograd.grad(loss(m(x), *args), list(params.values()))
    s = Stoke(
        model=_model(8, device, torch.float32),
        optimizer=StokeOptimizer(optimizer=torch.optim.SGD,
                                 optimizer_kwargs={"lr": 0.5}),
        loss=loss, batch_size_per_device=4, grad_accum_steps=accum,
        gpu=device == "cuda", verbose=False)
    s.model_access.train()
    for _ in range(accum):  # the same batch: the mean is its gradient
        value = s.loss(s.model(x), *args)
        assert value.dim() == 0
        s.backward(value)
        s.step()
    got = s.model_access.state_dict()
    for (n, p), g in zip(params.items(), grads):
        # halves of equal gradients add up to them, the step rounds once more;
        # the library may add a gradient's parts up in another order
        off = (got[n] - (want[n] - 0.5 * g)).abs()
        size = want[n].abs() + g.abs()
        assert bool((off <= 4 * 2.0 ** -24 * size + 1e-6 * g.abs().max()
                     ).all()), n
        assert bool((got[n] != want[n]).any()), n


def _operators(w):
    """Each operator on tensors made of the leaf w [4, 64]."""
    t = torch.zeros(4, dtype=torch.int64, device=w.device)
    v = torch.zeros(4, device=w.device)
    c = torch.ones(4, 8, device=w.device)

    def heads(y):
        q = y.view(1, 4, 4, 16)
        return qk_norm_rope(q, q, None, None, c, c)[0]

    return [
        lambda y: token_logprobs(y, t),
        lambda y: fused_policy_loss(y, t, v, v),
        lambda y: fused_preference_loss(y[:, None], t[:, None],
                                        v[:, None])[0],
        heads,
        lambda y: swiglu(y, y, save_bits=8),
    ]


@pytest.mark.gpu
def test_gpu_capture_over_a_live_graph_behind_other_operators():
    """The leaf is reached through what was computed in the capture, or the
    input itself was computed before it."""
    _skip("cuda")
    w = torch.randn(4, 64, device="cuda",
                    generator=torch.Generator("cuda").manual_seed(0))
    w.requires_grad_(True)
    alive = w * 2.0  # a graph of the default stream
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        inside = (w * 0.5).view(4, 64)
        for fn in _operators(w):
            for y in (inside, alive):
                with pytest.raises(RuntimeError, match="drop that graph"):
                    fn(y)
            with torch.no_grad():
                out = fn(inside)
            assert not out.requires_grad
    del alive, inside, y


@pytest.mark.gpu
def test_gpu_capture_over_a_live_graph_of_a_side_stream():
    """A warm-up whose result was kept: its stream takes no part in the
    capture."""
    _skip("cuda")
    w = torch.randn(4, 64, device="cuda",
                    generator=torch.Generator("cuda").manual_seed(0))
    w.requires_grad_(True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        alive = w * 2.0
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        inside = w * 0.5
        for fn in _operators(w):
            for y in (inside, alive):
                with pytest.raises(RuntimeError, match="drop that graph"):
                    fn(y)
        out = inside.detach() + 1
    graph.replay()
    assert torch.equal(out, w.detach() * 0.5 + 1)


@pytest.mark.gpu
def test_gpu_capture_behind_other_operators_and_over_a_fork():
    _skip("cuda")
    w = torch.randn(4, 64, device="cuda",
                    generator=torch.Generator("cuda").manual_seed(0))
    w.requires_grad_(True)

    def step():
        outs = [fn((w * 0.5).view(4, 64)) for fn in _operators(w)]
        return torch.autograd.grad(sum(o.sum() for o in outs), w)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(3):
        with torch.no_grad():
            w.mul_(1.25)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, step()), i
    # a stream that the capture has forked belongs to it
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        with torch.cuda.stream(side):
            inside = w * 0.5
        main.wait_stream(side)
        outs = [fn(inside) for fn in _operators(w)]
    assert all(o.requires_grad for o in outs)
    graph.replay()
    torch.cuda.synchronize()
    want = [fn(w.detach() * 0.5) for fn in _operators(w)]
    assert all(torch.equal(a, b) for a, b in zip(outs, want))


@pytest.mark.parametrize("device", DEVICES)
def test_example_runs(device):
    _skip(device)
    cmd = [sys.executable, os.path.join(REPO, "examples", "llm", "train.py"),
           "--layers", "2", "--dim", "256", "--steps", "2", "--batch", "4",
           "--act-ckpt", "--act-bits", "8", "--qk-norm"]
    if device == "cpu":
        cmd.append("--cpu")
    env = {k: v for k, v in os.environ.items() if k != "WORLD_SIZE"}
    r = subprocess.run(cmd, cwd=REPO, env=env, capture_output=True,
                       text=True, timeout=110)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-2000:]
    assert "done: 2 steps" in r.stdout


@pytest.mark.parametrize("flags,swiglu_bits", [
    ("--act-bits 8", 8), ("--act-bits 8 --act-ckpt", 16), ("--act-ckpt", 16),
    ("", 16)])
def test_example_holds_an_activation_once(flags, swiglu_bits):
    """SwiGLU inputs inside a recomputed block stay as they are."""
    spec = importlib.util.spec_from_file_location(
        "llm_train", os.path.join(REPO, "examples", "llm", "train.py"))
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    m = ex.build_model(ex.parse_args(
        ["--layers", "2", "--dim", "256", *flags.split()]))
    assert [b.act_bits for b in m.blocks] == [swiglu_bits] * 2
    held = [getattr(b, "_stoke_act_ckpt_bits", None) for b in m.blocks]
    bits = 8 if "8" in flags else 16
    assert held == ([bits] * 2 if "--act-ckpt" in flags else [None] * 2)
