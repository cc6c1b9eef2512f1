"""``AttentionComm`` with ``attn_mode="multihead"``: messages and every gradient
against the same composition in float64 autograd, ragged teams, types, and what
it refuses."""

from __future__ import annotations

import math

import pytest
import torch
import torch.nn.functional as F

import heads_reference as H


def _module(n_agents=12, msg_dim=64, **more):
    from tarmac.agents import AttentionComm, MAPPOConfig
    torch.manual_seed(5)
    return AttentionComm(MAPPOConfig(obs_dim=18, n_actions=5, n_agents=n_agents, use_comm=True,
                                     msg_dim=msg_dim, attn_mode="multihead", **more), 32)


def _composed(m, x, lengths):
    """The module in float64: (messages, leaves by name)."""
    cfg = m.cfg
    p = {n: t.detach().double().requires_grad_() for n, t in m.named_parameters() if "k_gate" not in n}
    p["x"] = x.detach().double().requires_grad_()
    B, N, _ = x.shape
    h, g = cfg.n_heads, cfg.n_kv_heads or cfg.n_heads
    qkv = (p["x"] @ p["qkv.weight"].T + p["qkv.bias"]).view(B, N, h + 2 * g, -1)
    q, k, v = qkv.split([h, g, g], 2)
    table = None if m._rotary is None else m._rotary.to(x.device)
    q, k = (H.norm_rope(t, p.get(n), table, None, 1e-6) for t, n in ((q, "q_norm"), (k, "k_norm")))
    k, v = (t.repeat_interleave(h // g, 2).transpose(1, 2) for t in (k, v))
    s = q.transpose(1, 2) @ k.transpose(2, 3) / math.sqrt(q.shape[-1])
    ok = H.allowed(B, N, N, x.device, exclude_self=True, lengths=lengths, q_lengths=lengths)[:, None]
    w = torch.softmax(s.masked_fill(~ok, -1e30), -1) * ok
    msg = (w @ v).transpose(1, 2).reshape(B, N, cfg.msg_dim)
    return F.gelu(msg) @ p["proj.weight"].T + p["proj.bias"], p


@pytest.mark.gpu
@pytest.mark.parametrize("more", [dict(n_heads=4), dict(n_heads=8, n_kv_heads=2),
                                  dict(n_heads=4, qk_norm=True), dict(n_heads=2, n_kv_heads=1, rotary=True),
                                  dict(n_heads=4, n_kv_heads=2, qk_norm=True, rotary=True)])
@pytest.mark.parametrize("ragged", [False, True])
def test_messages_and_gradients(more, ragged):
    m = _module(**more).cuda()
    with torch.no_grad():
        for n, t in m.named_parameters():
            if n.endswith("_norm"):
                t += 0.1 * torch.randn_like(t)
    m.collect_info = False
    x = torch.randn(5, 12, 32, device="cuda", requires_grad=True)
    lengths = torch.tensor([12, 1, 0, 7, 2], dtype=torch.int32, device="cuda") if ragged else None
    dout = torch.randn(5, 12, 64, device="cuda")
    msg, info = m(x, lengths=lengths)
    assert not info
    names = [n for n, _ in m.named_parameters() if "k_gate" not in n]
    got = dict(zip(["x", *names], torch.autograd.grad(msg, [x, *(m.get_parameter(n) for n in names)], dout)))
    want, leaves = _composed(m, x, lengths)
    grads = dict(zip(leaves, torch.autograd.grad(want, list(leaves.values()), dout.double())))
    # fp32 throughout: some hundred roundings a value, independent of each other
    for name, value in [("msg", want.detach()), *grads.items()]:
        mine = (msg if name == "msg" else got[name]).detach()
        rel = float((mine.double() - value).norm() / value.norm())
        assert rel <= 5e-6, (name, rel)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,tol", [(torch.bfloat16, 3e-2), (torch.float16, 4e-3)])
def test_half_precision(dtype, tol):
    """In half precision each stage rounds (projections, norm and rotation, weights,
    messages, gelu): about ten roundings of half a step each, 2^-8 and 2^-11."""
    m = _module(n_heads=4, n_kv_heads=2, qk_norm=True, rotary=True).cuda().to(dtype)
    m.collect_info = False
    x = torch.randn(4, 12, 32, device="cuda").to(dtype)
    msg, _ = m(x)
    assert msg.dtype == dtype
    want, _ = _composed(m, x, None)
    assert float(((msg.double() - want).norm() / want.norm()).detach()) <= tol
    msg.float().square().mean().backward()
    assert m.q_norm.grad.dtype == dtype and torch.isfinite(m.qkv.weight.grad).all()


@pytest.mark.gpu
def test_inference_is_the_training_forward_and_info():
    m = _module(n_heads=4, qk_norm=True, rotary=True).cuda()
    x = torch.randn(3, 12, 32, device="cuda")
    n = torch.tensor([12, 5, 1], dtype=torch.int32, device="cuda")
    with torch.no_grad():
        a, info = m(x, lengths=n)
    b, _ = m(x.requires_grad_(), lengths=n)
    assert torch.equal(a, b.detach())
    assert 0.0 < info["mean_attn_entropy"] <= math.log(11) + 1e-6
    # what stands in a padded team's other rows changes nothing of the team's
    y = x.detach().clone()
    y[1, 5:] = 7.0
    with torch.no_grad():
        c, _ = m(y, lengths=n)
    assert torch.equal(a[1, :5], c[1, :5]) and torch.equal(a[0], c[0])


def test_refusals_and_shapes():
    for more in (dict(n_heads=0), dict(n_heads=3), dict(n_heads=16), dict(n_heads=4, n_kv_heads=3)):
        with pytest.raises(ValueError):
            _module(**more)
    with pytest.raises(ValueError, match="up to 128"):
        _module(msg_dim=512, n_heads=2)
    m = _module(n_heads=4)
    assert m.qkv.weight.shape == (192, 32) and m.q_norm is None and m._rotary is None
    assert set(m.state_dict()) == {f"{a}.{b}" for a in ("qkv", "proj", "k_gate") for b in ("weight", "bias")}
    assert _module(n_heads=8, n_kv_heads=2).qkv.weight.shape == (64 + 2 * 16, 32)
    from tarmac.agents import AttentionComm, MAPPOConfig
    dense = AttentionComm(MAPPOConfig(obs_dim=18, n_actions=5, n_agents=6), 32)
    with pytest.raises(ValueError, match="lengths"):
        dense(torch.zeros(2, 6, 32), lengths=torch.tensor([6, 6], dtype=torch.int32))


@pytest.mark.gpu
def test_second_derivatives_are_refused():
    m = _module(n_heads=4, qk_norm=True).cuda()
    m.collect_info = False
    x = torch.randn(2, 12, 32, device="cuda", requires_grad=True)
    g, = torch.autograd.grad(m(x)[0].square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()


@pytest.mark.gpu
def test_gradients_captured_and_replayed():
    """Norm, rotation, attention and the way back through autograd in one graph,
    captured while no eager graph of the same tensors lives, replayed on other
    values between eager work."""
    from tarmac.agents.mappo import _HeadsCore, _NormRope
    from tarmac.kernels import rotary_table
    table = rotary_table(40, 16, device="cuda")
    n = torch.tensor([40, 17, 0], dtype=torch.int32, device="cuda")
    leaves = [torch.randn(3, 40, h, 16, device="cuda").requires_grad_() for h in (4, 2, 2)]
    leaves += [torch.rand(16, device="cuda").add_(0.5).requires_grad_() for _ in "qk"]
    dout = torch.randn(3, 40, 4, 16, device="cuda")

    def step():
        q, k, v, wq, wk = leaves
        q, k = _NormRope.apply(q, k, wq, wk, table)
        out = _HeadsCore.apply(q, k, v, n)
        return [out.detach(), *torch.autograd.grad(out, leaves, dout)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(3):
        with torch.no_grad():
            for t in (*leaves, dout):
                t.copy_(torch.randn_like(t))
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
