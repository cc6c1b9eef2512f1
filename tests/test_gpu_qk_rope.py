"""Norm and rotation of queries and keys, and their gradient, on the GPU against
float64: widths, partial rotation, positions far and outside the table, strides,
and a run through attention and back."""

from __future__ import annotations

import math

import pytest
import torch

import heads_reference as H

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _case(seed, B, N, Hq, Hkv, d, rot, dtype, weights="f32", rows=4096, positions=True):
    from tarmac.kernels import rotary_table
    g = torch.Generator().manual_seed(seed)
    dt = DTYPES[dtype]

    def normal(*s):
        return torch.randn(*s, generator=g).to("cuda", dt)

    q, k, dq, dk = normal(B, N, Hq, d), normal(B, N, Hkv, d), normal(B, N, Hq, d), normal(B, N, Hkv, d)
    wq, wk = (None if weights is None else
              (1 + 0.2 * torch.randn(d, generator=g)).to("cuda", DTYPES[weights]) for _ in range(2))
    table = rotary_table(rows, rot, device="cuda") if rot else None
    pos = torch.randint(0, rows, (B, N), generator=g).cuda() if rot and positions else None
    return q, k, dq, dk, wq, wk, table, pos


def _reference(q, k, dq, dk, wq, wk, table, pos, eps):
    res = {}
    for name, x, w, dz in (("q", q, wq, dq), ("k", k, wk, dk)):
        x64 = x.double().requires_grad_()
        w64 = None if w is None else w.double().requires_grad_()
        z = H.norm_rope(x64, w64, table, pos, eps)
        grads = torch.autograd.grad(z, (x64,) if w is None else (x64, w64), dz.double())
        res[name], res["d" + name] = z.detach(), grads[0]
        res["dw" + name] = None if w is None else grads[1]
    return res


def _run(q, k, dq, dk, wq, wk, table, pos, eps):
    from tarmac.kernels import qk_norm_rope, qk_norm_rope_backward
    got = dict(zip(("q", "k"), qk_norm_rope(q, k, wq, wk, table, pos, eps=eps)))
    got.update(zip(("dq", "dk", "dwq", "dwk"),
                   qk_norm_rope_backward(dq, dk, q, k, wq, wk, table, pos, eps=eps)))
    return got


def _check(got, want, dtype, d, terms):
    """An output is rounded once (r relative). Before that, fp32: the sum of
    squares (d terms), root, two products and a rotation, or the gradient's two
    sums of d terms: at most (2 d + 16) 2^-24 of the largest magnitude of its head
    (factors of at most about 4 between a value and what it is formed of). A
    weight's gradient: the same on each term, and ``terms`` additions."""
    e = (2 * d + 16) * 2.0 ** -24 * 4
    r = H.HALF_STEP[DTYPES[dtype]]
    for name, value in want.items():
        x = got[name]
        if value is None:
            assert x is None
            continue
        x = x.double()
        assert x.shape == value.shape
        if name.startswith("dw"):
            # a sum of terms of magnitude up to 5 x 5 that partly cancel
            assert float((x - value).abs().max()) <= (e + 2.0 ** -24 * math.sqrt(terms) * 8) * terms ** 0.5 * 8 + \
                2.0 ** -24 * float(value.abs().max()) * 8
            continue
        bound = r * value.abs() + e * value.abs().amax(-1, keepdim=True) + e
        bad = ~((x - value).abs() <= bound)
        assert not bad.any(), (name, int(bad.sum()), float(((x - value).abs() / bound).max()))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("d,rot", [(8, 8), (16, 16), (24, 24), (24, 8), (32, 16), (40, 40), (64, 64),
                                   (80, 40), (96, 96), (104, 56), (128, 128), (128, 8), (128, 0)])
def test_widths_and_partial_rotation(dtype, d, rot):
    t = _case(d + rot, 2, 19, 6, 2, d, rot, dtype)
    _check(_run(*t, 1e-6), _reference(*t, 1e-6), dtype, d, 2 * 19 * 6)


@pytest.mark.parametrize("B,N,Hq,Hkv", [(1, 1, 1, 1), (3, 1, 5, 2), (1, 700, 3, 3), (17, 33, 8, 1), (2, 5, 1, 7)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_sizes(dtype, B, N, Hq, Hkv):
    t = _case(B + N, B, N, Hq, Hkv, 64, 64, dtype)
    _check(_run(*t, 1e-5), _reference(*t, 1e-5), dtype, 64, B * N * max(Hq, Hkv))


@pytest.mark.parametrize("which", ["q", "k", "none"])
def test_one_weight_or_none(which):
    """Without its weight an input is rotated only, and has no weight gradient."""
    q, k, dq, dk, wq, wk, table, pos = _case(3, 2, 40, 4, 2, 64, 32, "bf16")
    wq = wq if which == "q" else None
    wk = wk if which == "k" else None
    t = (q, k, dq, dk, wq, wk, table, pos)
    _check(_run(*t, 1e-6), _reference(*t, 1e-6), "bf16", 64, 320)


def test_weights_of_the_heads_type_and_int32_positions():
    t = _case(4, 2, 40, 4, 2, 64, 64, "bf16", weights="bf16")
    want = _reference(*t, 1e-6)
    _check(_run(*t, 1e-6), want, "bf16", 64, 320)
    t = t[:7] + (t[7].int(),)
    _check(_run(*t, 1e-6), want, "bf16", 64, 320)


def test_positions_default_to_the_tokens_index():
    t = _case(5, 3, 50, 2, 2, 32, 32, "f32", positions=False)
    got, at = _run(*t, 1e-6), torch.arange(50, device="cuda").expand(3, 50).contiguous()
    want = _run(*t[:7], at, 1e-6)
    for name in got:
        assert torch.equal(got[name], want[name]), name
    _check(got, _reference(*t, 1e-6), "f32", 32, 300)


def test_far_positions():
    """The table's angles are formed in 64 bits: a rotation by position 10^6 is
    as exact as one by 10."""
    from tarmac.kernels import qk_norm_rope, rotary_table
    table = rotary_table(1_000_001, 16, device="cuda")
    x = torch.randn(1, 1, 1, 16, device="cuda")
    pos = torch.full((1, 1), 1_000_000, device="cuda")
    got, _ = qk_norm_rope(x, x, table=table, positions=pos)
    a = 1_000_000 * torch.pow(torch.tensor(10000.0, dtype=torch.float64), -torch.arange(8).double() / 8)
    y = x.cpu().double().flatten()
    want = torch.cat([y[:8] * a.cos() - y[8:] * a.sin(), y[8:] * a.cos() + y[:8] * a.sin()])
    # table entries rounded to fp32, three fp32 operations
    assert float((got.cpu().double().flatten() - want).abs().max()) <= 6 * 2.0 ** -24 * float(y.abs().max()) * 2


def test_positions_outside_the_table():
    """Never dereferenced: their rows are NaN, the others as they would be."""
    q, k, dq, dk, wq, wk, table, pos = _case(6, 2, 10, 2, 1, 32, 16, "bf16", rows=64)
    good = _run(q, k, dq, dk, wq, wk, table, pos, 1e-6)
    for bad in (-1, 64, 2 ** 31 - 1, -2 ** 31, 2 ** 40, -2 ** 62):
        p = pos.clone()
        p[1, 3] = bad
        got = _run(q, k, dq, dk, wq, wk, table, p, 1e-6)
        for name in ("q", "k", "dq", "dk"):
            assert torch.isnan(got[name][1, 3]).all(), (name, bad)
            same = torch.ones(2, 10, dtype=torch.bool)
            same[1, 3] = False
            assert torch.equal(got[name][same.cuda()], good[name][same.cuda()]), (name, bad)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_views_of_a_packed_projection(dtype):
    g = torch.Generator().manual_seed(2)
    packed = torch.randn(2, 30, 10, 48, generator=g).to("cuda", DTYPES[dtype])
    up = torch.randn(2, 6, 30, 48, generator=g).to("cuda", DTYPES[dtype]).transpose(1, 2)
    _, _, _, _, wq, wk, table, pos = _case(7, 2, 30, 6, 2, 48, 48, dtype)
    q, k = packed[:, :, :6], packed[:, :, 6:8]
    got = _run(q, k, up, up[:, :, 2:4], wq, wk, table, pos, 1e-6)
    want = _run(q.contiguous(), k.contiguous(), up.contiguous(), up[:, :, 2:4].contiguous(), wq, wk,
                table, pos, 1e-6)
    for name in got:
        assert torch.equal(got[name], want[name]), name


def test_zeros_and_empty():
    """A head of zeros has a norm of sqrt(eps) and no NaN; no tokens, no launch."""
    q, k, dq, dk, wq, wk, table, pos = _case(8, 2, 6, 2, 2, 16, 16, "f32")
    z = torch.zeros_like(q)
    t = (z, z, dq, dk, wq, wk, table, pos)
    got, want = _run(*t, 1e-6), _reference(*t, 1e-6)
    assert not got["q"].any() and not got["dwq"].any()
    # dx = w dy / sqrt(eps), dy a sum of two products of dz with cosine and sine: at most
    # 2 max |dz| max w 10^3 before anything cancels, and eight roundings on the way (eps as
    # fp32, root, quotient, the two products and their sum, the weight, the factor)
    off = float((got["dq"].double() - want["dq"]).abs().max())
    assert off <= 8 * 2.0 ** -24 * 2e3 * float(dq.abs().max()) * float(wq.abs().max())
    from tarmac.kernels import qk_norm_rope, qk_norm_rope_backward
    e = q[:, :0]
    assert qk_norm_rope(e, e, wq, wk, table)[0].shape == (2, 0, 2, 16)
    assert not qk_norm_rope_backward(e, e, e, e, wq, wk, table)[2].any()


def test_captured_and_replayed():
    t = _case(9, 2, 300, 8, 2, 64, 64, "bf16")
    want = _run(*t, 1e-6)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _run(*t, 1e-6)
    for rep in range(3):
        for x in got.values():
            x.fill_(math.nan)
        _run(*_case(20 + rep, 2, 300, 8, 2, 64, 64, "bf16"), 1e-6)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for name in want:
            assert torch.equal(got[name], want[name]), (rep, name)


def test_norm_rotation_attention_and_back():
    """The operators in a row as a layer uses them, in fp32, against float64
    autograd through the same composition: projection views -> norm and rotation
    -> causal attention with shared heads on a padded batch -> all gradients."""
    from tarmac.kernels import (multihead_attention, multihead_attention_backward, qk_norm_rope,
                                qk_norm_rope_backward)
    B, N, Hq, Hkv, d = 3, 75, 4, 2, 32
    q, k, _, _, wq, wk, table, pos = _case(10, B, N, Hq, Hkv, d, d, "f32")
    g = torch.Generator().manual_seed(11)
    v = torch.randn(B, N, Hkv, d, generator=g).cuda()
    dout = torch.randn(B, N, Hq, d, generator=g).cuda()
    n = torch.tensor([75, 1, 40], dtype=torch.int32, device="cuda")
    mask = {"causal": True, "lengths": n, "q_lengths": n}
    qr, kr = qk_norm_rope(q, k, wq, wk, table, pos)
    out, lse = multihead_attention(qr, kr, v, return_lse=True, **mask)
    dqr, dkr, dv = multihead_attention_backward(qr, kr, v, out, lse, dout, **mask)
    got = dict(zip(("dq", "dk", "dwq", "dwk"), qk_norm_rope_backward(dqr, dkr, q, k, wq, wk, table, pos)))
    got.update(out=out, dv=dv)

    leaves = [t.double().requires_grad_() for t in (q, k, v, wq, wk)]
    q64, k64, v64, wq64, wk64 = leaves
    ok = H.allowed(B, N, N, q.device, **mask)
    qh = H.norm_rope(q64, wq64, table, pos, 1e-6).transpose(1, 2)
    kh = H.norm_rope(k64, wk64, table, pos, 1e-6).transpose(1, 2).repeat_interleave(2, 1)
    s = (qh @ kh.transpose(2, 3) / math.sqrt(d)).masked_fill(~ok[:, None], -1e30)
    w = torch.softmax(s, -1) * ok[:, None]
    ref = (w @ v64.transpose(1, 2).repeat_interleave(2, 1)).transpose(1, 2)
    grads = torch.autograd.grad(ref, leaves, dout.double())
    want = dict(zip(("dq", "dk", "dv", "dwq", "dwk"), grads), out=ref.detach())
    for name, value in want.items():
        # fp32 throughout, some hundred operations a value whose roundings are independent
        rel = float((got[name].double() - value).norm() / value.norm())
        assert rel <= 5e-6, (name, rel)
