"""Attention over heads and its gradient on the GPU against float64, element by
element within bounds that follow from the arithmetic (oracle/heads_reference.py):
widths, lengths from one token on, shared key heads, masks that leave rows empty,
padded batches with anything behind their ends, strides, streams, graphs."""

from __future__ import annotations

import math

import pytest
import torch

import heads_reference as H

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
DTYPES = {"f32": F32, "bf16": BF16, "f16": F16}


def _inputs(seed, B, Nq, Nk, Hq, Hkv, d, dtype):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(*s, generator=g).to("cuda", dtype)
            for s in ((B, Nq, Hq, d), (B, Nk, Hkv, d), (B, Nk, Hkv, d), (B, Nq, Hq, d))]


def _i32(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _run(q, k, v, dout, **mask):
    from tarmac.kernels import multihead_attention, multihead_attention_backward
    out, lse = multihead_attention(q, k, v, return_lse=True, **mask)
    dq, dk, dv = multihead_attention_backward(q, k, v, out, lse, dout, **mask)
    return {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}


def _check(got, want, only=None):
    for name, (value, bound) in want.items():
        if only and name not in only:
            continue
        x = got[name].double()
        inf = torch.isinf(value)
        assert torch.equal(torch.isinf(x), inf), f"{name}: infinities"
        off = torch.where(inf, 0.0, x - value).abs()
        bad = ~(off <= bound)
        assert not bad.any(), (f"{name}: {int(bad.sum())} of {bad.numel()} outside their bound, "
                               f"worst {float((off / bound).max()):.3g} times, at "
                               f"{[int(t) for t in bad.nonzero()[0]]}")


def _against_float64(seed, B, Nq, Nk, Hq, Hkv, d, dtype, scale=None, **mask):
    q, k, v, dout = _inputs(seed, B, Nq, Nk, Hq, Hkv, d, DTYPES[dtype])
    ok = H.allowed(B, Nq, Nk, q.device, **mask)
    got = _run(q, k, v, dout, scale=scale, **mask)
    want = H.attention(q, k, v, ok, scale, dout)
    _check(got, want)
    # as a whole: roundings do not add up to their bounds. A weight's relative error is its
    # score's absolute one, so it grows with the scores' size: their root mean square is
    # scale sqrt(d) for N(0, 1) heads, 1 at the default scale
    size = max(1.0, scale * math.sqrt(d)) if scale else 1.0
    for name, (value, _) in want.items():
        fine = torch.isfinite(value)
        n = value[fine].norm()
        if name != "lse" and n > 0 and Nq >= 8 and Nk >= 8:
            rel = float((got[name].double() - value)[fine].norm() / n)
            assert rel <= size * {"f32": 2e-6, "bf16": 5e-3, "f16": 6e-4}[dtype], (name, rel)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("d", [8, 16, 24, 32, 40, 64, 72, 80, 96, 104, 128])
def test_widths(dtype, d):
    _against_float64(d, 2, 70, 70, 4, 2, d, dtype, causal=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("mask", ["causal", "exclude_self", "both", "all"])
@pytest.mark.parametrize("N", [1, 2, 31, 32, 33, 64, 65, 127, 129, 300])
def test_lengths_and_masks(dtype, mask, N):
    """Rows that the mask leaves empty: N = 1 without its own place, and the first
    row in causal order without its own place."""
    _against_float64(N, 2, N, N, 3, 1, 64, dtype, causal=mask in ("causal", "both"),
                     exclude_self=mask in ("exclude_self", "both"))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (5, 1), (8, 8), (12, 4), (16, 1), (40, 1), (6, 2)])
def test_shared_heads(dtype, Hq, Hkv):
    _against_float64(Hq, 2, 45, 45, Hq, Hkv, 32, dtype, exclude_self=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("Nq,Nk", [(1, 1), (1, 7), (1, 64), (1, 65), (3, 500), (4, 1000), (1, 4097),
                                   (200, 33), (65, 1)])
def test_queries_and_keys_of_other_numbers(dtype, Nq, Nk):
    _against_float64(Nq + Nk, 2, Nq, Nk, 8, 2, 128, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("Nq", [1, 2, 5])
def test_new_tokens_over_a_cache(dtype, Nq):
    """The last tokens of sequences of several lengths, one of them as short as
    the tokens themselves, one that fills the cache."""
    lengths = _i32(Nq, 700, 64, 63, 129)
    _against_float64(7, 5, Nq, 700, 16, 4, 64, dtype, causal=True, lengths=lengths,
                     q_start=lengths - Nq)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("mask", ["causal", "exclude_self", "all"])
def test_padded_batches(dtype, mask):
    """Lengths of nothing, of one, of all, and ends outside the tensor."""
    n = _i32(0, 1, 70, 33, 64, -5, 1000)
    _against_float64(3, 7, 70, 70, 4, 2, 64, dtype, causal=mask == "causal",
                     exclude_self=mask == "exclude_self", lengths=n, q_lengths=n)


@pytest.mark.parametrize("mask", ["causal", "exclude_self"])
def test_places_before_and_behind_the_keys(mask):
    """Queries that stand before the first key (in causal order they see
    nothing), among the keys, behind the last, and at the far ends of int32."""
    start = _i32(-100, -20, 5, 400, 2 ** 31 - 1, -2 ** 31)
    _against_float64(9, 6, 50, 90, 2, 2, 32, "bf16", causal=mask == "causal",
                     exclude_self=mask == "exclude_self", q_start=start)


@pytest.mark.parametrize("scale", [1e-3, 0.37, 2.0])
def test_scales(scale):
    _against_float64(11, 2, 100, 100, 2, 2, 64, "f32", scale=scale, causal=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_what_stands_behind_the_ends_is_not_read(dtype):
    """NaN and infinities in the keys, values, queries and gradients behind a
    sequence's end change no bit of any output."""
    B, N = 4, 100
    q, k, v, dout = _inputs(5, B, N, N, 4, 2, 64, DTYPES[dtype])
    n = _i32(0, 1, 37, 100)
    for mask in ({}, {"causal": True}, {"exclude_self": True}):
        want = _run(q, k, v, dout, lengths=n, q_lengths=n, **mask)
        behind = (torch.arange(N, device="cuda")[None] >= n[:, None])[..., None, None]
        for junk in (math.nan, math.inf, -math.inf):
            t = [torch.where(behind, torch.full_like(x, junk), x) for x in (q, k, v, dout)]
            got = _run(*t, lengths=n, q_lengths=n, **mask)
            for name in want:
                assert torch.equal(got[name], want[name]), (name, junk, mask)


def test_empty_rows_and_tensors():
    from tarmac.kernels import multihead_attention
    q, k, v, dout = _inputs(1, 2, 5, 5, 2, 1, 16, BF16)
    got = _run(q, k, v, dout, lengths=_i32(0, 0))
    assert not any(got[n].any() for n in ("out", "dq", "dk", "dv"))
    assert (got["lse"] == -math.inf).all()
    for shape in ((0, 5, 5), (2, 0, 5), (2, 5, 0)):
        B, Nq, Nk = shape
        t = _inputs(1, B, Nq, Nk, 2, 1, 16, BF16)
        got = _run(*t)
        assert got["out"].shape == (B, Nq, 2, 16) and not got["out"].any()
        assert not got["dk"].any() and not got["dv"].any() and not got["dq"].any()
        assert (got["lse"] == -math.inf).all()
    assert multihead_attention(q, k, v).shape == q.shape


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_large_scores(dtype):
    """Scores of hundreds: weights of one key only, and differences that
    underflow."""
    q, k, v, dout = _inputs(2, 2, 80, 80, 2, 2, 64, DTYPES[dtype])
    q, k = q * 8, k * 8
    got = _run(q, k, v, dout, causal=True)
    ok = H.allowed(2, 80, 80, q.device, causal=True)
    _check(got, H.attention(q, k, v, ok, None, dout))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_scores_that_grow_along_the_keys(dtype):
    """Each tile's scores exceed the last one's: the running maximum moves in
    every tile, in steps smaller and larger than its slack."""
    q, k, v, dout = _inputs(4, 1, 64, 640, 2, 2, 32, DTYPES[dtype])
    q = q.abs()
    for step in (0.002, 0.02):
        kk = (k * 0.1 + step * torch.arange(640, device="cuda")[None, :, None, None]).to(k.dtype)
        got = _run(q, kk, v, dout)
        ok = H.allowed(1, 64, 640, q.device)
        _check(got, H.attention(q, kk, v, ok, None, dout))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strides(dtype):
    """Views of a packed projection, of a cache's slice, transposed heads, one
    key head expanded to several, rows off 16 bytes: the same bits as copies."""
    dt = DTYPES[dtype]
    g = torch.Generator().manual_seed(1)
    B, N, d = 2, 50, 32
    packed = torch.randn(B, N, 4 + 2 * 2, d, generator=g).to("cuda", dt)
    dout = torch.randn(B, N, 4, d, generator=g).to("cuda", dt)
    cache = torch.randn(B, 2, 200, d, generator=g).to("cuda", dt)
    odd = torch.randn(B, N, 2, d + 1, generator=g).to("cuda", dt)
    one = torch.randn(B, N, 1, d, generator=g).to("cuda", dt)
    views = [(packed[:, :, :4], packed[:, :, 4:6], packed[:, :, 6:]),
             (packed[:, :, :4], cache[:, :, 60:110].transpose(1, 2), cache[:, :, :50].transpose(1, 2)),
             (packed[:, :, :4], odd[..., 1:], odd[..., :d]),
             (packed[:, :, :4], one.expand(B, N, 2, d), one.expand(B, N, 4, d)[:, :, ::2])]
    for q, k, v in views:
        do = dout.transpose(1, 2).contiguous().transpose(1, 2)
        got = _run(q, k, v, do, causal=True)
        want = _run(q.contiguous(), k.contiguous(), v.contiguous(), dout, causal=True)
        for name in want:
            assert torch.equal(got[name], want[name]), name


def test_the_same_bits_on_every_call():
    t = _inputs(6, 3, 333, 333, 8, 2, 64, BF16)
    first = _run(*t, causal=True)
    for _ in range(3):
        again = _run(*t, causal=True)
        for name in first:
            assert torch.equal(first[name], again[name]), name


@pytest.mark.parametrize("shape", [(3, 200, 200, 4, 2, 64), (2, 1, 3000, 16, 2, 128)])
def test_captured_and_replayed(shape):
    """Two calls in one graph, replayed between eager work on other inputs."""
    mask = {"lengths": _i32(*([shape[2], shape[2] // 2, 5][:shape[0]]))}
    a = _inputs(1, *shape, BF16)
    b = _inputs(2, *shape, BF16)
    want = [_run(*t, **mask) for t in (a, b)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [_run(*t, **mask) for t in (a, b)]
    for rep in range(3):
        for g in got:
            for t in g.values():
                t.fill_(math.nan)
        _run(*_inputs(3 + rep, *shape, BF16), **mask)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            for name in w:
                assert torch.equal(g[name], w[name]), (rep, name)


def test_two_streams():
    a, b = _inputs(1, 2, 500, 500, 4, 2, 64, BF16), _inputs(2, 4, 1, 2000, 16, 2, 64, BF16)
    want = _run(*a, causal=True), _run(*b)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for n, (s, t, m) in enumerate(zip(streams, (a, b), ({"causal": True}, {}))):
            with torch.cuda.stream(s):
                got[n].append(_run(*t, **m))
    torch.cuda.synchronize()
    for n in range(2):
        for g in got[n]:
            for name in want[n]:
                assert torch.equal(g[name], want[n][name]), name


def test_gradients_against_differences():
    """dq, dk, dv along random directions against central differences of the
    kernel's own forward in fp32: with a loss of about 10^2 and steps of 2^-7 the
    differences carry about 2^-24 10^2 2^7 / 2 = 4e-4 of rounding and 2^-14 of a
    third derivative of order one."""
    from tarmac.kernels import multihead_attention
    q, k, v, dout = _inputs(8, 1, 40, 40, 2, 1, 16, F32)
    got = _run(q, k, v, dout, causal=True)
    h = 2.0 ** -7

    def loss(*t):
        return float((multihead_attention(*t, causal=True).double() * dout.double()).sum())

    g = torch.Generator().manual_seed(3)
    for n, name in enumerate(("dq", "dk", "dv")):
        t = [q, k, v]
        step = torch.randn(t[n].shape, generator=g).to("cuda")
        step = step / step.norm()
        up, down = list(t), list(t)
        up[n], down[n] = t[n] + h * step, t[n] - h * step
        slope = (loss(*up) - loss(*down)) / (2 * h)
        along = float((got[name].double() * step.double()).sum())
        assert abs(slope - along) <= 2e-3 * max(1.0, abs(along)), (name, slope, along)
