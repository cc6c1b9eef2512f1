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
    # dS = P dP - P D rounds each of its terms, so the gradients' errors are relative to the
    # terms: rows of one key, where they are equal, have errors and no gradient
    terms = H.before_the_difference(q, k, v, ok, scale, dout)
    for name, (value, _) in want.items():
        fine = torch.isfinite(value)
        n = max(float(value[fine].norm()), terms.get(name, 0.0))
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


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("d", [16, 40, 64, 96, 128])
@pytest.mark.parametrize("mask", ["all", "causal", "exclude_self", "both"])
def test_many_workgroups(dtype, d, mask):
    """Enough rows for workgroups of 128 of them in every pass; a group of two
    queries a key head, a last tile of two rows, keys that end inside a tile."""
    _against_float64(d, 64, 129, 129, 8, 4, d, dtype, causal=mask in ("causal", "both"),
                     exclude_self=mask in ("exclude_self", "both"))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("mask", ["all", "causal", "exclude_self"])
@pytest.mark.parametrize("Hq,Hkv", [(4, 4), (12, 4)])
def test_many_workgroups_of_padded_batches(dtype, mask, Hq, Hkv):
    """Every number of keys and of queries from none to all, among them rows whose
    keys end before their tile begins, and places that the queries start from."""
    B, N = 70, 140
    n = torch.arange(B, device="cuda", dtype=torch.int32) * 2 % (N + 3)
    m = torch.arange(B, device="cuda", dtype=torch.int32) * 37 % (N + 1)
    start = torch.arange(B, device="cuda", dtype=torch.int32) * 11 % 90 - 30
    _against_float64(Hq, B, N, N, Hq, Hkv, 64, dtype, causal=mask == "causal",
                     exclude_self=mask == "exclude_self", lengths=n, q_lengths=m, q_start=start)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_many_workgroups_leave_what_stands_behind_the_ends(dtype):
    B, N = 64, 135
    q, k, v, dout = _inputs(5, B, N, N, 8, 4, 64, DTYPES[dtype])
    n = torch.arange(B, device="cuda", dtype=torch.int32) * 3 % (N + 1)
    behind = (torch.arange(N, device="cuda")[None] >= n[:, None])[..., None, None]
    for mask in ({}, {"causal": True}):
        want = _run(q, k, v, dout, lengths=n, q_lengths=n, **mask)
        for junk in (math.nan, math.inf):
            t = [torch.where(behind, torch.full_like(x, junk), x) for x in (q, k, v, dout)]
            got = _run(*t, lengths=n, q_lengths=n, **mask)
            for name in want:
                assert torch.equal(got[name], want[name]), (name, junk, mask)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_four_waves_a_tile(dtype):
    """As many tiles of 32 rows as leave four waves to each."""
    _against_float64(3, 64, 45, 45, 8, 4, 64, dtype, causal=True)
    _against_float64(4, 100, 37, 70, 4, 4, 128, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("Nq,Nk,mask", [(1100, 1100, "causal"), (1100, 1100, "all"), (40, 2500, "all"),
                                        (2500, 40, "all"), (1030, 1030, "exclude_self")])
def test_long_sequences_of_few_heads(dtype, d, Nq, Nk, mask):
    """The streamed side in parts, forward and backward, with parts that a causal
    tile has nothing in."""
    _against_float64(Nq + d, 1, Nq, Nk, 4, 2, d, dtype, causal=mask == "causal",
                     exclude_self=mask == "exclude_self")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("causal", [False, True])
def test_long_sequences_of_several_lengths(dtype, causal):
    """Parts behind a row's end, and rows that end in the first part."""
    B, N = 5, 2100
    n, m = _i32(2100, 0, 1, 300, 1025), _i32(2100, 7, 2100, 300, 1)
    _against_float64(1, B, N, N, 2, 1, 64, dtype, causal=causal, lengths=n, q_lengths=m)
    _against_float64(2, B, 6, N, 8, 1, 64, dtype, causal=causal, lengths=n,
                     q_start=(n - 6).contiguous())


def test_a_cache_longer_than_32_bits_of_offsets():
    """Two heads of a cache of 128, the second batch row: places of 2.2 10^9
    elements and more, beyond 2^32 bytes. The same bits as from copies."""
    from tarmac.kernels import multihead_attention
    B, N, H, d = 2, 140_000, 128, 64
    g = torch.Generator().manual_seed(1)
    q, dout = (torch.randn(B, 3, 8, d, generator=g).to("cuda", BF16) for _ in "qd")
    cache = torch.zeros(B, N, H, d, dtype=BF16, device="cuda")
    some = torch.randn(2, B, N, 2, d, device="cuda").to(BF16)
    cache[:, :, 120:122], cache[:, :, 126:] = some[0], some[1]
    k, v = cache[:, :, 120:122], cache[:, :, 126:]
    n = _i32(N, N - 5)
    mask = dict(causal=True, lengths=n, q_start=n - 3)
    got = _run(q, k, v, dout, **mask)
    want = _run(q, some[0], some[1], dout, **mask)
    for name in want:
        assert torch.equal(got[name], want[name]), name
    # the last token alone sees only itself where the lengths leave one key
    one = multihead_attention(q[:, :1], k[:, N - 1:], v[:, N - 1:])
    assert torch.equal(one, v[:, N - 1:].repeat_interleave(4, 2))


def test_rows_far_apart():
    """Rows of 32 MiB and more apart are copied, ones just below are not."""
    d = 8
    for step in ((1 << 24) - 8, 1 << 24):
        base = torch.randn(3 * step + d, device="cuda").to(BF16)
        k = base.as_strided((1, 4, 1, d), (0, step, 0, 1))
        q, _, _, dout = _inputs(1, 1, 5, 4, 2, 1, d, BF16)
        got = _run(q, k, k, dout)
        want = _run(q, k.contiguous(), k.contiguous(), dout)
        for name in want:
            assert torch.equal(got[name], want[name]), (name, step)


def test_tensors_of_another_device():
    from tarmac.kernels import multihead_attention, multihead_attention_backward
    q, k, v, dout = _inputs(1, 2, 5, 5, 2, 1, 16, BF16)
    with pytest.raises(ValueError, match="k is on cpu"):
        multihead_attention(q, k.cpu(), v)
    with pytest.raises(ValueError, match="lengths is on cpu"):
        multihead_attention(q, k, v, lengths=_i32(5, 5).cpu())
    out, lse = multihead_attention(q, k, v, return_lse=True)
    with pytest.raises(ValueError, match="lse is on cpu"):
        multihead_attention_backward(q, k, v, out, lse.cpu(), dout)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_many_workgroups_captured_and_replayed(dtype):
    """The passes of 128 rows and the parts' joins in one graph."""
    calls = [_inputs(1, 64, 130, 130, 8, 4, 64, DTYPES[dtype]), _inputs(2, 1, 1200, 1200, 2, 1, 64, DTYPES[dtype])]
    want = [_run(*t, causal=True) for t in calls]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [_run(*t, causal=True) for t in calls]
    for rep in range(3):
        for g in got:
            for t in g.values():
                t.fill_(math.nan)
        _run(*_inputs(3 + rep, 4, 700, 700, 4, 2, 64, DTYPES[dtype]))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            for name in w:
                assert torch.equal(g[name], w[name]), (rep, name)


@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("f16", 72), ("f32", 128), ("f32", 40), ("bf16", 64)])
@pytest.mark.parametrize("mask", ["all", "causal", "exclude_self"])
def test_workgroups_of_many_rows_in_parts(dtype, d, mask):
    """Long sequences of few heads by 128 rows, the streamed side in parts: 17
    tiles, the last of one row; keys that end inside a part, and rows that end
    before it."""
    n = _i32(2049, 1500, 600, 0)
    _against_float64(d, 4, 2049, 2049, 4, 4, d, dtype, causal=mask == "causal", exclude_self=mask == "exclude_self",
                     lengths=n, q_lengths=_i32(2049, 130, 1999, 64))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("B,Nq,Nk,Hq,Hkv", [(8, 17, 4100, 32, 4), (3, 200, 3000, 8, 4), (2, 1200, 2100, 6, 3)])
def test_several_new_tokens_over_a_long_cache(dtype, B, Nq, Nk, Hq, Hkv):
    """A prompt's piece: enough rows for the wide tiles, over caches of several
    lengths, NaN behind them."""
    n = torch.arange(B, device="cuda", dtype=torch.int32) * 700 % (Nk - Nq) + Nq
    q, k, v, dout = _inputs(B, B, Nq, Nk, Hq, Hkv, 128, DTYPES[dtype])
    behind = (torch.arange(Nk, device="cuda")[None] >= n[:, None])[..., None, None]
    k, v = (t.masked_fill(behind, math.nan) for t in (k, v))
    mask = dict(causal=True, lengths=n, q_start=n - Nq)
    got = _run(q, k, v, dout, **mask)
    _check(got, H.attention(q, k, v, H.allowed(B, Nq, Nk, q.device, **mask), None, dout))


def test_parts_captured_and_replayed():
    """Three calls in parts in one graph: their workspaces are apart."""
    calls = [_inputs(n, 2, 2048, 2048, 4, 2, 128, BF16) for n in range(2)] + [_inputs(3, 1, 2100, 2100, 4, 4, 128, F32)]
    want = [_run(*t, causal=True) for t in calls]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [_run(*t, causal=True) for t in calls]
    for rep in range(3):
        for g in got:
            for t in g.values():
                t.fill_(math.nan)
        _run(*_inputs(5 + rep, 1, 2048, 2048, 4, 4, 128, BF16))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            for name in w:
                assert torch.equal(g[name], w[name]), (rep, name)


def test_rows_far_apart_in_a_whole_tile():
    """70 rows just below 32 MiB apart: offsets of a tile's last rows near 2^31."""
    d, step = 8, (1 << 24) - 8
    base = torch.zeros(70 * step + d, dtype=BF16, device="cuda")
    k = base.as_strided((1, 70, 1, d), (0, step, 0, 1))
    k.copy_(torch.randn(1, 70, 1, d, device="cuda"))
    q, _, _, dout = _inputs(1, 1, 40, 70, 2, 1, d, BF16)
    got = _run(q, k, k, dout)
    want = _run(q, k.contiguous(), k.contiguous(), dout)
    for name in want:
        assert torch.equal(got[name], want[name]), name


@pytest.mark.parametrize("dtype,d", [("bf16", 16), ("bf16", 32), ("f16", 64), ("f32", 8), ("f32", 32), ("bf16", 72)])
@pytest.mark.parametrize("Nk", [512, 700, 1023, 1024, 5000])
def test_eight_waves_over_a_cache(dtype, d, Nk):
    """A token of each of three caches, one with a key or two a wave, one with none
    for most waves: the waves' sums added in a workgroup, and over its parts."""
    n = _i32(Nk, 9, Nk // 2 + 1)
    _against_float64(d, 3, 1, Nk, 4, 2, d, dtype, causal=True, lengths=n, q_start=n - 1)
    _against_float64(d, 1, 40, Nk, 4, 2, d, dtype)


@pytest.mark.parametrize("dtype,d", [("bf16", 64), ("f16", 32), ("f32", 64), ("f32", 128), ("bf16", 128)])
@pytest.mark.parametrize("causal", [False, True])
def test_one_half_of_the_gradient_wide(dtype, d, causal):
    """Many rows of queries and few of keys, and the other way round: the halves of
    the gradient divide the work differently, in launches of their own."""
    _against_float64(d, 64, 100, 100, 8, 4, d, dtype, causal=causal)
    start = torch.arange(64, device="cuda", dtype=torch.int32) * 5
    _against_float64(d, 64, 5, 300, 4, 4, d, dtype, causal=causal, q_start=start,
                     lengths=torch.minimum(start + 7, torch.tensor(300, dtype=torch.int32, device="cuda")))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("mask", ["all", "causal", "exclude_self"])
def test_gradients_of_rows_of_few_keys(dtype, mask):
    """At most 1.6 times as far off, as a whole, as the exact gradient rounded once:
    its rounding, that of dS (each of half a step, a root of two together) and O's in D,
    which a row of few keys feels most, are 1.5 times it; a row of up to 128 keys has
    the second made up for."""
    for B, N in ((64, 20), (8, 128), (2, 700)):
        q, k, v, dout = _inputs(N, B, N, N, 4, 2, 64, DTYPES[dtype])
        m = dict(causal=mask == "causal", exclude_self=mask == "exclude_self")
        got = _run(q, k, v, dout, **m)
        want = H.attention(q, k, v, H.allowed(B, N, N, q.device, **m), None, dout)
        for name in ("dq", "dk", "dv"):
            value = want[name][0]
            once = (value.to(q.dtype).double() - value).norm()
            assert float((got[name].double() - value).norm() / once) <= 1.6, (name, N)
