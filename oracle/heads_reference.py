"""Attention over heads, the norm and rotation before it, and their gradients in
float64 torch operations, with bounds of what fp32 kernels with 16-bit operands
may be off by. No code of the framework is used.

Bounds. u is half a rounding step of the heads' type (0 for fp32, whose
operands are not rounded), e what fp32 arithmetic costs a weight, relative:

* a score is a sum of d products: off by at most d 2^-23 sum |q||k| (the matrix
  instructions cut at the accumulator's last place, 2^-23 relative), and its
  exponent adds 2^-22 of its magnitude and of the maximum's; a weight and the
  sum of weights each carry that once, hence the factor 2; the sum of N terms
  adds N 2^-23;
* out = sum w v: weights rounded (u), the result rounded (u);
* D = dO . out with the rounded out; dS = P (dP - D) rounded (u); each gradient
  rounded (u);
* below the smallest normal value, 2^-14 in float16, a rounding is off by up to
  half a subnormal step, 2^-25, however small the value (2^-134 in bfloat16 and
  2^-150 in fp32 are covered by the 1e-30 of every bound). Each weight and each dS
  that a product takes adds that times the other factor, each float16 result once
  more: with a single query over 120 keys, dS of 2^-17 is rounded at 2^-8 of
  itself and dk is that one product. The forward divides its weights by their sum
  after the rounding, and that sum is 1 at least.
"""

from __future__ import annotations

import math

import torch

HALF_STEP = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}
SMALLEST = {torch.float32: 1e-30, torch.bfloat16: 1e-30, torch.float16: 2.0 ** -25}


def allowed(B, Nq, Nk, device, causal=False, exclude_self=False, lengths=None, q_lengths=None,
            q_start=None):
    """[B, Nq, Nk] truth values: the pairs that count."""
    i = torch.arange(Nq, device=device).view(1, Nq, 1)
    j = torch.arange(Nk, device=device).view(1, 1, Nk)
    place = i + (0 if q_start is None else q_start.long().view(B, 1, 1))
    ok = torch.ones(B, Nq, Nk, dtype=torch.bool, device=device)
    if causal:
        ok = ok & (j <= place)
    if exclude_self:
        ok = ok & (j != place)
    if lengths is not None:
        ok = ok & (j < lengths.view(B, 1, 1))
    if q_lengths is not None:
        ok = ok & (i < q_lengths.view(B, 1, 1))
    return ok


def attention(q, k, v, ok, scale=None, dout=None):
    """{name: (value, bound)} of out, lse and, given dout, dq, dk, dv. What
    stands in rows that no pair uses may be anything: it is zeroed first."""
    dtype = q.dtype
    B, Nq, Hq, d = q.shape
    Nk, Hkv = k.shape[1], k.shape[2]
    G = Hq // Hkv
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    rows, keys = ok.any(2)[:, :, None, None], ok.any(1)[:, :, None, None]

    def heads(t, used):  # [B, N, H, d] -> [B, H, N, d], float64
        return torch.where(used, t.double(), 0.0).permute(0, 2, 1, 3)

    qh = heads(q, rows)
    kh, vh = (heads(t, keys).repeat_interleave(G, 1) for t in (k, v))
    ok = ok[:, None]
    s = qh @ kh.transpose(2, 3) * scale
    mag = (qh.abs() @ kh.abs().transpose(2, 3) * scale)
    some = ok.any(3, keepdim=True)
    s = s.masked_fill(~ok, -math.inf)
    m = torch.where(some, s.amax(3, keepdim=True), 0.0)
    p = torch.exp(s - m)
    total = p.sum(3, keepdim=True)
    w = torch.where(some, p / total.clamp_min(1e-300), 0.0)
    lse = torch.where(some, total.clamp_min(1e-300).log() + m, -math.inf)
    out = w @ vh

    u = 0.0 if dtype == torch.float32 else HALF_STEP[dtype]
    r = HALF_STEP[dtype]  # the rounding of a result
    tiny = SMALLEST[dtype]  # of a weight, of dS or of a result below the normal values
    near = ok.double() * tiny
    worst = torch.where(ok, mag, 0.0).amax(3, keepdim=True)
    e_s = d * 2.0 ** -23 * worst + 2.0 ** -22 * (worst + 1)
    e = 2 * e_s + Nk * 2.0 ** -23 + 2.0 ** -20
    A = w @ vh.abs()
    b_out = (u + e) * A * (1 + u) + near @ vh.abs() + r * out.abs() + tiny
    res = {"out": (out.permute(0, 2, 1, 3), b_out.permute(0, 2, 1, 3)),
           "lse": (lse.squeeze(3), (2 * e_s + Nk * 2.0 ** -23 + 2.0 ** -20
                                    + 2.0 ** -22 * lse.abs().nan_to_num(posinf=0)).squeeze(3))}
    if dout is None:
        return res
    do = heads(dout, rows)
    dv = w.transpose(2, 3) @ do
    dp = do @ vh.transpose(2, 3)
    dp_mag = do.abs() @ vh.abs().transpose(2, 3)
    D = (do * out).sum(3, keepdim=True)
    D_mag = (do.abs() * out.abs()).sum(3, keepdim=True)
    b_D = (do.abs() * b_out).sum(3, keepdim=True) + d * 2.0 ** -23 * D_mag
    ds = w * (dp - D)
    b_ds = (u * ds.abs() + w * b_D * (1 + u)
            + (e * (dp - D).abs() + d * 2.0 ** -23 * (dp_mag + D_mag)) * w * (1 + u)) + near
    b_w = (u + e) * w + near

    def over_group(t):  # the shared key heads' sums
        return t.view(B, Hkv, G, Nk, d).sum(2).permute(0, 2, 1, 3)

    sums = (Nq * G + Nk) * 2.0 ** -23  # accumulating a gradient in fp32
    dq = ds @ kh * scale
    b_dq = (b_ds + sums * ds.abs()) @ kh.abs() * scale + r * dq.abs() + tiny
    dk, dv = over_group(ds.transpose(2, 3) @ qh) * scale, over_group(dv)
    b_dk = over_group((b_ds + sums * ds.abs()).transpose(2, 3) @ qh.abs()) * scale
    b_dv = over_group((b_w + sums * w).transpose(2, 3) @ do.abs())
    res["dq"] = (dq.permute(0, 2, 1, 3), b_dq.permute(0, 2, 1, 3))
    res["dk"] = (dk, b_dk + r * dk.abs() + tiny)
    res["dv"] = (dv, b_dv + r * dv.abs() + tiny)
    return res


def before_the_difference(q, k, v, ok, scale, dout):
    """Norms of the gradients of q and k with P dP in place of dS = P dP - P D: what
    the roundings of the two terms are relative to. In a row with one key the
    terms are equal, dS and with it dq are zero, and all that is left of
    either is its rounding."""
    B, Nq, Hq, d = q.shape
    G = Hq // k.shape[2]
    rows, keys = ok.any(2)[:, :, None, None], ok.any(1)[:, :, None, None]
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    qh, do = (torch.where(rows, t.double(), 0.0).permute(0, 2, 1, 3) for t in (q, dout))
    kh, vh = (torch.where(keys, t.double(), 0.0).permute(0, 2, 1, 3).repeat_interleave(G, 1) for t in (k, v))
    s = (qh @ kh.transpose(2, 3) * scale).masked_fill(~ok[:, None], -math.inf)
    w = torch.where(rows.permute(0, 2, 1, 3), s.softmax(3), 0.0) * (do @ vh.transpose(2, 3))
    dk = (w.transpose(2, 3) @ qh).view(B, -1, G, k.shape[1], d).sum(2)
    return {"dq": float((w @ kh).norm()) * scale, "dk": float(dk.norm()) * scale}


def norm_rope(x, w, table, positions, eps):
    """One of queries and keys in float64 (differentiable): x [B, N, H, d]."""
    y = x.double()
    if w is not None:
        y = y / (y.pow(2).mean(-1, keepdim=True) + eps).sqrt() * w.double()
    if table is None:
        return y
    B, N = x.shape[:2]
    at = torch.arange(N, device=x.device).expand(B, N) if positions is None else positions.long()
    t = table.double()[at].unsqueeze(2)
    h = table.shape[1] // 2
    co, si = t[..., :h], t[..., h:]
    lo, hi = y[..., :h], y[..., h:2 * h]
    return torch.cat([lo * co - hi * si, hi * co + lo * si, y[..., 2 * h:]], -1)
