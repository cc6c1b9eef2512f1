"""Attention over several heads, and its gradient, as HIP kernels.

The reference's attention core has one head (``src/agents/mappo.py:31-86``
carries ``n_heads``, which nothing reads); these are the same function for
``[B, N, H, d]`` tensors, with what teams and sequences of several lengths need:
key heads shared by groups of query heads, causal order or the self pair left
out, padded batches, and one new token (or a few) over a cache.

Query ``i`` of batch row ``b`` stands at place ``q_start[b] + i`` among the keys
(``q_start`` None: ``i``) and attends to key ``j`` if

* ``j < lengths[b]`` and ``i < q_lengths[b]`` (None: all of them),
* ``causal``: ``j`` is not behind the query's place,
* ``exclude_self``: ``j`` is not the query's place.

A query that nothing is left to has a message of zeros, a logsumexp of -inf and
no gradient. Keys behind ``lengths`` and queries behind ``q_lengths`` are not
read, so a cache may hold anything there; in other masked places values have to
be finite.

``d`` is a multiple of 8 up to 128; float32 heads run on fp32 matrix
instructions, bfloat16 and float16 heads on those of their type, with statistics
and sums in fp32. Tensors may be views of any strides (a packed projection, a
cache's slice) as long as rows start on 16 bytes; others are copied.
"""

from __future__ import annotations

import math
import struct

import torch

from .. import _launch, _lib

#: struct tarmac_mha of include/tarmac.h.
_CALL = struct.Struct("@q" + 8 * "Pqqq" + "PPqPPP" + "9if")


def _sizes(q, k, v, causal, exclude_self, scale, lengths, q_lengths, q_start):
    """Checks every argument but the device; (sizes, scale)."""
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t.dim() != 4:
            raise ValueError(f"{name}: expected a [B, N, H, d] tensor, got shape {tuple(t.shape)}")
    B, Nq, Hq, d = q.shape
    Nk, Hkv = k.shape[1], k.shape[2]
    code = _launch.heads_dtype_code(q.dtype)
    _launch.check_heads("k", k, q, (B, Nk, Hkv, d))
    _launch.check_heads("v", v, q, (B, Nk, Hkv, d))
    if Hkv < 1 or Hq < 1 or Hq % Hkv:
        raise ValueError(f"the key heads must divide the query heads, got {Hkv} and {Hq}")
    if d < 8 or d > 128 or d % 8:
        raise NotImplementedError(f"head width must be a multiple of 8 up to 128, got {d}")
    if (causal or exclude_self) and q_start is None and Nq != Nk:
        raise ValueError(f"{Nq} queries over {Nk} keys: causal and exclude_self need q_start")
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    if not 0.0 < scale < math.inf:
        raise ValueError(f"scale must be positive and finite, got {scale}")
    _launch.check_per_row("lengths", lengths, q, B)
    _launch.check_per_row("q_lengths", q_lengths, q, B)
    _launch.check_per_row("q_start", q_start, q, B)
    return (B, Nq, Nk, Hq, Hkv, d, code, int(causal), int(exclude_self)), scale


def _per_row(lengths, q_lengths, q_start):
    return tuple(0 if t is None else t.data_ptr() for t in (lengths, q_lengths, q_start))


def multihead_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *,
                        causal: bool = False, exclude_self: bool = False,
                        scale: float | None = None,
                        lengths: torch.Tensor | None = None,
                        q_lengths: torch.Tensor | None = None,
                        q_start: torch.Tensor | None = None,
                        return_lse: bool = False):
    """``softmax(scale q k^T) v`` per head over the allowed keys (see the
    module's text). q ``[B, Nq, Hq, d]``; k, v ``[B, Nk, Hkv, d]``, Hkv dividing
    Hq; ``scale`` defaults to 1/sqrt(d); ``lengths``, ``q_lengths`` and
    ``q_start`` are int32 ``[B]`` on the device. Returns the messages
    ``[B, Nq, Hq, d]``, with ``return_lse`` also the logsumexp of the scaled
    scores, fp32 ``[B, Hq, Nq]``, which the backward takes."""
    sizes, scale = _sizes(q, k, v, causal, exclude_self, scale, lengths, q_lengths, q_start)
    _launch.on_gpu(q)
    B, Nq, Nk, Hq, Hkv, d = sizes[:6]
    out = torch.empty(B, Nq, Hq, d, device=q.device, dtype=q.dtype)
    lse = torch.empty(B, Hq, Nq, device=q.device, dtype=torch.float32)
    if B == 0 or Nq == 0 or Nk == 0:  # nothing to launch: no keys, no message
        out.zero_()
        lse.fill_(-math.inf)
        return (out, lse) if return_lse else out
    (q, fq), (k, fk), (v, fv), (_, fo) = map(_launch.heads, (q, k, v, out))
    rows = _per_row(lengths, q_lengths, q_start)
    none = 4 * _launch.NO_HEADS

    def call(ws, nbytes):
        return _CALL.pack(_CALL.size, *fq, *fk, *fv, *fo, *none, lse.data_ptr(), ws, nbytes,
                          *rows, *sizes, scale)

    with _launch.on_device_of(q):
        packed = call(0, 0)
        need = _lib.LIB.tarmac_mha_fwd_workspace(packed)
        if need:
            if need < 0:
                _lib.check(_lib.TARMAC_ERR_INVALID)
            ws = torch.empty(need, device=q.device, dtype=torch.uint8)
            packed = call(ws.data_ptr(), need)
        _lib.check(_lib.LIB.tarmac_mha_fwd(packed, _launch.stream(q)))
    return (out, lse) if return_lse else out


def multihead_attention_backward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                                 out: torch.Tensor, lse: torch.Tensor, dout: torch.Tensor, *,
                                 causal: bool = False, exclude_self: bool = False,
                                 scale: float | None = None,
                                 lengths: torch.Tensor | None = None,
                                 q_lengths: torch.Tensor | None = None,
                                 q_start: torch.Tensor | None = None):
    """Gradients (dq, dk, dv) of :func:`multihead_attention` called with the
    same arguments, given its ``out`` and ``lse`` and the messages' gradient
    ``dout``. The probabilities are formed again from ``lse``; a shared key
    head's gradient is summed over its query heads in a fixed order."""
    sizes, scale = _sizes(q, k, v, causal, exclude_self, scale, lengths, q_lengths, q_start)
    B, Nq, Nk, Hq, Hkv, d = sizes[:6]
    _launch.check_heads("out", out, q, (B, Nq, Hq, d))
    _launch.check_heads("dout", dout, q, (B, Nq, Hq, d))
    if lse.shape != (B, Hq, Nq) or lse.dtype != torch.float32 or not lse.is_contiguous():
        raise ValueError(f"lse must be the contiguous fp32 [{B}, {Hq}, {Nq}] tensor of the forward")
    if lse.device != q.device:
        raise ValueError(f"lse is on {lse.device}, expected {q.device}")
    _launch.on_gpu(q)
    dq = torch.empty(B, Nq, Hq, d, device=q.device, dtype=q.dtype)
    dk, dv = (torch.empty(B, Nk, Hkv, d, device=q.device, dtype=q.dtype) for _ in range(2))
    if B == 0 or Nq == 0 or Nk == 0:
        return dq.zero_(), dk.zero_(), dv.zero_()
    tensors, fields = zip(*map(_launch.heads, (q, k, v, out, dout, dq, dk, dv)))
    with _launch.on_device_of(q):
        need = 8 * B * Hq * Nq
        ws = torch.empty(need, device=q.device, dtype=torch.uint8)
        packed = _CALL.pack(_CALL.size, *(x for f in fields for x in f), lse.data_ptr(),
                            ws.data_ptr(), need, *_per_row(lengths, q_lengths, q_start),
                            *sizes, scale)
        _lib.check(_lib.LIB.tarmac_mha_bwd(packed, _launch.stream(q)))
    del tensors  # copies made for alignment live until the launch
    return dq, dk, dv
