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
be finite, as their scores.

``d`` is a multiple of 8 up to 128. Statistics and sums are fp32. bfloat16 and
float16 heads run on the matrix instructions of their type, with the weights and
the scores' gradients rounded to it; float32 heads on bfloat16 ones, each value
as three parts, to fp32's accuracy. Tensors may be views of any strides (a packed
projection, a cache's slice) as long as rows start on 16 bytes and are less than
32 MiB apart; others are copied. The functions record no autograd graph;
``AttentionComm`` with ``attn_mode="multihead"`` trains through them.
"""

from __future__ import annotations

import functools
import math
import struct

import torch

from .. import _launch, _lib

#: struct tarmac_mha of include/tarmac.h.
_CALL = struct.Struct("@q" + 8 * "Pqqq" + "PPqPPP" + "9if")
_NONE = 4 * _launch.NO_HEADS


def _sizes(q, k, v, causal, exclude_self, scale, lengths, q_lengths, q_start):
    """Checks every argument but that the device is a GPU: (sizes, scale, the
    addresses of the three arrays)."""
    if not q.dim() == k.dim() == v.dim() == 4:
        raise ValueError("expected [B, N, H, d] tensors, got shapes "
                         f"{tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    B, Nq, Hq, d = q.shape
    _, Nk, Hkv, _ = shape = k.shape
    code = _launch.heads_dtype_code(q.dtype)
    if shape[0] != B or shape[3] != d:
        raise ValueError(f"k: expected shape {(B, Nk, Hkv, d)}, got {tuple(shape)}")
    _launch.check_heads("k", k, q, shape)
    _launch.check_heads("v", v, q, shape)
    if Hkv < 1 or Hq < 1 or Hq % Hkv:
        raise ValueError(f"the key heads must divide the query heads, got {Hkv} and {Hq}")
    if d < 8 or d > 128 or d % 8:
        raise NotImplementedError(f"head width must be a multiple of 8 up to 128, got {d}")
    if Nq != Nk and (causal or exclude_self) and q_start is None:
        raise ValueError(f"{Nq} queries over {Nk} keys: causal and exclude_self need q_start")
    scale = d ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale < math.inf:
        raise ValueError(f"scale must be positive and finite, got {scale}")
    per_row = (_launch.per_row("lengths", lengths, q, B),
               _launch.per_row("q_lengths", q_lengths, q, B),
               _launch.per_row("q_start", q_start, q, B))
    return (B, Nq, Nk, Hq, Hkv, d, code, int(causal), int(exclude_self)), scale, per_row


@functools.lru_cache(maxsize=1024)
def _workspace(backward, sizes):
    """Bytes of workspace a call of these sizes takes."""
    fn = _lib.LIB.tarmac_mha_bwd_workspace if backward else _lib.LIB.tarmac_mha_fwd_workspace
    need = fn(_CALL.pack(_CALL.size, *_NONE, *_NONE, 0, 0, 0, 0, 0, 0, *sizes, 1.0))
    if need < 0:
        _lib.check(_lib.TARMAC_ERR_UNSUPPORTED)
    return need


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
    sizes, scale, per_row = _sizes(q, k, v, causal, exclude_self, scale, lengths, q_lengths,
                                   q_start)
    _launch.on_gpu(q)
    B, Nq, Nk, Hq, Hkv, d = sizes[:6]
    out, fo = _launch.new_heads(q, B, Nq, Hq, d)
    lse = q.new_empty((B, Hq, Nq), dtype=torch.float32)
    if not (B and Nq and Nk):  # nothing to launch: no keys, no message
        out.zero_()
        lse.fill_(-math.inf)
        return (out, lse) if return_lse else out
    (q, fq), (k, fk), (v, fv) = _launch.heads(q), _launch.heads(k), _launch.heads(v)
    with _launch.on_device_of(q):
        need = _workspace(False, sizes)
        ws = q.new_empty(need, dtype=torch.uint8) if need else None
        rc = _lib.LIB.tarmac_mha_fwd(
            _CALL.pack(_CALL.size, *fq, *fk, *fv, *fo, *_NONE, lse.data_ptr(),
                       ws.data_ptr() if need else 0, need, *per_row, *sizes, scale),
            _launch.stream(q))
    if rc:
        _lib.check(rc)
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
    sizes, scale, per_row = _sizes(q, k, v, causal, exclude_self, scale, lengths, q_lengths,
                                   q_start)
    B, Nq, Nk, Hq, Hkv, d = sizes[:6]
    _launch.check_heads("out", out, q, q.shape)
    _launch.check_heads("dout", dout, q, q.shape)
    if lse.shape != (B, Hq, Nq) or lse.dtype is not torch.float32 or not lse.is_contiguous():
        raise ValueError(f"lse must be the contiguous fp32 [{B}, {Hq}, {Nq}] tensor of the forward")
    if lse.device != q.device:
        raise ValueError(f"lse is on {lse.device}, expected {q.device}")
    _launch.on_gpu(q)
    dq, fdq = _launch.new_heads(q, B, Nq, Hq, d)
    dk, fdk = _launch.new_heads(q, B, Nk, Hkv, d)
    dv, fdv = _launch.new_heads(q, B, Nk, Hkv, d)
    if not (B and Nq and Nk):
        return dq.zero_(), dk.zero_(), dv.zero_()
    heads = _launch.heads  # copies made for alignment live until the launch
    (q, fq), (k, fk), (v, fv), (out, fo), (dout, fg) = map(heads, (q, k, v, out, dout))
    need = _workspace(True, sizes)
    ws = q.new_empty(need, dtype=torch.uint8)
    with _launch.on_device_of(q):
        rc = _lib.LIB.tarmac_mha_bwd(
            _CALL.pack(_CALL.size, *fq, *fk, *fv, *fo, *fg, *fdq, *fdk, *fdv, lse.data_ptr(),
                       ws.data_ptr(), need, *per_row, *sizes, scale), _launch.stream(q))
    if rc:
        _lib.check(rc)
    return dq, dk, dv
