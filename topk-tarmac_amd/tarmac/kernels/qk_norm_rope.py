"""Norm of queries and keys per head and their rotation to positions, in one
HIP pass, and its gradient: what stands between a projection and
:func:`tarmac.kernels.multihead_attention`.

``y = x / sqrt(mean(x^2) + eps) * w`` over a head's channels (where a weight is
given), then channels ``j`` and ``j + rot / 2`` (j < rot / 2) are turned by the
angle of the row's position; channels from ``rot`` on pass. Arithmetic is fp32
from the inputs to the one rounding of the outputs. No counterpart in the
reference, whose heads are neither normed nor rotated.
"""

from __future__ import annotations

import math
import struct

import torch

from .. import _launch, _lib

#: struct tarmac_qk_rope of include/tarmac.h.
_CALL = struct.Struct("@q" + 6 * "Pqqq" + "PPPPPPPqq" + "9if")
_NONE = 2 * _launch.NO_HEADS


def rotary_table(positions: int, rot: int, base: float = 10000.0, *,
                 device=None) -> torch.Tensor:
    """Cosines and sines for ``qk_norm_rope``: fp32 ``[positions, rot]``, row
    ``p`` holding cos(p w_j), then sin(p w_j), with w_j = base^(-2 j / rot), j <
    rot / 2. Angles are formed in 64 bits (in 32 those of far positions would be
    off by whole turns' fractions) and rounded once, as cosine and sine."""
    if rot < 8 or rot % 8:
        raise ValueError(f"rot must be a positive multiple of 8, got {rot}")
    if positions < 1:
        raise ValueError(f"need at least one position, got {positions}")
    if not 0.0 < base < math.inf:
        raise ValueError(f"base must be positive and finite, got {base}")
    j = torch.arange(rot // 2, dtype=torch.float64)
    a = torch.arange(positions, dtype=torch.float64).unsqueeze(-1) * base ** (-2.0 * j / rot)
    return torch.cat([a.cos(), a.sin()], -1).float().to(device)


def _aligned(t):
    """``t`` (contiguous), or a copy that starts on 16 bytes."""
    return t.clone() if t.data_ptr() & 15 else t


def _weight(w, d, like):
    """A weight [d] of heads ``like``, as the kernels read it."""
    if w.shape != (d,) or not w.is_contiguous():
        raise ValueError(f"weights must be contiguous of shape ({d},), got {tuple(w.shape)}")
    if w.dtype is not torch.float32 and w.dtype is not like.dtype:
        raise TypeError("weights must be float32 or of the heads' type, both alike")
    if w.device != like.device:
        raise ValueError(f"weights are on {w.device}, expected {like.device}")
    return _aligned(w)


def _sizes(q, k, q_weight, k_weight, table, positions, eps):
    """Checks every argument but that the device is a GPU: (rows of the table,
    the small tensors as the kernels read them, the call's sizes)."""
    if not q.dim() == k.dim() == 4:
        raise ValueError("expected [B, N, H, d] tensors, got shapes "
                         f"{tuple(q.shape)}, {tuple(k.shape)}")
    B, N, Hq, d = q.shape
    Hkv = k.shape[2]
    code = _launch.heads_dtype_code(q.dtype)
    _launch.check_heads("k", k, q, (B, N, Hkv, d))
    if Hq < 1 or Hkv < 1:
        raise ValueError(f"need at least one query and one key head, got {Hq} and {Hkv}")
    if d < 8 or d > 128 or d % 8:
        raise NotImplementedError(f"head width must be a multiple of 8 up to 128, got {d}")
    if q_weight is None and k_weight is None and table is None:
        raise ValueError("neither weights nor a table: nothing to do")
    if q_weight is not None:
        q_weight = _weight(q_weight, d, q)
    if k_weight is not None:
        k_weight = _weight(k_weight, d, q)
        if q_weight is not None and q_weight.dtype is not k_weight.dtype:
            raise TypeError("weights must be float32 or of the heads' type, both alike")
    given = k_weight if q_weight is None else q_weight
    w_code = _lib.DTYPE_F32 if given is None or given.dtype is torch.float32 else code
    rot = rows = 0
    if table is not None:
        if table.dim() != 2 or table.dtype is not torch.float32 or not table.is_contiguous():
            raise ValueError("table must be the contiguous fp32 [positions, rot] of rotary_table")
        rows, rot = table.shape
        if rows < 1 or rot < 8 or rot > d or rot % 8:
            raise ValueError(f"the table's rot must be a multiple of 8 up to {d}, got {rot}")
        if table.device != q.device:
            raise ValueError(f"table is on {table.device}, expected {q.device}")
        table = _aligned(table)
    pos_code = _lib.IDX_I32
    if positions is not None:
        if table is None:
            raise ValueError("positions without a table")
        if positions.dtype is torch.int64:
            pos_code = _lib.IDX_I64
        elif positions.dtype is not torch.int32:
            raise TypeError(f"positions must be int32 or int64, got {positions.dtype}")
        if positions.shape != (B, N):
            raise ValueError(f"positions must be [{B}, {N}], got {tuple(positions.shape)}")
        if positions.device != q.device:
            raise ValueError(f"positions are on {positions.device}, expected {q.device}")
        positions = positions.contiguous()
    elif table is not None and rows < N:
        raise ValueError(f"the table has {rows} positions, the heads {N}")
    if not 0.0 <= eps < math.inf:
        raise ValueError(f"eps must be finite and not negative, got {eps}")
    return rows, (q_weight, k_weight, table, positions), (B, N, Hq, Hkv, d, rot, code, w_code, pos_code)


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor | None = None,
                 k_weight: torch.Tensor | None = None, table: torch.Tensor | None = None,
                 positions: torch.Tensor | None = None, eps: float = 1e-6):
    """Queries ``[B, N, Hq, d]`` and keys ``[B, N, Hkv, d]`` normed per head (each
    where its ``[d]`` weight is given) and turned to their positions (where a
    ``table`` of :func:`rotary_table` is given; ``positions`` int32 or int64
    ``[B, N]``, default 0 .. N-1). Heads may be views of any strides, a packed
    projection's for instance. Returns new contiguous (q, k). A position outside
    the table gives a row of NaN."""
    rows, small, sizes = _sizes(q, k, q_weight, k_weight, table, positions, eps)
    _launch.on_gpu(q)
    B, N, Hq, Hkv, d = sizes[:5]
    q_out, fqo = _launch.new_heads(q, B, N, Hq, d)
    k_out, fko = _launch.new_heads(q, B, N, Hkv, d)
    if not (B and N):
        return q_out, k_out
    (q, fq), (k, fk) = _launch.heads(q), _launch.heads(k)
    wq, wk, table, positions = [0 if t is None else t.data_ptr() for t in small]
    with _launch.on_device_of(q):
        rc = _lib.LIB.tarmac_qk_rope_fwd(
            _CALL.pack(_CALL.size, *fq, *fk, *fqo, *fko, *_NONE, wq, wk, table, positions, 0, 0, 0,
                       0, rows, *sizes, eps), _launch.stream(q))
    if rc:
        _lib.check(rc)
    return q_out, k_out


def qk_norm_rope_backward(dq_out: torch.Tensor, dk_out: torch.Tensor, q: torch.Tensor,
                          k: torch.Tensor, q_weight: torch.Tensor | None = None,
                          k_weight: torch.Tensor | None = None,
                          table: torch.Tensor | None = None,
                          positions: torch.Tensor | None = None, eps: float = 1e-6):
    """Gradients (dq, dk, dq_weight, dk_weight) of :func:`qk_norm_rope` called
    with the same arguments, given its outputs' gradients. The weights'
    gradients are fp32, summed over tokens and heads in a fixed order (None
    where the weight is None)."""
    rows, small, sizes = _sizes(q, k, q_weight, k_weight, table, positions, eps)
    _launch.check_heads("dq_out", dq_out, q, q.shape)
    _launch.check_heads("dk_out", dk_out, k, k.shape)
    _launch.on_gpu(q)
    B, N, Hq, Hkv, d = sizes[:5]
    dq, fdq = _launch.new_heads(q, B, N, Hq, d)
    dk, fdk = _launch.new_heads(q, B, N, Hkv, d)
    dwq, dwk = (None if w is None else q.new_empty(d, dtype=torch.float32)
                for w in (q_weight, k_weight))
    if not (B and N):
        return dq, dk, *(None if w is None else w.zero_() for w in (dwq, dwk))
    heads = _launch.heads  # copies made for alignment live until the launch
    (q, fq), (k, fk), (dq_out, fqo), (dk_out, fko) = map(heads, (q, k, dq_out, dk_out))
    wq, wk, table, positions = [0 if t is None else t.data_ptr() for t in small]

    def call(ws, nbytes):
        return _CALL.pack(_CALL.size, *fq, *fk, *fqo, *fko, *fdq, *fdk, wq, wk, table, positions,
                          _ptr(dwq), _ptr(dwk), ws, nbytes, rows, *sizes, eps)

    with _launch.on_device_of(q):
        need = _lib.LIB.tarmac_qk_rope_bwd_workspace(call(0, 0))
        if need < 0:
            _lib.check(_lib.TARMAC_ERR_UNSUPPORTED)
        ws = q.new_empty(need, dtype=torch.uint8)
        rc = _lib.LIB.tarmac_qk_rope_bwd(call(ws.data_ptr(), need), _launch.stream(q))
    if rc:
        _lib.check(rc)
    return dq, dk, dwq, dwk
