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
    j = torch.arange(rot // 2, dtype=torch.float64)
    a = torch.arange(positions, dtype=torch.float64).unsqueeze(-1) * base ** (-2.0 * j / rot)
    return torch.cat([a.cos(), a.sin()], -1).float().to(device)


def _sizes(q, k, q_weight, k_weight, table, positions, eps):
    """Checks every argument but the device; what the call's fields need."""
    for name, t in (("q", q), ("k", k)):
        if t.dim() != 4:
            raise ValueError(f"{name}: expected a [B, N, H, d] tensor, got shape {tuple(t.shape)}")
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
    given = [w for w in (q_weight, k_weight) if w is not None]
    for w in given:
        if w.shape != (d,) or not w.is_contiguous():
            raise ValueError(f"weights must be contiguous of shape ({d},), got {tuple(w.shape)}")
        if w.dtype not in (torch.float32, q.dtype) or w.dtype != given[0].dtype:
            raise TypeError("weights must be float32 or of the heads' type, both alike")
        if w.device != q.device:
            raise ValueError(f"weights are on {w.device}, expected {q.device}")
    w_code = _launch.heads_dtype_code(given[0].dtype) if given else _lib.DTYPE_F32
    rot = rows = 0
    if table is not None:
        if table.dim() != 2 or table.dtype != torch.float32 or not table.is_contiguous():
            raise ValueError("table must be the contiguous fp32 [positions, rot] of rotary_table")
        rows, rot = table.shape
        if rows < 1 or rot < 8 or rot > d or rot % 8:
            raise ValueError(f"the table's rot must be a multiple of 8 up to {d}, got {rot}")
        if table.device != q.device:
            raise ValueError(f"table is on {table.device}, expected {q.device}")
    pos_code = _lib.IDX_I32
    if positions is not None:
        if table is None:
            raise ValueError("positions without a table")
        if positions.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"positions must be int32 or int64, got {positions.dtype}")
        if positions.shape != (B, N):
            raise ValueError(f"positions must be [{B}, {N}], got {tuple(positions.shape)}")
        if positions.device != q.device:
            raise ValueError(f"positions are on {positions.device}, expected {q.device}")
        if positions.dtype == torch.int64:
            pos_code = _lib.IDX_I64
    elif table is not None and rows < N:
        raise ValueError(f"the table has {rows} positions, the heads {N}")
    if not 0.0 <= eps < math.inf:
        raise ValueError(f"eps must be finite and not negative, got {eps}")
    return rows, (B, N, Hq, Hkv, d, rot, code, w_code, pos_code)


def _small(*ts):
    """Weights, table and positions as the kernels read them."""
    return tuple(None if t is None else _launch.ready(t) for t in ts)


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
    rows, sizes = _sizes(q, k, q_weight, k_weight, table, positions, eps)
    _launch.on_gpu(q)
    q_out, k_out = (torch.empty(t.shape, device=t.device, dtype=t.dtype) for t in (q, k))
    if sizes[0] == 0 or sizes[1] == 0:
        return q_out, k_out
    (q, fq), (k, fk), (_, fqo), (_, fko) = map(_launch.heads, (q, k, q_out, k_out))
    wq, wk, table, positions = _small(q_weight, k_weight, table, positions)
    with _launch.on_device_of(q):
        packed = _CALL.pack(_CALL.size, *fq, *fk, *fqo, *fko, *(2 * _launch.NO_HEADS), _ptr(wq),
                            _ptr(wk), _ptr(table), _ptr(positions), 0, 0, 0, 0, rows, *sizes, eps)
        _lib.check(_lib.LIB.tarmac_qk_rope_fwd(packed, _launch.stream(q)))
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
    rows, sizes = _sizes(q, k, q_weight, k_weight, table, positions, eps)
    _launch.check_heads("dq_out", dq_out, q, q.shape)
    _launch.check_heads("dk_out", dk_out, k, k.shape)
    _launch.on_gpu(q)
    dev, d = q.device, sizes[4]
    dq, dk = (torch.empty(t.shape, device=dev, dtype=t.dtype) for t in (q, k))
    dwq, dwk = (None if w is None else torch.empty(d, device=dev, dtype=torch.float32)
                for w in (q_weight, k_weight))
    if sizes[0] == 0 or sizes[1] == 0:
        return dq, dk, *(None if w is None else w.zero_() for w in (dwq, dwk))
    tensors, fields = zip(*map(_launch.heads, (q, k, dq_out, dk_out, dq, dk)))
    wq, wk, table, positions = _small(q_weight, k_weight, table, positions)

    def call(ws, nbytes):
        return _CALL.pack(_CALL.size, *(x for f in fields for x in f), _ptr(wq), _ptr(wk),
                          _ptr(table), _ptr(positions), _ptr(dwq), _ptr(dwk), ws, nbytes, rows,
                          *sizes, eps)

    with _launch.on_device_of(q):
        need = _lib.LIB.tarmac_qk_rope_bwd_workspace(call(0, 0))
        if need < 0:
            _lib.check(_lib.TARMAC_ERR_INVALID)
        ws = torch.empty(need, device=dev, dtype=torch.uint8)
        _lib.check(_lib.LIB.tarmac_qk_rope_bwd(call(ws.data_ptr(), need), _launch.stream(q)))
    del tensors  # copies made for alignment live until the launch
    return dq, dk, dwq, dwk
