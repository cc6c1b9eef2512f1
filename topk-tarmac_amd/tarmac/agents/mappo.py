"""``AttentionComm`` -- the TarMAC communication block, with its attention core
on the HIP kernels of :mod:`tarmac.kernels`.

Drop-in for ``src/agents/mappo.py:31-86`` (``MAPPOConfig``) and
``src/agents/mappo.py:138-420`` (``AttentionComm``): same constructor, same
parameters and initialisation, same ``forward(x, pos=None) -> (msg, info)``
contract, same errors. The qkv and output projections stay ``nn.Linear``
(hipBLASLt); the core between them -- the part the reference times -- is one
HIP launch per call:

=============  ==========================================================
attn_mode      core
=============  ==========================================================
dense          ``tarmac_dense_fwd``
dense_sdpa     ``tarmac_dense_fwd`` (the same function, ``mappo.py:174-190``)
topk           ``tarmac_topk_fused_fwd`` (masked top-k is the same function
               as the gathered one, ``mappo.py:374-382``)
topk_gather    ``tarmac_topk_fused_fwd``
zorder_k       ``tarmac_zorder_fwd`` (selector + attend in one launch)
random_k       k peers drawn uniformly without the self pair, exactly as
               ``mappo.py:233-263`` draws them (the same ``torch.rand``
               call), then ``tarmac_fixedset_fwd`` over that set
entmax         alpha-entmax over all peers by the reference's 24-step
               threshold bisection (``mappo.py:294-330``), dense torch ops
adaptive_topk  the Gumbel-softmax k gate over dense weights
               (``mappo.py:383-414``), dense torch ops
multihead      ``tarmac_mha_fwd``: dense attention of ``n_heads`` heads over
               all peers, key heads shared by groups of them, heads normed
               and rotated to agent indices if asked for
               (``tarmac_qk_rope_fwd``); teams of fewer agents in one batch
=============  ==========================================================

``entmax`` and ``adaptive_topk`` are training-study arms outside the timed
core; their dense (B, N, N) formulations run as torch operations on the
device, as in the reference. Any ``msg_dim`` up to 128 works: heads whose
width the kernels do not take (fp32: 8, 16, 32, 64, 128; bf16: 16, 32, 64,
128) are zero-padded to the next width, with q pre-scaled by
sqrt(width / msg_dim) so that scores keep the 1/sqrt(msg_dim) scale; that
padding and scaling happen
in fp32 (bf16 heads are widened first, exactly), so the only perturbation of
the scores is fp32 rounding. float16 heads run the fp32 kernels on exact
fp32 copies. Messages return in the heads' dtype.

The reference's Triton kernels are forward-only
(``scripts/bench_attention_core.py:172-176``) and its training differentiates
the PyTorch composition; here the core's backward runs on HIP kernels too
(:mod:`tarmac.kernels.backward`, fp32 arithmetic for every head dtype):
gradients reach q, k, v through the retained set of the top-k and Z-order
cores, and through every pair of the dense core.

``multihead`` is not the reference's: its ``n_heads`` is read by nothing there.
Heads are ``msg_dim / n_heads`` wide, a multiple of 8 up to 128, in float32,
bfloat16 or float16 on kernels of their type, forward and backward. With one
key head per head (the default) the parameters have the reference's shapes. Its
training step can be captured into a HIP graph, once no autograd graph of the
same parameters from before the capture is alive; it has no second derivatives.
"""

from __future__ import annotations

import math
from dataclasses import dataclass

import numpy as np
import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from ..kernels.backward import (dense_attention_backward, dense_attention_forward_stats,
                                fixedset_attention_backward)
from ..kernels.fused_dense_attention import fused_dense_attention
from ..kernels.fused_prescore_attention import fused_prescore_attention
from ..kernels.fused_topk_attention import topk_attention
from ..kernels.multihead_attention import multihead_attention, multihead_attention_backward
from ..kernels.prescore_selection import zorder_attention
from ..kernels.qk_norm_rope import qk_norm_rope, qk_norm_rope_backward, rotary_table

#: Morton bits per axis of the zorder_k selector (``select_morton_window``'s
#: default, ``src/kernels/prescore_selection.py:62``).
ZORDER_BITS = 10

HIP_MODES = ("dense", "dense_sdpa", "topk", "topk_gather", "zorder_k", "random_k")
TORCH_MODES = ("entmax", "adaptive_topk")

#: Head widths the HIP kernels take, per dtype.
_WIDTHS = {torch.float32: (8, 16, 32, 64, 128), torch.bfloat16: (16, 32, 64, 128),
           torch.float16: (8, 16, 32, 64, 128)}


@dataclass
class MAPPOConfig:
    """Field-for-field ``src/agents/mappo.py:31-86``, then what
    ``attn_mode="multihead"`` takes beside ``n_heads``: ``n_kv_heads`` key heads
    (0: as many as heads), a norm of queries and keys per head (``qk_norm``), and
    their rotation to agent indices (``rotary``, ``rotary_base``)."""
    obs_dim: int
    n_actions: int
    n_agents: int
    hidden: int = 64
    use_orthogonal_init: bool = True
    use_comm: bool = False
    msg_dim: int = 16
    n_heads: int = 1
    attn_mode: str = "dense"
    topk: int = 0
    entmax_alpha: float = 1.5
    n_kv_heads: int = 0
    qk_norm: bool = False
    rotary: bool = False
    rotary_base: float = 10000.0


def _ortho_init(layer: nn.Linear, gain: float = np.sqrt(2.0)) -> None:
    nn.init.orthogonal_(layer.weight, gain=gain)
    nn.init.zeros_(layer.bias)


class _DenseCore(torch.autograd.Function):
    """Dense core with the HIP backward (fp32 arithmetic)."""

    @staticmethod
    def forward(ctx, q, k, v):
        if q.dtype == torch.float32:
            out, stats = dense_attention_forward_stats(q, k, v)
        else:  # bf16 / float16: the backward recomputes the statistics in fp32
            out, stats = fused_dense_attention(q, k, v), None
        ctx.save_for_backward(q, k, v, out, stats)
        return out

    @staticmethod
    def backward(ctx, dout):
        q, k, v, out, stats = ctx.saved_tensors
        return dense_attention_backward(q, k, v, out, dout, stats)


class _SetCore(torch.autograd.Function):
    """A core that attends over a peer set it chooses itself (top-k,
    Z-order); the HIP backward treats that set as fixed, as autograd through
    ``torch.topk``'s gather does. ``fn`` returns (out, idx)."""

    @staticmethod
    def forward(ctx, fn, q, k, v, *extra):
        out, idx = fn(q, k, v, *extra)
        ctx.mark_non_differentiable(idx)
        ctx.save_for_backward(q, k, v, idx)
        ctx.n_extra = len(extra)
        return out, idx

    @staticmethod
    def backward(ctx, dout, _didx):
        q, k, v, idx = ctx.saved_tensors
        dq, dk, dv = fixedset_attention_backward(q, k, v, idx, dout)
        return (None, dq, dk, dv) + (None,) * ctx.n_extra


class _NormRope(torch.autograd.Function):
    """Norm and rotation of queries and keys with their HIP backward."""

    @staticmethod
    def forward(ctx, q, k, wq, wk, table):
        ctx.save_for_backward(q, k, wq, wk, table)
        return qk_norm_rope(q, k, wq, wk, table)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk):
        q, k, wq, wk, table = ctx.saved_tensors
        dq, dk, dwq, dwk = qk_norm_rope_backward(dq, dk, q, k, wq, wk, table)
        if wq is not None:
            dwq, dwk = dwq.to(wq.dtype), dwk.to(wk.dtype)
        return dq, dk, dwq, dwk, None


class _HeadsCore(torch.autograd.Function):
    """Attention over heads, the self pair excluded, with its HIP backward."""

    @staticmethod
    def forward(ctx, q, k, v, lengths):
        out, lse = multihead_attention(q, k, v, exclude_self=True, lengths=lengths,
                                       q_lengths=lengths, return_lse=True)
        ctx.save_for_backward(q, k, v, out, lse, lengths)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, out, lse, lengths = ctx.saved_tensors
        return (*multihead_attention_backward(q, k, v, out, lse, dout, exclude_self=True,
                                              lengths=lengths, q_lengths=lengths), None)


def _tracks_grad(*ts: torch.Tensor) -> bool:
    return torch.is_grad_enabled() and any(t.requires_grad for t in ts)


def _kernel_width(d: int, dtype: torch.dtype) -> int:
    for w in _WIDTHS.get(dtype, ()):
        if w >= d:
            return w
    raise NotImplementedError(
        f"msg_dim={d} ({dtype}): the HIP attention core takes head widths up to 128")


def _to_width(q, k, v):
    """Zero-pad the heads to a width the kernels take; q is scaled so that
    q'.k' / sqrt(width) = q.k / sqrt(d). Padded heads are fp32 (bf16 and
    float16 values widen exactly, so the scaling rounds once, at fp32).
    Returns (q', k', v', d)."""
    d = q.shape[-1]
    w = _kernel_width(d, q.dtype)
    if w == d:
        return q, k, v, d
    q, k, v = q.float(), k.float(), v.float()
    pad = (0, w - d)
    return (F.pad(q * math.sqrt(w / d), pad), F.pad(k, pad), F.pad(v, pad), d)


def _random_peers(B: int, N: int, kk: int, device) -> torch.Tensor:
    """k peers per agent uniformly without replacement, self excluded: the
    reference ranks uniform noise with self pushed to +inf and keeps the k
    smallest (``mappo.py:250-255``); the same draw gives the same sets."""
    noise = torch.rand(B, N, N, device=device)
    eye = torch.eye(N, device=device, dtype=torch.bool).unsqueeze(0)
    noise = noise.masked_fill(eye, float("inf"))
    return noise.topk(kk, dim=-1, largest=False, sorted=False).indices


def _entropy(w: torch.Tensor) -> float:
    w = w.clamp_min(1e-12)
    return float((-(w * w.log()).sum(-1)).mean().item())


class AttentionComm(nn.Module):
    """Inter-agent attention communication block (``src/agents/mappo.py:138-420``).

    Inputs (B, N, D_in) -> messages (B, N, msg_dim). ``collect_info`` gates the
    diagnostics that synchronise the device (entropy via ``.item()``); timed
    callers must set it False, as in the reference.
    """

    def __init__(self, cfg: MAPPOConfig, in_dim: int) -> None:
        super().__init__()
        self.cfg = cfg
        self.collect_info = True
        self.qkv = nn.Linear(in_dim, self._qkv_width(cfg))
        self.proj = nn.Linear(cfg.msg_dim, cfg.msg_dim)
        self.k_bins = max(cfg.n_agents - 1, 1)
        self.k_gate = nn.Linear(in_dim, self.k_bins)
        if cfg.use_orthogonal_init:
            for layer in (self.qkv, self.proj, self.k_gate):
                _ortho_init(layer)
        if cfg.attn_mode == "multihead":
            width = cfg.msg_dim // cfg.n_heads
            for name in ("q_norm", "k_norm"):
                self.register_parameter(name, nn.Parameter(torch.ones(width)) if cfg.qk_norm else None)
            # not a parameter, and fp32 whatever the module is cast to
            self._rotary = rotary_table(max(cfg.n_agents, 1), width, cfg.rotary_base) if cfg.rotary else None

    @staticmethod
    def _qkv_width(cfg: MAPPOConfig) -> int:
        if cfg.attn_mode != "multihead":
            return 3 * cfg.msg_dim
        H, G = cfg.n_heads, cfg.n_kv_heads or cfg.n_heads
        if H < 1 or cfg.msg_dim % H or cfg.msg_dim // H % 8 or cfg.msg_dim // H > 128:
            raise ValueError(f"attn_mode='multihead' needs heads of a multiple of 8 up to 128 "
                             f"channels: msg_dim={cfg.msg_dim}, n_heads={H}")
        if G < 1 or H % G:
            raise ValueError(f"n_kv_heads={G} must divide n_heads={H}")
        return cfg.msg_dim + 2 * G * (cfg.msg_dim // H)

    def _k_eff(self, N: int) -> int:
        return min(max(self.cfg.topk, 1), N - 1)

    # -- diagnostics (only with collect_info) --------------------------------
    @staticmethod
    def _dense_weights(q, k) -> torch.Tensor:
        N = q.shape[1]
        s = torch.matmul(q.float(), k.float().transpose(-1, -2)) / (q.shape[-1] ** 0.5)
        eye = torch.eye(N, device=q.device, dtype=torch.bool).unsqueeze(0)
        return torch.softmax(s.masked_fill(eye, float("-inf")), -1)

    @staticmethod
    def _set_weights(q, k, idx) -> torch.Tensor:
        B, N, d = q.shape
        kk = idx.shape[-1]
        flat = idx.long().reshape(B, N * kk, 1).expand(B, N * kk, d)
        kg = k.float().gather(1, flat).view(B, N, kk, d)
        s = torch.matmul(q.float().unsqueeze(-2), kg.transpose(-1, -2)).squeeze(-2) / d ** 0.5
        return torch.softmax(s, -1)

    # -- the torch-composed arms (outside the timed core) ---------------------
    def _entmax(self, q, k, v, N: int) -> tuple[torch.Tensor, dict]:
        """alpha-entmax over all peers (``mappo.py:294-330``): threshold tau
        found by 24 bisection steps on sum_j [(alpha-1) s_j - tau]_+^(1/(alpha-1)) = 1,
        starting from [max - 1, max]; the self pair sits far below any threshold."""
        alpha = self.cfg.entmax_alpha
        z = (torch.matmul(q, k.transpose(-1, -2).contiguous()) / math.sqrt(q.shape[-1])) * (alpha - 1.0)
        z.diagonal(dim1=-2, dim2=-1).fill_(torch.finfo(z.dtype).min / 4)
        power = 1.0 / (alpha - 1.0)
        hi = z.amax(dim=-1, keepdim=True)
        lo = hi - 1.0
        for _ in range(24):
            mid = 0.5 * (lo + hi)
            above = (z - mid).clamp_min(0).pow(power).sum(-1, keepdim=True) > 1.0
            lo = torch.where(above, mid, lo)
            hi = torch.where(above, hi, mid)
        p = (z - 0.5 * (lo + hi)).clamp_min(0).pow(power)
        p = p / p.sum(-1, keepdim=True).clamp_min(1e-8)
        info: dict = {}
        if self.collect_info:
            info["effective_k"] = float((p > 0).sum(-1).float().mean().item())
        return torch.matmul(p, v), info

    def _adaptive_topk(self, x, q, k, v, N: int) -> tuple[torch.Tensor, dict]:
        """Per-agent k from a hard Gumbel-softmax gate over k = 1..N-1, applied
        to the dense weights (``mappo.py:383-414``): the weights outside each
        row's chosen top k are zeroed and the rest renormalised; ``expected_k``
        stays a differentiable tensor."""
        w = self._dense_weights_like(q, k)
        info: dict = {}
        if self.collect_info:
            info["mean_attn_entropy"] = _entropy(w)
        gate = F.gumbel_softmax(self.k_gate(x), tau=1.0, hard=True)          # (B, N, K)
        ranked, order = w.sort(dim=-1, descending=True)
        # prefix[m, j] = 1 when rank j is within the first m + 1 ranks
        ranks = torch.arange(N, device=x.device)
        prefix = (ranks.view(1, N) <= torch.arange(self.k_bins, device=x.device).view(-1, 1))
        keep_ranked = torch.matmul(gate, prefix.to(w.dtype))                  # (B, N, N)
        keep = torch.zeros_like(w).scatter_(-1, order, keep_ranked)
        attn = w * keep
        attn = attn / attn.sum(-1, keepdim=True).clamp_min(1e-8)
        ks = torch.arange(1, self.k_bins + 1, device=x.device, dtype=gate.dtype)
        info["expected_k"] = (gate * ks).sum(-1).mean()
        if self.collect_info:
            info["mean_k"] = float(info["expected_k"].item())
        return torch.matmul(attn, v), info

    @staticmethod
    def _dense_weights_like(q, k) -> torch.Tensor:
        """softmax(q k^T / sqrt(d)) with the self pair masked, in q's dtype."""
        N = q.shape[1]
        s = torch.matmul(q, k.transpose(-1, -2).contiguous()) / math.sqrt(q.shape[-1])
        s = s.masked_fill(torch.eye(N, device=q.device, dtype=torch.bool).unsqueeze(0),
                          float("-inf"))
        return torch.softmax(s, -1)

    # -- attention over heads --------------------------------------------------
    def _multihead(self, qkv, lengths, B: int, N: int) -> tuple[torch.Tensor, dict]:
        cfg = self.cfg
        H, G = cfg.n_heads, cfg.n_kv_heads or cfg.n_heads
        # views of the projection: the kernels read them where they are
        q, k, v = qkv.view(B, N, H + 2 * G, cfg.msg_dim // H).split([H, G, G], 2)
        if cfg.qk_norm or cfg.rotary:
            table = self._rotary
            if table is not None and (table.device != q.device or table.shape[0] < N):
                table = self._rotary = rotary_table(max(N, table.shape[0]), table.shape[1],
                                                    cfg.rotary_base, device=q.device)
            args = (q, k, self.q_norm, self.k_norm, table)
            grad = _tracks_grad(*(t for t in args if t is not None))
            q, k = _NormRope.apply(*args) if grad else qk_norm_rope(*args)
        if _tracks_grad(q, k, v):
            msg = _HeadsCore.apply(q, k, v, lengths)
        else:
            msg = multihead_attention(q, k, v, exclude_self=True, lengths=lengths, q_lengths=lengths)
        info: dict = {}
        if self.collect_info:
            info["mean_attn_entropy"] = self._heads_entropy(q.detach(), k.detach(), lengths)
        return msg.reshape(B, N, cfg.msg_dim), info

    @staticmethod
    def _heads_entropy(q, k, lengths) -> float:
        """Mean entropy of the weights, over heads and agents that have a peer."""
        B, N, H, d = q.shape
        k = k.float().repeat_interleave(H // k.shape[2], 2).permute(0, 2, 3, 1).contiguous()
        s = torch.matmul(q.float().transpose(1, 2), k) / math.sqrt(d)
        i = torch.arange(N, device=q.device)
        ok = (i[:, None] != i).expand(B, 1, N, N)
        if lengths is not None:
            n = lengths.view(B, 1, 1, 1)
            ok = ok & (i < n) & (i[:, None] < n)
        some = ok.any(-1, keepdim=True)
        w = torch.softmax(s.masked_fill(~(ok | ~some), float("-inf")), -1)
        each = -(w * w.clamp_min(1e-12).log()).sum(-1)
        rows = some.squeeze(-1).expand_as(each)
        return float(torch.where(rows, each, 0.0).sum() / rows.sum().clamp_min(1))

    # -- forward -------------------------------------------------------------
    def forward(self, x: torch.Tensor, pos: torch.Tensor | None = None,
                lengths: torch.Tensor | None = None) -> tuple[torch.Tensor, dict]:
        """``lengths`` (int32 [B], ``multihead`` only): agents of each team; rows
        behind a team's end are padding: no agent attends to them, their message is
        zero, and they add nothing to a gradient as long as they are finite."""
        B, N, _ = x.shape
        mode = self.cfg.attn_mode
        if lengths is not None and mode != "multihead":
            raise ValueError(f"attn_mode={mode!r} takes no lengths")
        qkv = self.qkv(x)
        if mode == "multihead":
            msg, info = self._multihead(qkv, lengths, B, N)
            return self.proj(F.gelu(msg)), info
        # one copy into a [3, B, N, m] buffer: q, k and v are then contiguous
        # views (three .contiguous() chunks would be three launches)
        m = qkv.shape[-1] // 3
        q, k, v = qkv.view(B, N, 3, m).permute(2, 0, 1, 3).contiguous().unbind(0)

        if mode == "entmax":
            msg, info = self._entmax(q, k, v, N)
            return self.proj(F.gelu(msg)), info
        if mode == "adaptive_topk":
            msg, info = self._adaptive_topk(x, q, k, v, N)
            return self.proj(F.gelu(msg)), info
        if mode not in HIP_MODES:
            raise ValueError(f"unknown attn_mode {mode!r}")
        if mode == "zorder_k" and pos is None:
            raise ValueError("attn_mode='zorder_k' needs agent positions")
        qw, kw, vw, d = _to_width(q, k, v)
        msg, info = self._core(mode, q, k, qw, kw, vw, pos, B, N)
        return self.proj(F.gelu(msg[..., :d].to(q.dtype))), info

    def _core(self, mode, q, k, qw, kw, vw, pos, B: int, N: int) -> tuple[torch.Tensor, dict]:
        """The HIP core on kernel-width heads (qw, kw, vw); q, k are the
        unpadded heads for the diagnostics."""
        info: dict = {}
        grad = _tracks_grad(qw, kw, vw)
        if mode == "zorder_k":
            kk = self._k_eff(N)
            if grad:
                msg, idx = _SetCore.apply(
                    lambda a, b, c, p: zorder_attention(a, b, c, p, kk, ZORDER_BITS,
                                                        return_indices=True),
                    qw, kw, vw, pos)
            else:
                res = zorder_attention(qw, kw, vw, pos, kk, ZORDER_BITS,
                                       return_indices=self.collect_info)
                msg, idx = res if self.collect_info else (res, None)
            info["effective_k"] = float(kk)
            if self.collect_info:
                info["mean_attn_entropy"] = _entropy(self._set_weights(q, k, idx))
            return msg, info

        if mode == "random_k":
            kk = self._k_eff(N)
            peers = _random_peers(B, N, kk, qw.device)
            if grad:
                msg, _ = _SetCore.apply(
                    lambda a, b, c, ix: (fused_prescore_attention(a, b, c, ix), ix),
                    qw, kw, vw, peers)
            else:
                msg = fused_prescore_attention(qw, kw, vw, peers)
            info["effective_k"] = float(kk)
            return msg, info

        if mode in ("dense", "dense_sdpa"):
            msg = _DenseCore.apply(qw, kw, vw) if grad else fused_dense_attention(qw, kw, vw)
            if mode == "dense" and self.collect_info:
                info["mean_attn_entropy"] = _entropy(self._dense_weights(q, k))
            return msg, info

        kk = self._k_eff(N)  # topk, topk_gather
        if grad:
            msg, idx = _SetCore.apply(
                lambda a, b, c: topk_attention(a, b, c, kk, return_indices=True), qw, kw, vw)
        else:
            want_idx = self.collect_info and mode == "topk_gather"
            res = topk_attention(qw, kw, vw, kk, return_indices=want_idx)
            msg, idx = res if want_idx else (res, None)
        if mode == "topk":
            if self.collect_info:
                info["mean_attn_entropy"] = _entropy(self._dense_weights(q, k))
            info["effective_k"] = float(kk)
        else:
            if self.collect_info:
                info["effective_k"] = float(kk)
                info["mean_attn_entropy"] = _entropy(self._set_weights(q, k, idx))
        return msg, info
