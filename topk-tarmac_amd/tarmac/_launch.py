"""Tensor plumbing between PyTorch and the C ABI: device/dtype checks,
contiguity and alignment, stream handles. No compute happens here."""

from __future__ import annotations

import functools

import torch

from . import _lib

_DTYPES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16}


def dtype_code(t: torch.Tensor) -> int:
    try:
        return _DTYPES[t.dtype]
    except KeyError:
        raise TypeError(f"tarmac kernels take float32 or bfloat16 tensors (float16 through "
                        f"the Python wrappers), got {t.dtype}") from None


def on_gpu(*ts: torch.Tensor) -> None:
    for t in ts:
        if not t.is_cuda:
            raise RuntimeError(
                "tarmac kernels run on the GPU only (HIP); got a tensor on "
                f"{t.device}. There is no CPU path.")


def ready(t: torch.Tensor, align: int = 16) -> torch.Tensor:
    """Contiguous and ``align``-byte aligned (a copy only when needed)."""
    t = t.contiguous()
    if t.data_ptr() % align:
        t = t.clone()
    return t


def ptr(t: torch.Tensor | None) -> int | None:
    """A tensor's address, as a ``c_void_p`` argument takes it."""
    return None if t is None else t.data_ptr()


def stream(t: torch.Tensor) -> int:
    """The handle of the stream current on ``t``'s device (0: the default
    stream), read without building a ``torch.cuda.Stream``."""
    return torch._C._cuda_getCurrentRawStream(t.device.index)


class _NoGuard:
    def __enter__(self):
        return None

    def __exit__(self, *exc):
        return None


_NO_GUARD = _NoGuard()


def on_device_of(t: torch.Tensor):
    """A context in which ``t``'s device is current; nothing to do where it
    already is (one query, where entering ``torch.cuda.device`` and leaving it
    exchange the device twice). A call with a few microseconds of kernel is
    bound by such host work: top-k at B=256, N=6 11.8 -> 8.1 us a call."""
    if torch._C._cuda_getDevice() == t.device.index:
        return _NO_GUARD
    return torch.cuda.device(t.device)


def core(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor):
    """Validate and normalise a (q, k, v) triple: same shape, 3-D, same dtype,
    on the GPU. Returns the prepared tensors."""
    assert k.shape == v.shape == q.shape, "q, k and v must share shape [B, N, d]"
    if q.dim() != 3:
        raise ValueError(f"expected [B, N, d] tensors, got shape {tuple(q.shape)}")
    on_gpu(q, k, v)
    if not (q.dtype == k.dtype == v.dtype):
        raise TypeError("q, k and v must share a dtype")
    dtype_code(q)
    return ready(q), ready(k), ready(v)


def half_on_f32(fn):
    """Let a forward wrapper ``fn(q, k, v, ...)`` take float16 heads: they run
    the fp32 kernels on fp32 copies. Every float16 value is an fp32 value, so
    the scores and retained sets are those of the inputs themselves (the
    exact top k of their canonical fp32 scores); the output comes back as
    float16 (rounded once), indices unchanged."""

    @functools.wraps(fn)
    def wrapper(q, k, v, *args, **kwargs):
        if q.dtype != torch.float16:
            return fn(q, k, v, *args, **kwargs)
        if not (k.dtype == v.dtype == torch.float16):
            raise TypeError("q, k and v must share a dtype")
        res = fn(q.float(), k.float(), v.float(), *args, **kwargs)
        if isinstance(res, tuple):
            return (res[0].to(torch.float16),) + tuple(res[1:])
        return res.to(torch.float16)

    return wrapper


# -- tensors of heads ([B, N, H, d], any strides) -------------------------------

_HEAD_DTYPES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16,
                torch.float16: _lib.DTYPE_F16}


def heads_dtype_code(dtype: torch.dtype) -> int:
    try:
        return _HEAD_DTYPES[dtype]
    except KeyError:
        raise TypeError(f"the operators over heads take float32, bfloat16 or float16 tensors, "
                        f"got {dtype}") from None


def check_heads(name: str, t: torch.Tensor, like: torch.Tensor, shape: tuple) -> None:
    """``t`` is a tensor of ``shape``, of ``like``'s type and device."""
    if t.shape != shape:
        raise ValueError(f"{name}: expected shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.dtype is not like.dtype:
        raise TypeError(f"{name}: expected {like.dtype}, got {t.dtype}")
    if t.device != like.device:
        raise ValueError(f"{name} is on {t.device}, expected {like.device}")


def per_row(name: str, t: torch.Tensor | None, like: torch.Tensor, B: int) -> int:
    """The address of ``t``, a contiguous int32 [B] on ``like``'s device; 0 for None."""
    if t is None:
        return 0
    if not isinstance(t, torch.Tensor) or t.dtype is not torch.int32:
        raise TypeError(f"{name} must be an int32 tensor, got "
                        f"{t.dtype if isinstance(t, torch.Tensor) else type(t).__name__}")
    if t.shape != (B,) or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous of shape ({B},), got {tuple(t.shape)}")
    if t.device != like.device:
        raise ValueError(f"{name} is on {t.device}, expected {like.device}")
    return t.data_ptr()


def heads(t: torch.Tensor) -> tuple:
    """``t`` with rows the kernels can read in place (channels contiguous, rows on
    16 bytes and less than 32 MiB apart; a copy only when they are not), and its
    ``tarmac_heads`` fields."""
    size = t.element_size()
    off = 16 // size - 1
    sb, sn, sh, sd = t.stride()
    at = t.data_ptr()
    if sd == 1 and not ((sb | sn | sh) & off or at & 15) and sn * size < 1 << 25:
        return t, (at, sb, sn, sh)
    # strides of dimensions of one element mean nothing
    sb, sn, sh, sd = (s if n > 1 else 0 for s, n in zip((sb, sn, sh, sd), t.shape))
    if (sd != 1 and t.shape[3] > 1) or (sb | sn | sh) & off or sn * size >= 1 << 25 or at & 15:
        t = t.contiguous()
        if t.data_ptr() & 15:
            t = t.clone()
        return t, (t.data_ptr(), *t.stride()[:3])
    return t, (at, sb, sn, sh)


def new_heads(like: torch.Tensor, B: int, N: int, H: int, d: int) -> tuple:
    """An uninitialised contiguous [B, N, H, d] of ``like``'s type and device, and
    its ``tarmac_heads`` fields (an allocation starts on 16 bytes)."""
    t = like.new_empty((B, N, H, d))
    return t, (t.data_ptr(), N * H * d, H * d, d)


NO_HEADS = (0, 0, 0, 0)
