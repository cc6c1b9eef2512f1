"""What the operators over heads refuse, on the CPU: the Python wrappers before
they look at the device, the C entry points before any launch."""

from __future__ import annotations

import sys

import pytest
import torch


def _qkv(B=2, Nq=6, Nk=6, Hq=4, Hkv=2, d=16, dtype=torch.float32):
    return torch.zeros(B, Nq, Hq, d, dtype=dtype), *(torch.zeros(B, Nk, Hkv, d, dtype=dtype) for _ in "kv")


def _i32(*v):
    return torch.tensor(v, dtype=torch.int32)


@pytest.mark.parametrize("change,error,text", [
    (dict(q=torch.zeros(2, 6, 16)), ValueError, "B, N, H, d"),
    (dict(k=torch.zeros(2, 5, 2, 16)), ValueError, "v: expected shape"),
    (dict(k=torch.zeros(3, 6, 2, 16)), ValueError, "k: expected shape"),
    (dict(v=torch.zeros(2, 6, 2, 24)), ValueError, "v: expected shape"),
    (dict(k=torch.zeros(2, 6, 2, 16, dtype=torch.float16)), TypeError, "expected torch.float32"),
    (dict(q=torch.zeros(2, 6, 3, 16)), ValueError, "divide"),
    (dict(scale=0.0), ValueError, "scale"),
    (dict(scale=-1.0), ValueError, "scale"),
    (dict(scale=float("inf")), ValueError, "scale"),
    (dict(scale=float("nan")), ValueError, "scale"),
    (dict(lengths=torch.tensor([1, 2])), TypeError, "lengths must be an int32"),
    (dict(lengths=[1, 2]), TypeError, "lengths must be an int32"),
    (dict(q_lengths=_i32(1, 2, 3)), ValueError, "q_lengths must be contiguous"),
    (dict(q_start=_i32(1, 5, 2, 5)[::2][:1]), ValueError, "q_start must be contiguous"),
    (dict(q_start=_i32(1, 5, 2, 5)[::2]), ValueError, "q_start must be contiguous"),
])
def test_attention(change, error, text):
    from tarmac.kernels import multihead_attention
    q, k, v = _qkv()
    args = {"q": q, "k": k, "v": v, **change}
    with pytest.raises(error, match=text):
        multihead_attention(args.pop("q"), args.pop("k"), args.pop("v"), **args)


@pytest.mark.parametrize("d", [4, 12, 136, 256])
def test_widths(d):
    from tarmac.kernels import multihead_attention, qk_norm_rope
    q, k, v = _qkv(d=d)
    with pytest.raises(NotImplementedError, match="multiple of 8"):
        multihead_attention(q, k, v)
    with pytest.raises(NotImplementedError, match="multiple of 8"):
        qk_norm_rope(q, k, torch.ones(d))


def test_types_places_and_device():
    from tarmac.kernels import multihead_attention
    q, k, v = (t.double() for t in _qkv())
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        multihead_attention(q, k, v)
    q, k, v = _qkv(Nq=2)
    for mask in ({"causal": True}, {"exclude_self": True}):
        with pytest.raises(ValueError, match="q_start"):
            multihead_attention(q, k, v, **mask)
    with pytest.raises(RuntimeError, match="GPU only"):
        multihead_attention(q, k, v)


@pytest.mark.parametrize("change,error,text", [
    (dict(out=torch.zeros(2, 6, 4, 8)), ValueError, "out: expected"),
    (dict(dout=torch.zeros(2, 6, 4, 16, dtype=torch.bfloat16)), TypeError, "dout: expected"),
    (dict(lse=torch.zeros(2, 6, 4)), ValueError, "lse must be"),
    (dict(lse=torch.zeros(2, 4, 6, dtype=torch.float64)), ValueError, "lse must be"),
    (dict(lse=torch.zeros(2, 6, 4).transpose(1, 2)), ValueError, "lse must be"),
    ({}, RuntimeError, "GPU only"),
])
def test_backward(change, error, text):
    from tarmac.kernels import multihead_attention_backward
    q, k, v = _qkv()
    args = {"out": q, "lse": torch.zeros(2, 4, 6), "dout": q, **change}
    with pytest.raises(error, match=text):
        multihead_attention_backward(q, k, v, args["out"], args["lse"], args["dout"])


@pytest.mark.parametrize("change,error,text", [
    (dict(q=torch.zeros(2, 6, 16)), ValueError, "B, N, H, d"),
    (dict(k=torch.zeros(2, 5, 2, 16)), ValueError, "k: expected shape"),
    (dict(q_weight=None, k_weight=None, table=None), ValueError, "nothing to do"),
    (dict(q_weight=torch.ones(8)), ValueError, "weights must be contiguous"),
    (dict(q_weight=torch.ones(16).double()), TypeError, "weights must be float32"),
    (dict(q_weight=torch.ones(16).bfloat16()), TypeError, "weights must be float32"),
    (dict(table=torch.ones(16)), ValueError, "table must be"),
    (dict(table=torch.ones(4, 24)), ValueError, "multiple of 8 up to 16"),
    (dict(table=torch.ones(4, 12)), ValueError, "multiple of 8 up to 16"),
    (dict(table=torch.ones(4, 16).double()), ValueError, "table must be"),
    (dict(table=torch.ones(4, 16)), ValueError, "4 positions"),
    (dict(positions=torch.zeros(2, 6)), TypeError, "positions must be int32"),
    (dict(positions=torch.zeros(2, 5, dtype=torch.int32)), ValueError, "positions must be"),
    (dict(table=None, positions=torch.zeros(2, 6, dtype=torch.int32)), ValueError, "without a table"),
    (dict(eps=-1.0), ValueError, "eps"),
    (dict(eps=float("nan")), ValueError, "eps"),
    ({}, RuntimeError, "GPU only"),
])
def test_norm_and_rotation(change, error, text):
    from tarmac.kernels import qk_norm_rope
    q, k, _ = _qkv()
    args = {"q": q, "k": k, "q_weight": torch.ones(16), "k_weight": torch.ones(16),
            "table": torch.ones(8, 16), **change}
    with pytest.raises(error, match=text):
        qk_norm_rope(**args)


def test_norm_and_rotation_backward_and_table():
    from tarmac.kernels import qk_norm_rope_backward, rotary_table
    q, k, _ = _qkv()
    with pytest.raises(ValueError, match="dq_out: expected"):
        qk_norm_rope_backward(k, k, q, k, torch.ones(16))
    with pytest.raises(RuntimeError, match="GPU only"):
        qk_norm_rope_backward(q, k, q, k, torch.ones(16))
    for rot in (0, 4, 12):
        with pytest.raises(ValueError, match="multiple of 8"):
            rotary_table(4, rot)
    with pytest.raises(ValueError, match="position"):
        rotary_table(0, 8)
    t = rotary_table(5, 8, 100.0)
    assert t.shape == (5, 8) and t.dtype == torch.float32
    a = 3 * 100.0 ** (-2 * 1 / 8)
    assert abs(float(t[3, 1]) - torch.tensor(a, dtype=torch.float64).cos()) <= 2 ** -24
    assert abs(float(t[3, 5]) - torch.tensor(a, dtype=torch.float64).sin()) <= 2 ** -24


# -- the C entry points ----------------------------------------------------------

HEADS = (256, 64, 64, 64)  # never dereferenced: refused before any launch


def _mha(size=None, q=HEADS, lse=256, ws=256, nbytes=1 << 20, lengths=0,
         sizes=(2, 6, 6, 4, 2, 16, 0, 0, 0), scale=1.0):
    _CALL = sys.modules["tarmac.kernels.multihead_attention"]._CALL
    return _CALL.pack(_CALL.size if size is None else size, *q, *(7 * HEADS), lse, ws, nbytes,
                      lengths, 0, 0, *sizes, scale)


@pytest.fixture(autouse=True, scope="module")
def _modules():
    import tarmac.kernels  # noqa: F401  (its attributes of these names are the functions)
    for m in ("multihead_attention", "qk_norm_rope"):
        assert "tarmac.kernels." + m in sys.modules


@pytest.mark.parametrize("change,code,text", [
    (dict(size=8), 1, "not a tarmac_mha"),
    (dict(q=(0, 64, 64, 64)), 1, "null q"),
    (dict(q=(264, 64, 64, 64)), 1, "aligned"),
    (dict(q=(256, 64, 62, 64)), 1, "strides"),
    (dict(lse=0), 1, "lse"),
    (dict(lengths=258), 1, "misaligned"),
    (dict(sizes=(0, 6, 6, 4, 2, 16, 0, 0, 0)), 1, "B, Nq, Nk"),
    (dict(sizes=(2, 6, 0, 4, 2, 16, 0, 0, 0)), 1, "B, Nq, Nk"),
    (dict(sizes=(2, 6, 6, 4, 3, 16, 0, 0, 0)), 1, "divide"),
    (dict(sizes=(2, 6, 6, 4, 2, 12, 0, 0, 0)), 2, "head width"),
    (dict(sizes=(2, 6, 6, 4, 2, 136, 0, 0, 0)), 2, "head width"),
    (dict(sizes=(2, 6, 6, 4, 2, 16, 3, 0, 0)), 1, "dtype"),
    (dict(sizes=(1 << 20, 6, 1 << 20, 4, 2, 16, 0, 0, 0)), 2, "2\\^31"),
    (dict(scale=0.0), 1, "scale"),
    (dict(scale=float("nan")), 1, "scale"),
])
def test_c_attention(change, code, text):
    import re
    from tarmac import _lib
    call = _mha(**change)
    for fn in (_lib.LIB.tarmac_mha_fwd, _lib.LIB.tarmac_mha_bwd):
        assert fn(call, None) == code
        assert re.search(text, _lib.last_error()), _lib.last_error()


def test_c_attention_workspace():
    from tarmac import _lib
    assert _lib.LIB.tarmac_mha_bwd_workspace(_mha()) >= 4 * 2 * 4 * 6
    assert _lib.LIB.tarmac_mha_fwd_workspace(_mha()) >= 0
    for fn in (_lib.LIB.tarmac_mha_fwd_workspace, _lib.LIB.tarmac_mha_bwd_workspace):
        assert fn(_mha(scale=0.0)) == -1 and "scale" in _lib.last_error()
        assert fn(None) == -1
    for bad in (dict(ws=0), dict(nbytes=16), dict(ws=260)):
        assert _lib.LIB.tarmac_mha_bwd(_mha(**bad), None) == 1
        assert "workspace" in _lib.last_error()


def _rope(size=None, q=HEADS, w=(256, 256), table=256, pos=0, dw=(256, 256), ws=256, nbytes=1 << 24,
          rows=100, sizes=(2, 6, 4, 2, 16, 16, 0, 0, 0), eps=1e-6):
    _CALL = sys.modules["tarmac.kernels.qk_norm_rope"]._CALL
    return _CALL.pack(_CALL.size if size is None else size, *q, *(5 * HEADS), *w, table, pos, *dw, ws,
                      nbytes, rows, *sizes, eps)


@pytest.mark.parametrize("change,code,text", [
    (dict(size=8), 1, "not a tarmac_qk_rope"),
    (dict(q=(0, 64, 64, 64)), 1, "null q"),
    (dict(q=(256, 64, 64, 63)), 1, "aligned"),
    (dict(w=(0, 0), dw=(0, 0), table=0), 1, "nothing to do"),
    (dict(w=(260, 256)), 1, "weights"),
    (dict(table=260), 1, "table"),
    (dict(rows=0), 1, "table"),
    (dict(pos=258), 1, "positions"),
    (dict(sizes=(2, 6, 4, 2, 16, 24, 0, 0, 0)), 1, "table"),
    (dict(sizes=(2, 6, 4, 2, 16, 12, 0, 0, 0)), 1, "table"),
    (dict(sizes=(2, 6, 0, 2, 16, 16, 0, 0, 0)), 1, "B, N, Hq"),
    (dict(sizes=(2, 6, 4, 2, 20, 16, 0, 0, 0)), 2, "head width"),
    (dict(sizes=(2, 6, 4, 2, 16, 16, 5, 0, 0)), 1, "dtype"),
    (dict(sizes=(2, 6, 4, 2, 16, 16, 0, 1, 0)), 1, "weights"),
    (dict(sizes=(2, 6, 4, 2, 16, 16, 0, 0, 7)), 1, "pos_dtype"),
    (dict(sizes=(1 << 15, 1 << 15, 4, 2, 16, 16, 0, 0, 0)), 2, "2\\^31"),
    (dict(eps=-1.0), 1, "eps"),
])
def test_c_norm_and_rotation(change, code, text):
    import re
    from tarmac import _lib
    call = _rope(**change)
    for fn in (_lib.LIB.tarmac_qk_rope_fwd, _lib.LIB.tarmac_qk_rope_bwd):
        assert fn(call, None) == code
        assert re.search(text, _lib.last_error()), _lib.last_error()


def test_c_norm_and_rotation_backward():
    from tarmac import _lib
    need = _lib.LIB.tarmac_qk_rope_bwd_workspace(_rope())
    assert need > 0
    for bad in (dict(ws=0), dict(nbytes=need - 1), dict(ws=264)):
        assert _lib.LIB.tarmac_qk_rope_bwd(_rope(**bad), None) == 1
        assert "workspace" in _lib.last_error()
    assert _lib.LIB.tarmac_qk_rope_bwd(_rope(dw=(0, 256)), None) == 1
    assert "come together" in _lib.last_error()


@pytest.mark.parametrize("sizes,fine", [
    ((1 << 24, 1, 1, 1, 1, 8, 1, 0, 0), False),       # a workgroup of the gradient each
    ((1 << 23, 1, 1, 1, 1, 8, 1, 0, 0), True),
    ((1 << 23, 1, 33, 1, 1, 8, 1, 0, 0), False),      # eight waves a tile forward
    (((1 << 23) - 1, 1, 33, 1, 1, 8, 1, 0, 0), True),
    ((1 << 24, 100, 100, 1, 1, 8, 1, 0, 0), False),
])
def test_c_attention_more_than_a_launch_holds(sizes, fine):
    from tarmac import _lib
    need = _lib.LIB.tarmac_mha_fwd_workspace(_mha(sizes=sizes))
    if fine:
        assert need >= 0
    else:
        assert need == -1 and "one launch" in _lib.last_error()
        assert _lib.LIB.tarmac_mha_fwd(_mha(sizes=sizes), None) == 2
        assert _lib.LIB.tarmac_mha_bwd(_mha(sizes=sizes), None) == 2


def test_c_norm_and_rotation_more_than_a_launch_holds():
    from tarmac import _lib
    # eight lanes a head, eight heads of a token a wave: 4 tokens of a side a workgroup of 256
    sizes = ((1 << 25) - 4, 1, 8, 8, 128, 16, 0, 0, 0)
    assert _lib.LIB.tarmac_qk_rope_bwd_workspace(_rope(sizes=sizes)) >= 0
    sizes = (1 << 25, 1, 8, 8, 128, 16, 0, 0, 0)
    assert _lib.LIB.tarmac_qk_rope_bwd_workspace(_rope(sizes=sizes)) == -1
    assert "one launch" in _lib.last_error()
    assert _lib.LIB.tarmac_qk_rope_fwd(_rope(sizes=sizes), None) == 2


@pytest.mark.parametrize("base", [0.0, -1.0, float("inf"), float("nan")])
def test_table_base(base):
    from tarmac.kernels import rotary_table
    with pytest.raises(ValueError, match="base"):
        rotary_table(4, 8, base)
