"""What the performance of the operators over attention heads is measured on:
attention of several heads ([B, N, H, d], key heads shared by groups of query
heads), its gradient, and the norm and position rotation of queries and keys
that comes before it.

``rotary``       queries and keys of a packed projection: normed per head and
                 rotated to their positions
``rotary_grad``  the gradient of that, weights included
``attend``       attention over whole sequences: causal, or over all peers but
                 oneself, padded batches
``decode``       one or a few new tokens over a cache of keys and values
``attend_grad``  a training pass: attention, then its gradient

With ``own`` false ``run`` computes each in elementary torch operations in 32
bits, rounded once at the end; with it true it calls :mod:`tarmac.kernels`.
Sequence lengths of a padded batch are part of the case (a fixed pattern over
the batch), everything else comes from the seed.
"""

import math
import os
import sys

import torch

own = False

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "topk-tarmac_amd"))

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZES = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-6
BASE = 10000.0


def listed():
    return [
        # one new token of each of 32 sequences, between the projection and the cache
        {"name": "rotary_token", "kind": "rotary", "B": 32, "N": 1, "Hq": 16, "Hkv": 4, "d": 64,
         "rot": 64, "dtype": "bf16"},
        # a training batch of four sequences of 4096 tokens
        {"name": "rotary_4k", "kind": "rotary", "B": 4, "N": 4096, "Hq": 32, "Hkv": 8, "d": 128,
         "rot": 128, "dtype": "bf16"},
        # fp32 heads of an odd width, only part of which is rotated; no size a multiple of anything
        {"name": "rotary_grad_odd", "kind": "rotary_grad", "B": 3, "N": 1237, "Hq": 6, "Hkv": 2,
         "d": 80, "rot": 40, "dtype": "f32"},
        # the gradient at the size of a training batch
        {"name": "rotary_grad_4k", "kind": "rotary_grad", "B": 4, "N": 4096, "Hq": 32, "Hkv": 8,
         "d": 128, "rot": 128, "dtype": "bf16"},
        # teams of up to 96 agents, four heads of 16, every peer but oneself: the communication block in fp32
        {"name": "attend_agents", "kind": "attend", "B": 256, "N": 96, "Hq": 4, "Hkv": 4, "d": 16,
         "dtype": "f32", "causal": False, "exclude_self": True, "ragged": True},
        # the largest forward: two sequences of 8192 tokens in causal order
        {"name": "attend_causal_8k", "kind": "attend", "B": 2, "N": 8192, "Hq": 16, "Hkv": 16,
         "d": 128, "dtype": "bf16", "causal": True, "exclude_self": False, "ragged": False},
        # a ragged prompt batch in half precision, shared key heads
        {"name": "attend_ragged", "kind": "attend", "B": 7, "N": 1111, "Hq": 12, "Hkv": 4, "d": 64,
         "dtype": "f16", "causal": True, "exclude_self": False, "ragged": True},
        # one token over a short cache of one sequence: latency
        {"name": "decode_one", "kind": "decode", "B": 1, "Nq": 1, "Nk": 700, "Hq": 16, "Hkv": 2,
         "d": 64, "dtype": "bf16"},
        # one token of each of 32 sequences over caches of up to 8192 tokens
        {"name": "decode_8k", "kind": "decode", "B": 32, "Nq": 1, "Nk": 8192, "Hq": 32, "Hkv": 8,
         "d": 128, "dtype": "bf16"},
        # training of the communication block's heads at the headline batch of agents
        {"name": "grad_agents", "kind": "attend_grad", "B": 64, "N": 256, "Hq": 4, "Hkv": 4,
         "d": 32, "dtype": "f32", "causal": False, "exclude_self": True, "ragged": True},
        # training over whole sequences in causal order
        {"name": "grad_causal_4k", "kind": "attend_grad", "B": 2, "N": 4096, "Hq": 16, "Hkv": 16,
         "d": 128, "dtype": "bf16", "causal": True, "exclude_self": False, "ragged": False},
        # the same with shared key heads, odd lengths and narrow heads
        {"name": "grad_shared", "kind": "attend_grad", "B": 3, "N": 1111, "Hq": 8, "Hkv": 2,
         "d": 64, "dtype": "bf16", "causal": True, "exclude_self": False, "ragged": True},
    ]


# -- drawn cases ---------------------------------------------------------------

#: What keeps a drawn case under the largest listed one's time: elements of q
#: and k, scores (in the plain forms they cost more than the products), elements
#: of a cache.
MOST = {"rotary": 8.3e7, "attend": 1.8e9, "attend_grad": 4.6e8, "decode": 2.6e8}


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng):
    shared = rng.choice([1, 1, 2, 3, 4, 8])
    kv = rng.choice([1, 2, 3, 4, 8])
    return {"Hq": kv * shared, "Hkv": kv}


def draw(rng):
    kind = rng.choice(["rotary", "rotary_grad", "attend", "attend", "decode", "decode",
                       "attend_grad", "attend_grad"])
    c = {"kind": kind, **_heads(rng), "d": rng.choice([16, 24, 32, 40, 64, 64, 80, 96, 128, 128]),
         "dtype": rng.choice(["f32", "bf16", "bf16", "f16"])}
    if kind in ("rotary", "rotary_grad"):
        c.update(N=_log_int(rng, 1, 8192), B=_log_int(rng, 1, 256),
                 rot=c["d"] if rng.random() < 0.6 else 8 * rng.randint(1, c["d"] // 8))
        c["B"] = max(1, min(c["B"], int(MOST["rotary"] / (c["N"] * (c["Hq"] + c["Hkv"]) * c["d"]))))
        return c
    if kind == "decode":
        c.update(B=_log_int(rng, 1, 64), Nq=rng.choice([1, 1, 1, 2, 4]), Nk=_log_int(rng, 8, 32768))
        c["B"] = max(1, min(c["B"], int(MOST["decode"] / (c["Nk"] * c["Hkv"] * c["d"])),
                            int(MOST["attend"] / (c["Nk"] * c["Nq"] * c["Hq"]))))
        return c
    mask = rng.choice(["causal", "causal", "exclude_self", "all"])
    # gradients of two or three tokens are mostly differences that vanish: from eight on
    c.update(N=_log_int(rng, 2, 8192) if kind == "attend" else _log_int(rng, 8, 4096),
             B=_log_int(rng, 1, 256),
             causal=mask == "causal", exclude_self=mask == "exclude_self", ragged=rng.random() < 0.5)
    c["N"] = min(c["N"], int(math.sqrt(MOST[kind] / c["Hq"])))
    c["B"] = max(1, min(c["B"], int(MOST[kind] / (c["N"] ** 2 * c["Hq"]))))
    return c


# -- inputs --------------------------------------------------------------------

def _lengths(case):
    """Valid tokens of each sequence: the whole length for the first, down to a
    third of it in an irregular order for the others."""
    B = case["B"]
    N = case["Nk"] if case["kind"] == "decode" else case["N"]
    if case["kind"] != "decode" and not case["ragged"]:
        return [N] * B
    least = max(1, case.get("Nq", 1), N // 3)
    return [N - (b * 7919) % (N - least + 1) for b in range(B)]


def _angles(positions, rot, dtype):
    """Rotation angles position * BASE^(-2 j / rot), in 64 bits."""
    j = torch.arange(rot // 2, device=positions.device, dtype=torch.float64)
    return (positions.double().unsqueeze(-1) * torch.pow(torch.tensor(BASE, dtype=torch.float64), -2 * j / rot)).to(dtype)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    B, Hq, Hkv, d = case["B"], case["Hq"], case["Hkv"], case["d"]
    dtype = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=dev).to(dtype)

    s = {"case": dict(case)}
    if case["kind"] in ("rotary", "rotary_grad"):
        N, rot = case["N"], case["rot"]
        # queries and keys are views of the packed projection, as a model's linear layer gives them
        packed = normal(B, N, Hq + 2 * Hkv, d)
        s["q"], s["k"] = packed[:, :, :Hq], packed[:, :, Hq:Hq + Hkv]
        s["wq"] = 1.0 + 0.1 * torch.randn(d, generator=gen, device=dev)
        s["wk"] = 1.0 + 0.1 * torch.randn(d, generator=gen, device=dev)
        room = max(4096, N)
        first = torch.randint(0, 2 * room - N, (B, 1), generator=gen, device=dev)
        s["positions"] = (first + torch.arange(N, device=dev)).to(torch.int32)
        a = _angles(torch.arange(2 * room, device=dev), rot, torch.float64)
        s["table"] = torch.cat([a.cos(), a.sin()], -1).float()
        if case["kind"] == "rotary_grad":
            s["dq"], s["dk"] = normal(B, N, Hq, d), normal(B, N, Hkv, d)
        return s
    lengths = torch.tensor(_lengths(case), dtype=torch.int32, device=dev)
    if case["kind"] == "decode":
        Nq, Nk = case["Nq"], case["Nk"]
        s["q"] = normal(B, Nq, Hq, d)
        s["k"], s["v"] = normal(B, Nk, Hkv, d), normal(B, Nk, Hkv, d)
        s["lengths"], s["start"] = lengths, lengths - Nq
        return s
    N = case["N"]
    s["q"], s["k"], s["v"] = normal(B, N, Hq, d), normal(B, N, Hkv, d), normal(B, N, Hkv, d)
    s["lengths"] = lengths if case["ragged"] else None
    if case["kind"] == "attend_grad":
        s["dout"] = normal(B, N, Hq, d)
    return s


# -- the plain forms -----------------------------------------------------------

def _plain_norm(x, w):
    x = x.float()
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    return x, r, x * r * w


def _plain_rotate(y, table, positions, back=False):
    half = table.shape[-1] // 2
    row = table[positions.long()].unsqueeze(2)
    c, s = row[..., :half], row[..., half:]
    if back:
        s = -s
    lo, hi, rest = y[..., :half], y[..., half:2 * half], y[..., 2 * half:]
    return torch.cat([lo * c - hi * s, hi * c + lo * s, rest], -1)


def _plain_rotary(x, w, s):
    return _plain_rotate(_plain_norm(x, w)[2], s["table"], s["positions"]).to(x.dtype)


def _plain_rotary_grad(dz, x, w, s):
    dy = _plain_rotate(dz.float(), s["table"], s["positions"], back=True)
    xf, r, _ = _plain_norm(x, w)
    xh = xf * r
    g = dy * w
    dx = r * (g - xh * (g * xh).mean(-1, keepdim=True))
    # the weights' sums run over every token and head: 64 bits
    return dx.to(x.dtype), (dy * xh).double().sum((0, 1, 2)).float()


def _by_head(x, groups):
    """[B, N, H, d] as fp32 [B * groups, H / groups * N, d]: the query heads that
    share a key head stand under each other."""
    B, N, H, d = x.shape
    return x.float().permute(0, 2, 1, 3).reshape(B * groups, H // groups * N, d)


def _from_head(x, like):
    B, N, H, d = like.shape
    return x.reshape(B, H, N, d).permute(0, 2, 1, 3).to(like.dtype).contiguous()


def _allowed(c, Nq, Nk, lengths, start, dev):
    """[B or 1, Nq, Nk]: which keys a query attends to."""
    i = torch.arange(Nq, device=dev).view(1, Nq, 1)
    j = torch.arange(Nk, device=dev).view(1, 1, Nk)
    pos = i if start is None else i + start.view(-1, 1, 1)
    ok = torch.ones(1, Nq, Nk, dtype=torch.bool, device=dev)
    if c.get("causal", c["kind"] == "decode"):
        ok = ok & (j <= pos)
    if c.get("exclude_self", False):
        ok = ok & (j != pos)
    if lengths is not None:
        ok = ok & (j < lengths.view(-1, 1, 1))
        if c["kind"] != "decode":  # a padded batch: rows behind a sequence's end attend to nothing
            ok = ok & (i < lengths.view(-1, 1, 1))
    return ok


def _plain_weights(c, q, k, ok):
    """exp(s - lse) [B, Hkv, shared, Nq, Nk] and lse; an empty row has weights of 0."""
    B, Nq, Hq, d = q.shape
    Nk, Hkv = k.shape[1], k.shape[2]
    kt = _by_head(k, Hkv).transpose(1, 2).contiguous()
    s = torch.bmm(_by_head(q, Hkv) * (1.0 / math.sqrt(d)), kt).view(B, Hkv, Hq // Hkv, Nq, Nk)
    s.masked_fill_(~ok[:, None, None], float("-inf"))
    m = s.amax(-1, keepdim=True)
    m = torch.where(m == float("-inf"), torch.zeros_like(m), m)
    p = s.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    p.div_(torch.where(total == 0, torch.ones_like(total), total))
    return p, (total.log() + m).reshape(B, Hq, Nq)


def _plain_attend(s):
    c, q, k, v = s["case"], s["q"], s["k"], s["v"]
    B, Nq, Hq, d = q.shape
    Nk, Hkv = k.shape[1], k.shape[2]
    ok = _allowed(c, Nq, Nk, s["lengths"], s.get("start"), q.device)
    p, lse = _plain_weights(c, q, k, ok)
    rows = p.view(B * Hkv, Hq // Hkv * Nq, Nk)
    vh = _by_head(v, Hkv)
    out = torch.bmm(rows, vh)
    result = {"out": _from_head(out, q), "lse": lse}
    if c["kind"] != "attend_grad":
        return result
    do = _by_head(s["dout"], Hkv)
    dv = torch.bmm(rows.transpose(1, 2).contiguous(), do)
    ds = torch.bmm(do, vh.transpose(1, 2).contiguous())
    ds.sub_((do * out).sum(-1, keepdim=True)).mul_(rows).mul_(1.0 / math.sqrt(d))
    dq = torch.bmm(ds, _by_head(k, Hkv))
    dk = torch.bmm(ds.transpose(1, 2).contiguous(), _by_head(q, Hkv))
    return {"out": result["out"], "dq": _from_head(dq, q), "dk": _from_head(dk, k),
            "dv": _from_head(dv, v)}


def _plain(s):
    kind = s["case"]["kind"]
    if kind == "rotary":
        return {"q": _plain_rotary(s["q"], s["wq"], s), "k": _plain_rotary(s["k"], s["wk"], s)}
    if kind == "rotary_grad":
        dq, dwq = _plain_rotary_grad(s["dq"], s["q"], s["wq"], s)
        dk, dwk = _plain_rotary_grad(s["dk"], s["k"], s["wk"], s)
        return {"dq": dq, "dk": dk, "dwq": dwq, "dwk": dwk}
    return _plain_attend(s)


# -- a pass --------------------------------------------------------------------

def run(s):
    if not own:
        return _plain(s)
    from tarmac import kernels as K

    c = s["case"]
    if c["kind"] == "rotary":
        q, k = K.qk_norm_rope(s["q"], s["k"], s["wq"], s["wk"], s["table"], s["positions"], eps=EPS)
        return {"q": q, "k": k}
    if c["kind"] == "rotary_grad":
        dq, dk, dwq, dwk = K.qk_norm_rope_backward(s["dq"], s["dk"], s["q"], s["k"], s["wq"], s["wk"],
                                                   s["table"], s["positions"], eps=EPS)
        return {"dq": dq, "dk": dk, "dwq": dwq, "dwk": dwk}
    if c["kind"] == "decode":
        out, lse = K.multihead_attention(s["q"], s["k"], s["v"], causal=True, lengths=s["lengths"],
                                         q_start=s["start"], return_lse=True)
        return {"out": out, "lse": lse}
    mask = {"causal": c["causal"], "exclude_self": c["exclude_self"], "lengths": s["lengths"],
            "q_lengths": s["lengths"]}
    out, lse = K.multihead_attention(s["q"], s["k"], s["v"], return_lse=True, **mask)
    if c["kind"] == "attend":
        return {"out": out, "lse": lse}
    dq, dk, dv = K.multihead_attention_backward(s["q"], s["k"], s["v"], out, lse, s["dout"], **mask)
    return {"out": out, "dq": dq, "dk": dk, "dv": dv}


# -- work ----------------------------------------------------------------------

def _pairs(case):
    """Allowed (query, key) pairs of one head, over the batch."""
    total = 0
    for n in _lengths(case):
        if case["kind"] == "decode":
            nq = case["Nq"]
            total += nq * n - nq * (nq - 1) // 2
        elif case["causal"]:
            total += n * (n + 1) // 2
        else:
            total += n * n - (n if case["exclude_self"] else 0)
    return total


def work(case):
    """Each input read once and each output written once: of a padded batch's
    inputs the valid tokens, of its outputs every row."""
    B, Hq, Hkv, d, size = case["B"], case["Hq"], case["Hkv"], case["d"], SIZES[case["dtype"]]
    if case["kind"] in ("rotary", "rotary_grad"):
        x = B * case["N"] * (Hq + Hkv) * d
        # a token's row of the table is shared by its heads; consecutive positions of a batch may overlap
        small = 4 * min(B * case["N"], 2 * max(4096, case["N"])) * case["rot"] + 4 * B * case["N"] + 8 * d
        if case["kind"] == "rotary":
            return {"bytes": 2 * x * size + small, "flops": 10 * x}
        return {"bytes": 3 * x * size + small + 8 * d, "flops": 20 * x}
    valid = sum(_lengths(case))
    pairs = _pairs(case) * Hq * d
    if case["kind"] == "decode":
        nq = case["Nq"]
        return {"bytes": size * (2 * B * nq * Hq * d + 2 * valid * Hkv * d) + 4 * B * Hq * nq,
                "flops": 4 * pairs}
    rows = B * case["N"]
    if case["kind"] == "attend":
        return {"bytes": size * (valid * (Hq + 2 * Hkv) * d + rows * Hq * d) + 4 * rows * Hq,
                "flops": 4 * pairs}
    # q, k, v, dout in; out, dq, dk, dv out; two products forward, five backward
    return {"bytes": size * (valid * (2 * Hq + 2 * Hkv) * d + rows * (2 * Hq + 2 * Hkv) * d),
            "flops": 14 * pairs}


# -- the same in 64 bits -------------------------------------------------------

def _exact_rotary(x, w, s):
    """The definition with complex numbers: a pair (y_j, y_{j + rot/2}) times
    e^(i angle)."""
    rot = s["case"]["rot"]
    y = x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * w
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=x.device),
                       _angles(s["positions"], rot, torch.float64)).unsqueeze(2)
    z = torch.complex(y[..., :rot // 2].contiguous(), y[..., rot // 2:rot].contiguous()) * turn
    return torch.cat([z.real, z.imag, y[..., rot:]], -1)


def _exact_head(q, k, v, ok, scale):
    """Attention of one key head [B, N, d] and its query heads [B, N, G, d]."""
    s = (torch.matmul(q.transpose(1, 2), k.transpose(1, 2).unsqueeze(1)) * scale)
    any_ = ok.any(-1)[:, None]
    s = s.masked_fill(~(ok | ~ok.any(-1, keepdim=True))[:, None], float("-inf"))
    lse = torch.logsumexp(s, -1)
    w = torch.exp(s - lse.unsqueeze(-1)) * any_.unsqueeze(-1)
    return torch.matmul(w, v.unsqueeze(1)).transpose(1, 2), lse.masked_fill(~any_, float("-inf"))


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind in ("rotary", "rotary_grad"):
        got = {}
        for name in ("q", "k"):
            outs, grads = [], []
            w = s["w" + name].double().requires_grad_()
            dw = torch.zeros_like(w)
            whole, places = s[name], s["positions"]
            step = max(1, (1 << 25) // whole[0].numel())
            for b in range(0, case["B"], step):
                x = whole[b:b + step].double().requires_grad_()
                s["positions"] = places[b:b + step]
                z = _exact_rotary(x, w, s)
                outs.append(z.detach())
                if kind == "rotary_grad":
                    dx, part = torch.autograd.grad(z, (x, w), s["d" + name][b:b + step].double())
                    grads.append(dx)
                    dw = dw + part
            s["positions"] = places
            if kind == "rotary":
                got[name] = torch.cat(outs)
            else:
                got["d" + name], got["dw" + name] = torch.cat(grads), dw.detach()
        return got
    q, k, v = s["q"], s["k"], s["v"]
    B, Nq, Hq, d = q.shape
    Nk, Hkv = k.shape[1], k.shape[2]
    G = Hq // Hkv
    lens = torch.tensor(_lengths(case), device=q.device).view(-1, 1, 1)
    i = torch.arange(Nq, device=q.device).view(1, -1, 1)
    j = torch.arange(Nk, device=q.device).view(1, 1, -1)
    if kind == "decode":
        ok = (j < lens) & (j <= lens - Nq + i)
    else:
        ok = (j < lens) & (i < lens)
        if case["causal"]:
            ok = ok & (i >= j)
        if case["exclude_self"]:
            ok = ok & (i != j)
    grad = kind == "attend_grad"
    got = {"out": torch.zeros(B, Nq, Hq, d, dtype=torch.float64, device=q.device),
           "lse": torch.zeros(B, Hq, Nq, dtype=torch.float64, device=q.device)}
    if grad:
        got.update(dq=torch.zeros_like(got["out"]), dk=torch.zeros_like(k, dtype=torch.float64),
                   dv=torch.zeros_like(v, dtype=torch.float64))
    step = max(1, (1 << 28) // (G * Nq * Nk))
    for h in range(Hkv):
        heads = slice(h * G, h * G + G)
        for b in range(0, B, step):
            r = slice(b, b + step)
            a = [t.double().contiguous().requires_grad_(grad)
                 for t in (q[r, :, heads], k[r, :, h], v[r, :, h])]
            out, lse = _exact_head(*a, ok[r], 1.0 / math.sqrt(d))
            got["out"][r, :, heads], got["lse"][r, heads] = out.detach(), lse.detach()
            if grad:
                dq, dk, dv = torch.autograd.grad(out, a, s["dout"][r, :, heads].double())
                got["dq"][r, :, heads], got["dk"][r, :, h], got["dv"][r, :, h] = dq, dk, dv
    if grad:
        del got["lse"]
    return got
