"""The operators beside the block in 64 bits, from their definitions, and bounds on what rounding may change.

Half a step of a type is ``finfo.eps / 2`` relative to the value: 2^-8 in bf16, 2^-24 in fp32.
"""

from __future__ import annotations

import math

import torch

E32 = 2.0 ** -24
FLUSH = 2.0 ** -126      # smallest normal fp32 number: exponentials below it may come out as zero


def half_step(dtype) -> float:
    return torch.finfo(dtype).eps / 2


# ---------------------------------------------------------------------------------------
# relative position bias
# ---------------------------------------------------------------------------------------
def bucket_of(d: int, kind: str, count: int, top: int) -> int:
    """Bucket of one distance, in whole numbers."""
    if kind == "clip":
        return max(-top, min(top, d)) + top
    half = count // 2 if kind == "log" else count
    near = half // 2
    n = abs(d) if kind == "log" else max(d, 0)
    if n < near:
        u = n
    else:       # largest k with (n / near)^(half - near) >= (top / near)^k
        m, k = half - near, 0
        while k < m - 1 and n ** m * near ** (k + 1) >= near ** m * top ** (k + 1):
            k += 1
        u = near + k
    return u + (half if kind == "log" and d < 0 else 0)


def bucket_matrix(q_pos, k_pos, kind, count, top, q_seg=None, k_seg=None):
    """``[(B,) Lq, Lk]`` buckets on the CPU."""
    q, k = q_pos.cpu().long(), k_pos.cpu().long()
    d = q[..., :, None] - k[..., None, :]
    values, index = torch.unique(d, return_inverse=True)
    u = torch.tensor([bucket_of(int(v), kind, count, top) for v in values])[index]
    if q_seg is not None:
        u = torch.where(q_seg.cpu()[..., :, None] == k_seg.cpu()[..., None, :], u, count)
    return u


# ---------------------------------------------------------------------------------------
# cross attention
# ---------------------------------------------------------------------------------------
def attention64(q, k, v, bias=None, mask=None, scale=None, grad=None):
    """``{name: (value, bound)}`` in 64 bits for out and, with ``grad``, dq, dk, dv, dbias.  The bounds count, with r
    half a step of the inputs' type and e = 2^-24 of the arithmetic: r for the probabilities and score gradients that
    enter a product, r for each result, and for every fp32 sum its length times e of the sum of absolute values.  The
    score of a pair is off by dx = e ((D + 3) scale sum|q||k| + 3|x| + 3|max|), a probability relatively by dx, the row's
    largest dx (through its sum), and (Lk + 8) e; one below 2^-126 may be zero, so 2^-126 is added to each
    probability's error and goes wherever the probability goes (into ds times |dp - delta|, which is far from 1)."""
    dtype = q.dtype
    r = half_step(dtype) if dtype != torch.float32 else 0.0
    last = half_step(dtype)
    B, Lq, H, D = q.shape
    Lk, Hk = k.shape[1], k.shape[2]
    G = H // Hk
    scale = D ** -0.5 if scale is None else scale
    keep = torch.ones(B, Lk, dtype=torch.bool, device=q.device) if mask is None else mask.bool()
    clean = lambda t: torch.where(keep[:, :, None, None], t.double(), 0.0)     # masked keys hold anything
    Q = q.double().transpose(1, 2)
    K, V = (clean(t).transpose(1, 2).repeat_interleave(G, 1) for t in (k, v))
    x = Q @ K.transpose(-1, -2) * scale
    size = Q.abs() @ K.abs().transpose(-1, -2) * abs(scale)
    b64 = None
    if bias is not None:
        b64 = bias.double()[(None,) * (4 - bias.dim())]
        x = x + torch.where(keep[:, None, None, :], b64, 0.0)
        size = size + torch.where(b64.abs() == math.inf, 0.0, b64.abs())
    x = x.masked_fill(~keep[:, None, None, :], -math.inf)
    m = x.amax(-1, keepdim=True)
    m0 = torch.where(m == -math.inf, 0.0, m)
    p = torch.exp(x - m0)
    l = p.sum(-1, keepdim=True)
    p = p / torch.where(l == 0, 1.0, l)
    xa = torch.where(x == -math.inf, 0.0, x.abs())
    dx = E32 * ((D + 3) * size + 3 * xa + 3 * m0.abs())
    R = dx + torch.where(p > 0, dx, 0.0).amax(-1, keepdim=True) + (Lk + 8) * E32
    o = p @ V
    o_err = (p * (R + r + Lk * E32) + FLUSH) @ V.abs()
    res = {"out": (o, o_err + last * o.abs())}
    if grad is not None:
        g = grad.double().transpose(1, 2)
        dp = g @ V.transpose(-1, -2)
        Eg = E32 * D * (g.abs() @ V.abs().transpose(-1, -2))
        delta = (g * o).sum(-1, keepdim=True)
        Ed = (g.abs() * (o_err + r * r * o.abs() + E32 * D * o.abs())).sum(-1, keepdim=True)
        ds = p * (dp - delta)
        dse = (p * R + FLUSH) * (dp - delta).abs() + p * (Eg + Ed) + r * ds.abs()
        dq = ds @ K * scale
        dq_e = (dse + Lk * E32 * ds.abs()) @ K.abs() * abs(scale) + last * dq.abs()
        dk = ds.transpose(-1, -2) @ Q * scale
        dk_e = (dse + Lq * G * E32 * ds.abs()).transpose(-1, -2) @ Q.abs() * abs(scale)
        dv = p.transpose(-1, -2) @ g
        dv_e = (p * (R + r + Lq * G * E32) + FLUSH).transpose(-1, -2) @ g.abs()
        dk, dk_e, dv, dv_e = (t.unflatten(1, (Hk, G)).sum(2) for t in (dk, dk_e, dv, dv_e))
        res |= {"dq": (dq, dq_e), "dk": (dk, dk_e + last * dk.abs()), "dv": (dv, dv_e + last * dv.abs())}
        if bias is not None:
            dse = dse + B * H * E32 * ds.abs()
            for axis in (0, 1):
                if b64.shape[axis] == 1:
                    ds, dse = ds.sum(axis, keepdim=True), dse.sum(axis, keepdim=True)
            res["dbias"] = (ds.reshape(bias.shape), (dse + last * ds.abs()).reshape(bias.shape))
    for name in ("out", "dq", "dk", "dv"):
        if name in res:
            res[name] = tuple(t.transpose(1, 2) for t in res[name])
    return res


def check(got, want, name):
    value, bound = want
    assert got.shape == value.shape, (name, got.shape, value.shape)
    off = (got.double() - value).abs()
    # what underflows in fp32 or in bf16's subnormals is not part of the relative steps
    bad = ~(off <= bound + 1e-37)
    assert not bad.any(), (f"{name}: {int(bad.sum())} of {bad.numel()} values off, the worst by "
                           f"{float((off / (bound + 1e-37)).nan_to_num(math.inf).max()):.3g} times its bound")
