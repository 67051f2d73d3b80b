"""Two operators that stand beside the pair stack's triangle multiplication, as cases that can be timed.

``bias``   the learned relative position bias by buckets: as the pair tensor's input embedding
           (channel-last, added to the pair tensor) and as the per-head additive bias of an attention
           (``[H, Lq, Lk]``), forward alone or with the gradient of its table.
``cross``  attention of tokens to the states of an encoder, which have a length of their own: with an
           additive bias, padded keys and key heads shared by several query heads, forward alone or with
           all gradients, and for single query rows.

With ``own`` false the operators are computed in their plain form, elementary torch operations in 32
bits; with ``own`` true through the package's entry points.
"""

from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _bias(layout, lq, lk, c, *, b=0, rule="clip32", chains=1, dtype="bf16", train=False, name=None):
    """``b`` = 0: positions shared by the batch (no batch axis), else one set of positions per batch element."""
    case = {} if name is None else {"name": name}
    case.update(op="bias", layout=layout, b=b, lq=lq, lk=lk, c=c, rule=rule, chains=chains, dtype=dtype, train=train)
    return case


def _cross(b, lq, lk, h, d, *, hk=None, bias="none", mask="none", dtype="bf16", train=False, name=None):
    """``bias``: none, shared (one for the whole batch) or batch (one per batch element); ``mask``: none,
    tail (padded encoder states) or holes (a twentieth of the keys, scattered)."""
    case = {} if name is None else {"name": name}
    case.update(op="cross", b=b, lq=lq, lk=lk, h=h, hk=h if hk is None else hk, d=d, bias=bias, mask=mask, dtype=dtype,
                train=train)
    return case


def listed():
    return [
        # a short peptide's per-head bias: launches and host time are all there is
        _bias("heads", 64, 64, 8, name="bias_heads_peptide"),
        # pair embedding of a 384-token crop of a complex (three chains), added to the pair tensor
        _bias("pair", 384, 384, 128, b=1, chains=3, name="bias_pair_crop"),
        # training step of the pair embedding of a 768-token complex: its table's gradient too
        _bias("pair", 768, 768, 128, b=1, chains=3, train=True, name="bias_pair_train"),
        # odd token counts, queries and keys of different lengths, training
        _bias("heads", 449, 577, 16, rule="log32_128", train=True, name="bias_heads_odd_train"),
        # per-head bias of a large complex in training, logarithmic buckets
        _bias("heads", 2048, 2048, 16, rule="log32_128", train=True, name="bias_heads_large_train"),
        # one new token attends to a padded batch of encoder states, key heads shared by pairs of query heads
        _cross(8, 1, 4096, 16, 64, hk=8, mask="tail", name="cross_one_token"),
        # ligand atoms to a pocket: small, odd, with a bias
        _cross(1, 61, 77, 8, 32, bias="batch", name="cross_pocket"),
        # tokens of a 768-token complex to padded encoder states, with the shared position bias
        _cross(2, 768, 1024, 16, 64, bias="shared", mask="tail", name="cross_complex"),
        # a large complex to the states of a long sequence encoder
        _cross(1, 4096, 8192, 16, 128, name="cross_long"),
        # training step of a crop's attention with the learned bias: every gradient, the bias's summed over the batch
        _cross(4, 512, 768, 16, 64, bias="shared", mask="tail", train=True, name="cross_train_bias"),
        # training step on long encoder states, four query heads to a key head, scattered unresolved residues
        _cross(1, 2048, 4096, 16, 128, hk=4, mask="holes", train=True, name="cross_train_long"),
        # full precision check of a small domain, training
        _cross(2, 256, 320, 8, 32, bias="batch", mask="tail", dtype="fp32", train=True, name="cross_fp32_train"),
    ]


def _spread(rng, lo, hi):
    """A length between lo and hi, even over the logarithm; half of them odd or ragged."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5:
        n = n // 8 * 8
    return max(lo, min(hi, n))


def draw(rng):
    train = rng.random() < 0.5
    dtype = "fp32" if rng.random() < 0.2 else "bf16"
    if rng.random() < 0.45:
        rule = rng.choice(["clip32", "clip32", "clip16", "log32_128", "log64_512", "causal32_128"])
        b, chains = rng.choice([0, 1, 2, 3]), rng.choice([1, 1, 2, 4])
        if rng.random() < 0.5:
            lq, lk, c = _spread(rng, 16, 700), _spread(rng, 16, 700), rng.choice([32, 64, 128, 128, 192, 256])
            b, layout = min(b, 1) if lq * lk * c > 4e7 else b, "pair"
        else:
            lq, lk, c = _spread(rng, 1, 2048), _spread(rng, 16, 2048), rng.choice([4, 8, 12, 16])
            b, layout = min(b, 1) if lq * lk > 1.5e6 else b, "heads"
        return _bias(layout, lq, lk, c, b=b, rule=rule, chains=chains, dtype=dtype, train=train)
    d = rng.choice([16, 24, 32, 48, 64, 64, 96, 128, 128])
    h = rng.choice([4, 8, 16])
    hk = rng.choice([h, h, h // 2, h // 4])
    b = rng.choice([1, 2, 3, 4])
    top = 512 if dtype == "fp32" else 2048
    lq, lk = _spread(rng, 1, top), _spread(rng, 1, 2 * top)
    while b > 1 and b * lq * lk * h * d > 8e9:
        b -= 1
    lk = max(1, min(lk, int(8e9 / (lq * h * d))))
    if train:       # with a single key the scores' gradient is zero, and what either side returns is rounding
        lk = max(lk, 4)
    return _cross(b, lq, lk, h, d, hk=hk, bias=rng.choice(["none", "shared", "batch"]),
                  mask=rng.choice(["none", "tail", "holes"]), dtype=dtype, train=train)


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def _rule(name):
    """(kind, buckets of the distances, largest distance told apart) of a rule's name."""
    if name.startswith("clip"):
        r = int(name[4:])
        return "clip", 2 * r + 1, r
    kind, rest = ("log", name[3:]) if name.startswith("log") else ("causal", name[6:])
    n, top = rest.split("_")
    return kind, int(n), int(top)


def _positions(n, b, chains, gen):
    """Residue numbers and chain numbers as structure files have them: each chain counts from its own
    start, with a few numbers left out where residues are unresolved."""
    rows = max(b, 1)
    step = 1 + (torch.rand(rows, n, generator=gen, device="cuda") < 0.02).int() * 5
    pos = step.cumsum(1)
    cuts = torch.rand(rows, max(chains - 1, 1), generator=gen, device="cuda") * n
    seg = torch.zeros(rows, n, dtype=torch.int32, device="cuda")
    if chains > 1:
        seg = (torch.arange(n, device="cuda")[None, :, None] >= cuts[:, None, :]).sum(-1).int()
        first = torch.cat([torch.ones(rows, 1, dtype=torch.bool, device="cuda"), seg[:, 1:] != seg[:, :-1]], 1)
        start = torch.where(first, pos, 0).cummax(1).values
        pos = pos - start + 1
    pos = pos.int()
    return (pos, seg) if b else (pos[0], seg[0])


def _lengths(case):
    """Valid keys of each batch element of a padded batch: the first is full, the others shorter."""
    b, lk = case["b"], case["lk"]
    return [lk - (lk * i) // (2 * b) if case["mask"] == "tail" else lk for i in range(b)]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = _DTYPES[case["dtype"]]

    def normal(*shape, to=dtype):
        return torch.randn(shape, generator=gen, device="cuda").to(to)

    state = {"case": dict(case)}
    lq, lk, b = case["lq"], case["lk"], case["b"]
    if case["op"] == "bias":
        kind, count, top = _rule(case["rule"])
        segments = case["chains"] > 1
        state["q_pos"], state["q_seg"] = _positions(lq, b, case["chains"], gen)
        # a square case is one sequence with itself; otherwise the keys have positions of their own
        state["k_pos"], state["k_seg"] = ((state["q_pos"], state["q_seg"]) if lq == lk
                                          else _positions(lk, b, case["chains"], gen))
        state["table"] = normal(count + segments, case["c"], to=torch.float32) * 0.5
        lead = (b,) if b else ()
        if case["layout"] == "pair":
            state["add"] = normal(*lead, lq, lk, case["c"])
            state["grad"] = normal(*lead, lq, lk, case["c"]) if case["train"] else None
        else:
            state["grad"] = normal(*lead, case["c"], lq, lk) if case["train"] else None
        if kind != "clip":
            half = count // 2 if kind == "log" else count
            state["thresholds"] = torch.tensor(_thresholds(half, half // 2, top), device="cuda")
        return state
    h, hk, d = case["h"], case["hk"], case["d"]
    state["q"], state["k"], state["v"] = normal(b, lq, h, d), normal(b, lk, hk, d), normal(b, lk, hk, d)
    state["bias"] = None
    if case["bias"] != "none":
        state["bias"] = normal(b if case["bias"] == "batch" else 1, h, lq, lk)
    state["mask"] = None
    if case["mask"] == "tail":
        state["mask"] = (torch.arange(lk, device="cuda")[None, :]
                         < torch.tensor(_lengths(case), device="cuda")[:, None])
    elif case["mask"] == "holes":
        state["mask"] = torch.rand(b, lk, generator=gen, device="cuda") >= 0.05
    state["grad"] = normal(b, lq, h, d) if case["train"] else None
    return state


# ------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if own:
        return _own_bias(state, case) if case["op"] == "bias" else _own_cross(state, case)
    return _plain_bias(state, case) if case["op"] == "bias" else _plain_cross(state, case)


def _own_bias(s, case):
    from miniworld_engine_b200 import (PositionBuckets, relative_position_bias_b200,
                                       relative_position_bias_backward_b200)
    (kind, count, top), segments = _rule(case["rule"]), case["chains"] > 1
    buckets = (PositionBuckets.clipped(top, segments=segments) if kind == "clip" else
               PositionBuckets.logarithmic(count, top, bidirectional=kind == "log", segments=segments))
    seg = {"q_segment": s["q_seg"], "k_segment": s["k_seg"]} if segments else {}
    out = relative_position_bias_b200(s["table"], buckets, s["q_pos"], s["k_pos"], layout=case["layout"],
                                      add=s.get("add"), dtype=_DTYPES[case["dtype"]], **seg)
    if not case["train"]:
        return out
    return out, relative_position_bias_backward_b200(s["grad"], buckets, s["q_pos"], s["k_pos"],
                                                     layout=case["layout"], **seg)


def _own_cross(s, case):
    from miniworld_engine_b200 import cross_attention_b200, cross_attention_backward_b200, cross_attention_forward_b200
    kw = {"bias": s["bias"], "key_mask": s["mask"]}
    if not case["train"]:
        return cross_attention_b200(s["q"], s["k"], s["v"], **kw)
    out, stats = cross_attention_forward_b200(s["q"], s["k"], s["v"], **kw)
    dq, dk, dv, dbias = cross_attention_backward_b200(s["grad"], s["q"], s["k"], s["v"], out, stats, **kw)
    return (out, dq, dk, dv) if dbias is None else (out, dq, dk, dv, dbias)


def _thresholds(n, first, top):
    """Smallest distances of buckets first + 1 ... n - 1 of ``n`` logarithmic ones, in whole numbers: the
    smallest t with t^(n-first) >= first^(n-first-k) * top^k."""
    out = []
    for k in range(1, n - first):
        want, t = first ** (n - first - k) * top ** k, first
        while t ** (n - first) < want:
            t += 1
        out.append(t)
    return out


def _plain_buckets(s, case):
    kind, count, top = _rule(case["rule"])
    delta = s["q_pos"].long()[..., :, None] - s["k_pos"].long()[..., None, :]
    if kind == "clip":
        u = delta.clamp(-top, top) + top
    else:
        half = count // 2 if kind == "log" else count
        dist = delta.abs() if kind == "log" else delta.clamp(min=0)
        first = half // 2
        u = dist.clamp(max=first) + torch.bucketize(dist, s["thresholds"], right=True)
        if kind == "log":
            u = u + (delta < 0) * half
    if case["chains"] > 1:
        u = torch.where(s["q_seg"][..., :, None] == s["k_seg"][..., None, :], u, count)
    return u


def _plain_bias(s, case):
    dtype, c = _DTYPES[case["dtype"]], case["c"]
    u, table = _plain_buckets(s, case), s["table"]
    out = table[u]
    if case["layout"] == "pair":
        out = (s["add"].float() + out).to(dtype)
    else:
        out = out.to(dtype).movedim(-1, -3).contiguous()
    if not case["train"]:
        return out
    grad = s["grad"] if case["layout"] == "pair" else s["grad"].movedim(-3, -1)
    # sums of up to millions of values a bucket: as one product with the buckets' indicators, in 64 bits
    which = (u.reshape(-1, 1) == torch.arange(table.shape[0], device="cuda")).double()
    return out, (which.T @ grad.reshape(-1, c).double()).to(table.dtype)


def _plain_cross(s, case):
    dtype, d, group = _DTYPES[case["dtype"]], case["d"], case["h"] // case["hk"]
    scale = d ** -0.5
    q, k, v = (s[n].float().transpose(1, 2) for n in ("q", "k", "v"))
    if group > 1:
        k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    x = (q @ k.transpose(-1, -2)) * scale
    if s["bias"] is not None:
        x = x + s["bias"].float()
    if s["mask"] is not None:
        x = x.masked_fill(~s["mask"][:, None, None, :], -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    o = p @ v
    out = o.transpose(1, 2).to(dtype).contiguous()
    if not case["train"]:
        return out
    g = s["grad"].float().transpose(1, 2)
    dv = p.transpose(-1, -2) @ g
    ds = p * (g @ v.transpose(-1, -2) - (g * o).sum(-1, keepdim=True))
    dq, dk = (ds @ k) * scale, (ds.transpose(-1, -2) @ q) * scale
    if group > 1:
        dk, dv = (t.unflatten(1, (-1, group)).sum(2) for t in (dk, dv))
    grads = tuple(t.transpose(1, 2).to(dtype).contiguous() for t in (dq, dk, dv))
    if s["bias"] is None:
        return (out, *grads)
    if case["bias"] == "shared":
        ds = ds.sum(0, keepdim=True)
    return (out, *grads, ds.to(dtype))


# ------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return _exact_bias(s, case) if case["op"] == "bias" else _exact_cross(s, case)


def _exact_bias(s, case):
    kind, count, top = _rule(case["rule"])
    qp, kp = s["q_pos"].double(), s["k_pos"].double()
    qp, kp = (t if t.dim() == 2 else t[None] for t in (qp, kp))
    d = qp.unsqueeze(2) - kp.unsqueeze(1)
    if kind == "clip":
        u = torch.clip(d, -top, top) + top
    else:
        half = count / 2 if kind == "log" else float(count)
        near = math.floor(half / 2)
        n = torch.abs(d) if kind == "log" else torch.relu(d)
        # a billionth above the logarithm: at a whole power the floor must not fall to the bucket below
        far = near + torch.floor(torch.log(n.clip(min=1) / near) / math.log(top / near) * (half - near) + 1e-9)
        u = torch.where(n < near, n, far.clip(max=half - 1))
        if kind == "log":
            u = torch.where(d < 0, u + half, u)
    if case["chains"] > 1:
        qs, ks = (t if t.dim() == 2 else t[None] for t in (s["q_seg"], s["k_seg"]))
        u[qs.unsqueeze(2) != ks.unsqueeze(1)] = count
    u = u.long()
    table = s["table"].double()
    grad = s["grad"]
    total = torch.zeros_like(table)
    outs = []
    for i in range(u.shape[0]):
        if case["layout"] == "pair":
            add = s["add"] if case["b"] else s["add"][None]
            outs.append(add[i].double() + torch.nn.functional.embedding(u[i], table))
        else:
            outs.append(torch.stack([torch.take(table[:, c].contiguous(), u[i]) for c in range(case["c"])]))
        if case["train"]:
            g = (grad if case["b"] else grad[None])[i].double()
            g = g if case["layout"] == "pair" else g.permute(1, 2, 0)
            total.index_add_(0, u[i].flatten(), g.reshape(-1, case["c"]))
    out = torch.stack(outs) if case["b"] else outs[0]
    return (out, total) if case["train"] else out


def _exact_cross(s, case):
    b, h, hk, d = case["b"], case["h"], case["hk"], case["d"]
    q, k, v = s["q"], s["k"], s["v"]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    dq, dk, dv = torch.zeros_like(out), k.double() * 0, v.double() * 0
    dbias = None if s["bias"] is None else s["bias"].double() * 0
    for i in range(b):
        keep = slice(None) if s["mask"] is None else s["mask"][i].nonzero()[:, 0]
        for a in range(h):
            c = a * hk // h
            qa, ka, va = q[i, :, a].double() / math.sqrt(d), k[i, keep, c].double(), v[i, keep, c].double()
            x = torch.einsum("id,jd->ij", qa, ka)
            if x.shape[1] == 0:
                continue
            ib = 0 if case["bias"] == "shared" else i
            if dbias is not None:
                x += s["bias"][ib, a][:, keep].double()
            p = torch.softmax(x, 1)
            out[i, :, a] = torch.einsum("ij,jd->id", p, va)
            if not case["train"]:
                continue
            g = s["grad"][i, :, a].double()
            gp = torch.einsum("id,jd->ij", g, va)
            ds = p * (gp - (p * gp).sum(1, keepdim=True))
            dq[i, :, a] = torch.einsum("ij,jd->id", ds, ka) / math.sqrt(d)
            dk[i, keep, c] += torch.einsum("ij,id->jd", ds, qa)
            dv[i, keep, c] += torch.einsum("ij,id->jd", p, g)
            if dbias is not None:
                dbias[ib, a][:, keep] += ds
    if not case["train"]:
        return out
    return (out, dq, dk, dv) if dbias is None else (out, dq, dk, dv, dbias)


# ------------------------------------------------------------------------------------------------
def work(case):
    """Bias: the tensor it is added to and the gradient are read once, the result written once; an add per
    element and direction.  Cross: queries, keys, values, bias and upstream gradient are read once, outputs
    and gradients written once; two products of the kept keys forward, five backward.  Padded keys need no work."""
    size = 2 if case["dtype"] == "bf16" else 4
    lq, lk, b = case["lq"], case["lk"], case["b"]
    if case["op"] == "bias":
        n = max(b, 1) * lq * lk * case["c"]
        kind, count, _ = _rule(case["rule"])
        passes = 1 + (case["layout"] == "pair") + case["train"]
        small = (count + (case["chains"] > 1)) * case["c"] * 4 * (1 + case["train"]) + max(b, 1) * (lq + lk) * 4
        return {"bytes": n * size * passes + small, "flops": n * ((case["layout"] == "pair") + case["train"])}
    h, hk, d = case["h"], case["hk"], case["d"]
    keys = sum(_lengths(case))                      # kept keys of the whole batch
    rows = b * lq * h * d * size                    # a tensor of the queries' shape
    kv = 2 * keys * hk * d * size                   # the kept keys and values
    bias = {"none": 0, "shared": h * lq * lk, "batch": h * lq * keys}[case["bias"]] * size
    mask = 0 if case["mask"] == "none" else b * lk
    product = 2 * keys * lq * h * d
    if not case["train"]:
        return {"bytes": 2 * rows + kv + bias + mask, "flops": 2 * product}
    return {"bytes": 4 * rows + 2 * kv + 2 * bias + mask, "flops": 7 * product}
