"""Cross attention on the GPU against its definition in 64 bits, with bounds that count roundings (``_ops64``)."""

import math

import pytest
import torch

from _ops64 import attention64, check

pytestmark = pytest.mark.gpu
BF16, FP32 = torch.bfloat16, torch.float32


def _inputs(B, Lq, Lk, H, Hk, D, bias, mask, dtype, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=gen, device="cuda").to(dtype)
    q, k, v, g = r(B, Lq, H, D), r(B, Lk, Hk, D), r(B, Lk, Hk, D), r(B, Lq, H, D)
    b = None if bias is None else r(*[{"B": B, "H": H}.get(c, 1) for c in bias], Lq, Lk)
    m = None
    if mask == "tail":
        m = torch.arange(Lk, device="cuda")[None] < torch.tensor([Lk - (Lk * i) // (2 * B) for i in range(B)], device="cuda")[:, None]
    elif mask == "holes":
        m = torch.rand(B, Lk, generator=gen, device="cuda") > 0.3
    elif mask == "empty":                    # the last batch element keeps nothing
        m = torch.ones(B, Lk, dtype=torch.bool, device="cuda")
        m[-1] = False
    return q, k, v, g, b, m


def _both(q, k, v, g, b, m, scale=None, **kw):
    """Forward and backward through the explicit calls."""
    from miniworld_engine_b200 import cross_attention_backward_b200, cross_attention_b200, cross_attention_forward_b200
    args = dict(bias=b, key_mask=m, scale=scale, **kw)
    out, state = cross_attention_forward_b200(q, k, v, **args)
    dq, dk, dv, db = cross_attention_backward_b200(g, q, k, v, out, state, **args)
    got = {"out": out, "dq": dq, "dk": dk, "dv": dv}
    if b is not None:
        got["dbias"] = db
    bare = cross_attention_b200(q, k, v, **args)             # without the backward pass's state
    return got, bare


def _check_all(q, k, v, g, b, m, scale=None, **kw):
    want = attention64(q, k, v, b, m, scale, g)
    got, bare = _both(q, k, v, g, b, m, scale, **kw)
    for name, w in want.items():
        check(got[name], w, name)
    check(bare, want["out"], "out alone")
    return got


SHAPES = [
    # B, Lq, Lk, H, Hk, D, bias, mask
    (1, 1, 1, 1, 1, 64, None, None),
    (2, 1, 300, 4, 2, 64, None, "tail"),
    (1, 3, 77, 4, 1, 32, "1H", None),
    (2, 61, 77, 4, 4, 32, "BH", "holes"),
    (2, 128, 128, 2, 2, 64, None, None),
    (1, 129, 257, 4, 2, 128, None, "holes"),
    (2, 300, 130, 4, 4, 64, "1H", "tail"),
    (3, 65, 200, 2, 1, 128, "B1", "empty"),
    (1, 256, 384, 2, 2, 128, "1H", None),
    (2, 130, 513, 4, 4, 48, "11", "holes"),
    (1, 200, 100, 3, 3, 24, "BH", None),
    (1, 40, 50, 2, 2, 8, None, "tail"),
    (1, 70, 90, 2, 2, 96, "1H", "tail"),
    (1, 17, 33, 2, 1, 20, "BH", "holes"),
    (1, 33, 40, 2, 2, 136, None, "tail"),
    (1, 20, 35, 2, 2, 256, "1H", None),
    (1, 9, 11, 1, 1, 1, None, None),
    (1, 520, 1030, 2, 1, 64, None, "holes"),
]


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("B,Lq,Lk,H,Hk,D,bias,mask", SHAPES)
def test_against_the_definition(B, Lq, Lk, H, Hk, D, bias, mask, dtype):
    _check_all(*_inputs(B, Lq, Lk, H, Hk, D, bias, mask, dtype))


@pytest.mark.parametrize("B,Lq,Lk,H,Hk,D,bias,mask", SHAPES[3:9])
def test_cuda_core_kernels_in_bf16(B, Lq, Lk, H, Hk, D, bias, mask):
    _check_all(*_inputs(B, Lq, Lk, H, Hk, D, bias, mask, BF16), plain_kernels=True)


@pytest.mark.parametrize("Lq", [1, 2, 5, 8, 15, 16, 17, 64])
@pytest.mark.parametrize("Lk", [2, 31, 128, 1000, 5000])
@pytest.mark.parametrize("H,Hk,D", [(4, 4, 64), (8, 2, 128)])
def test_few_query_rows(Lq, Lk, H, Hk, D):
    q, k, v, g, b, m = _inputs(2, Lq, Lk, H, Hk, D, "1H", "tail", BF16, seed=Lq)
    _check_all(q, k, v, g, b, m)
    _check_all(q, k, v, g, None, None)


@pytest.mark.parametrize("dtype,D", [(BF16, 64), (BF16, 128), (FP32, 32)])
def test_masked_places_may_hold_anything(dtype, D):
    q, k, v, g, b, m = _inputs(2, 150, 300, 2, 2, D, "BH", "holes", dtype)
    m[1] = False
    m[1, :20] = True
    clean = _both(q, k, v, g, b, m)
    k2, v2, b2 = k.clone(), v.clone(), b.clone()
    k2[~m], v2[~m] = math.nan, math.inf
    b2.masked_fill_(~m[:, None, None, :], math.nan)
    dirty = _both(q, k2, v2, g, b2, m)
    for name in clean[0]:
        assert torch.equal(clean[0][name], dirty[0][name]), name
    assert torch.equal(clean[1], dirty[1])
    assert not dirty[0]["dk"][~m].any() and not dirty[0]["dv"][~m].any()
    _check_all(q, k2, v2, g, torch.where(m[:, None, None, :], b2, 0), m)


@pytest.mark.parametrize("dtype,Lq,D", [(BF16, 150, 64), (BF16, 150, 128), (BF16, 1, 64), (FP32, 40, 32)])
def test_rows_masked_by_the_bias(dtype, Lq, D):
    """Minus infinity on whole rows: zeros.  The type's lowest value on whole rows: it swallows every score, and each key
    gets the same share."""
    q, k, v, g, b, m = _inputs(1, Lq, 200, 2, 2, D, "BH", None, dtype)
    b[0, 0, ::3] = -math.inf
    b[0, 1, ::3] = torch.finfo(dtype).min
    b[0, :, :, 50:60] = -math.inf
    got = _check_all(q, k, v, g, b, m)
    assert not got["out"][0, ::3, 0].any() and not got["dq"][0, ::3, 0].any()
    share = v.double()[0, :, 1].mean(0) * 200 / 190 - v.double()[0, 50:60, 1].sum(0) / 190
    assert (got["out"][0, 0, 1].double() - share).abs().max() < 0.01
    b[:] = torch.finfo(dtype).min
    _check_all(q, k, v, g, b, m)
    b[:] = -math.inf
    got = _check_all(q, k, v, g, b, m)
    assert not any(t.any() for t in got.values())


def test_nothing_kept_at_all():
    for dtype in (BF16, FP32):
        q, k, v, g, b, _ = _inputs(2, 140, 150, 2, 1, 64, "11", None, dtype)
        got = _check_all(q, k, v, g, b, torch.zeros(2, 150, dtype=torch.bool, device="cuda"))
        assert not any(t.any() for t in got.values())


@pytest.mark.parametrize("shape", [(0, 4, 5), (2, 0, 5), (2, 4, 0)])
def test_empty(shape):
    B, Lq, Lk = shape
    q, k, v, g, b, _ = _inputs(B, Lq, Lk, 4, 2, 64, "1H", None, BF16)
    got, bare = _both(q, k, v, g, b, None)
    assert bare.shape == q.shape and not bare.any()
    assert all(not t.any() for t in got.values()) and got["dbias"].shape == b.shape and got["dk"].shape == k.shape


def test_large_scores_and_scale():
    q, k, v, g, b, m = _inputs(1, 140, 260, 2, 2, 64, "1H", "holes", BF16)
    _check_all(q * 8, k * 8, v, g, b, m)                  # nearly one-hot rows
    _check_all(q, k, v, g, b, m, scale=-0.3)
    _check_all(q, k, v, g, b, m, scale=0.0)
    rising = torch.linspace(0, 400, 260, device="cuda").bfloat16().expand(1, 1, 140, 260)      # maxima grow tile by tile
    _check_all(q, k, v, g, rising.contiguous(), m)
    _check_all(q, k, v, g, rising.flip(-1).contiguous(), m)


@pytest.mark.parametrize("D", [64, 128, 32])
def test_layouts(D):
    q, k, v, g, b, m = _inputs(2, 70, 150, 4, 2, D, "BH", "tail", BF16)
    got, bare = _both(q, k, v, g, b, m)
    heads_first = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v, g)]
    packed = torch.cat([k, v], -1)                        # one projection, split
    wide = torch.zeros(2, 4, 80, 170, device="cuda").bfloat16()
    wide[:, :, 3:73, 5:155] = b
    odd = torch.empty(q.numel() + 1, dtype=BF16, device="cuda")[1:].view(q.shape).copy_(q)
    strided_mask = torch.zeros(2, 300, dtype=torch.bool, device="cuda")[:, ::2].copy_(m)
    for args in ((*heads_first, b, m), (q, packed[..., :D], packed[..., D:], g, b, m),
                 (q, k, v, g, wide[:, :, 3:73, 5:155], m), (odd, k, v, g, b, m),
                 (q, k, v, g, b.transpose(2, 3).contiguous().transpose(2, 3), strided_mask),
                 (q.transpose(1, 3).contiguous().transpose(1, 3), k, v, g, b, m)):
        other, bare2 = _both(*args)
        assert torch.equal(bare, bare2)
        for name in got:
            assert torch.equal(got[name], other[name]), name
    # repeated in place: a key head for all, a gradient of ones
    one = k[:, :, :1].expand(2, 150, 2, D)
    _check_all(q, one, one, torch.ones(1, 1, 1, 1, device="cuda").bfloat16().expand_as(q), b, m)


def test_shared_bias_gradient_is_the_sum_over_what_shares_it():
    for bias in ("11", "1H", "B1"):
        for dtype in (BF16, FP32):
            _check_all(*_inputs(3, 90, 75, 4, 2, 64, bias, "holes", dtype))
    q, k, v, g, b, m = _inputs(2, 50, 60, 2, 2, 64, "1H", None, BF16)
    flat = b[0]                                           # [H, Lq, Lk]
    want = attention64(q, k, v, flat, m, None, g)
    got, _ = _both(q, k, v, g, flat, m)
    assert got["dbias"].shape == flat.shape
    check(got["dbias"], want["dbias"], "dbias")


@pytest.mark.parametrize("dtype,D", [(BF16, 64), (BF16, 128), (FP32, 32)])
def test_same_bits_every_time(dtype, D):
    args = _inputs(2, 333, 700, 4, 2, D, "1H", "holes", dtype)
    first, bare = _both(*args)
    for _ in range(3):
        again, bare2 = _both(*args)
        assert torch.equal(bare, bare2) and all(torch.equal(first[n], again[n]) for n in first)


def test_autograd_matches_the_explicit_calls_and_differences():
    from miniworld_engine_b200 import cross_attention_b200
    q, k, v, g, b, m = _inputs(2, 30, 40, 4, 2, 16, "1H", "tail", FP32)
    got, _ = _both(q, k, v, g, b, m)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v, b)]
    cross_attention_b200(*leaves[:3], bias=leaves[3], key_mask=m).backward(g)
    for t, name in zip(leaves, ("dq", "dk", "dv", "dbias")):
        assert torch.equal(t.grad, got[name]), name
    # central differences of the 64-bit definition in a random direction agree with the kernels' gradients
    gen = torch.Generator(device="cuda").manual_seed(5)
    for i, name in enumerate(("dq", "dk", "dv", "dbias")):
        base = [t.double() for t in (q, k, v, b)]
        step = torch.randn(base[i].shape, generator=gen, device="cuda", dtype=torch.float64)
        if name in ("dk", "dv"):
            step[~m] = 0
        values = []
        for sign in (1, -1):
            moved = list(base)
            moved[i] = base[i] + sign * 1e-5 * step
            out = attention64(*moved[:3], moved[3], m)["out"][0]
            values.append((out * g.double()).sum())
        diff = float(values[0] - values[1]) / 2e-5
        mine = float((got[name].double() * step).sum())
        size = float((got[name].double() * step).abs().sum())
        assert abs(diff - mine) <= 1e-5 * size + 1e-6, name
    only_bias = b.clone().requires_grad_(True)
    cross_attention_b200(q, k, v, bias=only_bias, key_mask=m).sum().backward()
    with torch.no_grad():
        assert not cross_attention_b200(q, k, v, bias=only_bias, key_mask=m).requires_grad
    only_q = q.clone().requires_grad_(True)
    cross_attention_b200(only_q, k, v, bias=b).backward(g)
    assert only_q.grad is not None and b.grad is None


def test_streams_graphs_and_status():
    from miniworld_engine_b200 import read_status
    cases = [_inputs(2, 200, 300, 4, 2, 64, "1H", "holes", BF16, seed=s) for s in (1, 2)]
    few = [_inputs(2, 1, 3000, 4, 2, 64, None, "tail", BF16, seed=s) for s in (3, 4)]
    for pair in (cases, few):
        want = [_both(*c) for c in pair]
        graphs, outs = [], []
        for c in pair:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                outs.append(_both(*c))
            graphs.append(graph)
        streams = [torch.cuda.Stream() for _ in range(2)]
        torch.cuda.synchronize()
        for _ in range(4):
            for s, graph in zip(streams, graphs):
                with torch.cuda.stream(s):
                    graph.replay()
        torch.cuda.synchronize()
        for (got, bare), (w, wb) in zip(outs, want):
            assert torch.equal(bare, wb) and all(torch.equal(got[n], w[n]) for n in w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, bare = _both(*cases[0])
    side.synchronize()
    want, wb = _both(*cases[0])
    assert torch.equal(bare, wb) and all(torch.equal(got[n], want[n]) for n in want)
    assert read_status()[0] == 0


def test_learned_bias_and_attention_together():
    """A training step as the two operators are used: table -> bias -> attention, odd lengths, two chains."""
    from miniworld_engine_b200 import PositionBuckets, RelativePositionBiasB200, cross_attention_b200
    torch.manual_seed(0)
    B, Lq, Lk, H, D = 2, 131, 203, 4, 64
    q, k, v, g, _, m = _inputs(B, Lq, Lk, H, H, D, None, "tail", BF16)
    mod = RelativePositionBiasB200(PositionBuckets.logarithmic(32, 128, segments=True), H, dtype=BF16).cuda()
    with torch.no_grad():
        mod.weight.normal_()
    qp, kp = torch.arange(Lq, device="cuda"), torch.arange(Lk, device="cuda") - 20
    qs, ks = (torch.arange(n, device="cuda") > 90 for n in (Lq, Lk))
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    bias = mod(qp, kp, qs.int(), ks.int())
    cross_attention_b200(*leaves, bias=bias, key_mask=m).backward(g)
    from _ops64 import bucket_matrix
    u = bucket_matrix(qp, kp, "log", 32, 128, qs, ks).cuda()
    want = attention64(q, k, v, bias.detach(), m, None, g)
    for t, name in zip(leaves, ("dq", "dk", "dv")):
        check(t.grad, want[name], name)
    sums = lambda t: torch.zeros(33, H, dtype=torch.float64, device="cuda").index_add_(
        0, u.flatten(), t.movedim(0, -1).reshape(-1, H))
    value, bound = (sums(t) for t in want["dbias"])
    n = torch.bincount(u.flatten(), minlength=33)[:, None] * 2.0 ** -24
    check(mod.weight.grad, (value, bound + n * sums(want["dbias"][0].abs())), "table")


@pytest.mark.parametrize("Lq", [1, 40])
def test_offsets_beyond_32_bits(Lq):
    """Keys, values and a bias whose rows lie more than 2^31 elements apart in all."""
    step = 1 << 26
    Lk, H, D = 40, 2, 64
    big = torch.empty(Lk * step, dtype=BF16, device="cuda")                # 5.4 GB
    q, k, v, g, b, m = _inputs(1, Lq, Lk, H, H, D, "1H", "holes", BF16)
    far = lambda t, at: torch.as_strided(big, t.shape, (Lk * step, step, D, 1), at).copy_(t)
    k2, v2 = far(k, 0), far(v, 1024)
    rows = torch.as_strided(big, b.shape, (Lk * step, Lq * step, step, 1), 4096) if Lq <= 20 else b
    if rows is not b:
        rows.copy_(b)
    got, bare = _both(q, k2, v2, g, rows, m)
    want, wb = _both(q, k, v, g, b, m)
    assert torch.equal(bare, wb) and all(torch.equal(got[n], want[n]) for n in want)


def test_first_calls_inside_a_capture_and_backward_twice():
    """Gradients accumulate as autograd has it, and the explicit calls may be captured without a call before."""
    from miniworld_engine_b200 import cross_attention_b200
    q, k, v, g, b, m = _inputs(1, 77, 93, 2, 2, 40, "1H", "tail", BF16)       # a head dimension no other test has
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, bare = _both(q, k, v, g, b, m)
    graph.replay()
    torch.cuda.synchronize()
    want = attention64(q, k, v, b, m, None, g)
    for name in want:
        check(got[name], want[name], name)
    leaves = [t.float().requires_grad_(True) for t in (q, k, v, b)]
    for _ in range(2):
        cross_attention_b200(*leaves[:3], bias=leaves[3], key_mask=m).backward(g.float())
    once = [t.clone().requires_grad_(True) for t in (x.detach() for x in leaves)]
    cross_attention_b200(*once[:3], bias=once[3], key_mask=m).backward(g.float())
    for a, c in zip(leaves, once):
        assert torch.equal(a.grad, 2 * c.grad)


@pytest.mark.parametrize("dtype,plain", [(BF16, False), (BF16, True), (FP32, False)])
@pytest.mark.parametrize("B,Lq,Lk,H,Hk,D,bias", [
    (1, 61, 2100, 2, 2, 64, "1H"),
    (1, 2100, 61, 4, 2, 128, None),
    (2, 40, 1500, 2, 1, 96, "BH"),
    (1, 900, 10, 2, 2, 32, "11"),
    (1, 1030, 1700, 1, 1, 40, "BH"),
    (2, 9, 700, 1, 1, 136, "1H"),
])
def test_loops_that_several_blocks_share(B, Lq, Lk, H, Hk, D, bias, dtype, plain):
    """Few tiles on one side and many on the other; masks that leave some blocks' shares without a key."""
    q, k, v, g, b, _ = _inputs(B, Lq, Lk, H, Hk, D, bias, None, dtype, seed=Lk)
    _check_all(q, k, v, g, b, None, plain_kernels=plain)
    mask = torch.zeros(B, Lk, dtype=torch.bool, device="cuda")
    mask[:, Lk // 2:Lk // 2 + 3] = True
    mask[0, -1] = True
    first = _check_all(q, k, v, g, b, mask, plain_kernels=plain)
    again, _ = _both(q, k, v, g, b, mask, plain_kernels=plain)
    for name in first:
        assert torch.equal(first[name], again[name]), name
    mask[-1] = False
    _check_all(q, k, v, g, b, mask, plain_kernels=plain)


@pytest.mark.parametrize("Lq,D", [(1, 96), (9, 64), (40, 20)])
def test_shared_bias_gradient_of_a_small_call_is_rounded_once(Lq, D):
    """Half a bf16 step of the sum (2^-8), and of every summand the fp32 arithmetic and the 16 bits of ``o`` in delta: far
    below 2^-12 of p (|dout . v| + |delta|).  Rounding every summand to bf16 first would be off by up to 2^-8 of those.
    delta is taken from the result that the forward pass returned: its probabilities are rounded to bf16 on their way into
    the product with v, which moves delta by up to 2^-8 of sum p |dout . v| and is no part of this rounding."""
    from miniworld_engine_b200 import cross_attention_backward_b200, cross_attention_forward_b200
    q, k, v, g, b, _ = _inputs(4, Lq, 70, 2, 2, D, "1H", None, BF16, seed=Lq)
    out, state = cross_attention_forward_b200(q, k, v, bias=b)
    got = cross_attention_backward_b200(g, q, k, v, out, state, bias=b)[3].double()
    o = out.double() + state.rounding.double()
    q, k, v, g, o = (t.double().transpose(1, 2) for t in (q, k, v, g, o))
    p = (q @ k.mT * D ** -0.5 + b.double()).softmax(-1)
    dp = g @ v.mT
    delta = (g * o).sum(-1, keepdim=True)
    want, size = (p * (dp - delta)).sum(0), (p * (dp.abs() + delta.abs())).sum(0)
    assert (((got - want).abs() - 2.0 ** -8 * want.abs()) <= 2.0 ** -12 * size).all()


@pytest.mark.parametrize("plain", [False, True])
@pytest.mark.parametrize("B,H,Lq,Lk,D,bias", [(4, 8, 300, 400, 64, "1H"), (2, 4, 270, 514, 128, "B1"), (3, 5, 400, 333, 32, "11")])
def test_shared_bias_gradient_of_a_large_call_is_rounded_once(B, H, Lq, Lk, D, bias, plain):
    """As for small calls, with summands that nearly cancel: batch elements (heads) come in pairs of the same inputs, the
    second one's upstream gradient minus 0.9 times the first one's.  Bounds as there; half a step of every summand would be
    up to 2^-8 of 1.9 |ds| against a sum of 0.1 |ds|."""
    from miniworld_engine_b200 import cross_attention_backward_b200, cross_attention_forward_b200
    q, k, v, g, b, _ = _inputs(B, Lq, Lk, H, H, D, bias, None, BF16, seed=B)
    for t in (q, k, v):
        if bias != "B1":
            t[1] = t[0]
        else:
            t[:, :, 1] = t[:, :, 0]
    if bias != "B1":
        g[1] = -0.9 * g[0]
        g[2:] *= 0.01                        # and little beside the pair
    else:
        g[:, :, 1] = -0.9 * g[:, :, 0]
        g[:, :, 2:] *= 0.01
    out, state = cross_attention_forward_b200(q, k, v, bias=b, plain_kernels=plain)
    got = cross_attention_backward_b200(g, q, k, v, out, state, bias=b, plain_kernels=plain)[3].double()
    o = out.double() + state.rounding.double()
    q, k, v, g, o = (t.double().transpose(1, 2) for t in (q, k, v, g, o))
    p = (q @ k.mT * D ** -0.5 + b.double()).softmax(-1)
    dp = g @ v.mT
    delta = (g * o).sum(-1, keepdim=True)
    want, size = p * (dp - delta), p * (dp.abs() + delta.abs())
    for axis in (0, 1):
        if b.shape[axis] == 1:
            want, size = want.sum(axis, keepdim=True), size.sum(axis, keepdim=True)
    assert got.shape == want.shape
    assert (((got - want).abs() - 2.0 ** -8 * want.abs()) <= 2.0 ** -12 * size).all()


@pytest.mark.parametrize("D", [128, 96, 64])
@pytest.mark.parametrize("bias", [None, "11"])
def test_first_calls_on_cold_inputs(D, bias):
    """Keys and values that come late and in any order: fresh inputs, nothing of them in the L2, a mask with holes or a
    tail.  The call is right, and the same bits come again when the inputs are warm."""
    from miniworld_engine_b200 import cross_attention_b200, read_status
    flush = torch.empty(1 << 28, dtype=torch.uint8, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(D)
    r = lambda *s: torch.randn(s, generator=gen, device="cuda").bfloat16()
    for step in range(40):
        Lq = (5, 129, 300)[step % 3]
        q, k, v = r(5, Lq, 4, D), r(5, 4100, 4, D), r(5, 4100, 4, D)
        b = None if bias is None else r(1, 1, Lq, 4100)
        m = (torch.rand(5, 4100, generator=gen, device="cuda") > 0.4 if step % 2 else
             torch.arange(4100, device="cuda")[None] < torch.randint(1, 4101, (5, 1), generator=gen, device="cuda"))
        flush.zero_()
        first = cross_attention_b200(q, k, v, bias=b, key_mask=m)
        again = cross_attention_b200(q, k, v, bias=b, key_mask=m)
        assert torch.equal(first, again), step
        if step < 6:
            check(first, attention64(q, k, v, b, m)["out"], "out")
    assert read_status()[0] == 0
