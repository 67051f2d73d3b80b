"""The relative position bias on the GPU against its definition.

Forward results are one rounding of an fp32 value, so they are compared for equality with the same value rounded
by torch.  Gradients are tested with whole-number upstream values (every fp32 sum is then exact, so a missing or
doubled element shows) and with random ones, where a sum of n terms in any order is off by at most n 2^-24 times the
sum of their absolute values.
"""

import pytest
import torch

from _ops64 import bucket_matrix

pytestmark = pytest.mark.gpu

RULES = {"clip4": ("clip", 9, 4), "clip32": ("clip", 65, 32), "log32": ("log", 32, 128), "causal": ("causal", 32, 128),
         "log_wide": ("log", 64, 4000), "clip300": ("clip", 601, 300), "clip0": ("clip", 1, 0)}


def _rule(name, segments):
    from miniworld_engine_b200 import PositionBuckets
    kind, count, top = RULES[name]
    if kind == "clip":
        return PositionBuckets.clipped(top, segments=segments)
    return PositionBuckets.logarithmic(count, top, bidirectional=kind == "log", segments=segments)


def _case(rule, B, Lq, Lk, segments, wide=False, seed=0, spread=3):
    """Positions (shuffled, with repeats), segments, and the expected buckets."""
    gen = torch.Generator().manual_seed(seed)
    to = torch.int64 if wide else torch.int32
    shape = lambda n: (B, n) if B else (n,)
    q, k = (torch.randint(-spread * n, spread * n + 1, shape(n), generator=gen).to(to) for n in (Lq, Lk))
    kind, count, top = RULES[rule]
    qs = ks = None
    if segments:
        qs, ks = (torch.randint(0, 3, shape(n), generator=gen).to(to) for n in (Lq, Lk))
    u = bucket_matrix(q, k, kind, count, top, qs, ks)
    dev = lambda t: None if t is None else t.cuda()
    return _rule(rule, segments), dev(q), dev(k), {"q_segment": dev(qs), "k_segment": dev(ks)}, u.cuda()


SHAPES = [("clip32", 0, 64, 64, False, False), ("clip4", 0, 1, 1, False, False), ("log32", 2, 33, 65, True, True),
          ("causal", 0, 7, 300, False, True), ("clip32", 3, 129, 40, True, False), ("log_wide", 0, 70, 9, False, False),
          ("clip300", 1, 40, 77, True, False), ("clip0", 0, 5, 1027, False, False), ("clip32", 0, 300, 1, False, False)]


@pytest.mark.parametrize("rule,B,Lq,Lk,segments,wide", SHAPES)
@pytest.mark.parametrize("channels", [1, 4, 12, 16])
@pytest.mark.parametrize("dtype,table_dtype", [(torch.bfloat16, torch.float32), (torch.float32, torch.float32),
                                               (torch.bfloat16, torch.bfloat16)])
def test_heads(rule, B, Lq, Lk, segments, wide, channels, dtype, table_dtype):
    from miniworld_engine_b200 import relative_position_bias_b200, relative_position_bias_backward_b200
    buckets, q, k, seg, u = _case(rule, B, Lq, Lk, segments, wide)
    gen = torch.Generator(device="cuda").manual_seed(1)
    table = torch.randn(buckets.rows, channels, generator=gen, device="cuda").to(table_dtype)
    out = relative_position_bias_b200(table, buckets, q, k, dtype=dtype, **seg)
    want = table[u].to(dtype).movedim(-1, -3)
    assert out.dtype == dtype and out.shape == want.shape and torch.equal(out, want)
    assert out.stride(-2) * out.element_size() % 16 == 0

    whole = torch.randint(-3, 4, want.shape, generator=gen, device="cuda").to(dtype)
    sums = torch.zeros(buckets.rows, channels, dtype=torch.float64, device="cuda")
    sums.index_add_(0, u.flatten(), whole.movedim(-3, -1).reshape(-1, channels).double())
    for g in (whole, _like(whole, out)):                       # dense rows, and rows on 16 bytes as the result has
        got = relative_position_bias_backward_b200(g, buckets, q, k, **seg)
        assert got.dtype == torch.float32 and torch.equal(got.double(), sums)


def _like(values, layout):
    t = torch.empty_strided(layout.shape, layout.stride(), dtype=layout.dtype, device="cuda")
    return t.copy_(values)


@pytest.mark.parametrize("rule,B,Lq,Lk,segments,wide", SHAPES)
@pytest.mark.parametrize("channels", [3, 8, 64, 128, 192, 520])
@pytest.mark.parametrize("dtype,table_dtype", [(torch.bfloat16, torch.float32), (torch.float32, torch.float32),
                                               (torch.float32, torch.bfloat16)])
def test_pair(rule, B, Lq, Lk, segments, wide, channels, dtype, table_dtype):
    from miniworld_engine_b200 import relative_position_bias_b200, relative_position_bias_backward_b200
    buckets, q, k, seg, u = _case(rule, B, Lq, Lk, segments, wide, seed=2)
    gen = torch.Generator(device="cuda").manual_seed(3)
    table = torch.randn(buckets.rows, channels, generator=gen, device="cuda").to(table_dtype)
    add = torch.randn(*u.shape, channels, generator=gen, device="cuda").to(dtype)
    out = relative_position_bias_b200(table, buckets, q, k, layout="pair", add=add, **seg)
    assert torch.equal(out, (add.float() + table.float()[u]).to(dtype))
    bare = relative_position_bias_b200(table, buckets, q, k, layout="pair", dtype=dtype, **seg)
    assert torch.equal(bare, table[u].to(dtype))

    whole = torch.randint(-3, 4, out.shape, generator=gen, device="cuda").to(dtype)
    sums = torch.zeros(buckets.rows, channels, dtype=torch.float64, device="cuda")
    sums.index_add_(0, u.flatten(), whole.reshape(-1, channels).double())
    got = relative_position_bias_backward_b200(whole, buckets, q, k, layout="pair", **seg)
    assert torch.equal(got.double(), sums)


@pytest.mark.parametrize("layout", ["heads", "pair"])
@pytest.mark.parametrize("chains", [False, True])
def test_residue_numbers_in_order(layout, chains):
    """Positions as structures have them: runs of consecutive numbers, where most of a row shares a bucket."""
    from miniworld_engine_b200 import relative_position_bias_b200, relative_position_bias_backward_b200
    n, c = 611, 16 if layout == "heads" else 128
    pos = torch.arange(n, device="cuda", dtype=torch.int32) - (torch.arange(n, device="cuda") >= 400).int() * 400
    seg = (torch.arange(n, device="cuda") >= 400).long()
    kw = {"q_segment": seg} if chains else {}
    buckets = _rule("clip32", chains)
    u = bucket_matrix(pos, pos, "clip", 65, 32, seg if chains else None, seg if chains else None).cuda()
    table = torch.randn(buckets.rows, c, device="cuda")
    want = table[u].bfloat16()
    want = want if layout == "pair" else want.movedim(-1, 0)
    assert torch.equal(relative_position_bias_b200(table, buckets, pos, layout=layout, dtype=torch.bfloat16, **kw), want)
    g = torch.randn(want.shape, device="cuda").bfloat16()
    flat = (g if layout == "pair" else g.movedim(0, -1)).reshape(-1, c).double()
    sums, size = (torch.zeros(buckets.rows, c, dtype=torch.float64, device="cuda").index_add_(0, u.flatten(), t)
                  for t in (flat, flat.abs()))
    count = torch.bincount(u.flatten(), minlength=buckets.rows)[:, None]
    got = relative_position_bias_backward_b200(g, buckets, pos, layout=layout, **kw)
    assert ((got.double() - sums).abs() <= count * 2.0 ** -24 * size).all()
    again = relative_position_bias_backward_b200(g, buckets, pos, layout=layout, **kw)
    assert torch.equal(got, again)
    low = relative_position_bias_backward_b200(g, buckets, pos, layout=layout, dtype=torch.bfloat16, **kw)
    assert torch.equal(low, got.bfloat16())


def test_far_positions_and_broadcast_batches():
    from miniworld_engine_b200 import relative_position_bias_b200
    buckets = _rule("clip32", False)
    q = torch.tensor([[2 ** 30, -2 ** 30, 5], [2 ** 62, -2 ** 62, 0]], device="cuda")
    k = torch.tensor([-2 ** 30, 2 ** 30, 7, 2 ** 40], device="cuda")
    table = torch.randn(65, 8, device="cuda")
    lim = 2 ** 30
    u = bucket_matrix(q.clamp(-lim, lim), k.clamp(-lim, lim), "clip", 65, 32).cuda()
    assert torch.equal(relative_position_bias_b200(table, buckets, q, k), table[u].movedim(-1, -3))
    wide = k[None].expand(2, 4)                                  # repeated in place along the batch
    assert torch.equal(relative_position_bias_b200(table, buckets, q, wide), table[u].movedim(-1, -3))
    every_other = torch.arange(20, device="cuda")[::2]
    u = bucket_matrix(every_other, every_other, "clip", 65, 32).cuda()
    assert torch.equal(relative_position_bias_b200(table, buckets, every_other), table[u].movedim(-1, -3))


def test_strides_of_the_gradient():
    from miniworld_engine_b200 import relative_position_bias_backward_b200
    buckets, q, k, _, u = _case("clip4", 2, 37, 50, False)
    big = torch.randint(-3, 4, (2, 5, 40, 60), device="cuda").bfloat16()
    for g in (big[:, :4, 1:38, 3:53], big.transpose(2, 3)[:, :4, :37, :40].expand(2, 4, 37, 40),
              torch.ones(1, 1, 1, 1, device="cuda").bfloat16().expand(2, 4, 37, 50)):
        lk = g.shape[-1]
        sums = torch.zeros(9, 4, dtype=torch.float64, device="cuda")
        sums.index_add_(0, u[..., :lk].flatten(), g.movedim(1, -1).reshape(-1, 4).double())
        assert torch.equal(relative_position_bias_backward_b200(g, buckets, q, k[:, :lk]).double(), sums)


@pytest.mark.parametrize("layout,shape", [("heads", (0, 5)), ("heads", (5, 0)), ("pair", (0, 0))])
def test_empty(layout, shape):
    from miniworld_engine_b200 import relative_position_bias_b200, relative_position_bias_backward_b200
    buckets = _rule("clip4", False)
    q, k = (torch.arange(n, device="cuda") for n in shape)
    out = relative_position_bias_b200(torch.ones(9, 8, device="cuda"), buckets, q, k, layout=layout)
    assert out.numel() == 0 and out.shape == ((8, *shape) if layout == "heads" else (*shape, 8))
    assert not relative_position_bias_backward_b200(out, buckets, q, k, layout=layout).any()


@pytest.mark.parametrize("layout", ["heads", "pair"])
def test_autograd_and_module(layout):
    from miniworld_engine_b200 import PositionBuckets, RelativePositionBiasB200
    torch.manual_seed(0)
    n, c = 45, 8
    mod = RelativePositionBiasB200(PositionBuckets.clipped(4, segments=True), c, layout=layout).cuda()
    pos, seg = torch.arange(n, device="cuda").repeat(2, 1), (torch.arange(n, device="cuda") > 20).int().repeat(2, 1)
    add = torch.randn(2, n, n, c, device="cuda", requires_grad=True) if layout == "pair" else None
    out = mod(pos, q_segment=seg, add=add)
    g = torch.randint(-2, 3, out.shape, device="cuda").float()
    out.backward(g)
    u = bucket_matrix(pos, pos, "clip", 9, 4, seg, seg).cuda()
    w = mod.weight.detach().clone().requires_grad_(True)
    ref = w[u] + add.detach() if layout == "pair" else w[u].movedim(-1, 1)
    ref.backward(g)
    assert torch.equal(out.detach(), ref.detach()) and torch.equal(mod.weight.grad, w.grad)
    if add is not None:
        assert torch.equal(add.grad, g)
    # against differences: the result is linear in the table
    step = torch.zeros_like(mod.weight)
    step[3, 2] = 1.0
    with torch.no_grad():
        base = mod(pos, q_segment=seg, add=add)
        mod.weight += step
        moved = mod(pos, q_segment=seg, add=add)
    diff = ((moved.double() - base.double()) * g).sum()
    assert abs(float(diff) - float(w.grad[3, 2])) <= 1e-3 * float(g.abs().sum() + 1)


def test_streams_and_graphs():
    from miniworld_engine_b200 import relative_position_bias_b200, relative_position_bias_backward_b200
    buckets, q, k, _, u = _case("clip32", 0, 130, 200, False)
    tables = [torch.randn(65, 8, device="cuda") for _ in range(2)]
    grads = [torch.randint(-3, 4, (8, 130, 200), device="cuda").bfloat16() for _ in range(2)]

    def call(t, g):
        return (relative_position_bias_b200(t, buckets, q, k),
                relative_position_bias_backward_b200(g, buckets, q, k))

    want = [call(t, g) for t, g in zip(tables, grads)]
    graphs, outs = [], []
    for t, g in zip(tables, grads):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(call(t, g))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):                        # both at once: they share no workspace
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert torch.equal(o[0], w[0]) and torch.equal(o[1], w[1])


@pytest.mark.parametrize("layout", ["heads", "pair"])
def test_offsets_beyond_32_bits(layout):
    """Results and gradients of more than 2^31 elements: the last rows are right, and every element is counted."""
    from miniworld_engine_b200 import relative_position_bias_b200, relative_position_bias_backward_b200
    n, c = (12000, 16) if layout == "heads" else (4200, 128)
    pos = torch.arange(n, device="cuda")
    buckets = _rule("clip32", False)
    table = torch.randn(65, c, device="cuda")
    out = relative_position_bias_b200(table, buckets, pos, layout=layout, dtype=torch.bfloat16)
    assert out.numel() > 2 ** 31
    last = bucket_matrix(pos[-3:], pos, "clip", 65, 32).cuda()
    if layout == "heads":
        assert torch.equal(out[:, -3:], table[last].bfloat16().movedim(-1, 0))
    else:
        assert torch.equal(out[-3:], table[last].bfloat16())
    out.fill_(2.0 ** -10)
    got = relative_position_bias_backward_b200(out, buckets, pos, layout=layout)
    d = torch.arange(-32, 33, device="cuda")
    pairs = n - d.abs()
    pairs[0] = pairs[-1] = (n - 32) * (n - 31) // 2
    # counts up to 7e7 do not fit into 24 bits: exact within a part (less than 2^24 elements), then at most 2^10 parts are
    # added, each addition off by 2^-24 of the sum.  A row left out would be 2^-13.6 of it
    want = (pairs.double() * 2.0 ** -10)[:, None]
    assert ((got.double() - want).abs() <= 2.0 ** -14 * want).all()


def _far_ids(to):
    """Segment ids that agree in what a clamp, a low word or a sign would leave of them."""
    if to is torch.int32:
        return [2 ** 30, 2 ** 30 + 1, 2 ** 31 - 1, -2 ** 30, -2 ** 30 - 1, -2 ** 31, 0x41414141, 0x42414141, 0, -1]
    return [2 ** 30, 2 ** 30 + 1, 2 ** 32, 2 ** 33, 5, 2 ** 32 + 5, 2 ** 40 + 5, -2 ** 32 + 5, 2 ** 63 - 1, -2 ** 63, -1, 2 ** 32 - 1]


@pytest.mark.parametrize("layout,channels", [("heads", 8), ("heads", 1), ("pair", 64), ("pair", 3)])
@pytest.mark.parametrize("q_type,k_type", [(torch.int32, torch.int32), (torch.int64, torch.int64), (torch.int64, torch.int32),
                                           (torch.int32, torch.int64)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_segments_are_told_apart_whatever_their_numbers(layout, channels, q_type, k_type, dtype):
    from miniworld_engine_b200 import relative_position_bias_b200, relative_position_bias_backward_b200
    gen = torch.Generator().manual_seed(9)
    ids = lambda to: torch.tensor(_far_ids(to), dtype=torch.int64)
    Lq, Lk = 75, 130
    qs = ids(q_type)[torch.randint(len(ids(q_type)), (Lq,), generator=gen)]
    ks = ids(k_type)[torch.randint(len(ids(k_type)), (Lk,), generator=gen)]
    ks[40:80] = ids(k_type)[0]                                  # runs of one segment: the gradients add them up together
    qs[20:60] = ids(q_type)[1]
    q, k = torch.randint(-9, 10, (Lq,), generator=gen), torch.arange(Lk) - 60
    u = bucket_matrix(q, k, "clip", 9, 4, qs, ks).cuda()
    buckets = _rule("clip4", True)
    kw = {"q_segment": qs.to(q_type).cuda(), "k_segment": ks.to(k_type).cuda(), "layout": layout}
    assert (kw["q_segment"].cpu().long() == qs).all() and (kw["k_segment"].cpu().long() == ks).all()
    table = torch.randn(10, channels, device="cuda")
    want = table[u].to(dtype)
    want = want if layout == "pair" else want.movedim(-1, 0)
    assert torch.equal(relative_position_bias_b200(table, buckets, q.cuda(), k.cuda(), dtype=dtype, **kw), want)
    g = torch.randint(-3, 4, want.shape, device="cuda").to(dtype)
    flat = (g if layout == "pair" else g.movedim(0, -1)).reshape(-1, channels).double()
    sums = torch.zeros(10, channels, dtype=torch.float64, device="cuda").index_add_(0, u.flatten(), flat)
    got = relative_position_bias_backward_b200(g, buckets, q.cuda(), k.cuda(), **kw)
    assert torch.equal(got.double(), sums)


@pytest.mark.parametrize("layout,channels", [("heads", 1), ("heads", 2), ("heads", 16), ("pair", 128), ("pair", 5)])
@pytest.mark.parametrize("rule", ["clip32", "log32", "clip300"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("chains", [False, True])
def test_runs_of_one_bucket_add_up_exactly(layout, channels, rule, dtype, chains):
    """Residue numbers in order: most of a row shares a bucket, whose elements are summed in registers.  Upstream values of
    1 to 3 make every sum a whole number below 3 * 1100^2 < 2^24, exact in fp32 in any order; an element left out or taken
    twice shows."""
    from miniworld_engine_b200 import relative_position_bias_backward_b200
    n = 1100 if layout == "heads" else 420
    i = torch.arange(n, device="cuda", dtype=torch.int32)
    pos, seg = i - (i >= 400).int() * 400, (i >= 400).int() + (i >= 405).int()
    kw = {"q_segment": seg} if chains else {}
    kind, count, top = RULES[rule]
    u = bucket_matrix(pos, pos, kind, count, top, seg if chains else None, seg if chains else None).cuda()
    buckets = _rule(rule, chains)
    gen = torch.Generator(device="cuda").manual_seed(n)
    g = torch.randint(1, 4, (n, n, channels), generator=gen, device="cuda").to(dtype)
    want = torch.zeros(buckets.rows, channels, dtype=torch.float64, device="cuda")
    want.index_add_(0, u.flatten(), g.reshape(-1, channels).double())
    # the fullest bucket is full: at least the 120 * 121 / 2 = 7260 pairs of 420 that lie 300 or more apart, of mean 2
    assert want.max() > 7260 and want.max() < 2 ** 24
    g = g if layout == "pair" else g.movedim(-1, 0)
    for grad in (g, g.contiguous()):
        got = relative_position_bias_backward_b200(grad, buckets, pos, layout=layout, **kw)
        assert torch.equal(got.double(), want)
