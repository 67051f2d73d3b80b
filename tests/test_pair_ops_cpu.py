"""Checks of the operators beside the block that need no GPU: bucket rules, refusals, the C ABI's argument checks."""

import ctypes as C

import pytest
import torch

from _ops64 import bucket_of
from miniworld_engine_b200 import (PositionBuckets, RelativePositionBiasB200, cross_attention_b200,
                                   relative_position_bias_b200, relative_position_bias_backward_b200)
from miniworld_engine_b200 import _lib


@pytest.fixture(scope="module")
def lib():
    from miniworld_engine_b200 import build
    build.build()
    return _lib.load()


def _buckets_of(rule, d):
    """What the kernels compute from the rule's struct."""
    if rule.kind == _lib.BUCKETS_CLIPPED:
        return max(-rule.max_distance, min(rule.max_distance, d)) + rule.max_distance
    half = rule.count // 2 if rule.kind == _lib.BUCKETS_LOG else rule.count
    n = abs(d) if rule.kind == _lib.BUCKETS_LOG else max(d, 0)
    u = min(n, half // 2) + sum(t <= n for t in rule.thresholds)
    return u + (half if rule.kind == _lib.BUCKETS_LOG and d < 0 else 0)


@pytest.mark.parametrize("kind,count,top", [("clip", 65, 32), ("clip", 1, 0), ("log", 32, 128), ("log", 64, 512),
                                            ("log", 16, 9), ("log", 4, 2), ("log", 10, 100), ("causal", 32, 128),
                                            ("causal", 2, 2), ("causal", 256, 4096)])
def test_rules_follow_their_definition(kind, count, top):
    rule = (PositionBuckets.clipped(top) if kind == "clip" else
            PositionBuckets.logarithmic(count, top, bidirectional=kind == "log"))
    assert rule.rows == count
    for d in list(range(-700, 701)) + [s * (top + o) for s in (-1, 1) for o in (-1, 0, 1, 10 ** 6)]:
        u = _buckets_of(rule, d)
        assert 0 <= u < count and u == bucket_of(d, kind, count, top), (d, u)


def test_segments_add_a_row_and_rules_are_shared():
    assert PositionBuckets.clipped(32, segments=True).rows == 66
    assert PositionBuckets.clipped(32) is PositionBuckets.clipped(32)
    assert "66" in repr(PositionBuckets.clipped(32, segments=True))


@pytest.mark.parametrize("make,error", [
    (lambda: PositionBuckets.clipped(-1), ValueError),
    (lambda: PositionBuckets.clipped(512), NotImplementedError),
    (lambda: PositionBuckets.logarithmic(31, 128), ValueError),
    (lambda: PositionBuckets.logarithmic(2, 128), ValueError),
    (lambda: PositionBuckets.logarithmic(32, 8), ValueError),
    (lambda: PositionBuckets.logarithmic(32, 10 ** 6), NotImplementedError),
    (lambda: PositionBuckets.logarithmic(1024, 8000), NotImplementedError),
])
def test_rules_that_are_refused(make, error):
    with pytest.raises(error):
        make()


def test_bias_refuses_before_touching_a_device():
    rule = PositionBuckets.clipped(4)
    pos = torch.arange(5)
    with pytest.raises(RuntimeError, match="no CPU path"):
        relative_position_bias_b200(torch.zeros(9, 4), rule, pos)
    with pytest.raises(RuntimeError, match="no CPU path"):
        relative_position_bias_backward_b200(torch.zeros(4, 5, 5), rule, pos)
    with pytest.raises(ValueError, match="layout"):
        RelativePositionBiasB200(rule, 4, layout="rows")


def test_bias_checks_its_arguments(monkeypatch):
    from miniworld_engine_b200 import relpos
    monkeypatch.setattr(relpos, "_require_cuda", lambda t, name: None)       # CPU tensors stand in
    rule, seg = PositionBuckets.clipped(4), PositionBuckets.clipped(4, segments=True)
    t, pos = torch.zeros(9, 4), torch.arange(5)
    f = relative_position_bias_b200
    for bad, text in [
        (lambda: f(torch.zeros(8, 4), rule, pos), "table must be"),
        (lambda: f(torch.zeros(9), rule, pos), "table must be"),
        (lambda: f(t, rule, pos.float()), "int32 or int64"),
        (lambda: f(t, rule, pos[None, None]), r"\[L\] or \[B, L\]"),
        (lambda: f(t, rule, pos, layout="rows"), "layout"),
        (lambda: f(t, rule, pos, add=torch.zeros(4, 5, 5)), "pair layout"),
        (lambda: f(t, rule, pos, layout="pair", add=torch.zeros(5, 5, 3)), "add must be"),
        (lambda: f(t, rule, pos, layout="pair", add=torch.zeros(5, 5, 4), dtype=torch.bfloat16), "differs"),
        (lambda: f(t, rule, pos, q_segment=pos, k_segment=pos), "do not tell"),
        (lambda: f(torch.zeros(10, 4), seg, pos), "q_segment is needed"),
        (lambda: f(torch.zeros(10, 4), seg, pos, pos + 1, q_segment=pos), "without k_segment"),
        (lambda: f(torch.zeros(10, 4), seg, pos, q_segment=pos[:4]), "length"),
        (lambda: f(t, rule, pos.expand(2, 5), pos.expand(3, 5)), "batch sizes"),
        (lambda: relative_position_bias_backward_b200(torch.zeros(4, 5, 6), rule, pos), "grad must be"),
        (lambda: relative_position_bias_backward_b200(torch.zeros(5, 5), rule, pos), "dimensions"),
    ]:
        with pytest.raises(ValueError, match=text):
            bad()
    with pytest.raises(NotImplementedError):
        f(t, rule, pos, dtype=torch.float16)


def test_attention_checks_its_arguments(monkeypatch):
    from miniworld_engine_b200 import attention
    q, k = torch.zeros(2, 3, 4, 8), torch.zeros(2, 5, 2, 8)
    with pytest.raises(RuntimeError, match="no CPU path"):
        cross_attention_b200(q, k, k)
    monkeypatch.setattr(attention, "_require_cuda", lambda t, name: None)
    f = cross_attention_b200
    for bad, text in [
        (lambda: f(q[0], k, k), r"\[B, L, heads, D\]"),
        (lambda: f(q, k, k[:, :4]), "k and v must both be"),
        (lambda: f(q, k[..., :4], k[..., :4]), "k and v must both be"),
        (lambda: f(q, k[:1], k[:1]), "k and v must both be"),
        (lambda: f(q, k[:, :, :1].expand(2, 5, 3, 8), k[:, :, :1].expand(2, 5, 3, 8)), "multiple"),
        (lambda: f(q, k.bfloat16(), k), "like q"),
        (lambda: f(q, k, k, bias=torch.zeros(4, 3, 4)), "bias must be"),
        (lambda: f(q, k, k, bias=torch.zeros(3, 4, 3, 5)), "bias must be"),
        (lambda: f(q, k, k, bias=torch.zeros(4, 1, 5)), "bias must be"),
        (lambda: f(q, k, k, bias=torch.zeros(4, 3, 5).bfloat16()), "like q"),
        (lambda: f(q, k, k, bias=torch.zeros(5)), "bias must be"),
        (lambda: f(q, k, k, key_mask=torch.ones(2, 4)), "key_mask"),
        (lambda: f(q, k, k, scale=float("nan")), "finite"),
        (lambda: f(q[..., :0], k[..., :0], k[..., :0]), "empty"),
    ]:
        with pytest.raises(ValueError, match=text):
            bad()
    with pytest.raises(NotImplementedError):
        f(q.half(), k.half(), k.half())


def test_c_abi_checks_relpos(lib):
    rule = PositionBuckets.clipped(4)._struct

    def desc(**kw):
        d = _lib.RelposDesc(C.sizeof(_lib.RelposDesc), 0, 0, 1, 1, 8, 8, 4, 0, 0, 0, 0, 0, 0, 0, 64, 8)
        for n, v in kw.items():
            setattr(d, n, v)
        return d

    n = C.c_size_t()
    need = lambda d, b=rule: lib.trimul_b200_relpos_bias_grad_workspace_bytes(C.byref(d), C.byref(b), C.byref(n))
    assert need(desc()) == 0 and n.value >= 9 * 4 * 4
    for kw in ({"struct_bytes": 4}, {"layout": 2}, {"dtype": 5}, {"table_dtype": -1}, {"B": 0}, {"Lq": 0}, {"Lk": -1},
               {"channels": 0}, {"wide_index": 16}, {"stride_i": -8}):
        assert need(desc(**kw)) == _lib.E_INVALID, kw
    for kw in ({"channels": 10000}, {"Lk": 1 << 25}, {"B": 1 << 16, "Lq": 1 << 16}):
        assert need(desc(**kw)) == _lib.E_UNSUPPORTED, kw
    for kw in ({"count": 8}, {"count": 0}, {"kind": 3}, {"kind": 1}, {"max_distance": -1}):
        b = _lib.Buckets.from_buffer_copy(rule)
        for name, v in kw.items():
            setattr(b, name, v)
        assert need(desc(), b) == _lib.E_INVALID, kw
    b = _lib.Buckets.from_buffer_copy(PositionBuckets.logarithmic(32, 128)._struct)
    b.thresholds[3] = 2                                          # not ascending
    assert need(desc(), b) == _lib.E_INVALID
    b = _lib.Buckets.from_buffer_copy(PositionBuckets.logarithmic(32, 128)._struct)
    b.n_thresholds = 8                                           # a bucket too many
    assert need(desc(), b) == _lib.E_INVALID
    f = lib.trimul_b200_relpos_bias
    p = 4096
    assert f(C.byref(desc()), C.byref(rule), None, p, p, None, None, None, p, None) == _lib.E_INVALID
    assert f(C.byref(desc()), C.byref(rule), p, p, p, None, None, None, p + 2, None) == _lib.E_INVALID     # alignment
    assert f(C.byref(desc(stride_i=4)), C.byref(rule), p, p, p, None, None, None, p, None) == _lib.E_INVALID
    assert f(C.byref(desc(Lk=9)), C.byref(rule), p, p, p, None, None, None, p, None) == _lib.E_INVALID     # row too short
    assert f(C.byref(desc()), C.byref(rule), p, p, p, None, None, p, p, None) == _lib.E_INVALID            # add
    seg = PositionBuckets.clipped(4, segments=True)._struct
    assert f(C.byref(desc()), C.byref(seg), p, p, p, None, None, None, p, None) == _lib.E_INVALID
    g = lib.trimul_b200_relpos_bias_grad
    assert need(desc()) == 0
    assert g(C.byref(desc()), C.byref(rule), p, p, None, None, p, p, p, n.value - 1, None) == _lib.E_WORKSPACE
    assert g(C.byref(desc()), C.byref(rule), p, p, None, None, p, p, None, n.value, None) == _lib.E_INVALID


def test_c_abi_checks_attention(lib):
    def desc(**kw):
        d = _lib.AttnDesc()
        d.struct_bytes, d.dtype, d.scale = C.sizeof(_lib.AttnDesc), 0, 1.0
        d.B, d.Lq, d.Lk, d.H, d.Hk, d.D = 2, 16, 24, 4, 2, 64
        for n, v in kw.items():
            setattr(d, n, v)
        return d

    n = C.c_size_t()
    need = lambda d, b=1: lib.trimul_b200_attn_workspace_bytes(C.byref(d), b, C.byref(n))
    assert need(desc()) == 0 and n.value >= 2 * 4 * 16 * 4
    for kw in ({"struct_bytes": 8}, {"dtype": 3}, {"B": 0}, {"Lq": 0}, {"Lk": 0}, {"Hk": 3}, {"D": 0}, {"H": -4},
               {"bias": 4096, "bias_batch": 3, "bias_heads": 1}, {"bias": 4096, "bias_batch": 1, "bias_heads": 2},
               {"dbias": 4096, "bias_batch": 1, "bias_heads": 1},
               {"bias": 4096, "dbias": 4098, "bias_batch": 1, "bias_heads": 1, "dbias_i": 24},
               {"bias": 4096, "dbias": 4096, "bias_batch": 1, "bias_heads": 1, "dbias_i": 16}):
        assert need(desc(**kw)) == _lib.E_INVALID, kw
    for kw in ({"D": 264}, {"B": 70000}, {"Lk": 1 << 25}):
        assert need(desc(**kw)) == _lib.E_UNSUPPORTED, kw
    d = desc()
    assert lib.trimul_b200_attn_forward(C.byref(d), None, 0, None, None) == _lib.E_INVALID
    assert lib.trimul_b200_attn_backward(C.byref(d), None, 0, None, None) == _lib.E_INVALID
    for t in ("q", "k", "v", "o", "dout", "dq", "dk", "dv"):
        getattr(d, t).p = 4096
    assert lib.trimul_b200_attn_backward(C.byref(d), 4096, 1 << 20, None, None) == _lib.E_INVALID       # no state
    d.stats = 4096
    assert need(d) == 0
    assert lib.trimul_b200_attn_backward(C.byref(d), 4096, n.value - 1, None, None) == _lib.E_WORKSPACE


def test_c_abi_wants_the_statistics_on_eight_bytes(lib):
    d = _lib.AttnDesc()
    d.struct_bytes, d.dtype, d.scale = C.sizeof(_lib.AttnDesc), 0, 1.0
    d.B, d.Lq, d.Lk, d.H, d.Hk, d.D = 1, 4, 4, 1, 1, 8
    for t in ("q", "k", "v", "o", "dout", "dq", "dk", "dv"):
        getattr(d, t).p = 4096
    n = C.c_size_t()
    for stats, rc in ((4096, 0), (4100, _lib.E_INVALID)):
        d.stats = stats
        assert lib.trimul_b200_attn_workspace_bytes(C.byref(d), 1, C.byref(n)) == rc
    assert lib.trimul_b200_attn_forward(C.byref(d), 4096, 1 << 20, None, None) == _lib.E_INVALID
    assert lib.trimul_b200_attn_backward(C.byref(d), 4096, 1 << 20, None, None) == _lib.E_INVALID


# what a process does with a rule that came to it: the library reads it (here for the size of a workspace)
_READ_RULE = """
import ctypes as C, pickle, sys
from miniworld_engine_b200 import _lib
rules = pickle.loads(bytes.fromhex(sys.stdin.read()))
for rule in rules:
    desc = _lib.RelposDesc(C.sizeof(_lib.RelposDesc), 0, 0, 1, 1, 8, 8, 4, 0, 0, 0, 0, 0, 0, 0, 64, 8)
    n = C.c_size_t()
    rc = _lib.load().trimul_b200_relpos_bias_grad_workspace_bytes(C.byref(desc), rule._address, C.byref(n))
    print(rc, rule.rows, n.value)
"""


def _read_rule(lib, rule):
    desc = _lib.RelposDesc(C.sizeof(_lib.RelposDesc), 0, 0, 1, 1, 8, 8, 4, 0, 0, 0, 0, 0, 0, 0, 64, 8)
    n = C.c_size_t()
    return lib.trimul_b200_relpos_bias_grad_workspace_bytes(C.byref(desc), rule._address, C.byref(n)), rule.rows, n.value


def test_rules_survive_another_process(lib):
    import os
    import pickle
    import subprocess
    import sys
    rules = [PositionBuckets.clipped(20, segments=True), PositionBuckets.logarithmic(32, 128),
             RelativePositionBiasB200(PositionBuckets.clipped(7), 4).buckets]
    want = [_read_rule(lib, r) for r in rules]
    got = subprocess.run([sys.executable, "-c", _READ_RULE], input=pickle.dumps(rules).hex(), capture_output=True, text=True,
                         cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))), timeout=600)
    assert got.returncode == 0, got.stderr[-2000:]
    assert [tuple(int(x) for x in line.split()) for line in got.stdout.splitlines()] == want
    assert all(rc == 0 for rc, _, _ in want)


def test_copies_of_a_rule_do_not_need_the_original(lib):
    """A deep copy (an averaged model's) reads its own struct, also when the original and its memory are gone."""
    import copy
    import gc
    for make in (lambda: PositionBuckets(_lib.BUCKETS_CLIPPED, 19, 9, (), True),         # not kept by the factories' cache
                 lambda: PositionBuckets(_lib.BUCKETS_LOG, 8, 30, (4,), False)):
        for dup in (copy.deepcopy, copy.copy):
            rule = make()
            want = _read_rule(lib, rule)
            kept = dup(rule)
            size = C.sizeof(rule._struct)
            own = C.addressof(kept._struct)
            assert kept._address == own
            del rule
            gc.collect()
            filler = [C.create_string_buffer(b"\xff" * size, size) for _ in range(64)]        # likely to land on freed memory
            assert _read_rule(lib, kept) == want and want[0] == 0
            assert kept.rows == want[1] and len(filler) == 64
    module = RelativePositionBiasB200(PositionBuckets(_lib.BUCKETS_CLIPPED, 19, 9, (), True), 4)
    twin = copy.deepcopy(module)
    assert twin.buckets._address == C.addressof(twin.buckets._struct)
    want = _read_rule(lib, module.buckets)
    del module
    gc.collect()
    assert _read_rule(lib, twin.buckets) == want


@pytest.mark.parametrize("no_grad", [False, True])
def test_forward_mode_tangents_are_refused(no_grad):
    """A dual tensor does not require a gradient: the call must not return a result without its tangent."""
    import contextlib
    import torch.autograd.forward_ad as fwd
    rule, pos = PositionBuckets.clipped(4), torch.arange(5)
    q, k, b = torch.zeros(1, 5, 2, 8), torch.zeros(1, 5, 2, 8), torch.zeros(2, 5, 5)
    t, add = torch.zeros(9, 4), torch.zeros(5, 5, 4)
    f, attend = relative_position_bias_b200, cross_attention_b200
    with fwd.dual_level(), torch.no_grad() if no_grad else contextlib.nullcontext():
        dual = lambda x: fwd.make_dual(x, torch.ones_like(x))
        for call in (lambda: attend(dual(q), k, k), lambda: attend(q, dual(k), k), lambda: attend(q, k, dual(k)),
                     lambda: attend(q, k, k, bias=dual(b)), lambda: f(dual(t), rule, pos),
                     lambda: f(t, rule, pos, layout="pair", add=dual(add))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        for call in (lambda: attend(q, k, k, bias=b), lambda: f(t, rule, pos)):      # no tangent: the usual refusal on the CPU
            with pytest.raises(RuntimeError, match="no CPU path"):
                call()
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda x: attend(x, k, k), (q,), (q,))
    with pytest.raises(RuntimeError, match="no CPU path"):
        attend(q, k, k)


@pytest.mark.parametrize("count,top", [(32, 10 ** 9), (32, 10 ** 15), (4, 10 ** 18), (64, 2 ** 62)])
@pytest.mark.parametrize("bidirectional", [False, True])
def test_far_distances_are_refused_at_once(count, top, bidirectional):
    """A border beyond the look-up table is refused without counting up to it."""
    import signal

    def late(signum, frame):
        raise TimeoutError("still counting")

    before = signal.signal(signal.SIGALRM, late)
    signal.setitimer(signal.ITIMER_REAL, 10)
    try:
        with pytest.raises(NotImplementedError, match="must share a bucket"):
            PositionBuckets.logarithmic(count, top, bidirectional=bidirectional)
    finally:
        signal.setitimer(signal.ITIMER_REAL, 0)
        signal.signal(signal.SIGALRM, before)


@pytest.mark.parametrize("same", [False, True])
def test_positions_that_come_back_as_another_object(monkeypatch, same):
    """Saved-tensor hooks (checkpointing, offload) hand the backward pass copies: positions given once as queries' and keys'
    are still one set of positions there."""
    from miniworld_engine_b200 import relpos
    buckets, pos, seg = PositionBuckets.clipped(4, segments=True), torch.arange(5), torch.zeros(5, dtype=torch.int32)
    seen = []

    def backward(grad, rule, q_pos, k_pos=None, *, q_segment, k_segment, layout, dtype):
        call = relpos._Call(rule, q_pos, k_pos, q_segment, k_segment, layout, 1, 1, 4, q_pos.device)
        seen.append((call.lq, call.lk, call.keep[1] is call.keep[0], call.keep[3] is call.keep[2]))
        return torch.zeros(10, 4)

    monkeypatch.setattr(relpos, "_forward", lambda table, *args: torch.zeros(4, 5, 5))
    monkeypatch.setattr(relpos, "relative_position_bias_backward_b200", backward)
    table = torch.zeros(10, 4, requires_grad=True)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), lambda t: t):
        out = relative_position_bias_b200(table, buckets, pos, pos if same else None, q_segment=seg)
    out.sum().backward()
    assert seen == [(5, 5, True, True)]


@pytest.mark.parametrize("scale", [1e39, -1e300, 3.5e38])
def test_scales_beyond_32_bits_are_refused(monkeypatch, scale):
    from miniworld_engine_b200 import attention
    monkeypatch.setattr(attention, "_require_cuda", lambda t, name: None)
    q, k = torch.zeros(2, 3, 4, 8), torch.zeros(2, 5, 2, 8)
    with pytest.raises(ValueError, match="scale must be finite"):
        cross_attention_b200(q, k, k, scale=scale)
    with pytest.raises(ValueError, match="scale must be finite"):
        cross_attention_b200(q[:0], k[:0], k[:0], scale=scale)          # also where nothing is computed
    assert attention._Call(q, k, k, None, None, torch.finfo(torch.float32).max, False).pack((0, 0, 0, 0), 0, 0)


def test_attention_kernels_load_nothing_through_the_non_coherent_path():
    """They run while the kernel before them still writes; that path is for memory that is not written meanwhile."""
    import os
    import re
    csrc = os.path.join(os.path.dirname(_lib.__file__), "csrc")
    for name in sorted(os.listdir(csrc)):
        if name.startswith("attn_"):
            code = re.sub(r"//[^\n]*", "", open(os.path.join(csrc, name)).read())
            assert not re.search(r"__ldg|ld\.global\.nc|__restrict__", code), name
