"""NaN and infinity in places that are not masked: what depends on them comes out as NaN, never as the zeros of a row
without keys, and everything else keeps its bits."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, FP32 = torch.bfloat16, torch.float32

# name: dtype, Lq, Lk, D, plain_kernels.  One and several blocks to a row's keys ("split") for each kind of kernel
KERNELS = {
    "few rows": (BF16, 1, 300, 64, False),
    "few rows split": (BF16, 2, 5000, 128, False),
    "few rows fp32": (FP32, 1, 2000, 32, False),
    "up to 64": (BF16, 150, 300, 64, False),
    "up to 64 split": (BF16, 40, 4100, 40, False),
    "up to 128": (BF16, 150, 300, 128, False),
    "up to 128 split": (BF16, 40, 4100, 96, False),
    "CUDA cores": (BF16, 70, 60, 64, True),
    "CUDA cores split": (BF16, 40, 1000, 20, False),
    "CUDA cores fp32": (FP32, 70, 50, 72, False),
    "CUDA cores fp32 split": (FP32, 40, 900, 136, False),
}


def _inputs(kernel, bias, masked):
    dtype, Lq, Lk, D, plain = KERNELS[kernel]
    gen = torch.Generator(device="cuda").manual_seed(Lk)
    r = lambda *s: torch.randn(s, generator=gen, device="cuda").to(dtype)
    q, k, v, g = r(2, Lq, 4, D), r(2, Lk, 2, D), r(2, Lk, 2, D), r(2, Lq, 4, D)
    b = r(2, 4, Lq, Lk) if bias else None
    m = None
    if masked:
        m = torch.rand(2, Lk, generator=gen, device="cuda") > 0.3
        m[:, :3] = torch.tensor([True, False, True], device="cuda")
    return q, k, v, g, b, m, plain


def _both(q, k, v, g, b, m, plain):
    from miniworld_engine_b200 import cross_attention_backward_b200, cross_attention_b200, cross_attention_forward_b200
    kw = dict(bias=b, key_mask=m, plain_kernels=plain)
    out, state = cross_attention_forward_b200(q, k, v, **kw)
    assert torch.equal(out, cross_attention_b200(q, k, v, **kw)) or not out.isfinite().all()
    return dict(zip(("out", "dq", "dk", "dv", "db"), (out, *cross_attention_backward_b200(g, q, k, v, out, state, **kw))))


def _same_but(got, clean, nan):
    """``nan`` (bool, broadcast): NaN there, the clean call's bits elsewhere."""
    nan = nan.expand_as(got)
    assert got[nan].isnan().all(), f"{int((~got[nan].isnan()).sum())} of {int(nan.sum())} values are not NaN"
    assert torch.equal(got[~nan], clean[~nan])


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("kernel", KERNELS)
def test_nan_in_a_query_row(kernel, bias, masked):
    q, k, v, g, b, m, plain = _inputs(kernel, bias, masked)
    clean = _both(q, k, v, g, b, m, plain)
    Lq, D = q.shape[1], q.shape[3]
    row = torch.zeros(2, Lq, 4, 1, dtype=torch.bool, device="cuda")
    row[1, Lq // 2, 2] = True
    q2 = q.clone()
    q2[1, Lq // 2, 2, D - 1] = math.nan
    got = _both(q2, k, v, g, b, m, plain)
    _same_but(got["out"], clean["out"], row)
    _same_but(got["dq"], clean["dq"], row)
    kept = torch.ones(2, k.shape[1], dtype=torch.bool, device="cuda") if m is None else m
    hit = torch.zeros(2, k.shape[1], 2, 1, dtype=torch.bool, device="cuda")
    hit[1, :, 1] = kept[1, :, None]                            # the key head that this query head reads
    for name in ("dk", "dv"):
        _same_but(got[name], clean[name], hit)
    if bias:
        _same_but(got["db"], clean["db"], row.permute(0, 2, 1, 3) & kept[:, None, None, :])


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("keys", ["one", "all", "half a tile"])
def test_nan_in_keys(kernel, bias, keys):
    q, k, v, g, b, m, plain = _inputs(kernel, bias, True)
    clean = _both(q, k, v, g, b, m, plain)
    which = {"one": slice(2, 3), "all": slice(0, None), "half a tile": slice(64, 128) if k.shape[1] > 128 else slice(32, None)}[keys]
    k2 = k.clone()
    k2[0, which, 1] = math.nan                                 # query heads 2 and 3 of batch element 0
    got = _both(q, k2, v, g, b, m, plain)
    heads = torch.zeros(2, 1, 4, 1, dtype=torch.bool, device="cuda")
    heads[0, :, 2:] = True
    _same_but(got["out"], clean["out"], heads)
    for name in ("dk", "dv"):                                  # masked keys keep their zeros
        assert not got[name][~m].any()


@pytest.mark.parametrize("kernel", KERNELS)
def test_nan_queries_of_rows_without_keys_and_infinite_scores(kernel):
    q, k, v, g, b, m, plain = _inputs(kernel, True, True)
    m[1] = False
    clean = _both(q, k, v, g, b, m, plain)
    q2, b2 = q.clone(), b.clone()
    q2[1, 0] = math.nan                                        # no key is kept: zeros, whatever the query holds
    b2[0, 3, 0, 2] = math.inf                                  # inf - inf
    got = _both(q2, k, v, g, b2, m, plain)
    row = torch.zeros(2, q.shape[1], 4, 1, dtype=torch.bool, device="cuda")
    row[0, 0, 3] = True
    _same_but(got["out"], clean["out"], row)
    assert not got["out"][1].any()


@pytest.mark.parametrize("kernel", KERNELS)
def test_nan_and_infinity_in_values(kernel):
    """A column of the values goes into the same column of every row, and nowhere else."""
    q, k, v, g, b, m, plain = _inputs(kernel, False, True)
    clean = _both(q, k, v, g, b, m, plain)["out"]
    D = q.shape[3]
    for bad in (math.nan, math.inf):
        v2 = v.clone()
        v2[0, 2, 0, D // 2] = bad                              # a kept key; query heads 0 and 1
        got = _both(q, k, v2, g, b, m, plain)["out"]
        hit = torch.zeros(2, 1, 4, D, dtype=torch.bool, device="cuda").expand_as(got).clone()
        hit[0, :, :2, D // 2] = True
        assert torch.equal(got[~hit], clean[~hit]) and not got[hit].isfinite().any()
