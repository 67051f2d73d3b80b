"""The operators beside the block under torch's saved-tensor hooks: what was saved comes back as other tensor objects
(checkpointing, offload to the host), and the gradients are the same bits."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _step(around, positions, dtype):
    """A learned bias and the attention that takes it, forward under ``around``; result and gradients."""
    from miniworld_engine_b200 import PositionBuckets, cross_attention_b200, relative_position_bias_b200
    gen = torch.Generator(device="cuda").manual_seed(1)
    L, H, D = 70, 4, 32
    r = lambda *s: torch.randn(s, generator=gen, device="cuda")
    q, k, v = (r(2, L, H, D).to(dtype).requires_grad_(True) for _ in range(3))
    table, add = r(10, H).requires_grad_(True), r(L, L, H).requires_grad_(True)
    buckets = PositionBuckets.clipped(4, segments=True)
    pos, seg = torch.arange(L, device="cuda"), (torch.arange(L, device="cuda") > 30).int()
    keep = torch.rand(2, L, generator=gen, device="cuda") > 0.2
    args = {"once": (pos, None), "same object": (pos, pos), "own": (pos, pos + 1)}[positions]
    kw = {"q_segment": seg} if positions != "own" else {"q_segment": seg, "k_segment": seg}

    def body(q, k, v, table, add):
        bias = relative_position_bias_b200(table, buckets, *args, dtype=dtype, **kw)
        pair = relative_position_bias_b200(table, buckets, *args, layout="pair", add=add, **kw)
        return cross_attention_b200(q, k, v, bias=bias, key_mask=keep), pair

    out, pair = around(body, q, k, v, table, add)
    (out.float().square().sum() + pair.square().sum()).backward()
    return [out, pair, *(t.grad for t in (q, k, v, table, add))]


def _hooks(pack, unpack):
    def around(body, *args):
        with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
            return body(*args)
    return around


def _offload(body, *args):
    with torch.autograd.graph.save_on_cpu():
        return body(*args)


def _checkpoint(body, *args):
    return torch.utils.checkpoint.checkpoint(body, *args, use_reentrant=False)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("positions", ["once", "same object", "own"])
@pytest.mark.parametrize("around", [_hooks(lambda t: t.clone(), lambda t: t), _offload, _checkpoint],
                         ids=["clones", "offload", "checkpoint"])
def test_saved_tensors_may_come_back_as_others(around, positions, dtype):
    want = _step(lambda body, *args: body(*args), positions, dtype)
    for a, b in zip(_step(around, positions, dtype), want):
        assert torch.equal(a, b)
