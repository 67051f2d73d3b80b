"""How the tensor-core forward kernels tell that a key or value tile has come, as a model: loads that arrive in any order,
warps that go on in any order, barriers that are waited for by parity.

The ring's slots take key 0, value 0, key 1, value 1, ... in turn.  One warp (cleaner) waits for value tiles alone and signals
them to the issuer, which waits for key tiles and for those signals.  A parity wait passes whenever the barrier's current phase
has the other parity, so a warp may only wait on barriers whose every phase it sees.  The model also finds the fault of a
barrier per slot in a ring of an odd number of slots."""

import os
import random
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "miniworld_engine_b200", "csrc")


def _run(stages, tiles, per_tile, rng, in_flight=4):
    phase, slot, loading = {}, {}, []
    loads = cleaned = 0
    issued = -1                                               # -1: the first scores are still to come
    passed = lambda bar, parity: (phase.get(bar, 0) & 1) != parity

    def full(x):                                              # barrier and parity of load x
        if per_tile:
            return ("kv"[x & 1], (x >> 1) % in_flight), ((x >> 1) // in_flight) & 1
        return ("full", x % stages), (x // stages) & 1

    def flip(bar):
        phase[bar] = phase.get(bar, 0) + 1

    while True:
        steps = [("arrive", x) for x in loading]
        if loads < 2 * tiles and passed(("empty", loads % stages), ((loads // stages) & 1) ^ 1):
            steps.append(("load", loads))
        if cleaned < tiles and passed(*full(2 * cleaned + 1)):
            steps.append(("clean", 2 * cleaned + 1))
        if issued == -1:
            if passed(*full(0)):
                steps.append(("first", 0))
        elif issued < tiles and passed(("ok", issued % in_flight), (issued // in_flight) & 1) and (
                issued + 1 == tiles or passed(*full(2 * issued + 2))):
            steps.append(("issue", issued))
        if not steps:
            return "done" if issued == tiles and cleaned == tiles else "stuck"
        what, x = rng.choice(steps)
        if what == "load":
            slot[x % stages] = None
            loading.append(x)
            loads += 1
        elif what == "arrive":
            loading.remove(x)
            slot[x % stages] = x
            flip(full(x)[0])
        elif what == "clean":
            if slot.get(x % stages) != x:
                return "cleaned another tile"
            flip(("ok", cleaned % in_flight))
            cleaned += 1
        else:
            used = [0] if what == "first" else [2 * x + 1] + ([2 * x + 2] if x + 1 < tiles else [])
            for u in used:
                if slot.get(u % stages) != u:
                    return "product of another tile"
                flip(("empty", u % stages))
            issued += 1


def _outcomes(stages, per_tile, runs=400):
    rng = random.Random(stages)
    return {_run(stages, tiles, per_tile, rng) for _ in range(runs) for tiles in (1, 2, 3, 7, 14)}


@pytest.mark.parametrize("stages", [2, 3, 4, 5, 6, 7])
def test_a_barrier_per_tile_is_right_for_every_ring(stages):
    assert _outcomes(stages, True) == {"done"}


@pytest.mark.parametrize("stages", [4, 6])
def test_a_barrier_per_slot_is_right_where_a_slot_keeps_its_kind(stages):
    assert _outcomes(stages, False) == {"done"}


@pytest.mark.parametrize("stages", [3, 5])
def test_the_model_sees_what_is_wrong_with_a_barrier_per_slot(stages):
    assert "cleaned another tile" in _outcomes(stages, False)


def test_the_kernels_use_what_is_right_for_their_rings():
    """Both kernels' numbers of slots; where one is odd, the kernel has barriers per tile."""
    for name in ("attn_fwd_sm100.cuh", "attn_fwd64_sm100.cuh"):
        text = open(os.path.join(CSRC, name)).read()
        stages = [int(n) for n in re.search(r"kStages = kBias \? (\d) : (\d);", text).groups()]
        clean = int(re.search(r"kAfClean = (\d)", open(os.path.join(CSRC, "attn_fwd_sm100.cuh")).read()).group(1))
        assert all((s + 1) // 2 <= clean for s in stages)
        if any(s % 2 for s in stages):
            assert "v_full[j % kAfClean]" in text and "k_full[(j + 1) % kAfClean]" in text and "&full[" not in text, name
