"""Two warps that issue a ring's products in turn, each waiting by the parity of a stage's barrier only every other round: no order in
which boxes land, products end and warps run may let one take an earlier round's phase for its own (it would multiply a box that has
not come).  Every interleaving of a model of the kernels' waits, for the ring lengths that the sources allow, on the CPU."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(__file__), "..", "ferrum-torrens_b200", "csrc")


def constant(path, name):
    return int(re.search(rf"\b{name} = (\d+)\b", open(os.path.join(CSRC, path)).read()).group(1))


def too_early(stages, accumulators, box_first):
    """A block that some interleaving multiplies before its box has landed, or None.

    State: boxes asked for (in order), landed and multiplied (sets of blocks, as bits), blocks the epilogue has finished (in
    order), and for each issuer its next block and how many of its two waits are behind it."""
    blocks = stages + 8
    start = (0, 0, 0, 0, (0, 0), (1, 0))
    seen, todo = {start}, [start]
    while todo:
        asked, landed, done, finished, *issuers = todo.pop()
        after = []
        # the producer sees every round of every stage
        if asked < blocks and (asked < stages or done >> (asked - stages) & 1):
            after.append((asked + 1, landed, done, finished, *issuers))
        for b in range(max(0, asked - stages), asked):
            if not landed >> b & 1:
                after.append((asked, landed | 1 << b, done, finished, *issuers))
        # so does the epilogue
        if done >> finished & 1:
            after.append((asked, landed, done, finished + 1, *issuers))
        for i, (b, waits) in enumerate(issuers):
            if b >= blocks:
                continue
            if (waits == 0) == box_first:
                rounds = sum(landed >> r & 1 for r in range(b % stages, blocks, stages))       # phases the stage's barrier has completed
                passes = (rounds & 1) != (b // stages & 1)
                if passes and not landed >> b & 1:
                    return b
            else:
                passes = finished > b - accumulators            # (an issuer has every round of its own accumulators)
            if passes:
                moved = list(issuers)
                moved[i] = (b, 1) if waits == 0 else (b + 2, 0)
                after.append((asked, landed, done if waits == 0 else done | 1 << b, finished, *moved))
        for state in after:
            if state not in seen:
                seen.add(state)
                todo.append(state)
    return None


def test_the_model_finds_the_ring_that_is_too_short():
    assert too_early(3, 4, False) is not None


@pytest.mark.parametrize("stages", range(2, 13))
def test_rings_of_the_narrow_tiles(stages):
    least, most, accumulators = (constant("fp8_umma.cu", n) for n in ("kMinStages", "kMaxStages", "kMaxAcc"))
    if least <= stages <= most:
        assert too_early(stages, accumulators, False) is None


def test_ring_of_the_pairs():
    # two accumulators, the box waited for first
    assert too_early(constant("fp8_pair.cu", "kStages"), 2, True) is None
