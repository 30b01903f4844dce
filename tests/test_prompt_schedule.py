"""CPU: the ring of published work items of the prompt kernel, as its source has it.

A model of the ring under an adversarial order of steps: one producer that publishes items into slots, readers that wait for a
slot's phase by its parity, as an mbarrier wait does (a parity tells a phase from the next one, not from the one after that).
Readers may be held up for as long as nothing in the kernel waits for them."""
import random
import re
from pathlib import Path

import pytest

SOURCE = (Path(__file__).resolve().parents[1] / "nanopd_b200" / "csrc" / "prefill_kernel.cuh").read_text()
SLOTS = int(re.search(r"constexpr int kSchedSlots = (\d+);", SOURCE).group(1))


def run(items, readers, waits_for_readers, pick):
    """True when every reader has seen every item in order; False when one takes a later item for the awaited one or can
    make no further step."""
    published, slots, read = 0, [None] * SLOTS, [0] * readers
    while True:
        able = []
        if published < items:
            # the producer's wait: everyone has read what the slot held
            if not waits_for_readers or published < SLOTS or min(read) > published - SLOTS:
                able.append(-1)
        for r in range(readers):
            k = read[r]
            if k < items:
                phases = (published - k % SLOTS + SLOTS - 1) // SLOTS         # completed phases of slot k % SLOTS
                if phases > 0 and (phases - 1) % 2 == (k // SLOTS) % 2:
                    able.append(r)
        if not able:
            return published == items and all(k == items for k in read)
        step = pick(able)
        if step == -1:
            slots[published % SLOTS] = published
            published += 1
        else:
            if slots[read[step] % SLOTS] != read[step]:
                return False
            read[step] += 1


def late(able):
    """The reader 0 moves only when nobody else can."""
    others = [a for a in able if a != 0]
    return others[0] if others else 0


def test_a_reader_that_nobody_waits_for_loses_the_ring():
    assert not run(5 * SLOTS, 3, False, late)


@pytest.mark.parametrize("seed", range(20))
def test_the_producer_waits_for_every_reader(seed):
    assert run(5 * SLOTS, 3, True, late)
    rng = random.Random(seed)
    assert run(7 * SLOTS + 3, 4, True, rng.choice)


def test_the_kernel_has_that_wait():
    """The producer waits for the slot's reader before it writes there; the second softmax group, the only role that nothing
    else holds the producer for, arrives once per item, behind its last look at the item."""
    wait = SOURCE.index("wait_or_abort(smem_u32(&ctrl->sched_read[k % kSchedSlots]), (k / kSchedSlots - 1) & 1")
    assert wait < SOURCE.index("ctrl->sched_desc[k % kSchedSlots] = it;")
    assert "if (k >= kSchedSlots)" in SOURCE[wait - 200:wait]
    assert "mbar_init(smem_u32(&ctrl->sched_read[i]), kSchedReaders)" in SOURCE and "constexpr int kSchedReaders = 128;" in SOURCE
    softmax = SOURCE.index("softmax + correction (warps 0-7)")
    arrive = SOURCE.index("if (x == 1) mbar_arrive(smem_u32(&ctrl->sched_read[k % kSchedSlots]));")
    assert SOURCE.index("const ItemT it = ctrl->sched_desc[k % kSchedSlots];", softmax) < arrive
    assert SOURCE.count("mbar_arrive(smem_u32(&ctrl->sched_read") == 1
