"""What a block of the 8-bit kernels waits for before it ends with copies still on their way (csrc/tcgen05_util.cuh, `ring_last_parity`): the
last copy into every slot of its ring, wherever the loads ended.  The barriers are played here."""

import ctypes

import pytest

from ullm_b200.csrc.build import build


@pytest.fixture(scope="module")
def last_parity():
    f = ctypes.CDLL(build()).ullm_ring_last_parity
    f.argtypes, f.restype = [ctypes.c_int] * 3, ctypes.c_int
    return f


class Barrier:
    """A phase completes with each copy; a wait on a parity passes once the phase of that parity has (a fresh barrier passes on 1)."""

    def __init__(self):
        self.done = 0

    def passes(self, parity):
        return (self.done & 1) != parity


@pytest.mark.parametrize("slots", [1, 2, 5, 8, 12])
def test_the_last_copy_into_every_slot_is_waited_for(last_parity, slots):
    for copies in range(5 * slots + 2):
        s, parity = 0, 1  # as the loading warps count
        for _ in range(copies):
            s += 1
            if s == slots:
                s, parity = 0, parity ^ 1
        assert (s, parity) == (copies % slots, (copies // slots) & 1 ^ 1)  # as rows_int8_stream and a pair's plan do
        for t in range(slots):
            of_slot = (copies - t + slots - 1) // slots if copies > t else 0
            bar = Barrier()
            # a slot is filled again once its copy before has come: all but the last one are there
            bar.done = max(of_slot - 1, 0)
            assert bar.passes(last_parity(t, s, parity)) == (of_slot == 0)
            bar.done = of_slot
            assert bar.passes(last_parity(t, s, parity))
