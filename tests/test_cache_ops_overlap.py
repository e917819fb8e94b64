"""CPU test: an eviction whose list of kept slots lies in another buffer of the call is refused."""
import ctypes as C

import pytest

from fastforwardattention_amd import capi

M = 0x100000


@pytest.mark.parametrize("where", [1 * M, 2 * M + 64, 3 * M, 3 * M + 508, 4 * M + 64, 5 * M, 6 * M + 4, 8 * M, 9 * M + 4096, 10 * M, 13 * M,
                                   3 * M - 4, 3 * M - 476])
def test_kept_slots_in_another_buffer(where):
    """Two caches of two pairs of 64 slots: 16 KiB of K or V, 512 bytes of weights; kept is 480 bytes."""
    lib = capi.load()
    arrays = [(C.c_void_p * 2)(a * M, b * M) for a, b in ((1, 8), (2, 9), (3, 10), (4, 11), (5, 12), (6, 13))]
    assert lib.ffa_evict(16, 2, *arrays, 1, 2, 64, 64, 64, 60, 30, 10, None, None, where, None) == capi.FFA_ERR_OVERLAP


def test_message():
    assert b"kept" in capi.load().ffa_status_string(capi.FFA_ERR_OVERLAP)
