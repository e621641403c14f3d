"""CPU checks of the entry points around drafted tokens and the Q8_0 pool beyond
their refusals (no GPU work)."""
import ctypes as C
import os

import numpy as np
import pytest


@pytest.fixture(scope="module")
def hip():
    from lgml_amd import build, hip
    if not os.path.exists(hip.LIB_PATH):
        build.build()
    hip.lib()
    return hip


def store(hip, cells, blocks):
    """lgmlh_kv_store_q8's answer to cells that it refuses (it reads no other data)."""
    c, d = np.ascontiguousarray(cells, np.int64), C.c_void_p(256)
    return hip.lib().lgmlh_kv_store_q8(d, d, 64 * blocks, 1, 64, d, d, d, c.ctypes.data, len(c), None)


# blocks whose numbers, times 2^64 / the golden ratio, have high words that are
# multiples of 3: a table's share by the remainder would hold them all
THREES = [b for b in range(9000) if (b * 0x9e3779b97f4a7c15 % 2**64 >> 32) % 3 == 0]


@pytest.mark.parametrize("blocks", [THREES[:1500], range(0, 70000 * 64, 64), range(70000),
                                    np.random.default_rng(3).permutation(1 << 22)[:70000]])
def test_a_cell_twice_is_found_among_any_cells(hip, blocks):
    """Lone cells of any blocks are told apart (none are too many), and the one that
    comes again is found."""
    cells = np.asarray(list(blocks), np.int64) * 64 + 7
    top = int(cells.max()) // 64 + 1
    rng = np.random.default_rng(len(cells))
    for at in (0, len(cells) // 2, len(cells) - 1):
        assert store(hip, np.append(rng.permutation(cells), cells[at]), top) == hip.EINVAL
        assert "block %d is written twice" % (cells[at] // 64) in hip.last_error()


@pytest.mark.parametrize("kv", [65536, 130000, 1 << 28])
def test_pools_of_more_kv_heads_than_a_launch_takes_are_refused(hip, kv):
    """(The bytes of a block past 2^31 would not be counted right.)"""
    L, d, c = hip.lib(), C.c_void_p(256), np.zeros(1, np.int64)
    assert L.lgmlh_kv_store_q8(d, d, 64, kv, 256, d, d, d, c.ctypes.data, 1, None) == hip.EINVAL
    assert L.lgmlh_kv_gather_q8(d, 0, 64, kv, 256, d, 1, d, hip.F32, None) == hip.EINVAL
    assert L.lgmlh_kv_gather_q8(d, 1, 64, kv, 256, d, 0, d, hip.F32, None) == hip.EINVAL
