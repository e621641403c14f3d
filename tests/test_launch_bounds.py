"""CPU checks: calls of the quantised pools' operators that would take 2^32 threads in a
launch are refused by their checks of arguments (no GPU work)."""
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


D16 = C.c_void_p(256)


@pytest.mark.parametrize("items,kv", [(1 << 24, 1), (1 << 21, 8), ((1 << 25) // 3, 2)])
def test_attention_over_q4(hip, items, kv):
    """Four waves an item and KV head."""
    ub = hip.Ubatch()
    ub.n_items, ub.rows, ub.n_head_kv, ub.n_seq, ub.n_tokens, ub.max_blocks = items, 16, kv, 1, 1, 1
    assert hip.lib().lgmlh_paged_attention_q4(D16, 4 * kv, kv, 64, 0.1, D16, D16, C.byref(ub), D16, D16, 0,
                                              None) == hip.EINVAL
    assert "in one launch" in hip.last_error()


@pytest.mark.parametrize("kind", ["q4", "q8"])
@pytest.mark.parametrize("kv,n,D", [(65000, 8258, 256), (50000, 10736, 256)])
def test_rows_that_fill_their_last_workgroups_in_part(hip, kind, kv, n, D):
    """n KV heads times rows of 32 a workgroup, rounded up for each head."""
    L = hip.lib()
    cells = np.arange(n, dtype=np.int64)
    n_cells = (n + 63) // 64 * 64
    assert n < (1 << 29) // kv and (n + 31) // 32 * kv >= 1 << 24
    store, gather = getattr(L, "lgmlh_kv_store_" + kind), getattr(L, "lgmlh_kv_gather_" + kind)
    assert store(D16, D16, n_cells, kv, D, D16, D16, D16, cells.ctypes.data, n, None) == hip.EINVAL
    assert "workgroups in one launch" in hip.last_error()
    if kind == "q8":
        assert gather(D16, 0, n_cells, kv, D, D16, n, D16, hip.F32, None) == hip.EINVAL


@pytest.mark.parametrize("which,kv,n,D", [(0, 1, (1 << 29) - 1, 64), (0, 1, (1 << 28) - 1, 256),
                                          (0, 16384, (1 << 15) - 1, 128), (0, 60000, 4472, 256)])
def test_read_back_of_q4(hip, which, kv, n, D):
    """8 threads a row of K (16, heads of 256)."""
    L = hip.lib()
    for ty in (hip.F32, hip.F16):
        assert L.lgmlh_kv_gather_q4(D16, which, 64, kv, D, D16, n, D16, ty, None) == hip.EINVAL
