"""CPU checks of lgmlh_plan_tree and of the argument checks of the entry points
around drafted tokens and the Q8_0 pool (no GPU work)."""
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


def plan_tree(hip, seq_n, npast, parents, bt, H, Hkv, pool_blocks, bps=0, ids=None):
    L = hip.lib()
    info = hip.PlanInfo()
    keep = [np.ascontiguousarray(a, np.int32) for a in
            (seq_n, npast, parents, bt, np.zeros(sum(seq_n)) if ids is None else ids)]
    args = (len(seq_n), keep[0].ctypes.data, keep[1].ctypes.data, keep[2].ctypes.data,
            keep[3].ctypes.data, keep[3].shape[1], pool_blocks, keep[4].ctypes.data, H, Hkv, bps)
    rc = L.lgmlh_plan_tree(*args, None, 0, C.byref(info))
    if rc:
        return rc, None, None
    buf = np.full(info.bytes + 64, 0xA5, np.uint8)
    assert L.lgmlh_plan_tree(*args, buf.ctypes.data, info.bytes - 1, C.byref(info)) == hip.ENOMEM
    rc = L.lgmlh_plan_tree(*args, buf.ctypes.data, info.bytes, C.byref(info))
    assert (buf[info.bytes:] == 0xA5).all()
    return rc, info, buf[:info.bytes]


def arr(buf, off, n, dt):
    return buf[off:off + n * np.dtype(dt).itemsize].view(dt)


def tree(rng, n):
    return [-1] + [int(rng.integers(max(-1, j - 9), j)) for j in range(1, n)]


@pytest.mark.parametrize("H,Hkv", [(4, 4), (8, 4), (32, 8), (32, 4), (16, 1)])
@pytest.mark.parametrize("bps", [0, 2])
def test_masks_positions_and_cells(hip, H, Hkv, bps):
    rng = np.random.default_rng(H + bps)
    seq_n = [1, 9, 64, 0, 70, 130, 33]
    npast = [0, 63, 64, 5, 1000, 37, 127]
    nb = [max(1, (p + n + 63) // 64) for p, n in zip(npast, seq_n)]
    bt = np.full((len(seq_n), max(nb)), -1, np.int32)
    order, at = rng.permutation(sum(nb)), 0
    for s, k in enumerate(nb):
        bt[s, :k] = order[at:at + k]
        at += k
    parents = sum((tree(rng, n) if n else [] for n in seq_n), [])
    rc, info, buf = plan_tree(hip, seq_n, npast, parents, bt, H, Hkv, sum(nb), bps)
    assert rc == 0 and info.ring == hip.PLAN_TREE
    N, W = sum(seq_n), info.window
    assert info.n_tokens == N
    pos, cells = arr(buf, info.off_pos, N, np.int32), arr(buf, info.off_cells, N, np.int64)
    off_vis = (info.off_order + 4 * info.n_single + 15) // 16 * 16
    vis = arr(buf, off_vis, N * W, np.uint64).reshape(N, W)
    assert off_vis + 8 * N * W <= info.bytes
    t = 0
    for s, (n, p0) in enumerate(zip(seq_n, npast)):
        for j in range(n):
            line, a = set(), j
            while a >= 0:
                line.add(a)
                a = parents[t - j + a]
            assert pos[t] == p0 + len(line) - 1
            slot = p0 + j
            assert cells[t] == bt[s, slot // 64] * 64 + slot % 64
            for w in range(W):
                for c in range(64):
                    x = (p0 // 64 + w) * 64 + c  # the slot of bit c
                    want = x < p0 or (x - p0) in line
                    assert bool(int(vis[t, w]) >> c & 1) == want, (t, w, c)
            t += 1
    # the work list is the causal plan's over the slots
    causal = hip.PlanInfo()
    a = [np.ascontiguousarray(x, np.int32) for x in (seq_n, npast, bt)]
    assert hip.lib().lgmlh_plan(len(seq_n), a[0].ctypes.data, a[1].ctypes.data, a[2].ctypes.data,
                                bt.shape[1], sum(nb), None, H, Hkv, bps, None, 0,
                                C.byref(causal)) == 0
    assert (causal.n_items, causal.n_merge, causal.n_single, causal.n_shared) == \
        (info.n_items, info.n_merge, info.n_single, info.n_shared)


def test_tree_refusals(hip):
    bt = np.array([[0, 1]], np.int32)
    ok = plan_tree(hip, [3], [10], [-1, 0, 0], bt, 4, 2, 2)
    assert ok[0] == 0
    for bad in ([0, 0, 0], [-1, 1, 0], [-1, 0, 2], [-1, -2, 0], [-1, 0, 7]):
        assert plan_tree(hip, [3], [10], bad, bt, 4, 2, 2)[0] == hip.ERANGE, bad
        assert "parent" in hip.last_error()
    assert plan_tree(hip, [3], [126], [-1, 0, 0], bt, 4, 2, 2)[0] == hip.ERANGE  # a third block
    assert plan_tree(hip, [3], [10], [-1, 0, 0], np.array([[5, 1]], np.int32), 4, 2, 2)[0] == hip.ERANGE
    assert plan_tree(hip, [3], [10], [-1, 0, 0], bt, 5, 2, 2)[0] == hip.EINVAL
    assert plan_tree(hip, [3], [10], [-1, 0, 0], bt, 0, 2, 2)[0] == hip.EINVAL
    big = np.arange(40, dtype=np.int32)[None]
    assert plan_tree(hip, [hip.TREE_MAX], [10], [-1] * hip.TREE_MAX, big, 4, 2, 40)[0] == 0
    n = hip.TREE_MAX + 1
    assert plan_tree(hip, [n], [10], [-1] * n, big, 4, 2, 40)[0] == hip.EINVAL
    info = hip.PlanInfo()
    a = [np.ascontiguousarray(x, np.int32) for x in ([3], [10])]
    assert hip.lib().lgmlh_plan_tree(1, a[0].ctypes.data, a[1].ctypes.data, None, bt.ctypes.data, 2, 2,
                                     None, 4, 2, 0, None, 0, C.byref(info)) == hip.EINVAL


def test_q8_sizes_and_refusals(hip):
    L, d = hip.lib(), C.c_void_p(256)
    assert L.lgmlh_kv_q8_layer_bytes(128, 8, 128) == 2 * 8 * 68 * 128
    assert 32 * L.lgmlh_kv_q8_layer_bytes(640, 4, 64) == 17 * L.lgmlh_kv_layer_bytes(640, 4, 64)
    for bad in ((100, 8, 128), (0, 8, 128), (64, 0, 128), (64, 8, 96), (64, 8, 32)):
        assert L.lgmlh_kv_q8_layer_bytes(*bad) == -1

    def store(cells, n_cells=128, kv=8, dim=128, k=d):
        c = np.ascontiguousarray(cells, np.int64)
        return L.lgmlh_kv_store_q8(k, d, n_cells, kv, dim, d, d, d, c.ctypes.data, len(c), None)

    assert store([]) == hip.OK
    assert store([0, 128]) == hip.ERANGE and store([-1]) == hip.ERANGE
    assert store([3], dim=96) == hip.EINVAL and store([3], n_cells=100) == hip.EINVAL
    assert store([3], k=None) == hip.EINVAL and store([3], kv=0) == hip.EINVAL
    assert store([5, 6, 5]) == hip.EINVAL and "twice" in hip.last_error()
    assert store([5, 5]) == hip.EINVAL
    # a cell twice among many: whole blocks in a shuffled order, then one of their cells
    rng = np.random.default_rng(1)
    blocks = rng.permutation(5000)
    many = (blocks[:, None] * 64 + np.arange(64)[None]).reshape(-1)
    assert store(np.append(many, many[77777]), n_cells=5000 * 64) == hip.EINVAL
    lone = rng.permutation(5000 * 64)[:9000]
    assert store(np.append(lone, lone[1234]), n_cells=5000 * 64) == hip.EINVAL
    assert L.lgmlh_kv_store_q8(d, d, 128, 8, 128, d, d, d, None, 1, None) == hip.EINVAL
    g = L.lgmlh_kv_gather_q8
    assert g(d, 2, 128, 8, 128, d, 1, d, hip.F32, None) == hip.EINVAL
    assert g(d, 0, 128, 8, 128, d, 1, d, hip.Q8_0, None) == hip.EINVAL
    assert g(d, 0, 128, 8, 100, d, 1, d, hip.F32, None) == hip.EINVAL
    assert g(d, 0, 128, 8, 128, d, -1, d, hip.F32, None) == hip.EINVAL
    assert g(d, 0, 128, 8, 128, d, 0, d, hip.F16, None) == hip.OK


def test_move_refusals(hip):
    L, d = hip.lib(), C.c_void_p(256)

    def move(src, dst, ty=hip.F16, pools=4, n_cells=128, kv=2, dim=64, host=True):
        s, t = (np.ascontiguousarray(a, np.int64) for a in (src, dst))
        return L.lgmlh_kv_move(ty, d, pools, n_cells, kv, dim, d, d, s.ctypes.data if host else None,
                               t.ctypes.data, len(s), None)

    assert move([], []) == hip.OK
    assert move([1], [128]) == hip.ERANGE and move([128], [1]) == hip.ERANGE and move([-1], [1]) == hip.ERANGE
    assert move([1, 2], [7, 7]) == hip.EINVAL and "twice" in hip.last_error()
    assert move([1], [2], ty=hip.F32) == hip.EINVAL and move([1], [2], pools=3) == hip.EINVAL
    assert move([1], [2], pools=0) == hip.EINVAL and move([1], [2], n_cells=100) == hip.EINVAL
    assert move([1], [2], ty=hip.Q8_0, dim=32) == hip.EINVAL and move([1], [2], dim=40) == hip.EINVAL
    assert move([1], [2], host=False) == hip.EINVAL
    assert move(np.arange(1025), np.arange(1025), n_cells=6400) == hip.EINVAL


def test_log_probs_refusals(hip):
    L, d = hip.lib(), C.c_void_p(256)
    ws = L.lgmlh_log_probs_workspace

    def lp(rows=4, cols=1000, ids=d, n_ids=1, id_lp=d, ent=d, top=5, top_ids=d, top_lp=d, w=d, wb=1 << 30):
        return L.lgmlh_log_probs(d, rows, cols, ids, n_ids, id_lp, ent, top, top_ids, top_lp, w, wb, None)

    assert lp(rows=0) == hip.OK
    assert lp(rows=-1) == hip.EINVAL and lp(cols=0) == hip.EINVAL and lp(cols=(1 << 20) + 1) == hip.EINVAL
    assert lp(ids=None) == hip.EINVAL and lp(id_lp=None) == hip.EINVAL and lp(n_ids=65) == hip.EINVAL
    assert lp(top=65) == hip.EINVAL and lp(cols=4, top=5) == hip.EINVAL and lp(top=-1) == hip.EINVAL
    assert lp(top_ids=None, top_lp=None) == hip.EINVAL
    assert lp(w=None) == hip.ENOMEM and lp(wb=ws(4, 1000, 5) - 1) == hip.ENOMEM
    assert lp(w=C.c_void_p(264)) == hip.ENOMEM
    assert lp(rows=2**31 - 1, cols=1 << 20, wb=1 << 62) == hip.EINVAL  # the launch
    # a workspace for the largest call holds the smaller ones
    for cols in (1, 64, 8192, 128256, 151936, 1 << 20):
        size = [ws(n, cols, 20) for n in range(1, 700)]
        assert all(a < b for a, b in zip(size, size[1:]))
    assert ws(3, 1000, 0) < ws(3, 1000, 1) == ws(3, 1000, 64)


def test_attention_q8_refusals(hip):
    L, d = hip.lib(), C.c_void_p(256)
    rc, info, buf = plan_tree(hip, [3], [10], [-1, 0, 0], np.array([[0, 1]], np.int32), 4, 2, 2)
    ub = hip.Ubatch()
    assert L.lgmlh_plan_bind(C.byref(info), buf.ctypes.data, C.byref(ub)) == 0
    assert ub.ring == hip.PLAN_TREE
    for fn in (L.lgmlh_paged_attention_q8, L.lgmlh_paged_attention):
        assert fn(d, 4, 2, 96, 1.0, d, d, C.byref(ub), d, d, 1 << 20, None) == hip.EINVAL
        assert fn(d, 8, 2, 64, 1.0, d, d, C.byref(ub), None, d, 1 << 20, None) == hip.EINVAL
        assert fn(d, 0, 2, 64, 1.0, d, d, C.byref(ub), d, d, 1 << 20, None) == hip.EINVAL
        assert fn(d, 4, 4, 64, 1.0, d, d, C.byref(ub), d, d, 1 << 20, None) == hip.EINVAL  # another plan's
    assert L.lgmlh_paged_attention_q8(d, 4, 2, 32, 1.0, d, d, C.byref(ub), d, d, 1 << 20, None) == hip.EINVAL


def test_forward_refuses_a_tree_through_sliding_layers(hip):
    L = hip.lib()
    rc, info, buf = plan_tree(hip, [3], [10], [-1, 0, 0], np.array([[0, 1]], np.int32), 4, 2, 2)
    ub = hip.Ubatch()
    L.lgmlh_plan_bind(C.byref(info), buf.ctypes.data, C.byref(ub))
    layers = (hip.Layer * 1)()
    layers[0].swa = 1
    m = hip.Model()
    m.n_layer, m.n_embd, m.n_head, m.n_head_kv, m.head_dim = 1, 256, 4, 2, 64
    m.layers = layers
    d = C.c_void_p(256)
    assert L.lgmlh_forward(C.byref(m), C.byref(ub), C.byref(ub), None, 0, d, d, 1 << 30, None,
                           None) == hip.EINVAL
    assert "tree" in hip.last_error()


def test_refusals_of_more_than_a_launch_holds(hip):
    """Before anything of the arguments is read."""
    L, d = hip.lib(), C.c_void_p(256)
    n = (1 << 29) // 8
    assert L.lgmlh_kv_store_q8(d, d, 128, 8, 128, d, d, d, d, n, None) == hip.EINVAL
    assert L.lgmlh_kv_gather_q8(d, 0, 128, 8, 128, d, n, d, hip.F32, None) == hip.EINVAL
    assert L.lgmlh_kv_move(hip.F16, d, 2, 128, 1 << 16, 64, d, d, d, d, 1, None) == hip.EINVAL
    assert L.lgmlh_log_probs(d, 1 << 24, 1, None, 0, None, d, 0, None, None, d, 1 << 40, None) == hip.EINVAL


def test_q8_pools_off_their_alignment_are_refused(hip):
    L, d, odd = hip.lib(), C.c_void_p(256), C.c_void_p(264)
    c = np.array([3], np.int64)
    h = c.ctypes.data
    assert L.lgmlh_kv_store_q8(odd, d, 128, 8, 128, d, d, d, h, 1, None) == hip.EINVAL
    assert L.lgmlh_kv_store_q8(d, odd, 128, 8, 128, d, d, d, h, 1, None) == hip.EINVAL
    assert L.lgmlh_kv_gather_q8(odd, 0, 128, 8, 128, d, 1, d, hip.F32, None) == hip.EINVAL
    assert L.lgmlh_qkv_rope_store_q8(d, 1, 4, 2, 64, 64, 0, 1e4, None, None, None, 1e-5, d, d, odd, 128, d, d,
                                     None) == hip.EINVAL
    rc, info, buf = plan_tree(hip, [3], [10], [-1, 0, 0], np.array([[0, 1]], np.int32), 4, 2, 2)
    ub = hip.Ubatch()
    assert L.lgmlh_plan_bind(C.byref(info), buf.ctypes.data, C.byref(ub)) == 0
    assert L.lgmlh_paged_attention_q8(d, 4, 2, 64, 1.0, d, odd, C.byref(ub), d, d, 1 << 20, None) == hip.EINVAL
