"""CPU checks of the Q4_0 pool, copies of blocks, relocation and rope by several axes:
refusals, sizes, the bookkeeping of forks and compaction (no GPU work)."""
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


def test_sizes(hip):
    L = hip.lib()
    for d in (64, 128, 256):
        assert L.lgmlh_kv_q4_layer_bytes(64, 3, d) == 3 * 36 * d
        # as f16 heads of 9 D / 32, for the entry points that copy whole blocks
        assert L.lgmlh_kv_block_bytes(3, d * 9 // 32) == 3 * 36 * d
    assert L.lgmlh_kv_q4_layer_bytes(1 << 36, 8, 128) == (1 << 30) * 8 * 36 * 128
    for bad in ((64, 3, 32), (64, 3, 96), (63, 3, 64), (64, 0, 64), (0, 1, 64)):
        assert L.lgmlh_kv_q4_layer_bytes(*bad) == -1
    assert L.lgmlh_row_size(hip.Q4_0, 4096) == -1  # a type of pools only
    assert L.lgmlh_repacked_bytes(hip.Q4_0, 64, 256) < 0


def test_store_and_gather_refuse(hip):
    L = hip.lib()

    def store(kp=D16, vp=D16, cells_n=128, kv=2, d=64, ks=D16, vs=D16, dc=D16, h=(3, 5), n=None):
        c = None if h is None else np.array(h, np.int64)
        return L.lgmlh_kv_store_q4(kp, vp, cells_n, kv, d, ks, vs, dc, None if c is None else c.ctypes.data,
                                   len(c) if n is None else n, None)

    assert store(h=(), n=0) == hip.OK
    for kw in (dict(kp=None), dict(vp=None), dict(ks=None), dict(vs=None), dict(dc=None), dict(cells_n=100),
               dict(cells_n=0), dict(kv=0), dict(kv=65536), dict(d=96), dict(d=32), dict(n=-1), dict(h=None, n=1),
               dict(kp=C.c_void_p(260)), dict(vp=C.c_void_p(264)), dict(h=(3, 3)), dict(cells_n=(1 << 36) + 64),
               dict(n=1 << 29)):
        assert store(**kw) == hip.EINVAL, kw
    for h in ((-1, 3), (3, 128), (1 << 40, 2)):
        assert store(h=h) == hip.ERANGE, h

    def gather(pool=D16, which=0, cells_n=128, kv=2, d=64, dc=D16, n=0, out=D16, ty=hip.F32):
        return L.lgmlh_kv_gather_q4(pool, which, cells_n, kv, d, dc, n, out, ty, None)

    assert gather() == hip.OK
    for kw in (dict(pool=None), dict(which=2), dict(cells_n=65), dict(kv=70000), dict(d=16), dict(dc=None),
               dict(n=-2), dict(out=None), dict(ty=hip.Q4_0), dict(pool=C.c_void_p(8))):
        assert gather(**kw) == hip.EINVAL, kw


def test_attention_refuses(hip):
    L = hip.lib()
    info, ub = hip.PlanInfo(), hip.Ubatch()
    one, zero, tab = np.ones(1, np.int32), np.zeros(1, np.int32), np.zeros(1, np.int32)
    args = (1, one.ctypes.data, zero.ctypes.data, tab.ctypes.data, 1, 1, zero.ctypes.data, 8, 2, 0)
    hip.check(L.lgmlh_plan(*args, None, 0, C.byref(info)))
    buf = np.zeros(info.bytes, np.uint8)
    hip.check(L.lgmlh_plan(*args, buf.ctypes.data, buf.nbytes, C.byref(info)))
    hip.check(L.lgmlh_plan_bind(C.byref(info), buf.ctypes.data, C.byref(ub)))

    def call(q=D16, H=8, kv=2, d=64, kp=D16, vp=D16, out=D16):
        return L.lgmlh_paged_attention_q4(q, H, kv, d, 0.1, kp, vp, C.byref(ub), out, D16, 1 << 20, None)

    for kw in (dict(q=None), dict(H=6), dict(H=64), dict(kv=4), dict(d=32), dict(d=96), dict(kp=None), dict(vp=None),
               dict(out=None), dict(kp=C.c_void_p(8)), dict(vp=C.c_void_p(24))):
        assert call(**kw) == hip.EINVAL, kw
    m = hip.Model()
    m.n_layer, m.n_embd, m.n_head, m.n_head_kv, m.head_dim = 1, 64, 4, 4, 16
    layers = (hip.Layer * 1)()
    m.layers = layers
    assert L.lgmlh_forward_q4(C.byref(m), C.byref(ub), None, None, 1, D16, D16, 1 << 20, None, None) == hip.EINVAL
    assert "heads of 16" in hip.last_error()


def test_copies_refuse(hip):
    L = hip.lib()

    def copy(c, ty=hip.F16, pools=D16, n_pools=2, cells=64 * 10, kv=2, d=64, dc=D16, n=None, host=True):
        h = np.array(c, np.int32).reshape(-1, 3)
        return L.lgmlh_kv_copy_blocks(ty, pools, n_pools, cells, kv, d, dc, h.ctypes.data if host else None,
                                      len(h) if n is None else n, None)

    assert copy([]) == hip.OK
    for c in ([(0, 1, 64), (2, 1, 3)], [(0, 1, 64), (1, 2, 64)], [(1, 2, 64), (0, 1, 0)], [(4, 4, 64)],
              [(0, 1, 65)], [(0, 1, -1)], [(-1, 3, 64), (3, 5, 64)], [(-1, 3, 64), (-1, 3, 64)]):
        assert copy(c) == hip.EINVAL, c
    for c in ([(0, 10, 64)], [(10, 0, 64)], [(-2, 0, 64)], [(0, -1, 64)], [(2**31 - 1, 0, 1)]):
        assert copy(c) == hip.ERANGE, c
    ok = [(0, 1, 64)]
    for kw in (dict(ty=hip.F32), dict(ty=hip.Q4_K), dict(pools=None), dict(n_pools=0), dict(n_pools=3),
               dict(n_pools=65536), dict(cells=100), dict(cells=0), dict(kv=0), dict(d=12), dict(d=2048),
               dict(ty=hip.Q4_0, d=32), dict(ty=hip.Q8_0, d=96), dict(dc=None), dict(host=False), dict(n=-1),
               dict(n=1 << 40), dict(kv=65536)):
        assert copy(ok, **kw) == hip.EINVAL, kw


@pytest.mark.parametrize("n", [200, 5000])
def test_a_block_named_twice_is_found_among_many(hip, n):
    rng = np.random.default_rng(n)
    blocks = rng.permutation(1 << 20)[:2 * n].astype(np.int32)
    c = np.stack([blocks[:n], blocks[n:], np.full(n, 64, np.int32)], 1)

    def copy(c):
        c = np.ascontiguousarray(c)
        return hip.lib().lgmlh_kv_copy_blocks(hip.F16, D16, 2, 64 << 20, 1, 64, D16, c.ctypes.data, len(c), None)

    for at in (0, n // 2, n - 1):
        for bad in ((c[at, 0], c[at - 1, 1], 1), (c[at, 1], 1 << 19, 1), (7, c[at, 0], 1)):
            assert copy(np.vstack([c, [bad]]).astype(np.int32)) == hip.EINVAL


def test_rope_axes_refuses(hip):
    L = hip.lib()

    def call(ty=hip.F16, x=D16, n=0, H=8, kv=2, d=128, rot=128, sec=(16, 24, 24, 0), inter=0, base=1e4, pos=D16,
             kp=D16, vp=D16, cells_n=64, cells=D16, q=D16):
        s = None if sec is None else np.array(sec, np.int32)
        return L.lgmlh_qkv_rope_store_axes(ty, x, n, H, kv, d, rot, None if s is None else s.ctypes.data, inter, base,
                                           None, None, None, 1e-6, pos, kp, vp, cells_n, cells, q, None)

    assert call() == hip.OK and call(sec=(24, 20, 20, 0), inter=1) == hip.OK and call(rot=64, sec=(32, 0, 0, 0)) == hip.OK
    for kw in (dict(ty=hip.F32), dict(x=None), dict(n=-1), dict(H=0), dict(kv=0), dict(kv=70000), dict(d=96),
               dict(d=32), dict(rot=0), dict(rot=132), dict(rot=12, sec=(2, 2, 2, 0)), dict(sec=None),
               dict(sec=(16, 24, 23, 0)), dict(sec=(16, 24, 25, 0)), dict(sec=(-1, 40, 25, 0)),
               dict(sec=(2**31 - 1, 2**31 - 1, 66, 0)), dict(sec=(16, 16, 16, 16), inter=1), dict(base=0.0),
               dict(base=float("nan")), dict(pos=None), dict(kp=None), dict(vp=C.c_void_p(8)), dict(cells_n=65),
               dict(cells=None), dict(q=None), dict(n=1 << 23)):
        assert call(**kw) == hip.EINVAL, kw


# ---- bookkeeping -----------------------------------------------------------------
def test_relocate_takes_the_record_along(hip):
    from lgml_amd import kvpool
    p = kvpool.Pool(8, 64)
    for _ in range(6):
        p.take()
    toks = list(range(64))
    k = kvpool.key("root", toks)
    assert p.publish(5, k, "root", 1, toks, kvpool.HIGH)
    p.ref(5)
    assert p.publish_part(4, k, 2, [1, 2, 3], kvpool.LOW)
    p.unref(4)  # kept for its tokens
    p.unref(1)
    p.unref(2)
    used, cached = p.used, p.cached
    for src, dst in ((1, 7), (5, 0), (5, 4), (5, 5), (8, 1), (5, 8), (-1, 1), (5, -1)):
        with pytest.raises(hip.LgmlhError):
            p.relocate(src, dst)
    p.relocate(5, 1)
    p.relocate(4, 2)
    assert (p.used, p.cached) == (used, cached)
    assert p.lookup(k) == 1 and p.refs_of(1) == 2 and p.key_of(1) == k and p.key_of(5) is None and p.refs_of(5) == 0
    assert p.longest_kid(k, [1, 2, 9], 1, 3) == (2, 2) and p.refs_of(2) == 0 and p.in_use(2) and not p.in_use(4)
    assert p.longest_kid("root", toks, 1, 64) == (1, 64)
    assert p.take() == 4 and p.take() == 5 and p.take() == 6  # low went down to the freed places
    p.unref(1)
    p.unref(1)
    assert p.evict() == 2 and p.evict() == 1  # lowest priority first, as before
    assert p.lookup(k) is None


class _Model:
    def __init__(self, blocks):
        self.pool_blocks, self.n_cells = blocks, 64 * blocks
        self.calls = []

    def copy_blocks(self, src, dst, cells=64):
        self.calls.append((list(src), list(dst), cells))


def test_forks_share_full_blocks_and_copy_the_partial_one(hip):
    from lgml_amd import engine
    m = _Model(12)
    seqs = engine.PoolSeqs(m)
    c = engine.Seq(seqs, 2)
    seqs.reserve(c, 150)
    c.n_past = 150
    kids = seqs.fork(c, 3)
    assert m.calls == [([2, 2, 2], [3, 4, 5], 22)]
    assert [k.blocks for k in kids] == [[0, 1, 3], [0, 1, 4], [0, 1, 5]] and [k.prio for k in kids] == [2] * 3
    assert [seqs.alloc.refs_of(b) for b in range(6)] == [4, 4, 1, 1, 1, 1]
    more = seqs.fork(kids[0])  # a fork of a fork
    assert more[0].blocks == [0, 1, 6] and seqs.fork(c, 0) == []
    with pytest.raises(engine.PoolFull):
        seqs.fork(c, 6)  # five blocks are free
    assert seqs.alloc.used == 7 and seqs.alloc.refs_of(0) == 5
    c.n_past = 128
    k = seqs.fork(c, 2)
    assert len(m.calls) == 2 and all(x.blocks == [0, 1] for x in k)
    for x in [c] + kids + more + k:
        seqs.free(x)
    assert seqs.alloc.used == 0
    empty = seqs.fork(c, 2)
    assert [x.blocks for x in empty] == [[], []]


def test_compaction_keeps_tables_references_and_keys(hip):
    from lgml_amd import engine, kvpool
    rng = np.random.default_rng(5)
    m = _Model(60)
    seqs = engine.PoolSeqs(m)
    all_ = [engine.Seq(seqs) for _ in range(8)]
    for _ in range(5):
        for i in rng.permutation(8):
            c = all_[i]
            seqs.reserve(c, c.n_past + 64)
            c.n_past += 64
    content = {b: ("cells", b) for b in range(60)}
    toks = list(range(64))
    key = kvpool.key("root", toks)
    kept = all_[7].blocks[0]
    assert seqs.alloc.publish(kept, key, "root", 1, toks)
    for i in (0, 2, 7):
        seqs.free(all_[i])
    live = [all_[i] for i in (1, 3, 4, 5, 6)]
    live += seqs.fork(live[0])
    want = [[content[b] for b in c.blocks] for c in live]
    refs = [[seqs.alloc.refs_of(b) for b in c.blocks] for c in live]
    m.calls.clear()
    with pytest.raises(ValueError):
        seqs.compact(live[1:])
    assert m.calls == []
    n = seqs.compact(live)
    assert n == 26 and len(m.calls) == 1
    src, dst, cells = m.calls[0]
    assert cells == 64 and not set(src) & set(dst) and min(src) >= n > max(dst)
    for a, b in zip(src, dst):
        content[b] = content[a]
    assert [[content[b] for b in c.blocks] for c in live] == want
    assert [[seqs.alloc.refs_of(b) for b in c.blocks] for c in live] == refs
    assert content[seqs.alloc.lookup(key)] == ("cells", kept) and seqs.alloc.lookup(key) < n
    assert [seqs.alloc.in_use(b) for b in range(60)] == [True] * n + [False] * (60 - n)
    m.calls.clear()
    assert seqs.compact(live) == n and m.calls == []  # nothing left to move
    seqs.alloc.set_cap(n)
    with pytest.raises(engine.PoolFull):
        seqs.fork(c := live[0], 1) and seqs.reserve(c, 64 * 60)


def test_new_kernels_use_no_scratch():
    pytest.importorskip("msgpack")
    from tests.test_kernel_resources import kernels
    all_ = kernels()
    for name in ("paged_attn_q4_kernel", "kv_store_q4_kernel", "kv_gather_q4_k_kernel", "kv_gather_q4_v_kernel",
                 "kv_gather_q4_v_few_kernel", "merge_slices_kernel", "kv_copy_blocks_kernel", "qkv_rope_axes_kernel"):
        got = {n: k for n, k in all_.items() if name in n}
        assert got, name
        for n, k in got.items():
            assert k[".private_segment_fixed_size"] == 0 and k.get(".vgpr_spill_count", 0) == 0, n
