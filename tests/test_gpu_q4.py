"""The Q4_0 KV pool and attention over it, on the GPU, against plain 64-bit
implementations: store, read back, moves of cells, causal, ring and tree plans,
cells that a row does not see, scales of any size, rows in any group of rows,
pools past 4 GiB."""
import ctypes as C

import numpy as np
import pytest

from tests.test_gpu_draft import GAINS, SEQS, Pass, attend, bound, dev, seen, st, tree

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def L():
    from lgml_amd import hip
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    return hip.lib()


# ---- the plain forms -------------------------------------------------------------
def quants(x):
    """Q4_0 of (n, kv, D) f32 in its defined steps: (n uint8, d f16)."""
    n, kv, d = x.shape
    g = x.reshape(n, kv, d // 32, 32)
    m = np.take_along_axis(g, np.abs(g).argmax(-1)[..., None], -1)  # the first of the largest
    dd = m * np.float32(-0.125)
    with np.errstate(divide="ignore"):
        inv = np.where(dd != 0, np.float32(1) / dd, np.float32(0)).astype(np.float32)
    y = (g * inv).astype(np.float32) + np.float32(8.5)
    q = np.minimum(15, np.trunc(y))
    return q.reshape(n, kv, d).astype(np.uint8), dd[..., 0].astype(np.float16)


def values(x):
    q, d = quants(x)
    return (q.astype(np.float64) - 8) * np.repeat(d.astype(np.float64), 32, -1)


def k_tile(q, d, D):
    """A tile of K (36 D bytes) from 64 cells' n (64, D) and d (64, D / 32) f16."""
    U = min(4, D // 32)
    v = q.reshape(64, D // 32 // U, U, 4, 8).astype(np.uint32)
    word = sum(v[..., e] << np.uint32(4 * (e // 2) + 16 * (e % 2)) for e in range(8))
    word = np.ascontiguousarray(word.transpose(1, 0, 3, 2))
    return np.concatenate([word.reshape(-1).view(np.uint8), d.T.copy().reshape(-1).view(np.uint8)])


def v_tile(q, d, D):
    v = q.T.reshape(D // 32, 2, 16, 2, 4, 8)
    byte = np.zeros((D // 32, 16, 4, 2, 8), np.uint8)
    for e, p in enumerate([0, 2, 1, 3, 4, 6, 5, 7]):
        byte[..., p] = (v[:, 0, ..., e] | v[:, 1, ..., e] << 4).transpose(0, 1, 3, 2)
    return np.concatenate([byte.reshape(-1), d.T.copy().reshape(-1).view(np.uint8)])


def fill(L, P, kv, D, k, v):
    from lgml_amd import hip
    cells = np.arange(P.n_cells, dtype=np.int64)
    dc, kd, vd = dev(cells), dev(k), dev(v)
    nb = L.lgmlh_kv_q4_layer_bytes(P.n_cells, kv, D)
    pools = [torch.zeros(nb, dtype=torch.uint8, device="cuda") for _ in range(2)]
    hip.check(L.lgmlh_kv_store_q4(pools[0].data_ptr(), pools[1].data_ptr(), P.n_cells, kv, D, kd.data_ptr(),
                                  vd.data_ptr(), dc.data_ptr(), cells.ctypes.data, len(cells), st()))
    torch.cuda.synchronize()
    return pools, values(k), values(v)


def run_attention(L, P, H, kv, D, scale, q, pools):
    from lgml_amd import hip
    qd = dev(q)
    out = torch.full((len(q) + 1, H, D), 7.0, dtype=torch.float32, device="cuda")
    nb = L.lgmlh_attention_workspace(C.byref(P.info), D)
    ws = torch.full((nb + 256,), 0xA5, dtype=torch.uint8, device="cuda")
    hip.check(L.lgmlh_paged_attention_q4(qd.data_ptr(), H, kv, D, scale, pools[0].data_ptr(), pools[1].data_ptr(),
                                         C.byref(P.ub), out.data_ptr(), ws.data_ptr(), nb, st()))
    torch.cuda.synchronize()
    assert bool((out[-1] == 7.0).all()) and bool((ws[nb:] == 0xA5).all())
    return out[:-1].cpu().numpy().astype(np.float64)


# ---- the pool --------------------------------------------------------------------
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("kv", [1, 3, 8])
@pytest.mark.parametrize("many", [False, True])
def test_store_writes_the_defined_bytes(L, D, kv, many):
    """Every byte of the pool: runs of cells from odd offsets, lone cells, cells in any
    order, values at the borders of a step, ties of the largest of either sign, zero
    blocks, tiny and huge ones; cells not written stay."""
    from lgml_amd import hip
    rng = np.random.default_rng(D + kv)
    blocks = 70 if many else 7
    runs = [(64 + 3, 70), (200, 1), (5 * 64, 64), (6 * 64 + 1, 7), (6 * 64 + 9, 1), (6 * 64 + 20, 33), (2, 1)]
    cells = np.concatenate([np.arange(a, a + n) for a, n in runs]).astype(np.int64)
    if many:  # enough for the wider windows
        cells = np.concatenate([cells, 7 * 64 + rng.permutation(1000), np.arange(24 * 64 + 5, 69 * 64)])
    n = len(cells)
    x = [rng.standard_normal((n, kv, D)).astype(np.float32) for _ in range(2)]
    for w in range(2):
        x[w][0] = 0.0
        x[w][1, :, :32] = (np.arange(32) % 17 - 8) * np.float32(0.5) + np.float32(0.25) * (np.arange(32) % 2)
        x[w][1, :, 5] = -8.0  # d = 1: x + 8.5 on whole numbers
        x[w][2] *= np.float32(1e-30)
        x[w][3] *= np.float32(6e4)
        x[w][4, :, 32:64] = np.float32(2.0**-20) * rng.integers(-3, 4, (kv, 32))
        x[w][5, :, :32] = np.float32(0.3)
        x[w][5, :, [7, 20]] = np.array([2.5, -2.5], np.float32)[:, None]
        x[w][6, :, :32] = np.float32(0.3)
        x[w][6, :, [7, 20]] = np.array([-2.5, 2.5], np.float32)[:, None]
        x[w][7] = np.abs(x[w][7])
        x[w][8] = -np.float32(0.0)
    pool0 = rng.integers(0, 256, (2, blocks, kv, 36 * D)).astype(np.uint8)
    pools = [dev(pool0[w]) for w in range(2)]
    dc, xd = dev(cells), [dev(a) for a in x]
    hip.check(L.lgmlh_kv_store_q4(pools[0].data_ptr(), pools[1].data_ptr(), 64 * blocks, kv, D,
                                  xd[0].data_ptr(), xd[1].data_ptr(), dc.data_ptr(), cells.ctypes.data, n, st()))
    for w, make in enumerate((k_tile, v_tile)):
        q, d = quants(x[w])
        want = pool0[w].copy()
        for b in np.unique(cells // 64):
            for h in range(kv):
                tq, td = np.zeros((64, D), np.uint8), np.zeros((64, D // 32), np.float16)
                on_q, on_d = np.zeros((64, D), np.uint8), np.zeros((64, D // 32), np.float16)
                j = np.flatnonzero(cells // 64 == b)
                c = cells[j] % 64
                tq[c], td[c], on_q[c], on_d[c] = q[j, h], d[j, h], 15, np.uint16(0xffff).view(np.float16)
                on = make(on_q, on_d, D)
                want[b, h] = (make(tq, td, D) & on) | (want[b, h] & ~on)
        got = pools[w].cpu().numpy().reshape(want.shape)
        assert np.array_equal(got, want), (w, np.argwhere(got != want)[:4])


@pytest.mark.parametrize("D,kv,n", [(64, 2, 1), (64, 1, 33), (128, 8, 300), (256, 4, 77), (128, 8, 2100)])
@pytest.mark.parametrize("f16", [False, True])
def test_gather_reads_what_was_stored(L, D, kv, n, f16):
    """Rows in any order, repeated and outside the pool (zeros)."""
    from lgml_amd import hip
    rng = np.random.default_rng(n)
    blocks = 40

    class P:
        n_cells = 64 * blocks

    x = rng.standard_normal((64 * blocks, kv, D)).astype(np.float32)
    pools, kx, vx = fill(L, P, kv, D, x, -3 * x)
    for cells in (rng.integers(0, 64 * blocks, n), np.arange(5, 5 + n),
                  np.r_[np.arange(64, 64 + n), [7, 7, -1, 64 * blocks, -2**40, 2**40]]):
        cells = np.ascontiguousarray(cells, np.int64)
        dc = dev(cells)
        for w, want in enumerate((kx, vx)):
            out = torch.full((len(cells) + 1, kv, D), 5.0, dtype=torch.float16 if f16 else torch.float32,
                             device="cuda")
            hip.check(L.lgmlh_kv_gather_q4(pools[w].data_ptr(), w, 64 * blocks, kv, D, dc.data_ptr(), len(cells),
                                           out.data_ptr(), hip.F16 if f16 else hip.F32, st()))
            got = out.cpu().numpy()
            assert (got[-1] == 5.0).all()
            ok = (cells >= 0) & (cells < 64 * blocks)
            ref = np.where(ok[:, None, None], want[np.where(ok, cells, 0)], 0.0)
            ref = ref.astype(np.float32).astype(got.dtype)  # the f32 products are exact
            assert np.array_equal(got[:-1], ref)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("n", [1, 5, 40, 700, 1024])
def test_move_takes_the_cells_as_they_were(L, D, n):
    """Overlapping moves (a source that is another's target), every tensor; the
    other cells stay."""
    from lgml_amd import hip
    rng = np.random.default_rng(n + D)
    kv, blocks, layers = 3, 20, 2
    pools0 = rng.integers(0, 256, (2 * layers, blocks, kv, 36 * D)).astype(np.uint8)
    pools = dev(pools0)
    if n == 5:
        src, dst = np.array([131, 133, 134, 60, 70]), np.array([130, 131, 132, 60, 133])
    else:
        src, dst = rng.permutation(64 * blocks)[:n], rng.permutation(64 * blocks)[:n]
    src, dst = src.astype(np.int64), dst.astype(np.int64)
    addr = torch.tensor([p.data_ptr() for p in pools], dtype=torch.int64, device="cuda")
    ds, dt = dev(src), dev(dst)
    hip.check(L.lgmlh_kv_move(hip.Q4_0, addr.data_ptr(), 2 * layers, 64 * blocks, kv, D, ds.data_ptr(),
                              dt.data_ptr(), src.ctypes.data, dst.ctypes.data, n, st()))
    got = pools.cpu().numpy()
    at = [[cell_bytes(w, c, D) for c in range(64)] for w in range(2)]
    want = pools0.copy()
    for p in range(2 * layers):
        for a, b in zip(src, dst):
            want[p, b // 64][:, at[p % 2][b % 64]] = pools0[p, a // 64][:, at[p % 2][a % 64]]
    assert np.array_equal(got, want)


def cell_bytes(which, cell, D):
    """Where a cell's bytes are in its tile, found by the plain tiles."""
    q, d = np.zeros((64, D), np.uint8), np.zeros((64, D // 32), np.float16)
    q[cell], d[cell] = 15, np.uint16(0xffff).view(np.float16)
    t = (v_tile if which else k_tile)(q, d, D)
    assert set(np.unique(t)) <= {0, 255}  # whole bytes
    return np.flatnonzero(t)


# ---- attention -------------------------------------------------------------------
def check_attention(L, H, kv, D, seq_n, npast, parents, bps, seed, window=0, ring=0, q_gain=1.0):
    """Every row of a pass over random pools, against 64 bits; the outputs."""
    flat = None if parents is None else sum(parents, [])
    P = Pass(seq_n, npast, H, kv, flat, bps, seed, ring=ring, window=window)
    rng = np.random.default_rng(seed)
    k = rng.standard_normal((P.n_cells, kv, D)).astype(np.float32)
    v = rng.standard_normal((P.n_cells, kv, D)).astype(np.float32)
    k[:, :, ::17] *= 6
    q = (rng.standard_normal((sum(seq_n), H, D)) * q_gain).astype(np.float32)
    pools, kx, vx = fill(L, P, kv, D, k, v)
    scale = D ** -0.5
    got = run_attention(L, P, H, kv, D, scale, q, pools)
    t = 0
    for s, (n, p0) in enumerate(zip(seq_n, npast)):
        c = P.cells(s)
        for j in range(n):
            if parents is not None:
                vis = seen(parents[s], p0, j)
            else:
                vis = list(range(max(0, p0 + j - window + 1) if ring else 0, p0 + j + 1))
            qt = q[t].astype(np.float64)
            want = attend(qt, kx[c], vx[c], scale, vis)
            err = np.abs(got[t] - want).max()
            tol = bound(qt, kx[c][vis], vx[c][vis], scale, len(vis))
            assert err <= tol, (s, j, err, tol)
            t += 1
    return got


@pytest.mark.parametrize("H,kv,D", [(4, 2, 64), (8, 8, 64), (32, 8, 128), (16, 1, 128), (8, 4, 256), (32, 2, 64)])
@pytest.mark.parametrize("case", range(len(SEQS)))
@pytest.mark.parametrize("bps", [0, 2])
def test_tree_attention(L, H, kv, D, case, bps):
    seq_n, npast = SEQS[case]
    rng = np.random.default_rng(case)
    check_attention(L, H, kv, D, seq_n, npast, [tree(rng, n) for n in seq_n], bps, 3 + case)


@pytest.mark.parametrize("H,kv,D", [(4, 2, 64), (16, 2, 128), (8, 4, 256)])
@pytest.mark.parametrize("bps", [1, 0])
def test_tree_rows_that_see_nothing_of_whole_runs(L, H, kv, D, bps):
    seq_n, npast = [200, 1024, 3], [0, 37, 0]
    rng = np.random.default_rng(29)
    parents = [[-1 if j == 0 or rng.random() < 0.5 else int(rng.integers(max(0, j - 200), j)) for j in range(n)]
               for n in seq_n]
    check_attention(L, H, kv, D, seq_n, npast, parents, bps, 29)


@pytest.mark.parametrize("H,kv,D", [(4, 2, 64), (32, 4, 128), (8, 4, 256), (64, 4, 128)])
@pytest.mark.parametrize("seq_n,npast,bps", [([1] * 9, [0, 1, 63, 64, 65, 700, 1500, 12, 127], 0),
                                             ([1, 100, 1], [900, 0, 3], 3), ([130], [333], 2)])
def test_causal_attention(L, H, kv, D, seq_n, npast, bps):
    check_attention(L, H, kv, D, seq_n, npast, None, bps, 11)


@pytest.mark.parametrize("H,kv,D", [(8, 2, 64), (16, 2, 128), (8, 8, 128), (8, 4, 256)])
@pytest.mark.parametrize("is_tree", [False, True])
def test_many_splits(L, H, kv, D, is_tree):
    """Groups of 4 splits, 5, 16, 17 and more, of one row to sixteen, alone and together;
    in the tree, rows that see nothing of some."""
    seq_n, npast = [1, 1, 2, 16, 1, 7], [200, 300, 900, 1000, 1087, 4500]
    rng = np.random.default_rng(37)
    parents = [[-1] + [int(rng.integers(0, j)) for j in range(1, n)] for n in seq_n] if is_tree else None
    all_ = check_attention(L, H, kv, D, seq_n, npast, parents, 1, 41)
    assert np.isfinite(all_).all()


@pytest.mark.parametrize("H,kv,D", [(4, 2, 64), (16, 8, 128), (8, 4, 256)])
def test_ring_attention(L, H, kv, D):
    check_attention(L, H, kv, D, [1, 20, 1, 90], [1000, 37, 0, 100], None, 1, 13, window=100, ring=3)


def test_a_line_of_tokens_is_the_causal_plan(L):
    seq_n, npast = [9, 64, 1], [100, 3, 64]
    line = [[j - 1 for j in range(n)] for n in seq_n]
    for H, kv, D in ((8, 2, 64), (8, 2, 128), (8, 4, 256)):
        a = check_attention(L, H, kv, D, seq_n, npast, line, 2, 21)
        b = check_attention(L, H, kv, D, seq_n, npast, None, 2, 21)
        assert np.array_equal(a, b)


@pytest.mark.parametrize("gain", [1e-30, 1e-6, 1.0])
def test_small_queries(L, gain):
    rng = np.random.default_rng(1)
    check_attention(L, 8, 2, 128, [5], [200], [tree(rng, 5)], 0, 2, q_gain=gain)


@pytest.mark.parametrize("gain", list(GAINS))
@pytest.mark.parametrize("H,kv,D", [(8, 2, 64), (8, 2, 128), (8, 4, 256)])
def test_small_and_large_values(L, gain, H, kv, D):
    """V's scales inside and outside the range of the packed products, in one pass of
    decoding sequences, a chunk (shared runs) and long contexts; each 32 dims of a
    head held to their own size."""
    seq_n, npast = [1, 40, 1], [500, 70, 64]
    rng = np.random.default_rng(77)
    P = Pass(seq_n, npast, H, kv, None, 3, 77)
    k = rng.standard_normal((P.n_cells, kv, D)).astype(np.float32)
    v = rng.standard_normal((P.n_cells, kv, D)).astype(np.float32)
    v = (v * np.minimum(GAINS[gain](rng, v.shape), 8e4)).astype(np.float32)  # (d is an f16)
    q = rng.standard_normal((sum(seq_n), H, D)).astype(np.float32)
    pools, kx, vx = fill(L, P, kv, D, k, v)
    assert np.isfinite(vx).all()
    got = run_attention(L, P, H, kv, D, D ** -0.5, q, pools)
    t = 0
    for s, (n, p0) in enumerate(zip(seq_n, npast)):
        c = P.cells(s)
        for j in range(n):
            vis = list(range(p0 + j + 1))
            qt = q[t].astype(np.float64)
            want = attend(qt, kx[c], vx[c], D ** -0.5, vis)
            for b in range(D // 32):
                part = vx[c][vis][:, :, 32 * b:32 * b + 32]
                tol = bound(qt, kx[c][vis], part, D ** -0.5, len(vis))
                err = np.abs(got[t] - want)[:, 32 * b:32 * b + 32].max()
                assert err <= tol, (s, j, b, err, tol)
            t += 1


@pytest.mark.parametrize("gain", [None, "dims", "cells", "small"])
@pytest.mark.parametrize("H,kv,D", [(8, 2, 64), (16, 2, 128), (8, 4, 256)])
@pytest.mark.parametrize("bps", [2, 40])
def test_a_row_has_its_bits_in_any_group_of_rows(L, gain, H, kv, D, bps):
    """A chunk's tokens together, and each by itself with the later cells of its
    block as the chunk left them (quieter and louder ones among them)."""
    from lgml_amd import runtime
    n, past = 70, 45
    rng = np.random.default_rng(5)
    P = Pass([n], [past], H, kv, None, bps, 5)
    k = rng.standard_normal((P.n_cells, kv, D)).astype(np.float32)
    v = rng.standard_normal((P.n_cells, kv, D)).astype(np.float32)
    if gain:
        v = (v * GAINS[gain](rng, v.shape)).astype(np.float32)
    q = rng.standard_normal((n, H, D)).astype(np.float32)
    pools, _, _ = fill(L, P, kv, D, k, v)
    got = run_attention(L, P, H, kv, D, D ** -0.5, q, pools)
    for j in range(n):
        P.plan = runtime.Plan([1], [past + j], P.tab, np.zeros(1, np.int32), H, kv, P.blocks, bps)
        P.info, P.ub = P.plan.info, P.plan.ub
        one = run_attention(L, P, H, kv, D, D ** -0.5, q[j:j + 1], pools)
        assert np.array_equal(one[0], got[j]), j


def test_a_row_on_one_quiet_cell_keeps_its_bits(L):
    """V of the cell that a row attends to 1e-4 of the others': held to its own size."""
    H, kv, D, past = 4, 1, 128, 130
    rng = np.random.default_rng(9)
    P = Pass([1], [past], H, kv, None, 12, 9)
    c = P.cells(0)
    k = np.zeros((P.n_cells, kv, D), np.float32)
    k[:, :, 0] = -8.0
    quiet = c[77]
    k[quiet, :, 0] = 8.0
    v = rng.standard_normal((P.n_cells, kv, D)).astype(np.float32)
    v[quiet] *= np.float32(1e-4)
    q = np.zeros((1, H, D), np.float32)
    q[..., 0] = 20.0
    pools, kx, vx = fill(L, P, kv, D, k, v)
    got = run_attention(L, P, H, kv, D, D ** -0.5, q, pools)
    want = attend(q[0].astype(np.float64), kx[c], vx[c], D ** -0.5, list(range(past + 1)))
    # scores of -14 and 14 at most: the others weigh e^-28 in all
    assert np.abs(got[0] - want).max() <= np.abs(vx[quiet]).max() * 2.0**-18


@pytest.mark.parametrize("bits", [0x7e00, 0xffff, 0x7c00, 0xfc00, 0xbc00, 0x7bff, 0x0001])
@pytest.mark.parametrize("lone", [False, True])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("is_tree", [False, True])
def test_unseen_cells_of_any_scale(L, bits, lone, D, is_tree):
    """The cells past each sequence, or the last one alone, with scales of NaN,
    infinity, either sign, the largest and the smallest."""
    H, kv, seq_n, npast = 8, 2, [1, 40, 9], [70, 131, 3]
    rng = np.random.default_rng(19)
    parents = sum([tree(rng, n) for n in seq_n], []) if is_tree else None
    P = Pass(seq_n, npast, H, kv, parents, 2, 19)
    k, v = (rng.standard_normal((P.n_cells, kv, D)).astype(np.float32) for _ in range(2))
    q = rng.standard_normal((sum(seq_n), H, D)).astype(np.float32)
    pools, _, _ = fill(L, P, kv, D, k, v)
    want = run_attention(L, P, H, kv, D, D ** -0.5, q, pools)
    for s in range(len(seq_n)):
        last = int(P.cells(s)[-1])
        for w in range(2):
            scales = pools[w].view(-1, kv, 36 * D)[last // 64, :, 32 * D:].view(torch.int16).view(kv, D // 32, 64)
            scales[:, :, 63 if lone else slice(last % 64 + 1, 64)] = bits - (bits >> 15 << 16)
    assert np.isfinite(want).all()
    assert np.array_equal(run_attention(L, P, H, kv, D, D ** -0.5, q, pools), want)


@pytest.mark.parametrize("H,kv,D", [(4, 2, 64), (32, 8, 128), (8, 4, 256)])
def test_tree_nodes_a_row_does_not_see_change_nothing(L, H, kv, D):
    """Nodes 1 and 2 of each tree hold scales of infinity and NaN: rows that do not see
    them have the bits of clean pools."""
    seq_n, npast = [7, 12, 40], [60, 131, 257]
    parents = [[-1, 0, 0, 0, 3, 4, 3], [-1, 0, -1] + [0] + [3] * 8, [-1, 0, 0] + list(range(2, 39))]
    parents[2][3] = 0
    clean = check_attention(L, H, kv, D, seq_n, npast, parents, 2, 31)
    rng = np.random.default_rng(31)
    P = Pass(seq_n, npast, H, kv, sum(parents, []), 2, 31)
    k = rng.standard_normal((P.n_cells, kv, D)).astype(np.float32)
    v = rng.standard_normal((P.n_cells, kv, D)).astype(np.float32)
    k[:, :, ::17] *= 6
    q = rng.standard_normal((sum(seq_n), H, D)).astype(np.float32)
    pools, _, _ = fill(L, P, kv, D, k, v)
    for w in range(2):
        t = pools[w].view(-1, kv, 36 * D)
        for s, p0 in enumerate(npast):
            for i, c in enumerate(P.cells(s)[[p0 + 1, p0 + 2]]):
                x = t[int(c) // 64, :, 32 * D:].view(torch.float16).view(kv, D // 32, 64)
                x[:, :, int(c) % 64] = float("nan") if i else float("inf")
    got = run_attention(L, P, H, kv, D, D ** -0.5, q, pools)
    t = checked = 0
    for s, n in enumerate(seq_n):
        for j in range(n):
            if not set(x - npast[s] for x in seen(parents[s], npast[s], j)) & {1, 2}:
                assert np.array_equal(got[t], clean[t]), (s, j)
                checked += 1
            t += 1
    assert checked > 20


def test_another_dispatch_order_and_a_long_context(L):
    """order may be NULL or the caller's own; a context of many runs."""
    H, kv, D = 16, 2, 128
    P = Pass([1, 1, 3], [20000, 64, 9000], H, kv, None, 12, 4)
    rng = np.random.default_rng(4)
    k, v = (rng.standard_normal((P.n_cells, kv, D)).astype(np.float32) for _ in range(2))
    q = rng.standard_normal((5, H, D)).astype(np.float32)
    pools, kx, vx = fill(L, P, kv, D, k, v)
    want = run_attention(L, P, H, kv, D, D ** -0.5, q, pools)
    c = P.cells(0)
    ref = attend(q[0].astype(np.float64), kx[c], vx[c], D ** -0.5, list(range(20001)))
    assert np.abs(want[0] - ref).max() <= bound(q[0].astype(np.float64), kx[c], vx[c], D ** -0.5, 20001)
    own = dev(np.arange(P.info.n_single, dtype=np.int32)[::-1])
    for order in (own.data_ptr(), None):
        P.ub.order = order
        assert np.array_equal(run_attention(L, P, H, kv, D, D ** -0.5, q, pools), want)


def test_cells_behind_4_gib(L):
    """The last blocks of a pool whose tensors pass 4 GiB: stored, moved, copied, read
    back and attended to as in a small pool (the same bits)."""
    from lgml_amd import hip, runtime
    H, kv, D, n, past = 16, 8, 256, 40, 70
    per = 36 * D * kv
    big = (1 << 32) // per + 12
    rng = np.random.default_rng(8)
    k, v = (rng.standard_normal((past + n, kv, D)).astype(np.float32) for _ in range(2))
    q = rng.standard_normal((n, H, D)).astype(np.float32)
    parents = np.array(tree(rng, n), np.int32)
    src, dst = np.array([past + 3, past + 9, past + 20]), np.array([past, past + 1, past + 2])
    results = []
    for blocks in (8, big):
        tab = blocks - 1 - np.array([[3, 0]], np.int32)

        def cell(p):
            return tab[0][p // 64].astype(np.int64) * 64 + p % 64

        pools = [torch.full((blocks * per,), 0xFF, dtype=torch.uint8, device="cuda") for _ in range(2)]
        cells = cell(np.arange(past + n))
        dc, kd, vd = dev(cells), dev(k), dev(v)
        hip.check(L.lgmlh_kv_store_q4(pools[0].data_ptr(), pools[1].data_ptr(), 64 * blocks, kv, D, kd.data_ptr(),
                                      vd.data_ptr(), dc.data_ptr(), cells.ctypes.data, len(cells), st()))

        class P:
            plan = runtime.Plan([n], [past], tab, np.zeros(n, np.int32), H, kv, blocks, 2, parents=parents)

        P.info, P.ub = P.plan.info, P.plan.ub
        got = [run_attention(L, P, H, kv, D, D ** -0.5, q, pools)]
        one = runtime.Plan([1], [past], tab, np.zeros(1, np.int32), H, kv, blocks, 2)
        P.info, P.ub = one.info, one.ub
        got.append(run_attention(L, P, H, kv, D, D ** -0.5, q[:1], pools))
        addr = torch.tensor([p.data_ptr() for p in pools], dtype=torch.int64, device="cuda")
        a, b = cell(src), cell(dst)
        da, db = dev(a), dev(b)
        hip.check(L.lgmlh_kv_move(hip.Q4_0, addr.data_ptr(), 2, 64 * blocks, kv, D, da.data_ptr(), db.data_ptr(),
                                  a.ctypes.data, b.ctypes.data, 3, st()))
        copies = np.array([[blocks - 4, blocks - 2, 64], [blocks - 1, blocks - 3, 37], [blocks - 4, 1, 64]], np.int32)
        dcp = dev(copies)
        hip.check(L.lgmlh_kv_copy_blocks(hip.Q4_0, addr.data_ptr(), 2, 64 * blocks, kv, D, dcp.data_ptr(),
                                         copies.ctypes.data, 3, st()))
        read = np.concatenate([cells, (blocks - 2) * 64 + np.arange(64), (blocks - 3) * 64 + np.arange(37),
                               64 + np.arange(64)])
        dr = dev(read)
        for w in range(2):
            out = torch.empty((len(read), kv, D), dtype=torch.float16, device="cuda")
            hip.check(L.lgmlh_kv_gather_q4(pools[w].data_ptr(), w, 64 * blocks, kv, D, dr.data_ptr(), len(read),
                                           out.data_ptr(), hip.F16, st()))
            got.append(out.cpu().numpy())
        results.append(got)
        want = values(k).astype(np.float16)
        want[dst] = want[src]
        want = np.concatenate([want, want[:64], want[64:101], want[:64]])
        assert np.array_equal(got[2], want)
    for a, b in zip(*results):
        assert np.array_equal(a, b)
