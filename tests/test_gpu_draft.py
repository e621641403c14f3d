"""The operators of serving drafted tokens over a quantised cache, on the GPU,
against plain 64-bit implementations: the Q8_0 pool (store, gather), moves of
cells, attention of tree plans and over Q8_0 pools, log probabilities; and a
run of them together, captured and replayed too."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def L():
    from lgml_amd import hip
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    return hip.lib()


def st():
    return torch.cuda.current_stream().cuda_stream


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to("cuda")


# ---- the plain forms -------------------------------------------------------------
def quants(x):
    """Q8_0 of (n, kv, D) f32 in its defined steps: (q int8, d f16 as f64)."""
    n, kv, d = x.shape
    g = x.reshape(n, kv, d // 32, 32)
    dd = np.abs(g).max(-1) / np.float32(127)
    with np.errstate(divide="ignore"):
        inv = np.where(dd > 0, np.float32(1) / dd, np.float32(0)).astype(np.float32)
    y = (g * inv[..., None]).astype(np.float32).astype(np.float64)
    q = np.sign(y) * np.floor(np.abs(y) + 0.5)
    return q.reshape(n, kv, d).astype(np.int8), dd.astype(np.float16)


def values(x):
    q, d = quants(x)
    return q.astype(np.float64) * np.repeat(d.astype(np.float64), 32, -1)


def k_tile(q, d, D):
    """A tile of K (68 D bytes) from 64 cells' q (64, D) int8 and d (64, D / 32) f16."""
    v = q.reshape(64, D // 64, 2, 4, 8).transpose(1, 0, 3, 2, 4)
    return np.concatenate([v.reshape(-1).view(np.uint8), d.T.copy().reshape(-1).view(np.uint8)])


def v_tile(q, d, D):
    v = q.reshape(2, 4, 8, D).transpose(3, 1, 0, 2)
    return np.concatenate([v.reshape(-1).view(np.uint8), d.T.copy().reshape(-1).view(np.uint8)])


def tree(rng, n):
    return [-1] + [int(rng.integers(max(-1, j - 9), j)) for j in range(1, n)]


def seen(parents, past, j):
    line, a = [], j
    while a >= 0:
        line.append(past + a)
        a = parents[a]
    return list(range(past)) + sorted(line)


def attend(q, k, v, scale, vis):
    """q (H, D), k and v (cells, kv, D) f64; the cells vis."""
    H, D = q.shape
    kv = k.shape[1]
    ks, vs = k[vis].transpose(1, 2, 0), v[vis].transpose(1, 0, 2)
    x = np.matmul(q.reshape(kv, H // kv, D), ks) * scale
    e = np.exp(x - x.max(-1, keepdims=True))
    return (np.matmul(e, vs) / e.sum(-1, keepdims=True)).reshape(H, D)


def bound(q, k, v, scale, n):
    """How far an f32 computation of a row may be off. A score is a sum of D
    products of q (22 bits or more) in f32, at most D + 40 roundings of 2^-24 and
    2^-22 of sum |q k| scale, and 2^-22 of itself for its factor; p is off by
    that and 2^-21; a sum over n cells takes at most n / 16 + 64 roundings."""
    H, D = q.shape
    kv = k.shape[1]
    s = np.matmul(np.abs(q).reshape(kv, H // kv, D), np.abs(k).transpose(1, 2, 0)).max() * scale
    ds = s * ((D + 40) * 2.0**-24 + 2.0**-21)
    return np.abs(v).max() * 2 * (ds + 2.0**-20 + (n / 16 + 64) * 2.0**-24)


class Pass:
    """A pass's plan over a shuffled pool, and its cells."""

    def __init__(self, seq_n, npast, H, kv, parents=None, bps=0, seed=0, extra=2, ring=0, window=0):
        from lgml_amd import hip, runtime
        rng = np.random.default_rng(seed)
        if ring:
            nb = [ring] * len(seq_n)
        else:
            nb = [max(1, (p + n + 63) // 64) for p, n in zip(npast, seq_n)]
        self.blocks = sum(nb) + extra
        order, at = rng.permutation(self.blocks).astype(np.int32), 0
        self.tab = np.full((len(seq_n), max(nb)), -1, np.int32)
        for s, k in enumerate(nb):
            self.tab[s, :k] = order[at:at + k]
            at += k
        self.seq_n, self.npast, self.ring = seq_n, npast, ring
        self.n_cells = 64 * self.blocks
        self.plan = runtime.Plan(seq_n, npast, self.tab, np.zeros(sum(seq_n), np.int32), H, kv, self.blocks,
                                 bps, parents=parents, ring_tab=self.tab if ring else None, window=window)
        self.info, self.ub = self.plan.info, self.plan.ub
        self.hip = hip

    def cells(self, s):
        """The pool cells of a sequence's slots."""
        p = np.arange(self.npast[s] + self.seq_n[s])
        b = p // 64 % self.ring if self.ring else p // 64
        return self.tab[s][b].astype(np.int64) * 64 + p % 64


def fill(L, P, kv, D, k, v, q8):
    """Rows k, v (n_cells, kv, D) f32 into pools of one type: (pools, the f64
    values they hold)."""
    from lgml_amd import hip
    cells = np.arange(P.n_cells, dtype=np.int64)
    dc, kd, vd = dev(cells), dev(k), dev(v)
    nb = (L.lgmlh_kv_q8_layer_bytes if q8 else L.lgmlh_kv_layer_bytes)(P.n_cells, kv, D)
    pools = [torch.zeros(nb, dtype=torch.uint8, device="cuda") for _ in range(2)]
    fn = L.lgmlh_kv_store_q8 if q8 else L.lgmlh_kv_store
    hip.check(fn(pools[0].data_ptr(), pools[1].data_ptr(), P.n_cells, kv, D, kd.data_ptr(), vd.data_ptr(),
                 dc.data_ptr(), cells.ctypes.data, len(cells), st()))
    torch.cuda.synchronize()
    if q8:
        return pools, values(k), values(v)
    return pools, k.astype(np.float16).astype(np.float64), v.astype(np.float16).astype(np.float64)


def run_attention(L, P, H, kv, D, scale, q, pools, q8):
    from lgml_amd import hip
    qd = dev(q)
    out = torch.full((len(q) + 1, H, D), 7.0, dtype=torch.float32, device="cuda")
    nb = L.lgmlh_attention_workspace(C.byref(P.info), D)
    ws = torch.full((nb + 256,), 0xA5, dtype=torch.uint8, device="cuda")
    fn = L.lgmlh_paged_attention_q8 if q8 else L.lgmlh_paged_attention
    hip.check(fn(qd.data_ptr(), H, kv, D, scale, pools[0].data_ptr(), pools[1].data_ptr(), C.byref(P.ub),
                 out.data_ptr(), ws.data_ptr(), nb, st()))
    torch.cuda.synchronize()
    assert bool((out[-1] == 7.0).all()) and bool((ws[nb:] == 0xA5).all())
    return out[:-1].cpu().numpy().astype(np.float64)


# ---- the Q8_0 pool ---------------------------------------------------------------
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("kv", [1, 3, 8])
def test_store_q8_writes_the_defined_bytes(L, D, kv):
    """Every byte of the pool: runs of cells from odd offsets, lone cells, values
    at halves of a step, zero blocks, tiny and huge ones; cells not written stay."""
    from lgml_amd import hip
    rng = np.random.default_rng(D + kv)
    blocks = 7
    runs = [(64 + 3, 70), (200, 1), (5 * 64, 64), (6 * 64 + 1, 7), (6 * 64 + 9, 1), (6 * 64 + 20, 33), (2, 1)]
    cells = np.concatenate([np.arange(a, a + n) for a, n in runs]).astype(np.int64)
    n = len(cells)
    x = [rng.standard_normal((n, kv, D)).astype(np.float32) for _ in range(2)]
    x[0][0] = 0.0
    x[0][1, :, :32] = (np.arange(32) - 15.5) * np.float32(127 / 15.5 / 127)
    x[1][2] *= np.float32(1e-30)
    x[1][3] *= np.float32(1e5)
    x[0][4, :, 32:64] = np.float32(2.0**-20) * rng.integers(-3, 4, (kv, 32))
    pool0 = rng.integers(0, 256, (2, blocks, kv, 68 * D)).astype(np.uint8)
    pools = [dev(pool0[w]) for w in range(2)]
    dc, xd = dev(cells), [dev(a) for a in x]
    hip.check(L.lgmlh_kv_store_q8(pools[0].data_ptr(), pools[1].data_ptr(), 64 * blocks, kv, D,
                                  xd[0].data_ptr(), xd[1].data_ptr(), dc.data_ptr(), cells.ctypes.data, n, st()))
    for w, make in enumerate((k_tile, v_tile)):
        q, d = quants(x[w])
        want = pool0[w].copy()
        for b in range(blocks):
            for h in range(kv):
                tq, td = np.zeros((64, D), np.int8), np.zeros((64, D // 32), np.float16)
                on_q, on_d = np.zeros((64, D), np.int8), np.zeros((64, D // 32), np.float16)
                for j in np.flatnonzero(cells // 64 == b):
                    tq[cells[j] % 64], td[cells[j] % 64] = q[j, h], d[j, h]
                    on_q[cells[j] % 64], on_d[cells[j] % 64] = -1, np.uint16(0xffff).view(np.float16)
                on = make(on_q, on_d, D)
                want[b, h] = (make(tq, td, D) & on) | (want[b, h] & ~on)
        got = pools[w].cpu().numpy().reshape(want.shape)
        assert np.array_equal(got, want), (w, np.argwhere(got != want)[:4])


@pytest.mark.parametrize("D,kv,n", [(64, 2, 1), (64, 1, 33), (128, 8, 300), (256, 4, 77)])
@pytest.mark.parametrize("f16", [False, True])
def test_gather_q8_reads_what_was_stored(L, D, kv, n, f16):
    """Rows in any order, repeated and outside the pool (zeros)."""
    from lgml_amd import hip
    rng = np.random.default_rng(n)
    blocks = 8
    x = rng.standard_normal((64 * blocks, kv, D)).astype(np.float32)

    class P:
        n_cells = 64 * blocks

    pools, kx, vx = fill(L, P, kv, D, x, -3 * x, True)
    for cells in (rng.integers(0, 64 * blocks, n), np.arange(5, 5 + n), np.r_[np.arange(64, 64 + n), [7, 7, -1, 64 * blocks]]):
        cells = np.ascontiguousarray(cells, np.int64)
        dc = dev(cells)
        for w, want in enumerate((kx, vx)):
            out = torch.full((len(cells) + 1, kv, D), 5.0, dtype=torch.float16 if f16 else torch.float32, device="cuda")
            hip.check(L.lgmlh_kv_gather_q8(pools[w].data_ptr(), w, 64 * blocks, kv, D, dc.data_ptr(), len(cells),
                                           out.data_ptr(), hip.F16 if f16 else hip.F32, st()))
            got = out.cpu().numpy()
            assert (got[-1] == 5.0).all()
            ok = (cells >= 0) & (cells < 64 * blocks)
            ref = np.where(ok[:, None, None], want[np.where(ok, cells, 0)], 0.0)
            ref = ref.astype(np.float32).astype(got.dtype)  # the f32 products are exact
            assert np.array_equal(got[:-1], ref)


@pytest.mark.parametrize("q8,D", [(False, 16), (False, 64), (False, 128), (True, 64), (True, 128), (True, 256)])
@pytest.mark.parametrize("n", [1, 5, 40, 1024])
def test_move_takes_the_cells_as_they_were(L, q8, D, n):
    """Overlapping moves (a source that is another's target), every tensor; the
    other cells stay."""
    from lgml_amd import hip
    rng = np.random.default_rng(n + D)
    kv, blocks, layers = 3, 20, 2
    per = 68 * D if q8 else 128 * D
    pools0 = rng.integers(0, 256, (2 * layers, blocks, kv, per)).astype(np.uint8)
    pools = dev(pools0)
    if n == 5:
        src, dst = np.array([131, 133, 134, 60, 70]), np.array([130, 131, 132, 60, 133])
    else:
        src, dst = rng.permutation(64 * blocks)[:n], rng.permutation(64 * blocks)[:n]
    src, dst = src.astype(np.int64), dst.astype(np.int64)
    addr = torch.tensor([p.data_ptr() for p in pools], dtype=torch.int64, device="cuda")
    ds, dt = dev(src), dev(dst)
    hip.check(L.lgmlh_kv_move(hip.Q8_0 if q8 else hip.F16, addr.data_ptr(), 2 * layers, 64 * blocks, kv, D,
                              ds.data_ptr(), dt.data_ptr(), src.ctypes.data, dst.ctypes.data, n, st()))
    got = pools.cpu().numpy()

    def index(which, cell):
        """(bytes of the cell in its tile,)"""
        d = np.arange(D)
        if not q8:
            e = d * 64 + cell if which else cell * D + d
            return np.concatenate([2 * e, 2 * e + 1])
        if which:
            e = d * 64 + cell % 32 // 8 * 16 + cell // 32 * 8 + cell % 8
        else:
            e = ((d // 64 * 64 + cell) * 4 + d % 32 // 8) * 16 + d % 64 // 32 * 8 + d % 8
        s = 64 * D + 2 * (np.arange(D // 32) * 64 + cell)
        return np.concatenate([e, s, s + 1])

    want = pools0.copy()
    for p in range(2 * layers):
        for a, b in zip(src, dst):
            want[p, b // 64][:, index(p % 2, b % 64)] = pools0[p, a // 64][:, index(p % 2, a % 64)]
    assert np.array_equal(got, want)


# ---- attention -------------------------------------------------------------------
def check_attention(L, q8, H, kv, D, seq_n, npast, parents, bps, seed, q_gain=1.0, v_gain=None, window=0, ring=0):
    rng = np.random.default_rng(seed)
    flat = None if parents is None else sum(parents, [])
    P = Pass(seq_n, npast, H, kv, flat, bps, seed, ring=ring, window=window)
    k = rng.standard_normal((P.n_cells, kv, D)).astype(np.float32)
    v = rng.standard_normal((P.n_cells, kv, D)).astype(np.float32)
    k[:, :, ::17] *= 6
    if v_gain is not None:
        v *= v_gain(rng, v.shape).astype(np.float32)
    q = (rng.standard_normal((sum(seq_n), H, D)) * q_gain).astype(np.float32)
    pools, kx, vx = fill(L, P, kv, D, k, v, q8)
    scale = D ** -0.5
    got = run_attention(L, P, H, kv, D, scale, q, pools, q8)
    t, worst = 0, 0.0
    for s, (n, p0) in enumerate(zip(seq_n, npast)):
        c = P.cells(s)
        for j in range(n):
            if parents is not None:
                vis = seen(parents[s], p0, j)
            else:
                vis = list(range(max(0, p0 + j - window + 1) if window else 0, p0 + j + 1))
            qt = q[t].astype(np.float64)
            want = attend(qt, kx[c], vx[c], scale, vis)
            tol = bound(qt, kx[c][vis], vx[c][vis], scale, len(vis))
            err = np.abs(got[t] - want).max()
            assert err <= tol, (s, j, err, tol)
            worst = max(worst, err / tol)
            t += 1
    return got


SEQS = [([1], [0]), ([7], [0]), ([9, 1, 64], [63, 64, 130]), ([33, 16, 2, 70], [5, 1000, 127, 300])]


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("H,kv,D", [(4, 2, 64), (8, 8, 64), (32, 8, 128), (16, 1, 128), (8, 4, 256)])
@pytest.mark.parametrize("case", range(len(SEQS)))
@pytest.mark.parametrize("bps", [0, 2])
def test_tree_attention(L, q8, H, kv, D, case, bps):
    seq_n, npast = SEQS[case]
    rng = np.random.default_rng(case)
    check_attention(L, q8, H, kv, D, seq_n, npast, [tree(rng, n) for n in seq_n], bps, 3 + case)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("H,kv,D", [(4, 2, 64), (16, 2, 128), (8, 4, 256)])
@pytest.mark.parametrize("bps", [1, 0])
def test_tree_rows_that_see_nothing_of_whole_runs(L, q8, H, kv, D, bps):
    """Wide trees without a context, up to the largest: most of a sequence's blocks
    hold nothing that a token sees."""
    seq_n, npast = [200, 1024, 3], [0, 37, 0]
    rng = np.random.default_rng(29)
    parents = [[-1 if j == 0 or rng.random() < 0.5 else int(rng.integers(max(0, j - 200), j)) for j in range(n)]
               for n in seq_n]
    check_attention(L, q8, H, kv, D, seq_n, npast, parents, bps, 29)


@pytest.mark.parametrize("D", [16, 32])
def test_tree_attention_small_heads(L, D):
    rng = np.random.default_rng(D)
    seq_n, npast = SEQS[3]
    check_attention(L, False, 4, 2, D, seq_n, npast, [tree(rng, n) for n in seq_n], 2, 5)


@pytest.mark.parametrize("H,kv,D", [(4, 2, 64), (32, 4, 128), (8, 4, 256)])
@pytest.mark.parametrize("seq_n,npast,bps", [([1] * 9, [0, 1, 63, 64, 65, 700, 1500, 12, 127], 0),
                                             ([1, 100, 1], [900, 0, 3], 3), ([130], [333], 2)])
def test_q8_attention_of_causal_plans(L, H, kv, D, seq_n, npast, bps):
    check_attention(L, True, H, kv, D, seq_n, npast, None, bps, 11)


@pytest.mark.parametrize("H,kv,D", [(4, 2, 64), (16, 8, 128), (8, 4, 256)])
def test_q8_attention_of_ring_plans(L, H, kv, D):
    check_attention(L, True, H, kv, D, [1, 20, 1, 90], [1000, 37, 0, 100], None, 1, 13, window=100, ring=3)


@pytest.mark.parametrize("q8", [False, True])
def test_a_line_of_tokens_is_the_causal_plan(L, q8):
    """A tree without branches gives the bits of the causal plan."""
    seq_n, npast = [9, 64, 1], [100, 3, 64]
    line = [[j - 1 for j in range(n)] for n in seq_n]
    a = check_attention(L, q8, 8, 2, 64, seq_n, npast, line, 2, 21)
    b = check_attention(L, q8, 8, 2, 64, seq_n, npast, None, 2, 21)
    assert np.array_equal(a, b)


@pytest.mark.parametrize("q8", [False, True])
def test_a_tree_plan_in_another_dispatch_order(L, q8):
    """order, which picks only who runs an item, may be NULL or the caller's own."""
    H, kv, D, seq_n, npast = 16, 2, 64, [1, 2, 40, 1], [700, 64, 100, 5]
    rng = np.random.default_rng(21)
    P = Pass(seq_n, npast, H, kv, sum([tree(rng, n) for n in seq_n], []), 2, 21)
    k, v = (rng.standard_normal((P.n_cells, kv, D)).astype(np.float32) for _ in range(2))
    q = rng.standard_normal((sum(seq_n), H, D)).astype(np.float32)
    pools, _, _ = fill(L, P, kv, D, k, v, q8)
    want = run_attention(L, P, H, kv, D, D ** -0.5, q, pools, q8)
    own = dev(np.arange(P.info.n_single, dtype=np.int32)[::-1])
    for order in (own.data_ptr(), None):
        P.ub.order = order
        assert np.array_equal(run_attention(L, P, H, kv, D, D ** -0.5, q, pools, q8), want)


@pytest.mark.parametrize("gain", [1e-30, 1e-6, 3e3, 1e7])
def test_q8_attention_of_small_and_large_queries(L, gain):
    """q keeps its bits at any size (f16 parts of scaled rows); large scores leave
    a row to its largest."""
    rng = np.random.default_rng(1)
    H, kv, D = 8, 2, 128
    seq_n, npast = [5], [200]
    parents = [tree(rng, 5)]
    if gain <= 1:
        check_attention(L, True, H, kv, D, seq_n, npast, parents, 0, 2, q_gain=gain)
        return
    P = Pass(seq_n, npast, H, kv, parents[0], 0, 2)
    k = rng.standard_normal((P.n_cells, kv, D)).astype(np.float32)
    v = rng.standard_normal((P.n_cells, kv, D)).astype(np.float32)
    q = (rng.standard_normal((5, H, D)) * gain).astype(np.float32)
    pools, kx, vx = fill(L, P, kv, D, k, v, True)
    got = run_attention(L, P, H, kv, D, D ** -0.5, q, pools, True)
    c = P.cells(0)
    for j in range(5):
        vis = seen(parents[0], 200, j)
        x = np.einsum("hd,chd->hc", q[j].astype(np.float64), kx[c][vis].repeat(H // kv, 1)) * D ** -0.5
        for h in range(H):
            order = np.argsort(x[h])
            # the largest score is ahead of the next by more than both may be off
            if x[h][order[-1]] - x[h][order[-2]] > 40 + np.abs(x[h]).max() * 2.0**-15:
                want = vx[c[vis[order[-1]]], h // (H // kv)]
                assert np.abs(got[j, h] - want).max() <= np.abs(want).max() * 2.0**-20


GAINS = {
    "tiny": lambda rng, s: np.full(s, 2e-5), "small": lambda rng, s: np.full(s, 2e-3),
    "large": lambda rng, s: np.full(s, 1e3), "huge": lambda rng, s: np.full(s, 3e5),
    "zero": lambda rng, s: np.zeros(s),
    # some 32 dims of a head quiet, loud or 0 beside the others; some cells loud
    "dims": lambda rng, s: np.repeat(rng.choice([0, 1e-4, 1, 1, 300], s[:2] + (s[2] // 32,)), 32, -1),
    "cells": lambda rng, s: np.where(rng.random(s[:1] + (1, 1)) < 0.01, 1e4, 1.0) * np.ones(s),
}


@pytest.mark.parametrize("gain", list(GAINS))
@pytest.mark.parametrize("H,kv,D", [(8, 2, 64), (8, 2, 128), (8, 4, 256)])
def test_q8_attention_of_small_and_large_values(L, gain, H, kv, D):
    """V's scales inside and outside the range of the packed products, in one
    pass of decoding sequences, a chunk (shared runs) and long contexts. Quiet
    dims are held to their own size: each 32 dims of a head by itself."""
    seq_n, npast = [1, 40, 1], [500, 70, 64]
    rng = np.random.default_rng(77)
    P = Pass(seq_n, npast, H, kv, None, 3, 77)
    k = rng.standard_normal((P.n_cells, kv, D)).astype(np.float32)
    v = rng.standard_normal((P.n_cells, kv, D)).astype(np.float32)
    v = (v * GAINS[gain](rng, v.shape)).astype(np.float32)
    q = rng.standard_normal((sum(seq_n), H, D)).astype(np.float32)
    pools, kx, vx = fill(L, P, kv, D, k, v, True)
    got = run_attention(L, P, H, kv, D, D ** -0.5, q, pools, True)
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
def test_a_row_over_q8_has_its_bits_in_any_group_of_rows(L, gain, H, kv, D, bps):
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
    pools, _, _ = fill(L, P, kv, D, k, v, True)
    got = run_attention(L, P, H, kv, D, D ** -0.5, q, pools, True)
    for j in range(n):
        P.plan = runtime.Plan([1], [past + j], P.tab, np.zeros(1, np.int32), H, kv, P.blocks, bps)
        P.info, P.ub = P.plan.info, P.plan.ub
        one = run_attention(L, P, H, kv, D, D ** -0.5, q[j:j + 1], pools, True)
        assert np.array_equal(one[0], got[j]), j


def spoil_cells(q8, kv, D, which_cells):
    """Infinite and NaN contents for some cells: f16 values, or Q8_0 scales."""
    def spoil(P, pools):
        for w in range(2):
            if q8:
                t = pools[w].view(-1, kv, 68 * D)
                for c in which_cells(P):
                    s = t[c // 64, :, 64 * D:].view(torch.float16).view(kv, D // 32, 64)
                    s[:, :, c % 64] = float("nan") if c % 2 else float("inf")
            else:
                t = pools[w].view(torch.float16).view(-1, kv, 64 * D)
                for c in which_cells(P):
                    x = t[c // 64].view(kv, 64, D)[:, c % 64] if w == 0 else t[c // 64].view(kv, D, 64)[:, :, c % 64]
                    x[:] = float("nan") if c % 2 else (float("inf") if w else 60000.0)
    return spoil


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("H,kv,D", [(4, 2, 64), (32, 8, 128), (8, 4, 256)])
def test_cells_a_row_does_not_see_change_nothing(L, q8, H, kv, D):
    """Node 1 of each tree holds infinities and NaN, and node 2 and the cells past
    the sequence: rows that do not see them have the bits of clean pools (which
    are checked), rows that see node 1 may be anything."""
    seq_n, npast = [7, 12, 40], [60, 131, 257]
    parents = [[-1, 0, 0, 0, 3, 4, 3], [-1, 0, -1] + [0] + [3] * 8, [-1, 0, 0] + list(range(2, 39))]
    parents[2][3] = 0

    def bad(P):
        out = []
        for s, (n, p0) in enumerate(zip(seq_n, npast)):
            c = P.cells(s)
            out += [int(c[p0 + 1]), int(c[p0 + 2])]
            last = int(c[-1])
            out += range(last + 1, last // 64 * 64 + 64)
        return out

    flat = sum(parents, [])
    clean = check_attention(L, q8, H, kv, D, seq_n, npast, parents, 2, 31)
    rng = np.random.default_rng(31)
    P = Pass(seq_n, npast, H, kv, flat, 2, 31)
    k = rng.standard_normal((P.n_cells, kv, D)).astype(np.float32)
    v = rng.standard_normal((P.n_cells, kv, D)).astype(np.float32)
    k[:, :, ::17] *= 6
    q = rng.standard_normal((sum(seq_n), H, D)).astype(np.float32)
    pools, _, _ = fill(L, P, kv, D, k, v, q8)
    spoil_cells(q8, kv, D, bad)(P, pools)
    got = run_attention(L, P, H, kv, D, D ** -0.5, q, pools, q8)
    t = checked = 0
    for s, n in enumerate(seq_n):
        for j in range(n):
            line = set(x - npast[s] for x in seen(parents[s], npast[s], j))
            if not line & {1, 2}:
                assert np.array_equal(got[t], clean[t]), (s, j)
                checked += 1
            t += 1
    assert checked > 20


@pytest.mark.parametrize("bits", [0x7e00, 0xffff, 0x7c00, 0xfc00, 0xbc00, 0x7bff, 0x0001])
@pytest.mark.parametrize("lone", [False, True])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("is_tree", [False, True])
def test_unseen_q8_cells_of_any_scale(L, bits, lone, D, is_tree):
    """The cells past each sequence, or the last one alone, with scales of NaN,
    infinity, either sign, the largest and the smallest."""
    H, kv, seq_n, npast = 8, 2, [1, 40, 9], [70, 131, 3]
    rng = np.random.default_rng(19)
    parents = sum([tree(rng, n) for n in seq_n], []) if is_tree else None
    P = Pass(seq_n, npast, H, kv, parents, 2, 19)
    k, v = (rng.standard_normal((P.n_cells, kv, D)).astype(np.float32) for _ in range(2))
    q = rng.standard_normal((sum(seq_n), H, D)).astype(np.float32)
    pools, _, _ = fill(L, P, kv, D, k, v, True)
    want = run_attention(L, P, H, kv, D, D ** -0.5, q, pools, True)
    for s in range(len(seq_n)):
        last = int(P.cells(s)[-1])
        for w in range(2):
            scales = pools[w].view(-1, kv, 68 * D)[last // 64, :, 64 * D:].view(torch.int16).view(kv, D // 32, 64)
            scales[:, :, 63 if lone else slice(last % 64 + 1, 64)] = bits - (bits >> 15 << 16)
    assert np.isfinite(want).all()
    assert np.array_equal(run_attention(L, P, H, kv, D, D ** -0.5, q, pools, True), want)


# ---- log probabilities -----------------------------------------------------------
def log_probs(L, x, ids=None, top=0, entropy=True, lead=0):
    from lgml_amd import hip
    r, v = x.shape
    buf = torch.empty(lead + r * v, dtype=torch.float32, device="cuda")  # rows at any offset
    buf[lead:] = dev(x).reshape(-1)
    n_ids = 0 if ids is None else ids.shape[1]
    di = None if ids is None else dev(ids.astype(np.int32))
    lp = torch.full((r + 1, max(n_ids, 1)), 9.0, device="cuda")
    ent = torch.full((r + 1,), 9.0, device="cuda")
    ti = torch.full((r + 1, max(top, 1)), -7, dtype=torch.int32, device="cuda")
    tl = torch.full((r + 1, max(top, 1)), 9.0, device="cuda")
    nb = L.lgmlh_log_probs_workspace(r, v, top)
    ws = torch.full((nb + 64,), 0xA5, dtype=torch.uint8, device="cuda")
    hip.check(L.lgmlh_log_probs(buf.data_ptr() + 4 * lead, r, v, hip.ptr(di), n_ids, lp.data_ptr(),
                                ent.data_ptr() if entropy else None, top, ti.data_ptr(), tl.data_ptr(),
                                ws.data_ptr(), nb, st()))
    torch.cuda.synchronize()
    assert bool((ws[nb:] == 0xA5).all())
    out = [a.cpu().numpy() for a in (lp, ent, ti, tl)]
    assert (out[0][-1] == 9).all() and out[1][-1] == 9 and (out[2][-1] == -7).all() and (out[3][-1] == 9).all()
    return [a[:-1] for a in out]


def check_log_probs(L, x, ids=None, top=0, lead=0):
    """Rows without NaN or +inf and with a finite logit. Tolerances: x - M is
    rounded once, 2^-24 of up to 2 max|x|; each e^d is off by |d| 2^-23 + 2^-22,
    which weighs at most 2^-22 in Z, as do 64 roundings of a sum in a tree and
    log and log1p, 2^-22 of their value each: 2^-17 of log Z's 1 + n part is
    ample and still relative, since C and S stay apart; H also has sum p |d|."""
    r, v = x.shape
    lp, ent, ti, tl = log_probs(L, x, ids, top, lead=lead)
    y = x.astype(np.float64)
    m = y.max(1, keepdims=True)
    s = np.where(y == m, 0, np.exp(y - m)).sum(1, keepdims=True)
    c = (y == m).sum(1, keepdims=True)
    logz = np.log(c) + np.log1p(s / c)
    ref = y - m - logz
    with np.errstate(invalid="ignore"):
        tol = 2.0**-23 * np.abs(np.where(np.isfinite(y), y - m, 0)) + 2.0**-17 * logz
        p = np.exp(ref)
        h = -np.where(p > 0, p * ref, 0).sum(1)
    rows = np.arange(r)[:, None]
    if ids is not None:
        inside = (ids >= 0) & (ids < v)
        at = np.where(inside, ids, 0)
        want = np.where(inside, ref[rows, at], -np.inf)
        assert np.array_equal(np.isneginf(lp), np.isneginf(want))
        fin = np.isfinite(want)
        assert (np.abs(lp - want)[fin] <= tol[rows, at][fin]).all()
    assert (np.abs(ent - h) <= 2.0**-17 * np.maximum(h, logz[:, 0]) + 1e-37).all()
    if top:
        for i in range(r):
            order = np.lexsort((np.arange(v), -y[i]))[:top]
            assert np.array_equal(ti[i], order), i
            want = ref[i, order]
            fin = np.isfinite(want)
            assert np.array_equal(tl[i][~fin], want[~fin])
            assert (np.abs(tl[i] - want)[fin] <= tol[i, order][fin]).all()
    return lp, ent, ti, tl


@pytest.mark.parametrize("v", [1, 2, 3, 63, 64, 65, 257, 2047, 2049, 8192, 8197, 40001, 128256])
@pytest.mark.parametrize("top", [0, 1, 5, 20, 64])
@pytest.mark.parametrize("lead", [0, 1])
def test_log_probs(L, v, top, lead):
    rng = np.random.default_rng(v + top)
    r = 3
    x = (rng.standard_normal((r, v)) * 2.5).astype(np.float32)
    x[1, rng.integers(v)] += 25.0  # almost all of the mass: log p of 1e-8
    ids = rng.integers(0, v, (r, 4))
    ids[:, 0] = x.argmax(1)
    ids[0, 3], ids[1, 3] = -1, v
    check_log_probs(L, x, ids, min(top, v), lead)


def test_log_probs_of_many_rows(L):
    """Past the switch to the larger slices; a row's values do not change."""
    rng = np.random.default_rng(5)
    x = (rng.standard_normal((300, 20011)) * 3).astype(np.float32)
    ids = rng.integers(0, 20011, (300, 64))
    check_log_probs(L, x, ids, 7)


@pytest.mark.parametrize("v,top", [(300, 64), (5000, 20), (128256, 64), (1 << 20, 64)])
def test_log_probs_with_ties(L, v, top):
    """Equal logits go to the smaller id: all equal, few values, -0 and 0, and
    everything masked but a few."""
    rng = np.random.default_rng(v)
    few = rng.choice([0.5, -0.0, 0.0, 1.5], v).astype(np.float32)
    masked = np.full(v, -np.inf, np.float32)
    masked[[7, v // 2, v - 1]] = [0.0, 2.0, -1e30]
    low = np.full(v, np.finfo(np.float32).min, np.float32)
    low[v - 2] = 1.0
    x = np.stack([np.zeros(v, np.float32), few, masked, low, np.where(np.arange(v) % 2, -0.0, 0.0).astype(np.float32)])
    check_log_probs(L, x, rng.integers(0, v, (5, 3)), top)


def test_log_probs_of_rows_without_a_distribution(L):
    """Nothing but -inf; +inf; NaN."""
    v = 3000
    x = np.random.default_rng(2).standard_normal((5, v)).astype(np.float32)
    x[0] = -np.inf
    x[1, [5, 2500]] = np.inf
    x[2, 2999] = np.nan
    x[3], x[3, 9] = -np.inf, np.nan
    ids = np.tile(np.array([[5, 6]]), (5, 1))
    lp, ent, ti, tl = log_probs(L, x, ids, 3)
    assert (lp[0] == -np.inf).all() and ent[0] == 0 and list(ti[0]) == [0, 1, 2] and (tl[0] == -np.inf).all()
    half = np.log(0.5)
    assert abs(lp[1, 0] - half) < 1e-6 and lp[1, 1] == -np.inf and abs(ent[1] + half) < 1e-6
    assert list(ti[1][:2]) == [5, 2500] and tl[1, 2] == -np.inf
    for i in (2, 3):
        assert np.isnan(lp[i]).all() and np.isnan(ent[i]) and np.isnan(tl[i]).all()
    assert list(ti[2]) == list(np.lexsort((np.arange(v), -np.where(np.isnan(x[2]), -np.inf, x[2])))[:3])
    assert list(ti[3]) == [0, 1, 2]
    check_log_probs(L, x[4:], ids[4:], 3)


def test_log_probs_parts_alone(L):
    from lgml_amd import hip
    x = np.random.default_rng(3).standard_normal((2, 777)).astype(np.float32)
    a = log_probs(L, x, None, 0)
    b = log_probs(L, x, None, 9)
    assert np.array_equal(a[1], b[1])
    # either of the alternatives' outputs may be left out
    xd = dev(x)
    ws = torch.empty(L.lgmlh_log_probs_workspace(2, 777, 9), dtype=torch.uint8, device="cuda")
    ti = torch.empty(2, 9, dtype=torch.int32, device="cuda")
    tl = torch.empty(2, 9, device="cuda")
    for i, l in ((ti, None), (None, tl)):
        hip.check(L.lgmlh_log_probs(xd.data_ptr(), 2, 777, None, 0, None, None, 9, hip.ptr(i), hip.ptr(l),
                                    ws.data_ptr(), ws.numel(), st()))
    assert np.array_equal(ti.cpu().numpy(), b[2]) and np.array_equal(tl.cpu().numpy(), b[3])


@pytest.mark.parametrize("q8", [False, True])
def test_cells_behind_4_gib(L, q8):
    """The last blocks of a pool whose tensors pass 4 GiB: stored, moved, read
    back and attended to as in a small pool (the same bits)."""
    from lgml_amd import hip, runtime
    H, kv, D, n, past = 16, 8, 256, 40, 70
    per = (68 if q8 else 128) * D * kv
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

        # Memory never written is no input: a causal f16 plan takes 0 times the V of
        # unseen cells of a row's own blocks, and 0 x NaN is NaN. So the rest of the
        # pools is of defined bytes: finite f16, and NaN scales in Q8_0, where a row
        # holds whatever unseen cells hold.
        pools = [torch.full((blocks * per,), 0xFF if q8 else 0xA5, dtype=torch.uint8, device="cuda")
                 for _ in range(2)]
        cells = cell(np.arange(past + n))
        dc, kd, vd = dev(cells), dev(k), dev(v)
        hip.check((L.lgmlh_kv_store_q8 if q8 else L.lgmlh_kv_store)(
            pools[0].data_ptr(), pools[1].data_ptr(), 64 * blocks, kv, D, kd.data_ptr(), vd.data_ptr(),
            dc.data_ptr(), cells.ctypes.data, len(cells), st()))

        class P:
            plan = runtime.Plan([n], [past], tab, np.zeros(n, np.int32), H, kv, blocks, 2, parents=parents)

        P.info, P.ub = P.plan.info, P.plan.ub
        got = [run_attention(L, P, H, kv, D, D ** -0.5, q, pools, q8)]
        one = runtime.Plan([1], [past], tab, np.zeros(1, np.int32), H, kv, blocks, 2)
        P.info, P.ub = one.info, one.ub
        got.append(run_attention(L, P, H, kv, D, D ** -0.5, q[:1], pools, q8))
        addr = torch.tensor([p.data_ptr() for p in pools], dtype=torch.int64, device="cuda")
        a, b = cell(src), cell(dst)
        da, db = dev(a), dev(b)
        hip.check(L.lgmlh_kv_move(hip.Q8_0 if q8 else hip.F16, addr.data_ptr(), 2, 64 * blocks, kv, D,
                                  da.data_ptr(), db.data_ptr(), a.ctypes.data, b.ctypes.data, 3, st()))
        for w in range(2):
            out = torch.empty((len(cells), kv, D), dtype=torch.float16, device="cuda")
            if q8:
                hip.check(L.lgmlh_kv_gather_q8(pools[w].data_ptr(), w, 64 * blocks, kv, D, dc.data_ptr(),
                                               len(cells), out.data_ptr(), hip.F16, st()))
            else:
                hip.check(L.lgmlh_kv_gather(pools[w].data_ptr(), w, 64 * blocks, kv, D, dc.data_ptr(),
                                            len(cells), out.data_ptr(), st()))
            got.append(out.cpu().numpy())
        results.append(got)
        want = (values(k) if q8 else k).astype(np.float16)
        want[dst] = want[src]
        assert np.array_equal(got[2], want)
    for a, b in zip(*results):
        assert np.array_equal(a, b)


def test_log_probs_behind_the_32_bit_element(L):
    """The last row of more than 2^31 logits."""
    v = 1 << 20
    rows = (1 << 31) // v + 2
    x = torch.zeros((rows, v), dtype=torch.float32, device="cuda")
    last = np.random.default_rng(4).standard_normal(v).astype(np.float32)
    x[-1] = dev(last)
    from lgml_amd import runtime
    ids = torch.full((rows, 1), 77, dtype=torch.int32)
    got = runtime.log_probs(x, ids, 3)
    y = last.astype(np.float64)
    lz = np.log(np.exp(y).sum())
    order = np.lexsort((np.arange(v), -y))[:3]
    assert list(got["top_ids"][-1].cpu().numpy()) == list(order)
    # |x| up to 6 and log Z near 14.4, each a rounding or two; the sum's 2^-18 at most
    tol = 32 * 2.0**-23 + 2.0**-18
    assert np.abs(got["top_lp"][-1].cpu().numpy() - (y[order] - lz)).max() <= tol
    assert abs(got["lp"][-1, 0].item() - (y[77] - lz)) <= tol
    assert abs(got["lp"][0, 0].item() + np.log(v)) <= tol
