"""Copies of blocks in every pool tensor at once, on the GPU: every byte of pools of
each type, forks, cleared blocks, compaction of sequences and of an engine's pool."""
import numpy as np
import pytest

from oracle import models
from tests.gpu_util import lcg_ints
from tests.test_gpu_draft import dev, st
from tests.test_gpu_q4 import cell_bytes as q4_bytes
from tests.test_gpu_sched import GEMMA_TINY, R, UB, drive
from tests.test_gpu_spill import chat

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

TILE = {"F16": 128, "Q8_0": 68, "Q4_0": 36}


def cell_bytes(kind, which, cell, D):
    d = np.arange(D)
    if kind == "Q4_0":
        return q4_bytes(which, cell, D)
    if kind == "F16":
        e = 2 * (d * 64 + cell if which else cell * D + d)
        return np.concatenate([e, e + 1])
    if which:
        e = d * 64 + cell % 32 // 8 * 16 + cell // 32 * 8 + cell % 8
    else:
        e = ((d // 64 * 64 + cell) * 4 + d % 32 // 8) * 16 + d % 64 // 32 * 8 + d % 8
    s = 64 * D + 2 * (np.arange(D // 32) * 64 + cell)
    return np.concatenate([e, s, s + 1])


def copied(kind, pools, copies, D):
    """What the pools (n, blocks, kv, bytes) hold after the copies."""
    want = pools.copy()
    at = [[cell_bytes(kind, w, c, D) for c in range(64)] for w in range(2)]
    for p in range(len(pools)):
        for src, dst, n in copies:
            if n:
                b = np.concatenate(at[p % 2][:n])
                want[p, dst][:, b] = pools[p, src][:, b] if src >= 0 else 0
    return want


@pytest.mark.parametrize("kind,D,kv", [("F16", 8, 3), ("F16", 64, 1), ("F16", 128, 8), ("F16", 256, 2),
                                       ("Q8_0", 64, 3), ("Q8_0", 128, 8), ("Q8_0", 256, 1),
                                       ("Q4_0", 64, 1), ("Q4_0", 128, 3), ("Q4_0", 256, 8)])
def test_copies_take_the_first_cells(kind, D, kv):
    """Every count of cells, one source for several targets, cleared blocks, blocks at
    both ends; every other byte stays."""
    from lgml_amd import hip
    L = hip.lib()
    rng = np.random.default_rng(D + kv)
    blocks, layers = 140, 2
    pools0 = rng.integers(0, 256, (2 * layers, blocks, kv, TILE[kind] * D)).astype(np.uint8)
    pools = dev(pools0)
    addr = torch.tensor([p.data_ptr() for p in pools], dtype=torch.int64, device="cuda")
    order = rng.permutation(np.arange(1, blocks - 1))
    copies = [(int(order[i % 20]), int(order[30 + i]), i % 65) for i in range(0, 90)]
    copies += [(-1, int(order[120]), 64), (-1, int(order[121]), 13), (0, blocks - 1, 64), (0, int(order[122]), 0)]
    copies = np.array(copies, np.int32)
    d = dev(copies)
    hip.check(L.lgmlh_kv_copy_blocks(getattr(hip, kind), addr.data_ptr(), 2 * layers, 64 * blocks, kv, D,
                                     d.data_ptr(), copies.ctypes.data, len(copies), st()))
    got = pools.cpu().numpy()
    want = copied(kind, pools0, copies.tolist(), D)
    assert np.array_equal(got, want), np.argwhere(got != want)[:4]


def test_device_copies_that_the_host_copy_did_not_name_stay_in_the_pool():
    """Blocks outside the pool in the device's array are skipped."""
    from lgml_amd import hip
    L = hip.lib()
    kv, D, blocks = 2, 64, 6
    pools0 = np.random.default_rng(1).integers(0, 256, (2, blocks, kv, 128 * D)).astype(np.uint8)
    pools = dev(pools0)
    addr = torch.tensor([p.data_ptr() for p in pools], dtype=torch.int64, device="cuda")
    host = np.array([[0, 1, 64], [2, 3, 64], [4, 5, 64]], np.int32)
    d = dev(np.array([[0, blocks, 64], [-2, 3, 64], [4, 5, 90]], np.int32))
    hip.check(L.lgmlh_kv_copy_blocks(hip.F16, addr.data_ptr(), 2, 64 * blocks, kv, D, d.data_ptr(),
                                     host.ctypes.data, 3, st()))
    want = pools0.copy()
    want[:, 5] = pools0[:, 4]
    assert np.array_equal(pools.cpu().numpy(), want)


KINDS = ["F16", "Q8_0", "Q4_0"]


def model(kind, cells, **kw):
    from lgml_amd import hip, runtime
    hp, w = models.build("c1", seed=7)
    return runtime.DeviceModel(hp, w, cells, kv_type=getattr(hip, kind), **kw), hp["n_vocab"]


def step(m, seqs, toks):
    """Each sequence's tokens in one pass; the logits of its last."""
    for c, t in zip(seqs, toks):
        c.pool.reserve(c, c.n_past + len(t))
    tab = np.full((len(seqs), max(len(c.blocks) for c in seqs)), -1, np.int32)
    for i, c in enumerate(seqs):
        tab[i, :len(c.blocks)] = c.blocks
    plan = m.plan([len(t) for t in toks], [c.n_past for c in seqs], tab, np.concatenate(toks).astype(np.int32))
    out = m.forward(plan).cpu().numpy()
    for c, t in zip(seqs, toks):
        c.n_past += len(t)
    return out


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [64, 100])
def test_forks_go_on_as_their_sequence(kind, n):
    """Bit for bit the logits of sequences that ran the prompt themselves; the one they
    left goes on undisturbed; blocks come back when they end."""
    from lgml_amd import engine
    m, V = model(kind, 2048)
    seqs = engine.PoolSeqs(m)
    prompt = lcg_ints(1, n, 0, V)
    c = engine.Seq(seqs)
    step(m, [c], [prompt])
    kids = seqs.fork(c, 3)
    assert [k.n_past for k in kids] == [n] * 3 and seqs.alloc.used == (1 if n == 64 else 1 + 4)
    tails = [lcg_ints(5 + i, 9, 0, V) for i in range(4)]
    got = step(m, [c] + kids, tails)
    alone = engine.PoolSeqs(m2 := model(kind, 2048)[0])
    for i in range(4):
        s = engine.Seq(alone)
        step(m2, [s], [prompt])
        assert np.array_equal(step(m2, [s], [tails[i]])[0].view(np.uint32), got[i].view(np.uint32)), i
    for s in [c] + kids:
        seqs.free(s)
    assert seqs.alloc.used == 0


@pytest.mark.parametrize("kind", KINDS)
def test_sequences_compact_and_go_on(kind):
    """Blocks move down, shared ones once; the next logits have the bits they have
    without."""
    from lgml_amd import engine

    def run(compact):
        m, V = model(kind, 64 * 40)
        seqs = engine.PoolSeqs(m)
        all_ = [engine.Seq(seqs) for _ in range(6)]
        for r in range(3):  # blocks of the sequences in turn
            step(m, all_, [lcg_ints(10 * r + i, 64 if r < 2 else 20 + i, 0, V) for i in range(6)])
        for i in (0, 2, 3):
            seqs.free(all_[i])
        live = [all_[i] for i in (1, 4, 5)]
        live += seqs.fork(live[0], 2)
        if compact:
            m.clear_blocks([b for b in range(40) if not seqs.alloc.in_use(b)])
            with pytest.raises(ValueError):
                seqs.compact(live[:-1])
            n = seqs.compact(live)
            assert n == 11 and sorted({b for c in live for b in c.blocks}) == list(range(11))
            assert [seqs.alloc.in_use(b) for b in range(40)] == [True] * 11 + [False] * 29
            size = m.kpools[0].numel()
            assert m.shrink_pool(64 * n) == 64 * n and m.kpools[0].numel() * 40 == size * n
            seqs.alloc.set_cap(n)
            m.grow_pool(64 * 40)
            seqs.alloc.set_cap(40)
        return step(m, live, [lcg_ints(99 + i, 5, 0, V) for i in range(5)])

    assert np.array_equal(run(True).view(np.uint32), run(False).view(np.uint32))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("run_ahead", [False, True])
def test_an_engine_compacts_between_steps(kind, run_ahead):
    """A pool that grew for a peak is cut to the blocks in use, with passes in flight;
    replies, cached prefixes and later growth are those of an engine left alone."""
    from lgml_amd import engine

    def run(compact):
        m, V = model(kind, 64 * 64, kv_initial=128)
        eng = engine.Engine(m, 8, ubatch=64, prefix_cache=True, run_ahead=run_ahead)
        first = [engine.Request(lcg_ints(20 + i, 150 + 40 * i, 0, V), 3 + 9 * (i % 2)) for i in range(6)]
        for r in first:
            eng.submit(r)
        for _ in range(12):
            eng.step()
        cells = m.n_cells
        if compact:
            got = eng.compact(keep_cached=False)
            assert got < cells and got == 64 * max(1, len({b for r in eng.active for b in r.seq.blocks}))
        drive(eng, first)
        again = [engine.Request(first[0].prompt + lcg_ints(70, 30, 0, V), 5),
                 engine.Request(lcg_ints(71, 500, 0, V), 5)]
        for r in again:
            eng.submit(r)
        drive(eng, again)
        if compact:
            eng.compact()
            assert m.n_cells <= cells
        last = [engine.Request(first[1].prompt, 4)]
        eng.submit(last[0])
        drive(eng, last)
        return [r.out for r in first + again + last]

    assert run(True) == run(False)


def test_an_engine_with_rings_compacts_its_paged_layers():
    from lgml_amd import engine, hip, runtime
    hp, w = models.build(GEMMA_TINY, seed=91, init="normal")

    def run(compact):
        gm = runtime.DeviceModel(hp, w, 1024, ring_cells=2 * R * 64, kv_type=hip.F16)
        eng = engine.Engine(gm, 2, ubatch=UB)
        reqs = [engine.Request(lcg_ints(50 + i, n, 0, hp["n_vocab"]), 6 + 6 * i) for i, n in enumerate([90, 150])]
        for r in reqs:
            eng.submit(r)
        for _ in range(50):
            if reqs[0].done:
                break
            eng.step()
        if compact:
            assert eng.compact() < 1024
        drive(eng, reqs)
        return [r.out for r in reqs]

    assert run(True) == run(False)


def test_copies_are_queued_and_capture_is_refused():
    from lgml_amd import engine
    m, _ = model("Q4_0", 1024)
    before = [m.gather_kv(1, np.arange(1024), w) for w in (0, 1)]
    with pytest.raises(RuntimeError):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            m.copy_blocks([1], [2])
    for bad in (([1], [2, 3]), ([1.5], [2]), ([2**32], [2])):
        with pytest.raises(ValueError):
            m.copy_blocks(*bad)
    m.copy_blocks([], [])
    engine.PoolSeqs(m).copy_block(3, 3, 9)
    for w in (0, 1):
        assert np.array_equal(m.gather_kv(1, np.arange(1024), w), before[w])
