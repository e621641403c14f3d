"""CPU checks of pools that grow and shrink: what is left where memory for a tensor fails
part-way (no GPU work)."""
import ctypes as C
import types

import numpy as np
import pytest

torch = pytest.importorskip("torch")

LAYERS, KV, D = 4, 2, 64


@pytest.fixture
def runtime(monkeypatch):
    """The runtime over host memory; fail.after: allocations that succeed from now on."""
    from lgml_amd import runtime
    fail = types.SimpleNamespace(after=1 << 30)

    def spend():
        fail.after -= 1
        if fail.after < 0:
            raise torch.OutOfMemoryError("no memory")

    def grow(old, old_cells, new, cells, kv, d, _):
        C.memset(new, 0, 128 * kv * d * cells // 64)
        C.memmove(new, old, 128 * kv * d * old_cells // 64)
        return 0

    def empty(nbytes):
        spend()
        return torch.empty(nbytes, dtype=torch.uint8)

    clone = torch.Tensor.clone

    def cloned(t):
        spend()
        return clone(t)

    lib = types.SimpleNamespace(lgmlh_kv_layer_bytes=lambda cells, kv, d: 2 * cells * kv * d, lgmlh_kv_grow=grow)
    monkeypatch.setattr(runtime, "DEV", "cpu")
    monkeypatch.setattr(runtime, "_empty", empty)
    monkeypatch.setattr(runtime, "stream", lambda: None)
    monkeypatch.setattr(runtime.hip, "lib", lambda: lib)
    monkeypatch.setattr(torch.Tensor, "clone", cloned)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda: types.SimpleNamespace(synchronize=lambda: None))
    return types.SimpleNamespace(mod=runtime, fail=fail)


def pool(rt, blocks, ceiling):
    m = object.__new__(rt.mod.DeviceModel)
    m.kv_type, m.hp, m.swa = rt.mod.hip.F16, {"n_layer": LAYERS}, [i == 1 for i in range(LAYERS)]
    m.n_cells, m.max_cells, m.paged_dims = 64 * blocks, 64 * ceiling, (D, KV)
    m.m = types.SimpleNamespace(n_cells=m.n_cells)
    m.layers = [types.SimpleNamespace() for _ in range(LAYERS)]
    gen = torch.Generator().manual_seed(3)
    m.kpools, m.vpools = ([torch.randint(256, (128 * KV * D * blocks,), dtype=torch.uint8, generator=gen)
                           for _ in range(LAYERS)] for _ in range(2))
    for il in range(LAYERS):
        m.layers[il].kpool, m.layers[il].vpool = m.kpools[il].data_ptr(), m.vpools[il].data_ptr()
    m.pools_dev = torch.tensor([p.data_ptr() for il in range(LAYERS) if not m.swa[il]
                                for p in (m.kpools[il], m.vpools[il])])
    m.n_pools = len(m.pools_dev)
    return m


def holds(m, was, cells):
    """The pool has `cells` cells of what it was, in tensors that are all long enough, and
    every address is a tensor's own."""
    nb = 2 * cells * KV * D
    assert m.n_cells == m.m.n_cells == cells and m.pool_blocks == cells // 64
    addr = m.pools_dev.tolist()
    for il in range(LAYERS):
        for w, (pools, attr) in enumerate(((m.kpools, "kpool"), (m.vpools, "vpool"))):
            assert getattr(m.layers[il], attr) == pools[il].data_ptr()
            if m.swa[il]:
                assert torch.equal(pools[il], was[w][il])
                continue
            assert pools[il].numel() >= nb
            keep = min(nb, was[w][il].numel())
            assert torch.equal(pools[il][:keep], was[w][il][:keep])
            assert addr.pop(0) == pools[il].data_ptr()
    assert not addr


@pytest.mark.parametrize("after", range(6))
def test_a_pool_that_could_not_all_be_cut_counts_as_cut(runtime, after):
    m = pool(runtime, 6, 12)
    was = [[t + 0 for t in p] for p in (m.kpools, m.vpools)]
    runtime.fail.after = after
    with pytest.raises(torch.OutOfMemoryError):
        m.shrink_pool(128)
    holds(m, was, 128)
    runtime.fail.after = 1 << 30
    assert m.shrink_pool(128) == 128  # the rest is cut now
    holds(m, was, 128)
    assert all(m.kpools[il].numel() == (6 if m.swa[il] else 2) * 128 * KV * D for il in range(LAYERS))
    assert m.grow_pool(64 * 12) == 64 * 12
    holds(m, [[t if m.swa[il] else t[:256 * KV * D] for il, t in enumerate(p)] for p in was], 64 * 12)


@pytest.mark.parametrize("after", range(6))
def test_a_pool_that_could_not_all_grow_stays_as_it_was(runtime, after):
    m = pool(runtime, 6, 12)
    was = [[t + 0 for t in p] for p in (m.kpools, m.vpools)]
    runtime.fail.after = after
    with pytest.raises(torch.OutOfMemoryError):
        m.grow_pool()
    holds(m, was, 64 * 6)
    runtime.fail.after = 1 << 30
    assert m.grow_pool() == 64 * 12
    holds(m, was, 64 * 12)


def test_a_plan_of_blocks_that_were_cut_off_is_refused(runtime):
    """Such a pass would read behind the tensors."""
    m = pool(runtime, 6, 12)
    m.m = types.SimpleNamespace(n_cells=64 * 6)

    def plan(tab):
        return types.SimpleNamespace(seq_n=np.array([1, 2], np.int32), seq_npast=np.array([127, 63], np.int32),
                                     block_tab=np.array(tab, np.int32), pool_blocks=6)

    class Reached(Exception):
        pass

    def workspace(*_):
        raise Reached

    m.workspace = workspace
    rows = np.zeros(1, np.int32)
    high, low = plan([[0, 3], [1, 2]]), plan([[0, 1], [1, 2]])
    behind = plan([[0, 1, 5], [1, 2, -1]])  # (a place that no token takes)
    for p in (high, low, behind):
        with pytest.raises(Reached):
            m.forward(p, rows)
    m.shrink_pool(64 * 3)
    with pytest.raises(ValueError, match="block 3"):
        m.forward(high, rows)
    for p in (low, behind):
        with pytest.raises(Reached):
            m.forward(p, rows)
    m.grow_pool(64 * 6)
    with pytest.raises(Reached):
        m.forward(high, rows)


def test_cells_that_were_cut_off_are_not_read_back(runtime):
    """The f16 read back takes the cells it is given."""
    m = pool(runtime, 6, 12)
    m.dims, m.ring_cells = [(D, KV)] * LAYERS, 128

    def gather(*_):
        raise AssertionError("the device is reached")

    runtime.mod.hip.lib().lgmlh_kv_gather = gather
    m.shrink_pool(128)
    for layer, cells in ((0, [0, 128]), (0, [-1, 5]), (1, [128])):
        with pytest.raises(ValueError, match="of a pool of 128"):
            m.gather_kv(layer, cells)
    with pytest.raises(AssertionError, match="reached"):
        m.gather_kv(0, [0, 127])


def test_sizes_that_change_nothing(runtime):
    m = pool(runtime, 6, 12)
    was = [[t + 0 for t in p] for p in (m.kpools, m.vpools)]
    runtime.fail.after = 0
    assert m.shrink_pool(64 * 6) == m.shrink_pool(64 * 7) == m.grow_pool(64) == 64 * 6
    holds(m, was, 64 * 6)
    for bad in (0, -64, 100):
        with pytest.raises(ValueError):
            m.shrink_pool(bad)


def test_an_engine_whose_pool_could_not_all_be_cut_gives_out_its_blocks_alone():
    from lgml_amd import engine

    class Model:
        pool_blocks, max_blocks, n_cells = 8, 8, 512

        def shrink_pool(self, cells):
            self.n_cells, self.pool_blocks = cells, cells // 64
            raise torch.OutOfMemoryError("no memory")

    eng = object.__new__(engine.Engine)
    eng.model, eng.active = Model(), []
    eng.seqs = engine.PoolSeqs(eng.model)
    with pytest.raises(torch.OutOfMemoryError):
        eng.compact()
    assert eng.seqs.alloc.cap == 1
    assert eng.seqs.alloc.take() == 0 and eng.seqs.alloc.take() is None


def test_a_block_does_not_go_behind_the_cap():
    """The tensors hold no such block."""
    from lgml_amd import hip, kvpool
    p = kvpool.Pool(8, 64, cap=4)
    a, b = p.take(), p.take()
    for dst in (4, 7):
        with pytest.raises(hip.LgmlhError):
            p.relocate(a, dst)
    p.relocate(a, 3)
    assert p.refs_of(3) == 1 and p.take() == a and b == 1
