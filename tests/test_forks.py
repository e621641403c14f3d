"""CPU checks of forks of sequences: models they refuse, what a fork or another copy that
fails leaves behind, a source that goes while blocks are taken (no GPU work)."""
import pytest

torch = pytest.importorskip("torch")


class Model:
    def __init__(self, blocks, fail=None):
        self.pool_blocks = self.max_blocks = blocks
        self.n_cells = 64 * blocks
        self.calls, self.fail = [], fail

    def copy_blocks(self, src, dst, cells=64):
        if self.fail:
            raise self.fail
        self.calls.append((list(src), list(dst), cells))


def sequence(model, cells, **kw):
    from lgml_amd import engine
    seqs = engine.PoolSeqs(model, **kw)
    c = engine.Seq(seqs)
    seqs.reserve(c, cells)
    c.n_past = cells
    return seqs, c


@pytest.mark.parametrize("n_past", [128, 150])
def test_models_with_rings_are_refused(n_past):
    """A slot's rings hold the cells of its sliding layers: a fork would go on without."""
    m = Model(8)
    m.swa = [False, True]
    seqs, c = sequence(m, n_past)
    used = seqs.alloc.used
    with pytest.raises(ValueError, match="rings"):
        seqs.fork(c, 2)
    assert seqs.alloc.used == used and not m.calls
    m.swa = [False, False]
    assert len(seqs.fork(c, 2)) == 2


def test_a_copy_that_fails_leaves_no_references():
    m = Model(8, RuntimeError("captured"))
    seqs, c = sequence(m, 150)
    with pytest.raises(RuntimeError, match="captured"):
        seqs.fork(c, 3)
    assert [seqs.alloc.refs_of(b) for b in range(8)] == [1, 1, 1] + [0] * 5
    assert seqs.compact([c]) == 3
    m.fail = None
    assert [d.blocks for d in seqs.fork(c, 2)] == [[0, 1, 3], [0, 1, 4]]


def test_a_pool_that_cannot_grow_leaves_no_references():
    m = Model(4)
    m.max_cells, m.max_blocks = 64 * 16, 16

    def grow():
        raise torch.OutOfMemoryError("no memory")

    m.grow_pool = grow
    seqs, c = sequence(m, 150)
    with pytest.raises(torch.OutOfMemoryError):
        seqs.fork(c, 3)  # one block is free
    assert [seqs.alloc.refs_of(b) for b in range(4)] == [1, 1, 1, 0]
    assert seqs.compact([c]) == 3 and not m.calls


def test_a_source_that_pressure_frees_is_there_until_it_is_copied():
    m = Model(4)
    seqs, c = sequence(m, 150)
    more = []

    def pressure(pool, _):
        if not more:
            more.append(pool)
            pool.free(c)

    seqs.pressure = pressure
    from lgml_amd import engine
    with pytest.raises(engine.PoolFull):
        seqs.fork(c, 2)  # its blocks are held: there is no fifth
    assert more and c.blocks == [] and seqs.alloc.used == 0
    seqs, c = sequence(Model(5), 150)
    other = engine.Seq(seqs)
    seqs.reserve(other, 64)
    more.clear()

    def both(pool, _):
        pool.free(c)
        pool.free(other)

    seqs.pressure = both
    kids = seqs.fork(c, 2)
    assert [d.blocks for d in kids] == [[0, 1, 4], [0, 1, 3]] and seqs.model.calls == [([2, 2], [4, 3], 22)]
    assert [seqs.alloc.refs_of(b) for b in range(5)] == [2, 2, 0, 1, 1]


def test_a_cut_whose_copy_fails_leaves_no_references():
    """A shared block is copied before a sequence goes on in it."""
    from lgml_amd import engine
    m = Model(8)
    seqs, c = sequence(m, 128)
    d = seqs.fork(c)[0]
    m.fail, m.kv_type = RuntimeError("captured"), None
    with pytest.raises(RuntimeError):
        seqs.truncate(d, 100)
    assert seqs.alloc.used == 2 and [seqs.alloc.refs_of(b) for b in range(3)] == [2, 2, 0]
    m.fail = None
    seqs.truncate(d, 100)
    assert d.blocks == [0, 2] and m.calls == [([1], [2], 36)]
    assert isinstance(d, engine.Seq) and seqs.compact([c, d]) == 3


def test_an_attached_block_whose_copy_fails_is_let_go():
    from lgml_amd import engine
    m = Model(8, RuntimeError("captured"))
    m.kv_type = None
    seqs, c = sequence(m, 100)
    toks = list(range(100))
    eng = object.__new__(engine.Engine)
    eng.model, eng.seqs, eng.ram, eng.infos, eng.hits, eng.hit_blocks = m, seqs, None, {}, 0, 0
    req = engine.Request(toks, 1)
    req.seq = c
    eng.publish_tail(req, toks)
    seqs.free(c)
    assert (seqs.alloc.used, seqs.alloc.cached) == (0, 2)
    req = engine.Request(toks + [7], 1)
    req.seq = engine.Seq(seqs)
    with pytest.raises(RuntimeError):
        eng.attach(req)
    seqs.free(req.seq)
    assert (seqs.alloc.used, seqs.alloc.cached) == (0, 2)
    m.fail = None
    assert eng.attach(req) == 100 and m.calls == [([1], [2], 36)]


def test_a_request_whose_attach_fails_starts_from_nothing():
    """Blocks shared before the failure would put its first token behind them."""
    from lgml_amd import engine
    m = Model(8, RuntimeError("captured"))
    m.kv_type = None
    seqs, c = sequence(m, 100)
    toks = list(range(100))
    eng = object.__new__(engine.Engine)
    eng.model, eng.seqs, eng.ram, eng.infos, eng.hits, eng.hit_blocks = m, seqs, None, {}, 0, 0
    eng.active, eng.n_slots, eng.free_slots, eng._submitted, eng.prefix_cache = [], 2, [0, 1], 0, True
    req = engine.Request(toks, 1)
    req.seq = c
    eng.publish_tail(req, toks)
    seqs.free(c)
    req = engine.Request(toks + [7], 1)
    with pytest.raises(RuntimeError):
        eng.submit(req)
    assert (req.fed, req.seq.n_past, req.seq.blocks, req.seq.keys) == (0, 0, [], [])
    assert (seqs.alloc.used, seqs.alloc.cached) == (0, 2)
