"""Whole passes and the engine over Q8_0 pools and trees of drafted tokens: a tree
verified in one pass gives the logits of decoding its paths token by token, the
accepted path's cells moved behind the context go on as if decoded; Q8_0 pools
through the engine's sharing, spilling, growing and rings; captured and side
stream runs of the operators together."""
import ctypes as C

import numpy as np
import pytest

from oracle import models
from tests.gpu_util import Schedule, lcg_ints, rel_err
from tests.test_gpu_sched import GEMMA_TINY, R, UB, drive
from tests.test_gpu_spill import chat

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def kv_types():
    from lgml_amd import hip
    return {"f16": hip.F16, "q8_0": hip.Q8_0}


def st():
    return torch.cuda.current_stream().cuda_stream


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to("cuda")


# ---- the fused store ---------------------------------------------------------------
@pytest.mark.parametrize("H,kv,D,neox", [(4, 2, 64, 0), (8, 8, 128, 1), (8, 4, 256, 1)])
def test_qkv_rope_store_q8_stores_the_roped_rows(H, kv, D, neox):
    """Its pool bytes are lgmlh_kv_store_q8's of the same rows: K roped (read back
    as the q heads of a call with K in their place), V as given; a cell outside
    the pool is not written."""
    from lgml_amd import hip
    L = hip.lib()
    rng = np.random.default_rng(D)
    n, cells_n = 37, 256
    qkv = rng.standard_normal((n, (H + 2 * kv) * D)).astype(np.float32)
    pos = dev(rng.integers(0, 5000, n).astype(np.int32))
    cells = np.concatenate([np.arange(60, 96), [cells_n]]).astype(np.int64)
    qn, kn = (dev(1 + 0.1 * rng.standard_normal(D).astype(np.float32)) for _ in range(2))
    nb = L.lgmlh_kv_q8_layer_bytes(cells_n, kv, D)

    def pools():
        return [torch.full((nb,), 0x5A, dtype=torch.uint8, device="cuda") for _ in range(2)]

    got = pools()
    q = torch.empty(n, H * D, device="cuda")
    args = (D, neox, 1e4, None, qn.data_ptr(), kn.data_ptr(), 1e-5, pos.data_ptr())
    dq, dc = dev(qkv), dev(cells)
    hip.check(L.lgmlh_qkv_rope_store_q8(dq.data_ptr(), n, H, kv, D, *args, got[0].data_ptr(),
                                        got[1].data_ptr(), cells_n, dc.data_ptr(), q.data_ptr(), st()))
    # the f16 entry's q, and K's rows as the q heads of kv heads
    f16 = [torch.zeros(L.lgmlh_kv_layer_bytes(cells_n, kv, D), dtype=torch.uint8, device="cuda") for _ in range(2)]
    q2 = torch.empty_like(q)
    hip.check(L.lgmlh_qkv_rope_store(dq.data_ptr(), n, H, kv, D, *args, f16[0].data_ptr(), f16[1].data_ptr(),
                                     cells_n, dc.data_ptr(), q2.data_ptr(), st()))
    assert torch.equal(q, q2)
    k_as_q = dev(np.concatenate([qkv[:, H * D:(H + kv) * D], qkv[:, H * D:]], 1))
    roped = torch.empty(n, kv * D, device="cuda")
    args = (D, neox, 1e4, None, kn.data_ptr(), kn.data_ptr(), 1e-5, pos.data_ptr())
    hip.check(L.lgmlh_qkv_rope_store(k_as_q.data_ptr(), n, kv, kv, D, *args, f16[0].data_ptr(), f16[1].data_ptr(),
                                     cells_n, dc.data_ptr(), roped.data_ptr(), st()))
    want = pools()
    v = dev(qkv[:, (H + kv) * D:])
    hip.check(L.lgmlh_kv_store_q8(want[0].data_ptr(), want[1].data_ptr(), cells_n, kv, D, roped.data_ptr(),
                                  v.data_ptr(), dc.data_ptr(), cells.ctypes.data, n - 1, st()))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


# ---- a tree verified in one pass ------------------------------------------------------
class Decoder:
    """Sequences of one model over one pool."""

    def __init__(self, hp, w, kv_type, n_cells=2048, slots=3):
        from lgml_amd import runtime
        self.m = runtime.DeviceModel(hp, w, n_cells, kv_type=kv_type)
        self.sch = Schedule(n_cells // 64, slots)
        self.past = [0] * slots

    def run(self, which, toks, parents=None, rows=None):
        for s, t in zip(which, toks):
            self.sch.grow(s, self.past[s] + len(t))
        ids = np.concatenate([np.asarray(t, np.int32) for t in toks])
        plan = self.m.plan([len(t) for t in toks], [self.past[s] for s in which], self.sch.table(which), ids,
                           parents=None if parents is None else np.concatenate(parents))
        out = self.m.forward(plan, rows)
        if parents is None:
            for s, t in zip(which, toks):
                self.past[s] += len(t)
        return out, plan

    def cells(self, s, slots):
        b = self.sch.seqs[s].blocks
        return [b[p // 64] * 64 + p % 64 for p in slots]


@pytest.mark.parametrize("kind", ["f16", "q8_0"])
@pytest.mark.parametrize("shape,layers", [("c1", 2), ("c2", 2)])
def test_a_tree_is_verified_in_one_pass(kind, shape, layers):
    """Logits of a drafted path's nodes within 2e-3 of decoding its tokens one by
    one (the bar of whole passes here; a rounding of attention's last bits may
    move a K or V value to the next one its pool holds), the log probabilities
    of the drafted tokens, and the same again after the accepted cells moved."""
    from lgml_amd import runtime
    hp, w = models.build(shape, seed=21, n_layer=layers, init="normal")
    V = hp["n_vocab"]
    kv = kv_types()[kind]
    prompts = [lcg_ints(900 + i, n, 0, V) for i, n in enumerate([70, 17, 129])]
    a, b = Decoder(hp, w, kv), Decoder(hp, w, kv)
    la, lb = a.run([0, 1, 2], prompts)[0], b.run([0, 1, 2], prompts)[0]
    assert torch.equal(la, lb)  # a pass repeats its bits
    first = la.argmax(1).tolist()
    # token by token: six steps of greedy
    line, logits = [[t] for t in first], []
    for _ in range(6):
        lg = a.run([0, 1, 2], [[t[-1]] for t in line])[0]
        logits.append(lg.cpu().numpy())
        for s in range(3):
            line[s].append(int(lg[s].argmax()))
    # the tree: node 0 the last sampled token, a path of the right tokens among
    # others (sequence 1's path ends after two)
    trees, toks, path = [], [], []
    for s in range(3):
        t, par, right, at = [line[s][0]], [-1], [0], 0
        for d in range(1, 6):
            for wrong in range(2):
                t.append((line[s][d] + 1 + wrong) % V)
                par.append(at)
            ok = s != 1 or d < 3
            t.append(line[s][d] if ok else (line[s][d] + 5) % V)
            par.append(at)
            at = len(t) - 1
            if ok:
                right.append(at)
        trees.append(np.array(par, np.int32))
        toks.append(t)
        path.append(right)
    n = [len(t) for t in toks]
    off = np.cumsum([0] + n)
    lg, plan = b.run([0, 1, 2], toks, trees, rows=np.arange(off[-1]))
    got = lg.cpu().numpy()
    for s in range(3):
        for d, node in enumerate(path[s]):
            assert rel_err(got[off[s] + node][None], logits[d][s][None]) < 2e-3, (s, d)
    # the drafted tokens' log probabilities under their parents, and greedy
    for s in range(3):
        rows = lg[off[s]:off[s + 1]].contiguous()
        up = torch.from_numpy(trees[s][1:].astype(np.int64)).cuda()
        out = runtime.log_probs(rows[up].contiguous(), np.array(toks[s][1:], np.int32)[:, None], top=1)
        x = got[off[s]:off[s + 1]].astype(np.float64)[trees[s][1:]]
        ref = x - x.max(1, keepdims=True)
        ref -= np.log(np.exp(ref).sum(1, keepdims=True))
        want = ref[np.arange(n[s] - 1), toks[s][1:]]
        assert np.abs(out["lp"].cpu().numpy()[:, 0] - want).max() < 2e-5
        assert np.array_equal(out["top_ids"].cpu().numpy()[:, 0], x.argmax(1))
        keep, at = [0], 0
        while True:  # down the tree by greedy tokens
            kids = [j for j in range(1, n[s]) if trees[s][j] == at and toks[s][j] == int(got[off[s] + at].argmax())]
            if not kids:
                break
            at = kids[0]
            keep.append(at)
        assert keep == path[s]
        p0 = b.past[s]
        b.m.move_cells(b.cells(s, [p0 + j for j in keep]), b.cells(s, range(p0, p0 + len(keep))))
        b.past[s] += len(keep)
    # the next step goes on from the kept cells
    lg = b.run([0, 2], [[line[0][6]], [line[2][6]]])[0].cpu().numpy()
    want = a.run([0, 2], [[line[0][6]], [line[2][6]]])[0].cpu().numpy()
    assert b.past[0] == a.past[0] and rel_err(lg, want) < 2e-3


def test_tree_plans_and_move_cells_are_refused():
    from lgml_amd import hip, runtime
    hp, w = models.build("c1", seed=1)
    m = runtime.DeviceModel(hp, w, 256)
    tab = np.array([[0, 1]], np.int32)
    with pytest.raises(hip.LgmlhError):
        m.plan([3], [0], tab, [1, 2, 3], parents=[-1, 1, 0])
    with pytest.raises(ValueError):
        m.plan([3], [0], tab, [1, 2, 3], parents=[-1, 0])
    with pytest.raises(ValueError):
        m.move_cells([1, 2], [3])
    with pytest.raises(hip.LgmlhError):
        m.move_cells([1, 2], [3, 3])
    with pytest.raises(hip.LgmlhError):
        m.move_cells([1], [256])
    m.move_cells([], [])
    with pytest.raises(ValueError):
        runtime.DeviceModel(hp, w, 256, kv_type=hip.F32)
    g, wg = models.build(GEMMA_TINY, seed=91, init="normal")
    gm = runtime.DeviceModel(g, wg, 256, ring_cells=64 * R)
    with pytest.raises(ValueError):
        gm.plan([1], [0], tab, [1], ring_tab=np.arange(R, dtype=np.int32)[None], parents=[-1])


# ---- the engine over Q8_0 pools --------------------------------------------------------
def test_q8_engine_shares_spills_and_grows_like_a_fresh_run():
    """Shared prefixes (a partial block copied), evicted blocks spilled to RAM and
    back, a pool that grows: bit for bit the logits of a run without."""
    from lgml_amd import engine, hip, runtime
    hp, w = models.build("c1", seed=7)
    V = hp["n_vocab"]
    a, b = lcg_ints(7000, 460, 0, V), lcg_ints(7001, 470, 0, V)
    c, a2 = a[:100] + lcg_ints(7003, 30, 0, V), a + lcg_ints(7002, 5, 0, V)

    def model(cells, **kw):
        return runtime.DeviceModel(hp, w, cells, kv_type=hip.Q8_0, **kw)

    def fresh(prompt, n):
        return chat(engine.Engine(model(2048), 2), prompt, n)[0]

    def same(x, y):
        return all(ta == tb and np.array_equal(la.view(np.uint32), lb.view(np.uint32))
                   for (ta, la), (tb, lb) in zip(x, y))

    gm = model(768)
    assert gm.kpools[0].numel() * 32 == 17 * hip.lib().lgmlh_kv_layer_bytes(768, hp["n_head_kv"], hp["head_dim"])
    eng = engine.Engine(gm, 2, prefix_cache=True, ram=4 * gm.block_bytes_all)
    chat(eng, a, 3)
    rows, fed = chat(eng, c, 4)  # one block attached, the best partial match copied
    assert fed == 100 and same(rows, fresh(c, 4))
    chat(eng, b, 3)
    assert eng.ram.stats["spilled"] >= 3, eng.ram.stats
    rows, fed = chat(eng, a2, 4)
    assert eng.ram.stats["unspilled"] >= 1 and same(rows, fresh(a2, 4))
    grown = model(2048, kv_initial=128)
    rows, _ = chat(engine.Engine(grown, 2), a, 4)
    assert grown.n_cells > 128 and same(rows, fresh(a, 4))


def test_q8_rings_resume_with_their_cells():
    from lgml_amd import engine, hip, runtime
    hp, w = models.build(GEMMA_TINY, seed=91, init="normal")
    prompts = [lcg_ints(50 + i, n, 0, hp["n_vocab"]) for i, n in enumerate([90, 150])]

    def run(preempt):
        gm = runtime.DeviceModel(hp, w, 1024, ring_cells=2 * R * 64, kv_type=hip.Q8_0)
        eng = engine.Engine(gm, 2, ubatch=UB, run_ahead=True)
        reqs = [engine.Request(p, 12) for p in prompts]
        for r in reqs:
            eng.submit(r)
        done = not preempt
        for _ in range(200):
            if all(r.done for r in reqs):
                break
            if not done and len(reqs[0].out) >= 4:
                reqs[0].preempt = done = True
            eng.step()
        drive(eng, reqs)
        return [r.out for r in reqs], reqs[0].waits

    plain, _ = run(False)
    again, waits = run(True)
    assert waits >= 1 and again == plain and all(len(o) == 12 for o in plain)


# ---- together: a captured and a side stream's run ---------------------------------------
class Step:
    """A verification step on raw operators: rows stored, a tree's attention, log
    probabilities of a projection of it, cells moved; all buffers its own."""

    H, KV, D, V = 8, 2, 128, 3000

    def __init__(self, seed):
        from lgml_amd import hip, runtime
        self.L, self.hip = hip.lib(), hip
        rng = np.random.default_rng(seed)
        n, past = 21, 150
        par = [-1] + [int(rng.integers(max(0, j - 4), j)) for j in range(1, n)]
        tab = rng.permutation(6)[:3].astype(np.int32)[None]
        self.plan = runtime.Plan([n], [past], tab, np.zeros(n, np.int32), self.H, self.KV, 6, 2, parents=par)
        self.cells = self.plan.cells.copy()
        self.d_cells = dev(self.cells)
        self.src, self.dst = self.cells[[0, 3, 7, 8]].copy(), self.cells[[0, 1, 2, 3]].copy()
        self.d_src, self.d_dst = dev(self.src), dev(self.dst)
        nb = self.L.lgmlh_kv_q8_layer_bytes(384, self.KV, self.D)
        g = torch.Generator("cuda").manual_seed(seed)
        self.pools = torch.zeros(2, nb, dtype=torch.uint8, device="cuda")
        self.addr = torch.tensor([p.data_ptr() for p in self.pools], dtype=torch.int64, device="cuda")
        old = np.arange(384, dtype=np.int64)
        rows = [torch.randn(384, self.KV * self.D, generator=g, device="cuda") for _ in range(2)]
        hip.check(self.L.lgmlh_kv_store_q8(self.pools[0].data_ptr(), self.pools[1].data_ptr(), 384, self.KV, self.D,
                                           rows[0].data_ptr(), rows[1].data_ptr(), dev(old).data_ptr(),
                                           old.ctypes.data, 384, st()))
        self.n = n
        self.k, self.v = (torch.empty(n, self.KV * self.D, device="cuda") for _ in range(2))
        self.q = torch.empty(n, self.H * self.D, device="cuda")
        self.out = torch.empty(n, self.H * self.D, device="cuda")
        self.wgt = torch.randn(self.H * self.D, self.V, generator=g, device="cuda")
        self.logits = torch.empty(n, self.V, device="cuda")
        self.ids = torch.randint(self.V, (n, 2), generator=g, device="cuda", dtype=torch.int32)
        self.lp, self.ent = torch.empty(n, 2, device="cuda"), torch.empty(n, device="cuda")
        self.top = torch.empty(n, 5, dtype=torch.int32, device="cuda")
        self.top_lp = torch.empty(n, 5, device="cuda")
        self.back = torch.empty(2, 4, self.KV * self.D, device="cuda")
        self.ws = torch.empty(max(self.L.lgmlh_attention_workspace(C.byref(self.plan.info), self.D), 16),
                              dtype=torch.uint8, device="cuda")
        self.ws2 = torch.empty(self.L.lgmlh_log_probs_workspace(n, self.V, 5), dtype=torch.uint8, device="cuda")

    def inputs(self, seed):
        g = torch.Generator("cuda").manual_seed(1000 + seed)
        for t in (self.k, self.v, self.q):
            t.copy_(torch.randn(t.shape, generator=g, device="cuda"))

    def run(self):
        L, check, n = self.L, self.hip.check, self.n
        check(L.lgmlh_kv_store_q8(self.pools[0].data_ptr(), self.pools[1].data_ptr(), 384, self.KV, self.D,
                                  self.k.data_ptr(), self.v.data_ptr(), self.d_cells.data_ptr(),
                                  self.cells.ctypes.data, n, st()))
        check(L.lgmlh_paged_attention_q8(self.q.data_ptr(), self.H, self.KV, self.D, 0.09, self.pools[0].data_ptr(),
                                         self.pools[1].data_ptr(), C.byref(self.plan.ub), self.out.data_ptr(),
                                         self.ws.data_ptr(), self.ws.numel(), st()))
        torch.mm(self.out, self.wgt, out=self.logits)
        check(L.lgmlh_log_probs(self.logits.data_ptr(), n, self.V, self.ids.data_ptr(), 2, self.lp.data_ptr(),
                                self.ent.data_ptr(), 5, self.top.data_ptr(), self.top_lp.data_ptr(),
                                self.ws2.data_ptr(), self.ws2.numel(), st()))
        check(L.lgmlh_kv_move(self.hip.Q8_0, self.addr.data_ptr(), 2, 384, self.KV, self.D, self.d_src.data_ptr(),
                              self.d_dst.data_ptr(), self.src.ctypes.data, self.dst.ctypes.data, 4, st()))
        for w in range(2):
            check(L.lgmlh_kv_gather_q8(self.pools[w].data_ptr(), w, 384, self.KV, self.D, self.d_dst.data_ptr(), 4,
                                       self.back[w].data_ptr(), self.hip.F32, st()))

    def results(self):
        return [t.clone() for t in (self.out, self.lp, self.ent, self.top, self.top_lp, self.back, self.pools)]


def test_a_captured_step_replays_the_eager_one():
    eager, cap = Step(5), Step(5)
    cap.inputs(0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        cap.run()  # (torch.mm's own first use)
    torch.cuda.current_stream().wait_stream(s)
    eager.inputs(0)
    eager.run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cap.run()
    for i in range(1, 5):
        cap.inputs(i)
        eager.inputs(i)
        graph.replay()
        eager.run()
        torch.cuda.synchronize()
        for x, y in zip(cap.results(), eager.results()):
            assert torch.equal(x, y), i


def test_two_steps_on_two_streams_at_once():
    one, two, ref1, ref2 = Step(6), Step(7), Step(6), Step(7)
    for step, ref, seed in ((one, ref1, 3), (two, ref2, 4)):
        step.inputs(seed)
        ref.inputs(seed)
        ref.run()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        for step, s in ((one, streams[0]), (two, streams[1])):
            with torch.cuda.stream(s):
                step.run()
    torch.cuda.synchronize()
    # (a step's moved cells are stored anew by the next, so runs repeat)
    for step, ref in ((one, ref1), (two, ref2)):
        for x, y in zip(step.results(), ref.results()):
            assert torch.equal(x, y)


def test_log_probs_of_no_rows_and_of_host_rows():
    from lgml_amd import runtime
    none = runtime.log_probs(torch.empty((0, 100), device="cuda"), torch.empty((0, 2)), 4)
    assert none["lp"].shape == (0, 2) and none["top_ids"].shape == (0, 4)
    for bad in (torch.zeros(2, 8), torch.zeros(8, 2, device="cuda").t(), torch.zeros(2, 8, device="cuda").half()):
        with pytest.raises(ValueError):
            runtime.log_probs(bad, None, 1)
