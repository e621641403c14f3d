"""Whole passes and the engine over Q4_0 pools: the fused store, trees of drafted tokens
verified in one pass, sharing, spilling, growing and rings; the operators of a long
context together (rows turned by several axes and stored, a fork's copies, attention, the
read back), eager, captured and replayed, and on two streams at once."""
import ctypes as C

import numpy as np
import pytest

from oracle import models
from tests.gpu_util import lcg_ints, rel_err
from tests.test_gpu_draft import dev, st
from tests.test_gpu_draft_model import Decoder
from tests.test_gpu_sched import GEMMA_TINY, R, UB, drive
from tests.test_gpu_spill import chat

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("H,kv,D,neox", [(4, 2, 64, 0), (8, 8, 128, 1), (8, 4, 256, 1)])
def test_qkv_rope_store_q4_stores_the_roped_rows(H, kv, D, neox):
    """Its pool bytes are lgmlh_kv_store_q4's of the same rows: K roped (read back as
    the q heads of a call with K in their place), V as given; a cell outside the pool
    is not written."""
    from lgml_amd import hip
    L = hip.lib()
    rng = np.random.default_rng(D)
    n, cells_n = 37, 256
    qkv = rng.standard_normal((n, (H + 2 * kv) * D)).astype(np.float32)
    qkv[3, H * D:] = 0
    qkv[4, (H + kv) * D:(H + kv) * D + 32] = np.float32(2.5) * (-1) ** np.arange(32)  # ties: the first
    pos = dev(rng.integers(0, 5000, n).astype(np.int32))
    cells = np.concatenate([np.arange(60, 96), [cells_n]]).astype(np.int64)
    qn, kn = (dev(1 + 0.1 * rng.standard_normal(D).astype(np.float32)) for _ in range(2))
    nb = L.lgmlh_kv_q4_layer_bytes(cells_n, kv, D)

    def pools():
        return [torch.full((nb,), 0x5A, dtype=torch.uint8, device="cuda") for _ in range(2)]

    got = pools()
    q = torch.empty(n, H * D, device="cuda")
    args = (D, neox, 1e4, None, qn.data_ptr(), kn.data_ptr(), 1e-5, pos.data_ptr())
    dq, dc = dev(qkv), dev(cells)
    hip.check(L.lgmlh_qkv_rope_store_q4(dq.data_ptr(), n, H, kv, D, *args, got[0].data_ptr(),
                                        got[1].data_ptr(), cells_n, dc.data_ptr(), q.data_ptr(), st()))
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
    hip.check(L.lgmlh_kv_store_q4(want[0].data_ptr(), want[1].data_ptr(), cells_n, kv, D, roped.data_ptr(),
                                  v.data_ptr(), dc.data_ptr(), cells.ctypes.data, n - 1, st()))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_a_pass_attends_to_what_its_pools_hold():
    """A one-layer pass over a Q4_0 cache against 64 bits: the cells hold its K and V rows
    within a step of their scale, and the logits are those of attention over what they
    hold (within 2e-3, the bar of whole passes here)."""
    from lgml_amd import hip, runtime
    hp, w = models.build("c1", seed=21, n_layer=1, init="normal")
    L, V, H, kv, D = hip.lib(), hp["n_vocab"], hp["n_head"], hp["n_head_kv"], hp["head_dim"]
    n = 130
    m = runtime.DeviceModel(hp, w, 512, kv_type=hip.Q4_0)
    ids, tab = np.array(lcg_ints(5, n, 0, V), np.int32), np.array([[3, 0, 6]], np.int32)
    plan = m.plan([n], [0], tab, ids)
    got = m.forward(plan, np.arange(n)).cpu().numpy()
    dc = dev(plan.cells.copy())
    held = []
    for which, pool in enumerate((m.kpools[0], m.vpools[0])):
        out = torch.empty(n, kv, D, device="cuda")
        hip.check(L.lgmlh_kv_gather_q4(pool.data_ptr(), which, 512, kv, D, dc.data_ptr(), n, out.data_ptr(), hip.F32,
                                       st()))
        held.append(out.cpu().numpy().astype(np.float64))

    ly = w["layers"][0]
    mat = lambda name: np.asarray(ly[name][0], np.float64)
    norm = lambda x, g: x / np.sqrt((x * x).mean(-1, keepdims=True) + hp["eps"]) * np.asarray(g, np.float64)
    x = np.asarray(w["tok_embd"][0], np.float64)[ids]
    h = norm(x, ly["attn_norm"][0])
    q, k, v = ((h @ mat(name).T).reshape(n, -1, D) for name in ("wq", "wk", "wv"))
    theta = np.arange(n)[:, None] * hp["rope_base"] ** (-2.0 * np.arange(D // 2) / D)
    c, s_ = np.cos(theta)[:, None], np.sin(theta)[:, None]

    def turn(y):
        one, two = (slice(0, D // 2), slice(D // 2, D)) if hp["rope_neox"] else (slice(0, D, 2), slice(1, D, 2))
        out = y.copy()
        out[..., one], out[..., two] = y[..., one] * c - y[..., two] * s_, y[..., one] * s_ + y[..., two] * c
        return out

    q, k = turn(q), turn(k)
    for row, back in ((k, held[0]), (v, held[1])):
        step = np.abs(row.reshape(n, kv, D // 32, 32)).max(-1, keepdims=True) / 8
        # a value of the other sign than the largest may be 8 steps, kept as 7
        assert (np.abs(row - back).reshape(n, kv, D // 32, 32) <= step * 1.001 + 1e-7).all()
    o = np.empty((n, H, D))
    for t in range(n):
        sc = np.einsum("hd,chd->hc", q[t], held[0][:t + 1].repeat(H // kv, 1)) * D ** -0.5
        p = np.exp(sc - sc.max(1, keepdims=True))
        o[t] = np.einsum("hc,chd->hd", p / p.sum(1, keepdims=True), held[1][:t + 1].repeat(H // kv, 1))
    x = x + o.reshape(n, -1) @ mat("wo").T
    h = norm(x, ly["ffn_norm"][0])
    g = h @ mat("gate").T
    x = x + (g / (1 + np.exp(-g)) * (h @ mat("up").T)) @ mat("down").T
    want = norm(x, w["output_norm"][0]) @ np.asarray(w["output"][0], np.float64).T
    assert rel_err(got, want) < 2e-3


@pytest.mark.parametrize("shape,layers", [("c1", 2), ("c2", 2)])
def test_a_tree_is_verified_in_one_pass(shape, layers):
    """A drafted line and wrong branches behind it: bit for bit the logits of decoding the
    line token by token (its tokens take the same slots, and a row has its bits in any
    group of rows), and of the next step."""
    from lgml_amd import hip
    hp, w = models.build(shape, seed=21, n_layer=layers, init="normal")
    V = hp["n_vocab"]
    prompts = [lcg_ints(900 + i, n, 0, V) for i, n in enumerate([70, 17, 129])]
    a, b = Decoder(hp, w, hip.Q4_0), Decoder(hp, w, hip.Q4_0)
    la, lb = a.run([0, 1, 2], prompts)[0], b.run([0, 1, 2], prompts)[0]
    assert torch.equal(la, lb)  # a pass repeats its bits
    toks = [lcg_ints(40 + s, 4, 0, V) for s in range(3)]
    want = [a.run([0, 1, 2], [[t[d]] for t in toks])[0] for d in range(4)]
    drafted = [t + [(t[d] + 1 + i) % V for d in range(1, 4) for i in range(2)] for t in toks]
    trees = [np.array([-1, 0, 1, 2, 0, 0, 1, 1, 2, 2], np.int32)] * 3
    lg = b.run([0, 1, 2], drafted, trees, rows=np.arange(30))[0]
    for s in range(3):
        for d in range(4):
            assert torch.equal(lg[10 * s + d], want[d][s]), (s, d)
        b.past[s] += 4
    nxt = [[11 + s] for s in range(3)]
    assert torch.equal(b.run([0, 1, 2], nxt)[0], a.run([0, 1, 2], nxt)[0])


def test_the_engine_shares_spills_and_grows_like_a_fresh_run():
    """Shared prefixes (a partial block copied), evicted blocks spilled to RAM and
    back, a pool that grows: bit for bit the logits of a run without."""
    from lgml_amd import engine, hip, runtime
    hp, w = models.build("c1", seed=7)
    V = hp["n_vocab"]
    a, b = lcg_ints(7000, 460, 0, V), lcg_ints(7001, 470, 0, V)
    c, a2 = a[:100] + lcg_ints(7003, 30, 0, V), a + lcg_ints(7002, 5, 0, V)

    def model(cells, **kw):
        return runtime.DeviceModel(hp, w, cells, kv_type=hip.Q4_0, **kw)

    def fresh(prompt, n):
        return chat(engine.Engine(model(2048), 2), prompt, n)[0]

    def same(x, y):
        return all(ta == tb and np.array_equal(la.view(np.uint32), lb.view(np.uint32))
                   for (ta, la), (tb, lb) in zip(x, y))

    gm = model(768)
    assert gm.kpools[0].numel() * 32 == 9 * hip.lib().lgmlh_kv_layer_bytes(768, hp["n_head_kv"], hp["head_dim"])
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


def test_evicted_blocks_of_a_compacted_pool_come_back_from_ram():
    from lgml_amd import engine, hip, runtime
    hp, w = models.build("c1", seed=7)
    a = lcg_ints(7000, 300, 0, hp["n_vocab"])
    m = runtime.DeviceModel(hp, w, 1024, kv_type=hip.Q4_0, kv_initial=64)
    eng = engine.Engine(m, 2, prefix_cache=True, ram=8 * m.block_bytes_all)
    first, _ = chat(eng, a, 3)
    assert eng.compact(keep_cached=False) == 64 and eng.ram.stats["spilled"] >= 4
    rows, fed = chat(eng, a + [5], 3)
    assert fed >= 256 and eng.from_ram >= 4
    want, _ = chat(engine.Engine(runtime.DeviceModel(hp, w, 1024, kv_type=hip.Q4_0), 2), a + [5], 3)
    assert all(np.array_equal(x[1], y[1]) for x, y in zip(rows, want))


def test_rings_resume_with_their_cells():
    from lgml_amd import engine, hip, runtime
    hp, w = models.build(GEMMA_TINY, seed=91, init="normal")
    prompts = [lcg_ints(50 + i, n, 0, hp["n_vocab"]) for i, n in enumerate([90, 150])]

    def run(preempt):
        gm = runtime.DeviceModel(hp, w, 1024, ring_cells=2 * R * 64, kv_type=hip.Q4_0)
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


def test_models_take_and_refuse_a_q4_cache(tmp_path):
    from lgml_amd import hip, runtime
    from tests.test_gpu_gguf import c2_like_gguf
    path = str(tmp_path / "m.gguf")
    hp, w = c2_like_gguf(path)
    a = runtime.DeviceModel(hp, w, 256, kv_type=hip.Q4_0)
    b = runtime.load_gguf(path, 256, kv_type=hip.Q4_0)
    assert b.kpools[0].numel() == a.kpools[0].numel()
    ids, bt = np.array(lcg_ints(11, 37, 0, hp["n_vocab"]), np.int32), np.array([[0, 1]], np.int32)
    la, lb = (m.forward(m.plan([37], [0], bt, ids)).cpu().numpy() for m in (a, b))
    assert np.array_equal(la.view(np.uint32), lb.view(np.uint32))
    hp, w = models.build("c1", seed=7)
    runtime.DeviceModel(hp, w, 0, kv_type=hip.Q4_0)  # without cells
    hp = dict(hp, head_dim=hp["head_dim"] // 2, n_head=2 * hp["n_head"], n_head_kv=2 * hp["n_head_kv"],
              n_rot=hp["head_dim"] // 2)
    with pytest.raises(ValueError, match="a Q4_0 pool takes heads of 64, 128 or 256, not %d" % hp["head_dim"]):
        runtime.DeviceModel(hp, w, 128, kv_type=hip.Q4_0)


# ---- together: a captured and a side stream's run ---------------------------------------
class Step:
    """A pass of two forked sequences on raw operators: their partial block copied, rows
    turned by several axes and stored, attention, the cells read back; all buffers its
    own."""

    H, KV, D = 8, 2, 128

    def __init__(self, seed):
        from lgml_amd import hip, runtime
        self.L, self.hip = hip.lib(), hip
        rng = np.random.default_rng(seed)
        n, past = 21, 150
        self.blocks = 10
        order = rng.permutation(self.blocks).astype(np.int32)
        tab = np.array([[order[0], order[1], order[2]], [order[0], order[1], order[3]]], np.int32)
        self.plan = runtime.Plan([n, 1], [past, past], tab, np.zeros(n + 1, np.int32), self.H, self.KV, self.blocks, 2)
        self.cells = self.plan.cells.copy()
        self.d_cells = dev(self.cells)
        self.copies = np.array([[order[4], order[2], past % 64], [order[4], order[3], past % 64], [-1, order[5], 64]],
                               np.int32)
        self.d_copies = dev(self.copies)
        nb = self.L.lgmlh_kv_q4_layer_bytes(64 * self.blocks, self.KV, self.D)
        g = torch.Generator("cuda").manual_seed(seed)
        self.pools = torch.zeros(2, nb, dtype=torch.uint8, device="cuda")
        self.addr = torch.tensor([p.data_ptr() for p in self.pools], dtype=torch.int64, device="cuda")
        old = np.arange(64 * self.blocks, dtype=np.int64)
        rows = [torch.randn(len(old), self.KV * self.D, generator=g, device="cuda") for _ in range(2)]
        hip.check(self.L.lgmlh_kv_store_q4(self.pools[0].data_ptr(), self.pools[1].data_ptr(), len(old), self.KV,
                                           self.D, rows[0].data_ptr(), rows[1].data_ptr(), dev(old).data_ptr(),
                                           old.ctypes.data, len(old), st()))
        self.n = n + 1
        self.qkv = torch.empty(self.n, (self.H + 2 * self.KV) * self.D, device="cuda")
        self.pos = torch.empty(4, self.n, dtype=torch.int32, device="cuda")
        self.q = torch.empty(self.n, self.H * self.D, device="cuda")
        self.out = torch.empty(self.n, self.H * self.D, device="cuda")
        self.back = torch.empty(2, self.n, self.KV * self.D, device="cuda")
        self.sections = np.array([16, 24, 24, 0], np.int32)
        self.ws = torch.empty(max(self.L.lgmlh_attention_workspace(C.byref(self.plan.info), self.D), 16),
                              dtype=torch.uint8, device="cuda")

    def inputs(self, seed):
        g = torch.Generator("cuda").manual_seed(1000 + seed)
        self.qkv.copy_(torch.randn(self.qkv.shape, generator=g, device="cuda"))
        self.pos.copy_(torch.randint(4000, self.pos.shape, generator=g, device="cuda"))

    def run(self):
        L, check, cells = self.L, self.hip.check, 64 * self.blocks
        kp, vp = (p.data_ptr() for p in self.pools)
        check(L.lgmlh_kv_copy_blocks(self.hip.Q4_0, self.addr.data_ptr(), 2, cells, self.KV, self.D,
                                     self.d_copies.data_ptr(), self.copies.ctypes.data, 3, st()))
        check(L.lgmlh_qkv_rope_store_axes(self.hip.Q4_0, self.qkv.data_ptr(), self.n, self.H, self.KV, self.D, self.D,
                                          self.sections.ctypes.data, 0, 1e6, None, None, None, 1e-6,
                                          self.pos.data_ptr(), kp, vp, cells, self.d_cells.data_ptr(),
                                          self.q.data_ptr(), st()))
        check(L.lgmlh_paged_attention_q4(self.q.data_ptr(), self.H, self.KV, self.D, 0.09, kp, vp,
                                         C.byref(self.plan.ub), self.out.data_ptr(), self.ws.data_ptr(),
                                         self.ws.numel(), st()))
        for w in range(2):
            check(L.lgmlh_kv_gather_q4(self.pools[w].data_ptr(), w, cells, self.KV, self.D, self.d_cells.data_ptr(),
                                       self.n, self.back[w].data_ptr(), self.hip.F32, st()))

    def results(self):
        return [t.clone() for t in (self.q, self.out, self.back, self.pools)]


def test_a_captured_step_replays_the_eager_one():
    eager, cap = Step(5), Step(5)
    cap.inputs(0)
    torch.cuda.synchronize()
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
    for step, ref in ((one, ref1), (two, ref2)):
        for x, y in zip(step.results(), ref.results()):
            assert torch.equal(x, y)
