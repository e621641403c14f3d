"""Calls around drafted tokens and the Q8_0 pool at their edges, on the GPU:
products that end on a half of a step, moves and copies of cells behind a busy
stream, ids that no row holds, models without cells, rows that attend to a cell
much quieter than the others, lines of drafted tokens at every head size."""
import numpy as np
import pytest

from tests.test_gpu_draft import Pass, check_attention, dev, fill, k_tile, quants, run_attention, st, v_tile

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def L():
    from lgml_amd import hip
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    return hip.lib()


# ---- the rounding of the Q8_0 stores -----------------------------------------------
def half_block(rng):
    """32 f32 values of a block whose products with 1 / d end on k + 1/2 in f32, most
    of them with an exact product below it; the block's largest is the first."""
    a = np.float32(rng.uniform(0.3, 4.0))
    inv = np.float32(1) / (a / np.float32(127))
    y = (np.arange(126) + 0.5).astype(np.float32)
    x = (y / inv).astype(np.float32)
    near = np.stack([np.nextafter(x, np.float32(0)), x, np.nextafter(x, np.float32(9))])
    exact = near.astype(np.float64) * np.float64(inv)  # 48 bits at most
    tie = (near * inv).astype(np.float32) == y
    below, any_ = near[tie & (exact < y)], near[tie]
    take = rng.permutation(below)[:27]
    take = np.concatenate([take, rng.permutation(any_)[:31 - len(take)]])
    take = np.concatenate([take, np.full(31 - len(take), y[0] / inv, np.float32)])
    block = np.concatenate([[a], take * rng.choice([-1, 1], 31)]).astype(np.float32)
    return block


def halves(n, kv, D, seed):
    """Rows (n, kv, D) of such blocks; in every fourth d is 1 and the values are
    k + 1/2 and the numbers next to it."""
    rng = np.random.default_rng(seed)
    out = np.zeros((n * kv * D // 32, 32), np.float32)
    for i in range(len(out)):
        if i % 4:
            out[i] = half_block(rng)
        else:
            h = (rng.integers(0, 127, 31) + 0.5).astype(np.float32) * rng.choice([-1, 1], 31).astype(np.float32)
            to = rng.choice([-1000, 0, 1000], 31).astype(np.float32)
            h = np.where(to == 0, h, np.nextafter(h, to)).astype(np.float32)
            out[i] = np.concatenate([[127], h])
    out[0, 1:3] = 13.5, -13.5
    # a block of largest 0x1.62fe6p+1 takes -0x1.2de266p-2 to -13.5
    out[1, 0], out[1, 1] = float.fromhex("0x1.62fe6p+1"), float.fromhex("-0x1.2de266p-2")
    out[1, 2:] = 0
    rows = out.reshape(n, kv, D)
    g = rows.reshape(-1, 32)
    inv = np.float32(1) / (np.abs(g).max(1) / np.float32(127))
    y = np.abs((g * inv[:, None]).astype(np.float32))
    on_half = y % 1 == 0.5
    low = on_half & (np.abs(g.astype(np.float64) * inv[:, None].astype(np.float64)) < y)
    assert on_half.mean() > 0.4 and low.mean() > 0.1, (on_half.mean(), low.mean())
    return rows


def tiles_of(x, cells, blocks, D, make):
    """The pool bytes (blocks, kv, 68 D) of rows x in cells, zeros elsewhere."""
    q, d = quants(x)
    kv = x.shape[1]
    out = np.zeros((blocks, kv, 68 * D), np.uint8)
    for b in range(blocks):
        for h in range(kv):
            tq, td = np.zeros((64, D), np.int8), np.zeros((64, D // 32), np.float16)
            for j in np.flatnonzero(cells // 64 == b):
                tq[cells[j] % 64], td[cells[j] % 64] = q[j, h], d[j, h]
            out[b, h] = make(tq, td, D)
    return out


@pytest.mark.parametrize("D,kv", [(64, 2), (128, 1), (256, 2)])
def test_stores_round_the_f32_product(L, D, kv):
    """q is the f32 product x (1 / d) rounded with halves away from zero, in the plain
    store and in the fused one (at position 0, where the rope keeps K's rows)."""
    from lgml_amd import hip
    n, blocks, H = 40, 2, kv
    k, v = halves(n, kv, D, D), halves(n, kv, D, D + 1)
    cells = np.arange(70, 70 + n, dtype=np.int64)
    want = [tiles_of(k, cells, blocks, D, k_tile), tiles_of(v, cells, blocks, D, v_tile)]
    dc, kd, vd = dev(cells), dev(k), dev(v)
    pools = [torch.zeros(want[0].size, dtype=torch.uint8, device="cuda") for _ in range(4)]
    hip.check(L.lgmlh_kv_store_q8(pools[0].data_ptr(), pools[1].data_ptr(), 64 * blocks, kv, D, kd.data_ptr(),
                                  vd.data_ptr(), dc.data_ptr(), cells.ctypes.data, n, st()))
    qkv = dev(np.concatenate([k, k, v], 1).reshape(n, -1))
    pos = torch.zeros(n, dtype=torch.int32, device="cuda")
    q = torch.empty(n, H * D, device="cuda")
    hip.check(L.lgmlh_qkv_rope_store_q8(qkv.data_ptr(), n, H, kv, D, D, 0, 1e4, None, None, None, 1e-5,
                                        pos.data_ptr(), pools[2].data_ptr(), pools[3].data_ptr(), 64 * blocks,
                                        dc.data_ptr(), q.data_ptr(), st()))
    assert torch.equal(q.view(n, kv, D), kd)
    for i, p in enumerate(pools):
        got = p.cpu().numpy().reshape(want[0].shape)
        assert np.array_equal(got, want[i % 2]), (i, int((got != want[i % 2]).sum()))


# ---- moves of cells wait for nothing --------------------------------------------------
@pytest.mark.parametrize("kind", ["F16", "Q8_0"])
def test_moves_are_queued_behind_a_busy_stream(kind):
    """move_cells, and the engine's copy of a partial block, return while earlier
    work of the stream still runs, as lgmlh_kv_copy_block does, and move the cells
    that they were given then."""
    from lgml_amd import engine, hip, runtime
    from oracle import models
    hp, w = models.build("c1", seed=7)
    m = runtime.DeviceModel(hp, w, 1024, kv_type=getattr(hip, kind))
    seqs = engine.PoolSeqs(m)
    rng = np.random.default_rng(2)
    for pool in m.kpools + m.vpools:
        pool.copy_(dev(rng.integers(0, 60, pool.numel()).astype(np.uint8)))
    before = [m.gather_kv(1, np.arange(1024), which) for which in (0, 1)]
    seqs.copy_block(9, 10, 5)
    m.move_cells([900], [901])  # first uses
    a = torch.randn(8192, 8192, device="cuda")
    torch.mm(a, a)
    torch.cuda.synchronize()
    for _ in range(20):  # some 100 ms
        torch.mm(a, a)
    done = torch.cuda.Event()
    done.record()
    src, dst = np.array([70, 71, 3]), np.array([64, 65, 66])
    m.move_cells(src, dst)
    src[:], dst[:] = 0, 0
    seqs.copy_block(2, 5, 17)
    early = not done.query()
    for i in range(40):  # (their host memory is not used again too early)
        m.move_cells([200 + i], [300 + i])
    torch.cuda.synchronize()
    assert early
    frm = np.arange(1024)
    frm[64 * 10:64 * 10 + 5] = 64 * 9 + np.arange(5)
    frm[901] = 900
    frm[[64, 65, 66]] = [70, 71, 3]
    frm[64 * 5:64 * 5 + 17] = 64 * 2 + np.arange(17)
    frm[300:340] = np.arange(200, 240)
    for which in (0, 1):
        assert np.array_equal(m.gather_kv(1, np.arange(1024), which), before[which][frm])


def test_move_cells_of_a_captured_stream_is_refused():
    from lgml_amd import runtime
    from oracle import models
    hp, w = models.build("c1", seed=7)
    m = runtime.DeviceModel(hp, w, 256)
    x = torch.zeros(8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x += 1
        with pytest.raises(RuntimeError, match="lgmlh_kv_move"):
            m.move_cells([1], [2])
    graph.replay()
    torch.cuda.synchronize()
    assert bool((x == 1).all())


# ---- given ids of any integer type -----------------------------------------------------
def test_log_probs_of_ids_that_no_row_holds():
    """-inf for an id outside the row, of any width: none is taken for another."""
    from lgml_amd import runtime
    x = torch.randn(2, 300, generator=torch.Generator("cuda").manual_seed(3), device="cuda")
    ids = np.array([[7, 2**32 + 7, -1, 300], [2**33 + 5, -2**32 + 9, 5, 2**31 + 5]], np.int64)
    want = torch.log_softmax(x.double().cpu(), 1).numpy()
    for given in (ids, ids.tolist(), torch.from_numpy(ids), torch.from_numpy(ids).cuda()):
        lp = runtime.log_probs(x, given)["lp"].cpu().numpy()
        assert abs(lp[0, 0] - want[0, 7]) < 1e-5 and abs(lp[1, 2] - want[1, 5]) < 1e-5
        assert np.isneginf(lp).tolist() == [[False, True, True, True], [True, True, False, True]]
    small = runtime.log_probs(x, torch.tensor([[255], [5]], dtype=torch.uint8))["lp"].cpu().numpy()
    assert abs(small[0, 0] - want[0, 255]) < 1e-5 and abs(small[1, 0] - want[1, 5]) < 1e-5
    x = x[:, :200].contiguous()
    small = runtime.log_probs(x, torch.tensor([[255], [5]], dtype=torch.uint8))["lp"].cpu().numpy()
    assert np.isneginf(small).tolist() == [[True], [False]]


# ---- models -----------------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["F16", "Q8_0"])
def test_a_model_without_cells_is_built(kind):
    """And refuses tokens, not the heads of its pool."""
    from lgml_amd import hip, runtime
    from oracle import models
    hp, w = models.build("c1", seed=7)
    m = runtime.DeviceModel(hp, w, 0, kv_type=getattr(hip, kind))
    with pytest.raises(hip.LgmlhError):
        m.plan([1], [0], np.zeros((1, 1), np.int32), [1])


def test_q8_pools_of_other_heads_are_refused():
    from lgml_amd import hip, runtime
    from oracle import models
    hp, w = models.build("c1", seed=7)
    hp = dict(hp, head_dim=hp["head_dim"] // 2, n_head=2 * hp["n_head"], n_head_kv=2 * hp["n_head_kv"],
              n_rot=hp["head_dim"] // 2)
    runtime.DeviceModel(hp, w, 128)
    with pytest.raises(ValueError, match="heads of 64, 128 or 256, not %d" % hp["head_dim"]):
        runtime.DeviceModel(hp, w, 128, kv_type=hip.Q8_0)


def test_a_gguf_model_takes_a_q8_cache(tmp_path):
    from lgml_amd import hip, runtime
    from tests.gpu_util import lcg_ints
    from tests.test_gpu_gguf import c2_like_gguf
    path = str(tmp_path / "m.gguf")
    hp, w = c2_like_gguf(path)
    a = runtime.DeviceModel(hp, w, 256, kv_type=hip.Q8_0)
    b = runtime.load_gguf(path, 256, kv_type=hip.Q8_0)
    assert b.kpools[0].numel() == a.kpools[0].numel()
    ids, bt = np.array(lcg_ints(11, 37, 0, hp["n_vocab"]), np.int32), np.array([[0, 1]], np.int32)
    la, lb = (m.forward(m.plan([37], [0], bt, ids)).cpu().numpy() for m in (a, b))
    assert np.array_equal(la.view(np.uint32), lb.view(np.uint32))


# ---- parents of any integer type ---------------------------------------------------------
@pytest.mark.parametrize("bad", [[-1, 2**32, 0], [-1, -2**32, 0], [-1.0, 0.5, 0.0]])
def test_parents_past_32_bits_are_no_parents(bad):
    from lgml_amd import runtime
    tab, ids = np.array([[0, 1]], np.int32), np.zeros(3, np.int32)
    for good in ([-1, 0, 0], np.array([-1, 0, 0], np.int64), np.array([[-1, 0, 0]])):
        assert list(runtime.Plan([3], [10], tab, ids, 4, 2, 2, parents=good).parents) == [-1, 0, 0]
    with pytest.raises(ValueError):
        runtime.Plan([3], [10], tab, ids, 4, 2, 2, parents=np.array(bad))


# ---- rows whose weight is on quiet cells -----------------------------------------------
def bounds(q, k, v, scale):
    """(the output (H, D) in 64 bits, how far it may be off (H, D)): q (H, D), k and v
    (cells, kv, D) f64. A score is off by ds, as in the tests of attention; that
    turns p_i v_i by p_i |v_i - o| ds, and 2^-21 and the sum's n / 16 + 64 roundings
    come on sum p |v|; twice that for the terms of higher order. The f16 halves of
    P dv hold 22 bits (within the 2^-21) down to a place that is fixed, half of
    whose step each cell may be off: 2^-39 of the largest p dv of the cell's block,
    which is no more than the largest of the row, whose 127 steps are in the 32
    dims; or, where scales go by the packed products, 2^-42 times a value of up to
    127. Signs of n cells' roundings are as good as independent: 7.5 sqrt(n) of the
    latter (Hoeffding's bound for 1e-6 in all the values of these tests)."""
    (H, D), (n, kv, _) = q.shape, k.shape
    g = H // kv
    qs, ks, vs = q.reshape(kv, g, D), k.transpose(1, 2, 0), v.transpose(1, 0, 2)
    x = np.matmul(qs, ks) * scale
    ds = np.matmul(np.abs(qs), np.abs(ks)).max() * scale * ((D + 40) * 2.0**-24 + 2.0**-21)
    p = np.exp(x - x.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    o = np.matmul(p, vs)
    turn = np.stack([np.einsum("gc,gcd->gd", p[h], np.abs(vs[h][None] - o[h][:, None])) for h in range(kv)])
    size = np.matmul(p, np.abs(vs))
    big = size.reshape(kv, g, D // 32, 32).max(-1, keepdims=True)
    off = turn * ds + size * (2.0**-21 + (n / 16 + 64) * 2.0**-24)
    off = 2 * off.reshape(kv, g, D // 32, 32) + big * n * 2.0**-39 + 127 * 2.0**-42 * 7.5 * n ** 0.5
    return o.reshape(H, D), off.reshape(H, D)


@pytest.mark.parametrize("loud", [0.2, 1, 30, 600])
@pytest.mark.parametrize("quiet", [1e-2, 1e-4, 1e-5])
@pytest.mark.parametrize("H,kv,D", [(8, 2, 64), (8, 2, 128), (8, 4, 256)])
@pytest.mark.parametrize("n,past", [(1, 500), (40, 201)])
def test_q8_attention_keeps_the_bits_of_quiet_cells(L, loud, quiet, H, kv, D, n, past):
    """All but e^-12 to e^-20 of a row's weight on one cell whose V is far below the
    others': the row has the bits of that V, whatever the scales beside it."""
    rng = np.random.default_rng(int(loud) + D)
    P = Pass([n], [past], H, kv, None, 8, 3)
    k, v = (rng.standard_normal((P.n_cells, kv, D)).astype(np.float32) for _ in range(2))
    q = rng.standard_normal((n, H, D)).astype(np.float32)
    c = P.cells(0)
    way = rng.standard_normal((kv, D)).astype(np.float32)
    v *= np.float32(loud)
    k[c[3]], v[c[3]] = 2 * way, v[c[3]] * np.float32(quiet / loud)
    ahead = rng.choice([12, 20], (n, H, 1))
    w = np.repeat(2 * way, H // kv, 0)
    q = (q + ahead * w * (D ** 0.5 / (w * w).sum(1, keepdims=True))).astype(np.float32)
    pools, kx, vx = fill(L, P, kv, D, k, v, True)
    got = run_attention(L, P, H, kv, D, D ** -0.5, q, pools, True)
    for j in range(n):
        vis = c[:past + j + 1]
        want, tol = bounds(q[j].astype(np.float64), kx[vis], vx[vis], D ** -0.5)
        err = np.abs(got[j] - want)
        assert (err <= tol).all(), (j, (err / tol).max())


# ---- a line of drafted tokens --------------------------------------------------------
LINES = {
    "few": ([9, 64, 1], [100, 3, 64]),            # sets of a few query groups
    "many": ([300, 128, 257], [70, 640, 0]),      # sets of eight
    "edges": ([1, 2, 63, 65], [63, 62, 1, 191]),  # blocks that end with a token
}


@pytest.mark.parametrize("case", list(LINES))
@pytest.mark.parametrize("q8,H,kv,D", [(False, 4, 2, 16), (False, 4, 2, 32), (False, 8, 2, 64), (False, 32, 8, 128),
                                       (False, 8, 4, 256), (True, 8, 2, 64), (True, 32, 8, 128), (True, 8, 4, 256)])
@pytest.mark.parametrize("bps", [0, 2])
def test_a_line_of_tokens_is_the_causal_plan_at_every_head_size(L, case, q8, H, kv, D, bps):
    seq_n, npast = LINES[case]
    line = [[j - 1 for j in range(n)] for n in seq_n]
    a = check_attention(L, q8, H, kv, D, seq_n, npast, line, bps, 23)
    b = check_attention(L, q8, H, kv, D, seq_n, npast, None, bps, 23)
    assert np.array_equal(a, b), np.argwhere(a != b)[:4]
