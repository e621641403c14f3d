"""The forms that long calls take, on the GPU: windows of 64 tokens (32 of heads of 256)
in rope by several axes and in the read back of a Q4_0 pool, and passes over Q4_0 pools
whose attention splits and merges into the output product's operands."""
import numpy as np
import pytest

from oracle import core, models
from tests.gpu_util import lcg_ints, rel_err
from tests.test_gpu_draft import dev, st
from tests.test_gpu_q4 import L, test_gather_reads_what_was_stored as gather_reads  # noqa: F401
from tests.test_gpu_rope_axes import axis_of, run, turned

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def long_call(rng, n, kv, D):
    """n tokens and their cells: a run from an odd offset with a cell outside the pool in
    it, cells in any order, runs that end inside a group, a last window in part."""
    big = 32 if D > 128 else 64
    assert (n + big - 1) // big * kv >= 256  # windows of `big` tokens
    blocks = n // 64 + 6
    order = np.concatenate([np.arange(13, 13 + n // 2), rng.permutation(np.arange(13 + n // 2, 13 + n // 2 + 203)),
                            np.arange(13 + n // 2 + 203 + 5, 64 * blocks)])
    cells = order[:n].astype(np.int64)
    cells[[big + 7, n // 3, n - 2]] = [64 * blocks, -1, 1 << 40]
    return blocks, cells


WIDE = [(64, 4, 8, 2100, 64, (8, 12, 12, 0), 0), (128, 8, 8, 2090, 128, (24, 20, 20, 0), 1),
        (256, 2, 8, 1050, 192, (20, 30, 30, 16), 0), (256, 4, 4, 2077, 256, (64, 32, 32, 0), 1)]


@pytest.mark.parametrize("D,H,kv,n,rot,sections,inter", WIDE)
def test_wide_windows_of_turned_rows(D, H, kv, n, rot, sections, inter):
    """Every value of the f16 pools and of q, as in the short calls' test."""
    from lgml_amd import hip
    rng = np.random.default_rng(D + n)
    blocks, cells = long_call(rng, n, kv, D)
    x = (rng.standard_normal((n, H + 2 * kv, D)) * 3).astype(np.float32)
    pos = rng.integers(0, 5000, (4, n))
    kn = (1 + 0.3 * rng.standard_normal(D)).astype(np.float32)
    axes = axis_of(rot, sections, inter)
    wq, tq = turned(x[:, :H], rot, axes, pos, 1e4, None, None, 1e-6)
    wk, tk = turned(x[:, H:H + kv], rot, axes, pos, 1e4, None, kn, 1e-6)
    start = rng.integers(0, 2**16, (2, blocks, kv, 64 * D)).astype(np.uint16)
    pools = [dev(start[w].view(np.int16)) for w in range(2)]
    got = run(hip.F16, x, H, kv, D, rot, sections, inter, 1e4, None, None, kn, 1e-6, pos, pools, 64 * blocks, cells)
    assert (np.abs(got.cpu().numpy().astype(np.float64) - wq) <= tq).all()
    ok = (cells >= 0) & (cells < 64 * blocks)
    kp = pools[0].cpu().numpy().view(np.uint16).reshape(blocks, kv, 64, D)
    vp = pools[1].cpu().numpy().view(np.uint16).reshape(blocks, kv, D, 64)
    k = kp[cells[ok] // 64, :, cells[ok] % 64].view(np.float16).astype(np.float64)
    # the f16 of a value off by tk: half a step of it more (of 2^-24 near zero)
    assert (np.abs(k - wk[ok]) <= tk[ok] + (np.abs(wk[ok]) + tk[ok]) * 2.0**-11 + 2.0**-25).all()
    want = start[1].reshape(vp.shape).copy()
    want[cells[ok] // 64, :, :, cells[ok] % 64] = x[ok, H + kv:].astype(np.float16).view(np.uint16)
    assert np.array_equal(vp, want), np.argwhere(vp != want)[:4]
    rest = np.ones(64 * blocks, bool)
    rest[cells[ok]] = False
    rest = rest.reshape(blocks, 64)
    assert np.array_equal(kp.transpose(0, 2, 1, 3)[rest], start[0].reshape(kp.shape).transpose(0, 2, 1, 3)[rest])


@pytest.mark.parametrize("kind", ["Q8_0", "Q4_0"])
@pytest.mark.parametrize("D,H,kv,n,rot,sections,inter", WIDE)
def test_wide_windows_into_quantised_pools(L, kind, D, H, kv, n, rot, sections, inter):  # noqa: F811
    """The pools' bytes are those of storing the turned rows."""
    from lgml_amd import hip
    ty = getattr(hip, kind)
    rng = np.random.default_rng(D + n)
    blocks, cells = long_call(rng, n, kv, D)
    ok = (cells >= 0) & (cells < 64 * blocks)
    x = rng.standard_normal((n, H + 2 * kv, D)).astype(np.float32)
    pos = rng.integers(0, 3000, (4, n))
    kn = (1 + 0.1 * rng.standard_normal(D)).astype(np.float32)
    nb = (L.lgmlh_kv_q8_layer_bytes if kind == "Q8_0" else L.lgmlh_kv_q4_layer_bytes)(64 * blocks, kv, D)

    def pools():
        return [torch.full((nb,), 0x5A, dtype=torch.uint8, device="cuda") for _ in range(2)]

    got, other, want = pools(), pools(), pools()
    run(ty, x, H, kv, D, rot, sections, inter, 1e4, None, kn, kn, 1e-6, pos, got, 64 * blocks, cells)
    as_q = np.concatenate([x[:, H:H + kv], x[:, H:]], 1)
    k = run(ty, as_q, kv, kv, D, rot, sections, inter, 1e4, None, kn, kn, 1e-6, pos, other, 64 * blocks, cells)
    keep = torch.from_numpy(np.flatnonzero(ok)).cuda()
    k, v, c = k.index_select(0, keep).contiguous(), dev(x[ok, H + kv:].copy()), cells[ok].copy()
    dc = dev(c)
    fn = L.lgmlh_kv_store_q8 if kind == "Q8_0" else L.lgmlh_kv_store_q4
    hip.check(fn(want[0].data_ptr(), want[1].data_ptr(), 64 * blocks, kv, D, k.data_ptr(), v.data_ptr(), dc.data_ptr(),
                 c.ctypes.data, len(c), st()))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("D,kv,n", [(64, 8, 2100), (256, 8, 1050)])
@pytest.mark.parametrize("f16", [False, True])
def test_wide_windows_of_the_read_back(L, D, kv, n, f16):  # noqa: F811
    gather_reads(L, D, kv, n, f16)


@pytest.mark.parametrize("wtype", ["q4_K", "q8_0"])
@pytest.mark.parametrize("ggml", [False, True])
@pytest.mark.parametrize("D,H,kv", [(64, 8, 2), (128, 4, 1), (256, 2, 1)])
def test_passes_whose_attention_splits(wtype, ggml, D, H, kv):
    """One layer over the same pools with runs of one block (groups of 3, 10 and 30 splits,
    of one row and of many) and with one run for each context. The attention's outputs
    differ by its roundings, some 2^-20 of V's largest; averages over up to 1900 cells are
    1/20 of it, which makes 2e-5 of them, and 5e-4 is the bar. In ggml's arithmetic such a
    difference takes a value in 100 across a border of its 8 bits: a step of 1/127 of the
    largest value of 256 or 32 each, 1e-3 of the row's norm, and the bar is 2e-2 for some
    of them. (No FFN, and an output product in f32: nothing is rounded to 8 bits behind.)
    With V's cells cleared the logits are others altogether."""
    from lgml_amd import runtime, hip
    E = H * D
    hp, w = models.build(dict(arch="llama", n_layer=1, n_embd=E, n_head=H, n_head_kv=kv, head_dim=D, n_ff=256,
                              n_vocab=512, rope_base=1e4, eps=1e-6, wtype=wtype), seed=5, init="normal")
    hp = dict(hp, act_quant=ggml)
    ly, ty = w["layers"][0], core.Q4_K if wtype == "q4_K" else core.Q8_0
    rng = np.random.default_rng(D)
    ly["down"] = (core.quantize(ty, np.zeros((E, 256), np.float32)), ty)
    ly["wo"] = (core.quantize(ty, (0.2 * rng.standard_normal((E, E))).astype(np.float32)), ty)
    w["output"] = ((0.02 * rng.standard_normal((512, E))).astype(np.float32), core.F32)
    m = runtime.DeviceModel(hp, w, 64 * 80, kv_type=hip.Q4_0)
    past, n = [150, 640, 1900, 1200], [1, 1, 1, 20]
    order = np.random.default_rng(3).permutation(80).astype(np.int32)
    tab, at = np.full((4, 32), -1, np.int32), 0
    for s in range(4):
        need = (past[s] + n[s] + 63) // 64
        tab[s, :need] = order[at:at + need]
        at += need
    m.forward(m.plan(past, [0] * 4, tab, np.array(lcg_ints(1, sum(past), 0, 512), np.int32)))
    ids, rows = np.array(lcg_ints(2, sum(n), 0, 512), np.int32), np.arange(sum(n))

    def logits(bps):
        plan = m.plan(n, past, tab, ids, bps)
        assert (plan.info.n_merge > 0) == (bps == 1)
        return m.forward(plan, rows).cpu().numpy()

    one, many = logits(64), logits(1)
    for r in rows:
        assert rel_err(many[r:r + 1], one[r:r + 1]) < (2e-2 if ggml else 5e-4), r
    assert np.array_equal(logits(1).view(np.uint32), many.view(np.uint32))
    m.vpools[0].zero_()
    assert rel_err(logits(1), one) > 0.3
