"""lgmlh_qkv_rope_store_axes on the GPU against the formula in 64 bits: sections one
after the other and interleaved, norms, frequency factors, heads turned in part, far
and negative positions, pools of each type, cells outside the pool."""
import math

import numpy as np
import pytest

from tests.test_gpu_draft import dev, st

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def axis_of(rot, sections, interleaved):
    out = []
    for i in range(rot // 2):
        if interleaved:
            out.append(i % 3 if i < 3 * sections[i % 3] else 0)
        else:
            out.append(int(np.searchsorted(np.cumsum(sections), i, side="right")))
    return np.array(out)


def turned(x, rot, axes, pos, base, ff, w, eps):
    """Heads x (n, heads, D) f32 normed and turned, in 64 bits, and how far an f32
    computation may be off for each value. The norm's factor takes a sum of D squares
    (D + 8 roundings at most), a square root and a division, each side of a pair 3
    roundings more; the angle (made in 64 bits, rounded to f32 in turns of at most
    1/2: 2^-25 of them, 2 pi 2^-25 in its sine, whose f32 is off by 2 ulp, 2^-22 at
    most) 2^-21 of the pair, the products and their sum 3 roundings of it."""
    x = x.astype(np.float64)
    n, h, D = x.shape
    rel = np.zeros(x.shape)
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w.astype(np.float64)
        rel += (D / 2 + 12) * 2.0**-24
    theta = pos[axes].T.astype(np.float64) * base ** (-2.0 * np.arange(rot // 2) / rot)
    if ff is not None:
        theta = theta / ff.astype(np.float64)
    c, s = np.cos(theta)[:, None], np.sin(theta)[:, None]
    a, b = x[..., :rot // 2], x[..., rot // 2:rot]
    y = np.concatenate([a * c - b * s, a * s + b * c, x[..., rot:]], -1)
    pair = np.abs(a) + np.abs(b)
    tol = np.abs(x) * rel
    both = tol[..., :rot // 2] + tol[..., rot // 2:rot] + pair * (2.0**-21 + 3 * 2.0**-24)
    tol = np.concatenate([both, both, tol[..., rot:] + np.abs(x[..., rot:]) * 2.0**-24], -1)
    # an angle of 64 bits: pos times a frequency of 2^-52, past 2^30 turns
    far = np.abs(theta) * 2.0**-50
    tol[..., :rot] += np.concatenate([far, far], -1)[:, None] * np.concatenate([pair, pair], -1)
    return y, tol


def run(kv_type, x, H, kv, D, rot, sections, inter, base, ff, qn, kn, eps, pos, pools, n_cells, cells):
    from lgml_amd import hip
    n = len(x)
    q = torch.full((n + 1, H, D), 7.0, device="cuda")
    xd, pd, cd = dev(x), dev(pos.astype(np.int32)), dev(cells)
    ffd, qd, kd = (None if a is None else dev(a) for a in (ff, qn, kn))
    sec = np.array(sections, np.int32)
    hip.check(hip.lib().lgmlh_qkv_rope_store_axes(
        kv_type, xd.data_ptr(), n, H, kv, D, rot, sec.ctypes.data, inter, base, hip.ptr(ffd), hip.ptr(qd), hip.ptr(kd),
        eps, pd.data_ptr(), pools[0].data_ptr(), pools[1].data_ptr(), n_cells, cd.data_ptr(), q.data_ptr(), st()))
    assert torch.equal(xd, dev(x))  # the rows stay
    assert bool((q[-1] == 7.0).all())
    return q[:-1]


CASES = [  # n, H, kv, D, rot, sections, interleaved
    (1, 4, 2, 64, 64, (8, 12, 12, 0), 0), (7, 32, 8, 128, 128, (16, 24, 24, 0), 0),
    (300, 8, 4, 256, 256, (32, 48, 40, 8), 0), (33, 6, 1, 128, 64, (10, 11, 11, 0), 0),
    (70, 16, 4, 128, 128, (24, 20, 20, 0), 1), (5, 3, 3, 64, 8, (1, 1, 2, 0), 1),
    (2100, 4, 2, 64, 48, (24, 0, 0, 0), 0), (40, 70, 2, 256, 200, (0, 50, 50, 0), 0),
    (129, 9, 5, 128, 120, (20, 40, 0, 0), 1), (600, 40, 8, 128, 128, (16, 16, 16, 16), 0),
]


@pytest.mark.parametrize("case", range(len(CASES)))
@pytest.mark.parametrize("norms", [(0, 0), (1, 1), (1, 0), (0, 1)])
@pytest.mark.parametrize("far", [False, True])
def test_rows_turn_by_their_axes(case, norms, far):
    from lgml_amd import hip
    n, H, kv, D, rot, sections, inter = CASES[case]
    rng = np.random.default_rng(100 * case + 10 * norms[0] + norms[1])
    x = (rng.standard_normal((n, H + 2 * kv, D)) * 3).astype(np.float32)
    pos = rng.integers(-(1 << 22) if far else 0, (1 << 22) if far else 5000, (4, n))
    ff = (1 + 7 * rng.random(rot // 2)).astype(np.float32) if case % 2 else None
    qn, kn = ((1 + 0.3 * rng.standard_normal(D)).astype(np.float32) if on else None for on in norms)
    base, eps = (10000.0, 1e-6) if case % 3 else (1e6, 1e-5)
    blocks = n // 64 + 4
    if n < 50:  # tokens of as many sequences
        cells = rng.permutation(64 * blocks)[:n].astype(np.int64)
    else:
        cells = (np.arange(n) + 13).astype(np.int64)
    if n > 3:
        cells[2], cells[3] = 64 * blocks, -1  # outside the pool
    axes = axis_of(rot, sections, inter)
    wq, tq = turned(x[:, :H], rot, axes, pos, base, ff, qn, eps)
    wk, tk = turned(x[:, H:H + kv], rot, axes, pos, base, ff, kn, eps)
    start = rng.integers(0, 2**16, (2, blocks, kv, 64 * D)).astype(np.uint16)
    pools = [dev(start[w].view(np.int16)) for w in range(2)]
    got = run(hip.F16, x, H, kv, D, rot, sections, inter, base, ff, qn, kn, eps, pos, pools, 64 * blocks, cells)
    err = np.abs(got.cpu().numpy().astype(np.float64) - wq)
    assert (err <= tq).all(), float((err / tq).max())
    ok = (cells >= 0) & (cells < 64 * blocks)
    kp = pools[0].cpu().numpy().view(np.uint16).reshape(blocks, kv, 64, D)
    vp = pools[1].cpu().numpy().view(np.uint16).reshape(blocks, kv, D, 64)
    k = kp[cells[ok] // 64, :, cells[ok] % 64].view(np.float16).astype(np.float64)
    # the f16 of a value off by tk: half a step of it more (of 2^-24 near zero)
    assert (np.abs(k - wk[ok]) <= tk[ok] + (np.abs(wk[ok]) + tk[ok]) * 2.0**-11 + 2.0**-25).all()
    v = vp[cells[ok] // 64, :, :, cells[ok] % 64].view(np.float16)
    assert np.array_equal(v, x[ok, H + kv:].astype(np.float16))
    rest = np.ones(64 * blocks, bool)
    rest[cells[ok]] = False
    rest = rest.reshape(blocks, 64)
    assert np.array_equal(kp.transpose(0, 2, 1, 3)[rest], start[0].reshape(kp.shape).transpose(0, 2, 1, 3)[rest])
    assert np.array_equal(vp.transpose(0, 3, 1, 2)[rest], start[1].reshape(vp.shape).transpose(0, 3, 1, 2)[rest])


@pytest.mark.parametrize("kind", ["Q8_0", "Q4_0"])
@pytest.mark.parametrize("H,kv,D,rot,n", [(4, 2, 64, 64, 9), (8, 8, 128, 128, 300), (8, 4, 256, 128, 77),
                                          (5, 3, 128, 80, 2000)])
def test_quantised_pools_hold_the_turned_rows(kind, H, kv, D, rot, n):
    """The pools' bytes are those of storing the turned rows (K's as the q heads of a call
    with K in their place)."""
    from lgml_amd import hip
    L, ty = hip.lib(), getattr(hip, kind)
    rng = np.random.default_rng(D + n)
    x = rng.standard_normal((n, H + 2 * kv, D)).astype(np.float32)
    pos = rng.integers(0, 3000, (4, n))
    sections, blocks = (rot // 2 - 12, 6, 6, 0), n // 64 + 3
    cells = np.concatenate([np.arange(n - 1) + 60, [64 * blocks]]).astype(np.int64)
    kn = (1 + 0.1 * rng.standard_normal(D)).astype(np.float32)
    nb = (L.lgmlh_kv_q8_layer_bytes if kind == "Q8_0" else L.lgmlh_kv_q4_layer_bytes)(64 * blocks, kv, D)

    def pools():
        return [torch.full((nb,), 0x5A, dtype=torch.uint8, device="cuda") for _ in range(2)]

    got, other, want = pools(), pools(), pools()
    run(ty, x, H, kv, D, rot, sections, 0, 1e4, None, kn, kn, 1e-6, pos, got, 64 * blocks, cells)
    as_q = np.concatenate([x[:, H:H + kv], x[:, H:]], 1)
    k = run(ty, as_q, kv, kv, D, rot, sections, 0, 1e4, None, kn, kn, 1e-6, pos, other, 64 * blocks, cells)
    v, dc = dev(x[:, H + kv:]), dev(cells)
    fn = L.lgmlh_kv_store_q8 if kind == "Q8_0" else L.lgmlh_kv_store_q4
    hip.check(fn(want[0].data_ptr(), want[1].data_ptr(), 64 * blocks, kv, D, k.contiguous().data_ptr(), v.data_ptr(),
                 dc.data_ptr(), cells.ctypes.data, n - 1, st()))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_words_turn_as_by_one_position():
    """Tokens whose positions are alike: lgmlh_qkv_rope_store's rows, within what its running
    f32 product of an angle is off (pair i: i + 2 roundings of the angle)."""
    from lgml_amd import hip
    L = hip.lib()
    n, H, kv, D = 50, 8, 2, 128
    rng = np.random.default_rng(3)
    x = rng.standard_normal((n, H + 2 * kv, D)).astype(np.float32)
    p = rng.integers(0, 4000, n)
    cells = np.arange(n, dtype=np.int64)
    pools = [torch.zeros(64 * kv * D, dtype=torch.float16, device="cuda") for _ in range(2)]
    got = run(hip.F16, x, H, kv, D, D, (16, 24, 24, 0), 0, 1e4, None, None, None, 1e-6, np.stack([p] * 4), pools, 64,
              cells).cpu().numpy()
    xd, pd, cd = dev(x), dev(p.astype(np.int32)), dev(cells)
    q = torch.empty(n, H, D, device="cuda")
    hip.check(L.lgmlh_qkv_rope_store(xd.data_ptr(), n, H, kv, D, D, 1, 1e4, None, None, None, 1e-6, pd.data_ptr(),
                                     pools[0].data_ptr(), pools[1].data_ptr(), 64, cd.data_ptr(), q.data_ptr(), st()))
    i = np.arange(D // 2)
    theta = p[:, None] * 1e4 ** (-2.0 * i / D)
    off = theta * (i + 3) * 2.0**-23 + 2.0**-20
    pair = np.abs(x[:, :H, :D // 2]) + np.abs(x[:, :H, D // 2:])
    tol = pair * off[:, None]
    assert (np.abs(got - q.cpu().numpy()) <= np.concatenate([tol, tol], -1)).all()
