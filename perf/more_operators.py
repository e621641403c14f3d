"""Long contexts in a 4-bit cache, its blocks copied, and positions of several
axes: the operators, as cases to time and to check.

  cache      lgmlh_kv_store_q4 of a pass's K and V rows into a Q4_0 pool, and
             lgmlh_kv_gather_q4 of the same cells ("write"); or the read back
             of cells alone ("read")
  attention  lgmlh_paged_attention_q4 (decode, chunks and drafted trees)
  pages      lgmlh_kv_copy_blocks: blocks (or their first cells) to other
             blocks in every layer's K and V: forks of sequences, compaction
  rope       lgmlh_qkv_rope_store_axes: norms of q and k heads, rotation by
             positions of up to four axes (time, height, width, ...), K and V
             to their cells

`own` false: the plain forms, elementary torch operations in 32 bits on the
same buffers. Sizes are those of the repository's configurations (8B shape 32
/ 8 heads of 128, Gemma-4-style 8 / 4 heads of 256, MoE shape 32 / 4 heads of
128, tiny model 4 / 2 heads of 64).

The f16 pool is K [block][kv head][cell][D], V [block][kv head][D][cell]. A
(block, kv head) tile of the Q4_0 pool is 36 D bytes: 32 D of 4-bit values n,
which stand for (n - 8) d, then f16 scales d [D / 32][cell]. The values of K
are [D / (32 U)][cell][4][U][4], U = min(4, D / 32), dim 32 (U j + u) + 8 q + e
at (j, cell, q, u), its four bits at 4 (e / 2) + 16 (e % 2) of the 32; of V
[D / 32][16][4][2][8] bytes, dims 32 j + r and 32 j + 16 + r of cell 32 b + 8 q
+ e the low and the high half of byte (j, r, q, b, (0 2 1 3 4 6 5 7)[e]).
"""
import ctypes as C
import math
import random

import numpy as np
import torch

own = False
DEV = "cuda"


# ---- the cases ----------------------------------------------------------------
def listed():
    return [
        # the K / V rows of a decode step of 64 sequences, 8B shape
        dict(name="decode write", kind="cache", dir="write", seqs=64, tokens=1, kv=8, dim=128, out="f32"),
        # a long prompt's chunks: 4 sequences of 2048 tokens, at odd offsets
        dict(name="chunk write", kind="cache", dir="write", seqs=4, tokens=2048, kv=8, dim=128, out="f32"),
        # the context of 8 sequences of 4096 read back, 8B shape
        dict(name="long read", kind="cache", dir="read", seqs=8, tokens=4096, kv=8, dim=128, out="f16"),
        # the smallest attention: one token of one sequence of the tiny model
        dict(name="one token", kind="attention", heads=4, kv=2, dim=64, seqs=1, lo=333, hi=333, nodes=1,
             tree=False),
        # one decode step of 64 ragged sequences, 8B shape
        dict(name="decode", kind="attention", heads=32, kv=8, dim=128, seqs=64, lo=128, hi=4096, nodes=1,
             tree=False),
        # one decode step of 4 sequences far into long documents, MoE shape
        dict(name="long decode", kind="attention", heads=32, kv=4, dim=128, seqs=4, lo=32768, hi=131072,
             nodes=1, tree=False),
        # a prompt's chunk of 512 tokens after 2048, Gemma-4-style heads of 256
        dict(name="chunk", kind="attention", heads=8, kv=4, dim=256, seqs=1, lo=2048, hi=2048, nodes=512,
             tree=False),
        # a turn of the tiny model is forked: its last block's cells
        dict(name="fork one", kind="pages", pool="f16", layers=2, kv=2, dim=64, copies=1, parents=1, whole=False),
        # 32 replies branch off 4 prompts, whose last blocks are in part full; 8B shape, all 32 layers
        dict(name="fork a batch", kind="pages", pool="f16", layers=32, kv=8, dim=128, copies=32, parents=4,
             whole=False),
        # 64 blocks of the 8B shape move down into free places, all 32 layers
        dict(name="compact", kind="pages", pool="f16", layers=32, kv=8, dim=128, copies=64, parents=64, whole=True),
        # one decode step of 64 sequences that hold images, 8B shape
        dict(name="decode rope", kind="rope", tokens=64, heads=32, kv=8, dim=128, rot=128, sections="16 24 24 0",
             interleaved=False, norms=False),
        # an image of 64 x 64 patches in one pass, MoE shape with normed heads
        dict(name="image rope", kind="rope", tokens=4096, heads=32, kv=4, dim=128, rot=128, sections="24 20 20 0",
             interleaved=True, norms=True),
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """A case of the ranges above: every operator, one token to a long chunk,
    odd sizes and ragged contexts among them."""
    kind = rng.choice(["cache", "attention", "attention", "attention", "pages", "rope"])
    if kind == "cache":
        while True:
            kv, d = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 128, 256])
            seqs, tokens = _log(rng, 1, 64), _log(rng, 1, 4096)
            way = rng.choice(["write", "write", "read"])
            if seqs * tokens * kv * d <= (4 * 2048 if way == "write" else 8 * 4096) * 1024:
                return dict(kind=kind, dir=way, seqs=seqs, tokens=tokens, kv=kv, dim=d,
                            out=rng.choice(["f32", "f16"]))
    if kind == "attention":
        while True:
            d, kv, g = rng.choice([64, 128, 128, 256]), rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 8])
            tree = rng.random() < 0.3
            nodes = _log(rng, 2, 64) if tree else rng.choice([1, 1, _log(rng, 2, 512)])
            c = dict(kind=kind, heads=kv * g, kv=kv, dim=d, seqs=_log(rng, 1, 64), lo=_log(rng, 1, 1024),
                     hi=_log(rng, 1025, 65536), nodes=nodes, tree=tree)
            w = work(c)
            if w["bytes"] <= 1.8e8 and w["flops"] <= 9e9:
                return c
    if kind == "pages":
        while True:
            c = dict(kind=kind, pool=rng.choice(["f16", "f16", "q4"]), layers=_log(rng, 1, 32),
                     kv=rng.choice([1, 2, 4, 8]), dim=rng.choice([64, 128, 256]), copies=_log(rng, 1, 128),
                     parents=0, whole=rng.random() < 0.4)
            c["parents"] = c["copies"] if c["whole"] else rng.randint(1, c["copies"])
            if c["pool"] == "q4":
                c["layers"] = min(c["layers"], 4)
            if work(c)["bytes"] <= 1.1e9:
                return c
    while True:
        d, kv, g = rng.choice([64, 128, 128, 256]), rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 8])
        rot = rng.choice([d, d, d // 2])
        a = rng.randint(1, rot // 2 - 2)
        b = rng.randint(1, rot // 2 - a - 1)
        c = dict(kind="rope", tokens=_log(rng, 1, 4096), heads=kv * g, kv=kv, dim=d, rot=rot,
                 sections="%d %d %d 0" % (rot // 2 - a - b, a, b), interleaved=rng.random() < 0.4,
                 norms=rng.random() < 0.5)
        if work(c)["bytes"] <= 1.4e8:
            return c


# ---- inputs -------------------------------------------------------------------
def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)


def _cells(starts, counts, tab):
    """Pool cells of the positions start .. start + count of each sequence."""
    rows = [tab[s][np.arange(p, p + n) // 64].astype(np.int64) * 64 + np.arange(p, p + n) % 64
            for s, (p, n) in enumerate(zip(starts, counts))]
    return np.concatenate(rows)


def _tables(ends, seed):
    """Block tables over a shuffled pool, for sequences of `ends` cells."""
    need = [(n + 63) // 64 for n in ends]
    order = np.random.default_rng(seed + 11).permutation(sum(need)).astype(np.int32)
    tab, at = np.zeros((len(need), max(need)), np.int32), 0
    for s, n in enumerate(need):
        tab[s, :n] = order[at:at + n]
        at += n
    return tab, sum(need)


def _quants(x):
    """Q4_0 of (..., D) f32: values 0 .. 15 and f16 scales (..., D / 32). d is
    the value of largest size, the first of them, over -8."""
    x = x.unflatten(-1, (x.shape[-1] // 32, 32))
    size = x.abs()
    at = torch.where(size == size.amax(-1, keepdim=True), torch.arange(32, device=DEV), 32).amin(-1, keepdim=True)
    d = x.gather(-1, at) * -0.125
    inv = torch.where(d == 0, torch.zeros_like(d), 1.0 / d)
    y = x * inv
    y = y + 8.5
    return y.trunc().clamp(max=15).to(torch.uint8).flatten(-2), d.squeeze(-1).half()


# the byte of V's cell 8 q + e within its 8, and the nibble of K's dim 8 q + e
_V_BYTE = [0, 2, 1, 3, 4, 6, 5, 7]
_K_NIBBLE = [0, 4, 1, 5, 2, 6, 3, 7]


def _k_views(pool, d):
    """(bytes (blocks, 64, kv, D / 32 U, U, 4, 4), scales (blocks, 64, kv, D / 32)) of K tiles."""
    u = min(4, d // 32)
    q = pool[..., :32 * d].unflatten(-1, (d // 32 // u, 64, 4, u, 4))
    s = pool[..., 32 * d:].view(torch.float16).unflatten(-1, (d // 32, 64))
    return q.permute(0, 3, 1, 2, 5, 4, 6), s.permute(0, 3, 1, 2)


def _v_views(pool, d):
    """(bytes (blocks, 2, 4, 8, kv, D / 32, 16), scales (blocks, 64, kv, D / 32)) of V tiles."""
    q = pool[..., :32 * d].unflatten(-1, (d // 32, 16, 4, 2, 8))
    s = pool[..., 32 * d:].view(torch.float16).unflatten(-1, (d // 32, 64))
    return q.permute(0, 5, 4, 6, 1, 2, 3), s.permute(0, 3, 1, 2)


def _rows_in(pool, d, which, cells, x):
    """Rows x (n, kv, D) f32 into cells of a Q4_0 pool (blocks, kv, 36 D)."""
    q, s = _quants(x)
    b, c = cells // 64, cells % 64
    if which == 0:
        vals, sc = _k_views(pool, d)
        q = q.unflatten(-1, (d // 32, 4, 8))
        order = torch.tensor([_K_NIBBLE.index(i) for i in range(8)], device=DEV)
        q = q.index_select(-1, order).unflatten(-1, (4, 2))
        u = vals.shape[4]
        vals[b, c] = (q[..., 0] | (q[..., 1] << 4)).unflatten(2, (d // 32 // u, u))
    else:
        vals, sc = _v_views(pool, d)
        q = q.unflatten(-1, (d // 32, 2, 16))
        place = torch.tensor(_V_BYTE, device=DEV)[c % 8]
        vals[b, c // 32, c % 32 // 8, place] = q[:, :, :, 0] | (q[:, :, :, 1] << 4)
    sc[b, c] = s


def _rows_out(pool, d, which, cells):
    """Cells of a Q4_0 pool as (n, kv, D) f32."""
    b, c = cells // 64, cells % 64
    if which == 0:
        vals, sc = _k_views(pool, d)
        w = vals[b, c].flatten(2, 3)                                      # (n, kv, D / 32, 4, 4)
        q = torch.stack([w & 15, w >> 4], -1).flatten(-2)
        q = q.index_select(-1, torch.tensor(_K_NIBBLE, device=DEV)).flatten(2)
    else:
        vals, sc = _v_views(pool, d)
        w = vals[b, c // 32, c % 32 // 8, torch.tensor(_V_BYTE, device=DEV)[c % 8]]
        q = torch.stack([w & 15, w >> 4], -2).flatten(2)
    s = sc[b, c].float().unsqueeze(-1)
    return ((q.float() - 8.0).unflatten(-1, (d // 32, 32)) * s).flatten(-2)


def _block_rows(pool, d, which, table):
    """Whole blocks of a Q4_0 pool as (64 len(table), kv, D) f32."""
    cells = (table[:, None] * 64 + torch.arange(64, device=DEV)).flatten()
    return torch.cat([_rows_out(pool, d, which, part) for part in cells.split(16384)])


def _q4_pool(g, blocks, kv, d, which):
    """A Q4_0 pool of N(0, 1) rows."""
    pool = torch.empty(blocks, kv, 36 * d, dtype=torch.uint8, device=DEV)
    cells = torch.arange(64 * blocks, device=DEV)
    for at in range(0, 64 * blocks, 65536):
        part = cells[at:at + 65536]
        _rows_in(pool, d, which, part, _normal(g, len(part), kv, d))
    return pool


def _starts(c, seed):
    rng = random.Random(seed * 7919 + 5)
    return [rng.randint(0, 200) for _ in range(c["seqs"])]


def _cache_inputs(c, seed):
    g = torch.Generator(DEV).manual_seed(seed + 1)
    starts, counts = _starts(c, seed), [c["tokens"]] * c["seqs"]
    tab, blocks = _tables([p + n for p, n in zip(starts, counts)], seed)
    cells = _cells(starts, counts, tab)
    n, kv, d = len(cells), c["kv"], c["dim"]
    # keys have a few channels above the others
    gain = torch.where(torch.rand(kv, d, generator=g, device=DEV) < 0.05, 4.0, 1.0)
    return cells, blocks, _normal(g, n, kv, d) * gain, _normal(g, n, kv, d)


def _prep_cache(c, seed):
    cells, blocks, k, v = _cache_inputs(c, seed)
    kv, d = c["kv"], c["dim"]
    pools = [torch.zeros(blocks, kv, 36 * d, dtype=torch.uint8, device=DEV) for _ in range(2)]
    dev = torch.from_numpy(cells).to(DEV)
    if c["dir"] == "read":
        for w, x in enumerate((k, v)):
            _rows_in(pools[w], d, w, dev, x)
    dt = torch.float32 if c["out"] == "f32" else torch.float16
    out = [torch.empty(len(cells), kv * d, dtype=dt, device=DEV) for _ in range(2)]
    return dict(c=c, k=k, v=v, cells=dev, host=cells, pools=pools, n_cells=64 * blocks, out=out)


def _run_cache(s):
    c = s["c"]
    kv, d, n = c["kv"], c["dim"], len(s["host"])
    if own:
        from lgml_amd import hip
        L, st = hip.lib(), hip.stream()
        if c["dir"] == "write":
            hip.check(L.lgmlh_kv_store_q4(s["pools"][0].data_ptr(), s["pools"][1].data_ptr(), s["n_cells"], kv,
                                          d, s["k"].data_ptr(), s["v"].data_ptr(), s["cells"].data_ptr(),
                                          s["host"].ctypes.data, n, st))
        for w in range(2):
            hip.check(L.lgmlh_kv_gather_q4(s["pools"][w].data_ptr(), w, s["n_cells"], kv, d,
                                           s["cells"].data_ptr(), n, s["out"][w].data_ptr(),
                                           hip.F32 if c["out"] == "f32" else hip.F16, st))
        return s["out"]
    if c["dir"] == "write":
        _rows_in(s["pools"][0], d, 0, s["cells"], s["k"])
        _rows_in(s["pools"][1], d, 1, s["cells"], s["v"])
    dt = s["out"][0].dtype
    return [_rows_out(s["pools"][w], d, w, s["cells"]).to(dt).flatten(1) for w in range(2)]


def _contexts(c, seed):
    rng = random.Random(seed * 7919 + 5)
    past = [rng.randint(c["lo"], c["hi"]) for _ in range(c["seqs"])]
    past[0], past[-1] = c["lo"], c["hi"]
    return past


def _parents(c, seed):
    """A tree per sequence: node 0 follows the context, the others follow one
    of the eight before them (or the one before them: a line)."""
    rng = random.Random(seed * 7919 + 17)
    return [[-1] + [rng.randrange(max(0, j - 8), j) if c["tree"] else j - 1 for j in range(1, c["nodes"])]
            for _ in range(c["seqs"])]


def _attention_inputs(c, seed):
    g = torch.Generator(DEV).manual_seed(seed + 1)
    past = _contexts(c, seed)
    tab, blocks = _tables([p + c["nodes"] for p in past], seed)
    kv, d = c["kv"], c["dim"]
    q = _normal(g, c["seqs"] * c["nodes"], c["heads"], d)
    return past, tab, blocks, q, _q4_pool(g, blocks, kv, d, 0), _q4_pool(g, blocks, kv, d, 1)


def _prep_attention(c, seed):
    past, tab, blocks, q, k, v = _attention_inputs(c, seed)
    parents, n = _parents(c, seed), c["nodes"]
    masks = []
    for par in parents:
        m = np.zeros((n, n), bool)
        for j, p in enumerate(par):
            if p >= 0:
                m[j] = m[p]
            m[j, j] = True
        masks.append(torch.from_numpy(m).to(DEV))
    s = dict(c=c, q=q, k=k, v=v, past=past, masks=masks,
             tables=[torch.from_numpy(t.astype(np.int64)).to(DEV) for t in tab])
    if own:
        from lgml_amd import hip, runtime
        plan = runtime.Plan([n] * len(past), past, tab, np.zeros(n * len(past), np.int32), c["heads"], c["kv"],
                            blocks, 28 if c["dim"] >= 256 else 12,
                            parents=np.array(parents, np.int32).reshape(-1) if c["tree"] else None)
        ws = hip.lib().lgmlh_attention_workspace(C.byref(plan.info), c["dim"])
        s.update(plan=plan, ws=torch.empty(max(ws, 1), dtype=torch.uint8, device=DEV), out=torch.empty_like(q))
    return s


def _run_attention(s):
    c, q = s["c"], s["q"]
    h, kv, d, n = c["heads"], c["kv"], c["dim"], c["nodes"]
    if own:
        from lgml_amd import hip
        hip.check(hip.lib().lgmlh_paged_attention_q4(
            q.data_ptr(), h, kv, d, d ** -0.5, s["k"].data_ptr(), s["v"].data_ptr(), C.byref(s["plan"].ub),
            s["out"].data_ptr(), s["ws"].data_ptr(), s["ws"].numel(), hip.stream()))
        return s["out"]
    out = []
    for i, p in enumerate(s["past"]):
        t = s["tables"][i][:(p + n + 63) // 64]
        k = _block_rows(s["k"], d, 0, t)[:p + n].transpose(0, 1)
        v = _block_rows(s["v"], d, 1, t)[:p + n].transpose(0, 1)
        qs = q[i * n:(i + 1) * n].unflatten(1, (kv, h // kv)).permute(1, 2, 0, 3).flatten(1, 2)
        x = torch.matmul(qs, k.transpose(1, 2).contiguous()) * d ** -0.5               # (kv, g n, cells)
        seen = torch.cat([torch.ones(n, p, dtype=torch.bool, device=DEV), s["masks"][i]], 1)
        x = torch.where(seen.repeat(h // kv, 1), x, -math.inf)
        e = (x - x.amax(-1, keepdim=True)).exp()
        o = torch.matmul(e, v.contiguous()) / e.sum(-1, keepdim=True)
        out.append(o.unflatten(1, (h // kv, n)).permute(2, 0, 1, 3).flatten(1, 2))
    return torch.cat(out)


def _page_inputs(c, seed):
    """(source, target, cells) of each copy: targets are free blocks; in a fork
    several take the first cells of one source."""
    rng = random.Random(seed * 7919 + 5)
    n, m = c["copies"], c["parents"]
    blocks = n + m + 8
    order = list(range(blocks))
    rng.shuffle(order)
    if c["whole"]:  # from above into the places below
        src, dst = sorted(order[:m], reverse=True), sorted(order[m:m + n])
        return np.array([(a, b, 64) for a, b in zip(src, dst)], np.int32), blocks
    held = [rng.randint(1, 63) for _ in range(m)]
    return np.array([(order[i % m], order[m + i], held[i % m]) for i in range(n)], np.int32), blocks


def _page_pools(c, seed, blocks):
    g = torch.Generator(DEV).manual_seed(seed + 1)
    kv, d, n = c["kv"], c["dim"], 2 * c["layers"]
    if c["pool"] == "f16":
        return torch.randn(n, blocks, kv, 64 * d, generator=g, device=DEV, dtype=torch.float16)
    return torch.stack([_q4_pool(g, blocks, kv, d, p % 2) for p in range(n)])


def _target_cells(copies):
    return torch.from_numpy(np.concatenate([np.arange(64) + 64 * b for _, b, _ in copies]).astype(np.int64)).to(DEV)


def _prep_pages(c, seed):
    copies, blocks = _page_inputs(c, seed)
    pools = _page_pools(c, seed, blocks)
    s = dict(c=c, pools=pools, host=copies, n_cells=64 * blocks,
             addr=torch.tensor([p.data_ptr() for p in pools], dtype=torch.int64, device=DEV),
             copies=torch.from_numpy(copies).to(DEV))
    if c["pool"] == "q4":
        s["cells"] = _target_cells(copies)
        s["out"] = torch.empty(len(pools), len(s["cells"]), c["kv"] * c["dim"], device=DEV)
    return s


def _run_pages(s):
    c, pools, kv, d = s["c"], s["pools"], s["c"]["kv"], s["c"]["dim"]
    f16 = c["pool"] == "f16"
    if own:
        from lgml_amd import hip
        L, st = hip.lib(), hip.stream()
        hip.check(L.lgmlh_kv_copy_blocks(hip.F16 if f16 else hip.Q4_0, s["addr"].data_ptr(), len(pools),
                                         s["n_cells"], kv, d, s["copies"].data_ptr(), s["host"].ctypes.data,
                                         len(s["host"]), st))
        if f16:
            return pools
        for p in range(len(pools)):
            hip.check(L.lgmlh_kv_gather_q4(pools[p].data_ptr(), p % 2, s["n_cells"], kv, d, s["cells"].data_ptr(),
                                           len(s["cells"]), s["out"][p].data_ptr(), hip.F32, st))
        return s["out"]
    src, dst = s["copies"][:, 0].long(), s["copies"][:, 1].long()
    n = s["copies"][:, 2]
    held = torch.arange(64, device=DEV) < n[:, None]                                    # (copies, 64)
    if f16:
        k = pools[0::2].unflatten(-1, (64, d))
        v = pools[1::2].unflatten(-1, (d, 64))
        k[:, dst] = torch.where(held[None, :, None, :, None], k[:, src], k[:, dst])
        v[:, dst] = torch.where(held[None, :, None, None, :], v[:, src], v[:, dst])
        return pools
    i, cell = held.nonzero(as_tuple=True)
    a, b, rows = src[i], dst[i], []
    for p in range(len(pools)):
        if p % 2 == 0:
            vals, scale = _k_views(pools[p], d)
            vals[b, cell] = vals[a, cell]
        else:
            vals, scale = _v_views(pools[p], d)
            place = torch.tensor(_V_BYTE, device=DEV)[cell % 8]
            vals[b, cell // 32, cell % 32 // 8, place] = vals[a, cell // 32, cell % 32 // 8, place]
        scale[b, cell] = scale[a, cell]
        rows.append(_rows_out(pools[p], d, p % 2, s["cells"]).flatten(1))
    return torch.stack(rows)


def _axis_of(c):
    """The axis of each rotated pair: sections one after the other, or (of three
    axes) in turn, where what an axis has no pairs left for goes by time."""
    s = [int(x) for x in c["sections"].split()]
    if not c["interleaved"]:
        return [a for a in range(4) for _ in range(s[a])]
    return [i % 3 if i < 3 * s[i % 3] else 0 for i in range(c["rot"] // 2)]


def _rope_inputs(c, seed):
    """Rows of q, k and v, positions (4, tokens) of images between words, cells."""
    g = torch.Generator(DEV).manual_seed(seed + 1)
    rng = random.Random(seed * 7919 + 5)
    n, h, kv, d = c["tokens"], c["heads"], c["kv"], c["dim"]
    qkv = _normal(g, n, (h + 2 * kv) * d)
    if n <= 64:  # tokens of as many sequences: all axes alike, anywhere
        p = np.array([rng.randint(0, 100000) for _ in range(n)])
        pos = np.stack([p, p, p, p])
        blocks = n
        cells = np.array([64 * b + rng.randint(0, 63) for b in np.random.default_rng(seed + 3).permutation(n)])
    else:  # one sequence's image: its rows and columns
        t, w = rng.randint(0, 20000), max(1, math.isqrt(n))
        i = np.arange(n)
        pos = np.stack([np.full(n, t), t + i // w, t + i % w, np.zeros(n)])
        start = rng.randint(0, 200)
        tab, blocks = _tables([200 + n], seed)
        cells = _cells([start], [n], tab)
    norms = [1 + 0.2 * _normal(g, d) for _ in range(2)] if c["norms"] else [None, None]
    return qkv, pos.astype(np.int32), cells.astype(np.int64), blocks, norms


def _prep_rope(c, seed):
    qkv, pos, cells, blocks, norms = _rope_inputs(c, seed)
    kv, d = c["kv"], c["dim"]
    pools = [torch.zeros(blocks, kv, 64 * d, dtype=torch.float16, device=DEV) for _ in range(2)]
    return dict(c=c, qkv=qkv, pos=torch.from_numpy(pos).to(DEV), cells=torch.from_numpy(cells).to(DEV),
                n_cells=64 * blocks, norms=norms, pools=pools, axis=torch.tensor(_axis_of(c), device=DEV),
                sections=np.array([int(x) for x in c["sections"].split()], np.int32),
                q=torch.empty(c["tokens"], c["heads"], d, device=DEV))


def _run_rope(s):
    c, n = s["c"], s["c"]["tokens"]
    h, kv, d, rot = c["heads"], c["kv"], c["dim"], c["rot"]
    if own:
        from lgml_amd import hip
        hip.check(hip.lib().lgmlh_qkv_rope_store_axes(
            hip.F16, s["qkv"].data_ptr(), n, h, kv, d, rot, s["sections"].ctypes.data, int(c["interleaved"]),
            1000000.0, None, hip.ptr(s["norms"][0]), hip.ptr(s["norms"][1]), 1e-6, s["pos"].data_ptr(),
            s["pools"][0].data_ptr(), s["pools"][1].data_ptr(), s["n_cells"], s["cells"].data_ptr(),
            s["q"].data_ptr(), hip.stream()))
        return [s["q"], s["pools"][0], s["pools"][1]]
    # 64 bits: the angles of far positions
    freq = 1000000.0 ** (-2.0 / rot * torch.arange(rot // 2, device=DEV, dtype=torch.float64))
    angle = s["pos"].double()[s["axis"]].T * freq                                       # (n, rot / 2)
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    x = s["qkv"].unflatten(1, (h + 2 * kv, d))
    heads = []
    for part, w in ((x[:, :h], s["norms"][0]), (x[:, h:h + kv], s["norms"][1])):
        if w is not None:
            part = part * (1.0 / ((part * part).mean(-1, keepdim=True) + 1e-6).sqrt()) * w
        a, b = part[..., :rot // 2], part[..., rot // 2:rot]
        heads.append(torch.cat([a * cos - b * sin, a * sin + b * cos, part[..., rot:]], -1))
    b, cell = s["cells"] // 64, s["cells"] % 64
    s["pools"][0].unflatten(-1, (64, d))[b, :, cell] = heads[1].half()
    s["pools"][1].unflatten(-1, (d, 64))[b, :, :, cell] = x[:, h + kv:].half()
    return [heads[0], s["pools"][0], s["pools"][1]]


_PREPARE = dict(cache=_prep_cache, attention=_prep_attention, pages=_prep_pages, rope=_prep_rope)
_RUN = dict(cache=_run_cache, attention=_run_attention, pages=_run_pages, rope=_run_rope)


def prepare(case, seed):
    return _PREPARE[case["kind"]](case, seed)


def run(state):
    return _RUN[state["c"]["kind"]](state)


# ---- what a pass cannot do without --------------------------------------------
def work(case):
    c, kind = case, case["kind"]
    if kind == "cache":
        n = 2.0 * c["seqs"] * c["tokens"] * c["kv"] * c["dim"]
        out = 4.0 if c["out"] == "f32" else 2.0
        if c["dir"] == "read":
            return dict(bytes=n * (0.5625 + out), flops=n)
        return dict(bytes=n * (4 + 0.5625 + out), flops=4.0 * n)
    if kind == "attention":
        mean, n = (c["lo"] + c["hi"]) / 2, c["nodes"]
        return dict(bytes=c["seqs"] * (2 * (mean + n) * c["kv"] * c["dim"] * 0.5625 + 8.0 * n * c["heads"] * c["dim"]),
                    flops=4.0 * c["seqs"] * n * (mean + n / 2) * c["heads"] * c["dim"])
    if kind == "pages":
        cell = 2.0 * c["layers"] * c["kv"] * c["dim"] * (2.0 if c["pool"] == "f16" else 0.5625)
        cells = 64.0 if c["whole"] else 32.0
        return dict(bytes=cell * cells * (c["copies"] + c["parents"]), flops=0.0)
    n, kv, d = float(c["tokens"]), c["kv"], c["dim"]
    return dict(bytes=n * d * (4.0 * (2 * c["heads"] + 2 * kv) + 4.0 * kv), flops=4.0 * n * d * (c["heads"] + kv))


# ---- the definitions in 64 bits ------------------------------------------------
def _quantised(x):
    """The values that 4 bits keep of x (n, kv, D): its steps are the format's
    definition, 1 / d, x / d and its sum with 8.5 rounded to 32 bits, d kept in 16."""
    n, kv, d = x.shape
    g = x.double().view(n, kv, d // 32, 32)
    top, low = g.amax(3), g.amin(3)
    first = lambda v: torch.where(g == v[..., None], torch.arange(32, device=DEV), 32).amin(3)
    up = (top > -low) | ((top == -low) & (first(top) < first(low)))
    scale = torch.where(up, top, low) / -8
    inv = torch.where(scale != 0, (1 / scale).float().double(), 0.0)
    y = (g * inv[..., None]).float().double()
    n16 = ((y + 8.5).float().double().floor()).clamp(max=15.0)
    return ((n16 - 8) * scale.half().double()[..., None]).view(n, kv, d)


def _held(pool, d, which, cells):
    """What cells of a Q4_0 pool stand for, (n, kv, D), by each value's place in its tile."""
    x = torch.arange(d, device=DEV)
    cell = (cells % 64)[:, None]
    if which == 0:
        u = 4 if d >= 128 else 2
        word = ((x // (32 * u) * 64 + cell) * 4 + x % 32 // 8) * u + x // 32 % u
        at = 4 * word + x % 2 * 2 + x % 8 // 4
        shift = 4 * (x // 2 % 2)
    else:
        e = cell % 8
        at = ((x // 32 * 16 + x % 16) * 4 + cell % 32 // 8) * 16 + cell // 32 * 8 + e // 4 * 4 + e % 2 * 2 + e // 2 % 2
        shift = 4 * (x // 16 % 2)
    scale = 32 * d + 2 * (x // 32 * 64 + cell)
    n, kv = len(cells), pool.shape[1]
    t = pool[cells // 64].to(torch.int32)                                              # (n, kv, 36 D)
    byte = lambda i: t.gather(2, i[:, None].expand(n, kv, d))
    q = byte(at) >> shift & 15
    bits = byte(scale) + 256 * byte(scale + 1)
    bits = torch.where(bits > 32767, bits - 65536, bits).to(torch.int16)
    return (q - 8).double() * bits.view(torch.float16).double()


def _exact_cache(c, seed):
    _, _, k, v = _cache_inputs(c, seed)
    dt = torch.float64 if c["out"] == "f32" else torch.float16
    return [_quantised(x).flatten(1).to(dt).double() for x in (k, v)]


def _exact_attention(c, seed):
    past, tab, blocks, q, k, v = _attention_inputs(c, seed)
    h, kv, d, n = c["heads"], c["kv"], c["dim"], c["nodes"]
    out = torch.empty(len(q), h, d, dtype=torch.float64, device=DEV)
    for i, (p, par) in enumerate(zip(past, _parents(c, seed))):
        cells = torch.from_numpy(_cells([0], [p + n], tab[i:i + 1])).to(DEV)
        ks, vs = (torch.cat([_held(x, d, w, part) for part in cells.split(1024)]) for w, x in ((0, k), (1, v)))
        ks, vs = ks.permute(1, 2, 0).contiguous(), vs.permute(1, 0, 2).contiguous()
        far = torch.full((n, n), -math.inf, dtype=torch.float64)
        for j in range(n):
            at = j
            while at >= 0:
                far[j, at] = 0.0
                at = par[at]
        far = torch.cat([torch.zeros(n, p, dtype=torch.float64), far], 1).to(DEV)
        for t in range(0, n, 64):
            rows = q[i * n + t:i * n + min(n, t + 64)].double()
            m = len(rows)
            x = torch.bmm(rows.view(m, kv, h // kv, d).transpose(0, 1).reshape(kv, -1, d), ks) * d ** -0.5
            x = x + far[t:t + m].repeat_interleave(h // kv, 0)
            o = torch.bmm(torch.softmax(x, 2), vs).view(kv, m, h // kv, d)
            out[i * n + t:i * n + t + m] = o.transpose(0, 1).reshape(m, h, d)
    return out


def _exact_pages(c, seed):
    copies, blocks = _page_inputs(c, seed)
    pools = _page_pools(c, seed, blocks)
    kv, d = c["kv"], c["dim"]
    if c["pool"] == "q4":
        own_cells = _target_cells(copies)
        came = own_cells.clone()
        for i, (a, b, n) in enumerate(copies.tolist()):
            came[64 * i:64 * i + n] = torch.arange(64 * a, 64 * a + n, device=DEV)
        return torch.stack([_held(pools[p], d, p % 2, came).flatten(1) for p in range(len(pools))])
    new = pools.clone()
    for a, b, n in copies.tolist():
        new[0::2].view(-1, blocks, kv, 64, d)[:, b, :, :n] = pools[0::2].view(-1, blocks, kv, 64, d)[:, a, :, :n]
        new[1::2].view(-1, blocks, kv, d, 64)[:, b, ..., :n] = pools[1::2].view(-1, blocks, kv, d, 64)[:, a, ..., :n]
    return new.double()


def _exact_rope(c, seed):
    qkv, pos, cells, blocks, norms = _rope_inputs(c, seed)
    n, h, kv, d, rot = c["tokens"], c["heads"], c["kv"], c["dim"], c["rot"]
    x = qkv.double().view(n, h + 2 * kv, d)
    for at, m, w in ((0, h, norms[0]), (h, kv, norms[1])):
        if w is not None:
            part = x[:, at:at + m]
            x[:, at:at + m] = part / (part.pow(2).mean(2, keepdim=True) + 1e-6).sqrt() * w.double()
    v = x[:, h + kv:]
    turned = x[:, :h + kv].clone()
    p = torch.from_numpy(pos).to(DEV).double()
    t, hh, w, _ = (int(y) for y in c["sections"].split())
    for i in range(rot // 2):
        if c["interleaved"]:
            a = 1 if i in range(1, 3 * hh, 3) else 2 if i in range(2, 3 * w, 3) else 0
        else:
            a = (i >= t) + (i >= t + hh) + (i >= t + hh + w)
        angle = (p[a] * math.exp(-math.log(1000000.0) * 2 * i / rot))[:, None]
        a0, a1 = x[:, :h + kv, i], x[:, :h + kv, i + rot // 2]
        turned[:, :, i] = a0 * angle.cos() - a1 * angle.sin()
        turned[:, :, i + rot // 2] = a0 * angle.sin() + a1 * angle.cos()
    kp = torch.zeros(blocks, kv, 64, d, dtype=torch.float64, device=DEV)
    vp = torch.zeros(blocks, kv, d, 64, dtype=torch.float64, device=DEV)
    at = torch.from_numpy(cells).to(DEV)
    kp[at // 64, :, at % 64] = turned[:, h:]
    vp[at // 64, :, :, at % 64] = v
    return [turned[:, :h], kp.view(blocks, kv, 64 * d), vp.view(blocks, kv, 64 * d)]


def exact(case, seed):
    return dict(cache=_exact_cache, attention=_exact_attention, pages=_exact_pages,
                rope=_exact_rope)[case["kind"]](case, seed)
