"""Serving drafted tokens over a quantised cache: the operators, as cases to
time and to check.

  cache      lgmlh_kv_store_q8 of a pass's K and V rows into a Q8_0 pool, and
             lgmlh_kv_gather_q8 of the same cells ("write"); or the read back
             of cells alone ("read")
  move       lgmlh_kv_move: the cells of accepted drafted tokens to their
             places behind the context, in every layer's K and V
  attention  lgmlh_paged_attention over a tree plan (f16 pool), and
             lgmlh_paged_attention_q8 (decode, chunks and trees)
  logprobs   lgmlh_log_probs: log probabilities of given tokens, entropy, the
             most likely alternatives

`own` false: the plain forms, elementary torch operations in 32 bits on the
same buffers. Sizes are those of the repository's configurations (8B shape 32
/ 8 heads of 128 and a vocabulary of 128256, Gemma-4-style 8 / 4 heads of 256,
MoE shape 32 / 4 heads of 128 and 151936, tiny model 4 / 2 heads of 64).

The f16 pool is K [block][kv head][cell][D], V [block][kv head][D][cell]. A
(block, kv head) tile of the Q8_0 pool is 68 D bytes: 64 D int8 values, then
f16 scales [D / 32][cell]. The values of K are [D / 64][cell][4][2][8], dim 64
j + 32 b + 8 q + e at (j, cell, q, b, e); of V [D][4][2][8], cell 32 b + 8 q +
e at (d, q, b, e).
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
        # a short snapshot of the Gemma-4-style shape, odd length
        dict(name="short read", kind="cache", dir="read", seqs=1, tokens=777, kv=4, dim=256, out="f16"),
        # the context of 8 sequences of 4096 read back, 8B shape
        dict(name="long read", kind="cache", dir="read", seqs=8, tokens=4096, kv=8, dim=128, out="f32"),
        # one sequence of the tiny model keeps 4 of 9 drafted tokens
        dict(name="accept one", kind="move", pool="f16", layers=2, seqs=1, nodes=9, accept=4, kv=2, dim=64),
        # 64 sequences of the 8B shape keep 5 of 16 drafted tokens, all 32 layers
        dict(name="accept batch", kind="move", pool="f16", layers=32, seqs=64, nodes=16, accept=5, kv=8,
             dim=128),
        # the smallest attention: one sequence, a tree of 9 drafted tokens, tiny shape
        dict(name="one tree", kind="attention", pool="f16", heads=4, kv=2, dim=64, seqs=1, lo=333, hi=333,
             nodes=9, tree=True),
        # trees of 16 drafted tokens for 32 ragged sequences, 8B shape, f16 pool
        dict(name="trees of a batch", kind="attention", pool="f16", heads=32, kv=8, dim=128, seqs=32, lo=128,
             hi=4096, nodes=16, tree=True),
        # one decode step of 64 ragged sequences over the Q8_0 pool, 8B shape
        dict(name="decode q8", kind="attention", pool="q8", heads=32, kv=8, dim=128, seqs=64, lo=128, hi=4096,
             nodes=1, tree=False),
        # trees of 61 drafted tokens over long contexts, Gemma-4-style heads of 256, Q8_0 pool
        dict(name="trees q8", kind="attention", pool="q8", heads=8, kv=4, dim=256, seqs=8, lo=1024, hi=16384,
             nodes=61, tree=True),
        # one row of 128256 logits: its greedy token and 5 alternatives
        dict(name="one row", kind="logprobs", rows=1, vocab=128256, ids=1, top=5, masked=False),
        # 1000 rows (a prompt's tokens, or 64 trees) of 151936 logits, 3 given
        # tokens each and 20 alternatives
        dict(name="many rows", kind="logprobs", rows=1000, vocab=151936, ids=3, top=20, masked=False),
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """A case of the ranges above: every operator, one token to a long chunk,
    odd sizes and ragged contexts among them."""
    kind = rng.choice(["cache", "move", "attention", "attention", "attention", "logprobs"])
    if kind == "cache":
        while True:
            kv, d = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 128, 256])
            seqs, tokens = _log(rng, 1, 64), _log(rng, 1, 4096)
            way = rng.choice(["write", "write", "read"])
            if seqs * tokens * kv * d <= (4 * 2048 if way == "write" else 8 * 4096) * 1024:
                return dict(kind=kind, dir=way, seqs=seqs, tokens=tokens, kv=kv, dim=d,
                            out=rng.choice(["f32", "f16"]))
    if kind == "move":
        accept = _log(rng, 1, 12)
        pool = rng.choice(["f16", "f16", "q8"])
        return dict(kind=kind, pool=pool, layers=rng.randint(1, 2) if pool == "q8" else _log(rng, 1, 32),
                    seqs=_log(rng, 1, 64), nodes=2 * accept + rng.randint(0, 7), accept=accept,
                    kv=rng.choice([1, 2, 4, 8]), dim=rng.choice([64, 128]))
    if kind == "attention":
        while True:
            d, kv, g = rng.choice([64, 128, 128, 256]), rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 8])
            pool = rng.choice(["f16", "q8", "q8"])
            tree = pool == "f16" or rng.random() < 0.5
            nodes = _log(rng, 2, 64) if tree else rng.choice([1, 1, _log(rng, 2, 512)])
            c = dict(kind=kind, pool=pool, heads=kv * g, kv=kv, dim=d, seqs=_log(rng, 1, 64),
                     lo=_log(rng, 1, 1024), hi=_log(rng, 1025, 16384), nodes=nodes, tree=tree)
            w = work(c)
            if w["bytes"] <= 3.2e8 and w["flops"] <= 2.5e10:
                return c
    rows, vocab = _log(rng, 1, 1000), _log(rng, 8192, 262144)
    rows = min(rows, 1000 * 151936 // vocab)
    return dict(kind=kind, rows=rows, vocab=vocab, ids=rng.randint(1, 8), top=rng.choice([1, 5, 8, 20, 33]),
                masked=rng.random() < 0.3)


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
    """Q8_0 of (..., D) f32: int8 values and f16 scales (..., D / 32)."""
    x = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    d = x.abs().amax(-1, keepdim=True)
    d = d / torch.full_like(d, 127.0)  # (a scalar's reciprocal would be multiplied by)
    y = x * torch.where(d == 0, torch.zeros_like(d), 1.0 / d)
    a = y.abs()
    t = a.trunc()
    q = (t + (a - t >= 0.5)) * y.sign()
    return q.to(torch.int8).reshape(*x.shape[:-2], -1), d.squeeze(-1).half()


def _k_views(pool, d):
    """(values (blocks, 64, kv, D / 64, 2, 4, 8), scales (blocks, 64, kv, D / 32)) of K tiles."""
    q = pool[..., :64 * d].view(torch.int8).unflatten(-1, (d // 64, 64, 4, 2, 8))
    s = pool[..., 64 * d:].view(torch.float16).unflatten(-1, (d // 32, 64))
    return q.permute(0, 3, 1, 2, 5, 4, 6), s.permute(0, 3, 1, 2)


def _v_views(pool, d):
    """(values (blocks, 2, 4, 8, kv, D), scales (blocks, 64, kv, D / 32)) of V tiles."""
    q = pool[..., :64 * d].view(torch.int8).unflatten(-1, (d, 4, 2, 8))
    s = pool[..., 64 * d:].view(torch.float16).unflatten(-1, (d // 32, 64))
    return q.permute(0, 4, 3, 5, 1, 2), s.permute(0, 3, 1, 2)


def _rows_in(pool, d, which, cells, x):
    """Rows x (n, kv, D) f32 into cells of a Q8_0 pool (blocks, kv, 68 D)."""
    q, s = _quants(x)
    b, c = cells // 64, cells % 64
    if which == 0:
        vals, sc = _k_views(pool, d)
        vals[b, c] = q.unflatten(-1, (d // 64, 2, 4, 8))
    else:
        vals, sc = _v_views(pool, d)
        vals[b, c // 32, c % 32 // 8, c % 8] = q
    sc[b, c] = s


def _rows_out(pool, d, which, cells):
    """Cells of a Q8_0 pool as (n, kv, D) f32."""
    b, c = cells // 64, cells % 64
    if which == 0:
        vals, sc = _k_views(pool, d)
        q = vals[b, c].flatten(-4)
    else:
        vals, sc = _v_views(pool, d)
        q = vals[b, c // 32, c % 32 // 8, c % 8]
    s = sc[b, c].float().unsqueeze(-1)
    return (q.float().unflatten(-1, (d // 32, 32)) * s).flatten(-2)


def _block_rows(pool, d, which, table):
    """Whole blocks of a Q8_0 pool as (64 len(table), kv, D) f32."""
    t = pool[table]
    vals, sc = (_k_views if which == 0 else _v_views)(t, d)
    q = vals.flatten(-4) if which == 0 else vals.flatten(1, 3)
    return (q.float().unflatten(-1, (d // 32, 32)) * sc.float().unsqueeze(-1)).flatten(-2).flatten(0, 1)


def _q8_pool(g, blocks, kv, d, which):
    """A Q8_0 pool of N(0, 1) rows."""
    pool = torch.empty(blocks, kv, 68 * d, dtype=torch.uint8, device=DEV)
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
    # keys have a few channels far above the others
    gain = torch.where(torch.rand(kv, d, generator=g, device=DEV) < 0.05, 8.0, 1.0)
    return cells, blocks, _normal(g, n, kv, d) * gain, _normal(g, n, kv, d)


def _prep_cache(c, seed):
    cells, blocks, k, v = _cache_inputs(c, seed)
    kv, d = c["kv"], c["dim"]
    pools = [torch.zeros(blocks, kv, 68 * d, dtype=torch.uint8, device=DEV) for _ in range(2)]
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
            hip.check(L.lgmlh_kv_store_q8(s["pools"][0].data_ptr(), s["pools"][1].data_ptr(), s["n_cells"], kv,
                                          d, s["k"].data_ptr(), s["v"].data_ptr(), s["cells"].data_ptr(),
                                          s["host"].ctypes.data, n, st))
        for w in range(2):
            hip.check(L.lgmlh_kv_gather_q8(s["pools"][w].data_ptr(), w, s["n_cells"], kv, d,
                                           s["cells"].data_ptr(), n, s["out"][w].data_ptr(),
                                           hip.F32 if c["out"] == "f32" else hip.F16, st))
        return s["out"]
    if c["dir"] == "write":
        _rows_in(s["pools"][0], d, 0, s["cells"], s["k"])
        _rows_in(s["pools"][1], d, 1, s["cells"], s["v"])
    dt = s["out"][0].dtype
    return [_rows_out(s["pools"][w], d, w, s["cells"]).to(dt).flatten(1) for w in range(2)]


def _move_inputs(c, seed):
    """Cells from and to: sequence s keeps `accept` of its drafted tokens, the
    first among them, and each goes behind the context in order."""
    rng = random.Random(seed * 7919 + 5)
    starts = [rng.randint(0, 63) for _ in range(c["seqs"])]
    tab, blocks = _tables([63 + c["nodes"]] * c["seqs"], seed)
    src, dst = [], []
    for s, p in enumerate(starts):
        kept = [0] + sorted(rng.sample(range(c["accept"], c["nodes"]), c["accept"] - 1))
        at = [int(tab[s][(p + i) // 64]) * 64 + (p + i) % 64 for i in range(c["nodes"])]
        src += [at[i] for i in kept]
        dst += at[:c["accept"]]
    return np.array(src, np.int64), np.array(dst, np.int64), blocks


def _move_pools(c, seed, blocks):
    g = torch.Generator(DEV).manual_seed(seed + 1)
    kv, d, n = c["kv"], c["dim"], 2 * c["layers"]
    if c["pool"] == "f16":
        return torch.randn(n, blocks, kv, 64 * d, generator=g, device=DEV, dtype=torch.float16)
    return torch.stack([_q8_pool(g, blocks, kv, d, p % 2) for p in range(n)])


def _prep_move(c, seed):
    src, dst, blocks = _move_inputs(c, seed)
    pools = _move_pools(c, seed, blocks)
    n, kv, d = len(pools), c["kv"], c["dim"]
    addr = torch.tensor([p.data_ptr() for p in pools], dtype=torch.int64, device=DEV)
    out = torch.empty(n, len(src), kv * d, device=DEV) if c["pool"] == "q8" else None
    return dict(c=c, pools=pools, addr=addr, src=torch.from_numpy(src).to(DEV),
                dst=torch.from_numpy(dst).to(DEV), h_src=src, h_dst=dst, n_cells=64 * blocks, out=out)


def _run_move(s):
    c, pools, kv, d = s["c"], s["pools"], s["c"]["kv"], s["c"]["dim"]
    f16 = c["pool"] == "f16"
    if own:
        from lgml_amd import hip
        L, st = hip.lib(), hip.stream()
        hip.check(L.lgmlh_kv_move(hip.F16 if f16 else hip.Q8_0, s["addr"].data_ptr(), len(pools), s["n_cells"],
                                  kv, d, s["src"].data_ptr(), s["dst"].data_ptr(), s["h_src"].ctypes.data,
                                  s["h_dst"].ctypes.data, len(s["h_src"]), st))
        if f16:
            return pools
        for p in range(len(pools)):
            hip.check(L.lgmlh_kv_gather_q8(pools[p].data_ptr(), p % 2, s["n_cells"], kv, d, s["dst"].data_ptr(),
                                           len(s["h_src"]), s["out"][p].data_ptr(), hip.F32, st))
        return s["out"]
    sb, sc, db, dc = s["src"] // 64, s["src"] % 64, s["dst"] // 64, s["dst"] % 64
    if f16:
        k = pools[0::2].unflatten(-1, (64, d))
        v = pools[1::2].unflatten(-1, (d, 64))
        k[:, db, :, dc] = k[:, sb, :, sc]
        v[:, db, :, :, dc] = v[:, sb, :, :, sc]
        return pools
    rows = []
    for p in range(len(pools)):
        if p % 2 == 0:
            vals, scale = _k_views(pools[p], d)
            vals[db, dc] = vals[sb, sc]
        else:
            vals, scale = _v_views(pools[p], d)
            vals[db, dc // 32, dc % 32 // 8, dc % 8] = vals[sb, sc // 32, sc % 32 // 8, sc % 8]
        scale[db, dc] = scale[sb, sc]
        rows.append(_rows_out(pools[p], d, p % 2, s["dst"]).flatten(1))
    return torch.stack(rows)


def _contexts(c, seed):
    rng = random.Random(seed * 7919 + 5)
    past = [rng.randint(c["lo"], c["hi"]) for _ in range(c["seqs"])]
    past[0], past[-1] = c["lo"], c["hi"]
    return past


def _parents(c, seed):
    """A tree per sequence: node 0 follows the context, the others follow one
    of the eight before them."""
    rng = random.Random(seed * 7919 + 17)
    return [[-1] + [rng.randrange(max(0, j - 8), j) if c["tree"] else j - 1 for j in range(1, c["nodes"])]
            for _ in range(c["seqs"])]


def _attention_inputs(c, seed):
    g = torch.Generator(DEV).manual_seed(seed + 1)
    past = _contexts(c, seed)
    tab, blocks = _tables([p + c["nodes"] for p in past], seed)
    kv, d = c["kv"], c["dim"]
    q = _normal(g, c["seqs"] * c["nodes"], c["heads"], d)
    if c["pool"] == "f16":
        k = torch.randn(blocks, kv, 64, d, generator=g, device=DEV, dtype=torch.float16)
        v = torch.randn(blocks, kv, d, 64, generator=g, device=DEV, dtype=torch.float16)
    else:
        k, v = _q8_pool(g, blocks, kv, d, 0), _q8_pool(g, blocks, kv, d, 1)
    return past, tab, blocks, q, k, v


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
        L = hip.lib()
        fn = L.lgmlh_paged_attention if c["pool"] == "f16" else L.lgmlh_paged_attention_q8
        hip.check(fn(q.data_ptr(), h, kv, d, d ** -0.5, s["k"].data_ptr(), s["v"].data_ptr(),
                     C.byref(s["plan"].ub), s["out"].data_ptr(), s["ws"].data_ptr(), s["ws"].numel(),
                     hip.stream()))
        return s["out"]
    out = []
    for i, p in enumerate(s["past"]):
        t = s["tables"][i][:(p + n + 63) // 64]
        if c["pool"] == "f16":
            k = s["k"][t].float().transpose(0, 1).flatten(1, 2)[:, :p + n]              # (kv, cells, d)
            v = s["v"][t].float().permute(1, 0, 3, 2).flatten(1, 2)[:, :p + n]
        else:
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


def _logits(c, seed):
    """Rows of N(0, 2.5) logits, one token in half of them far above; masked:
    a grammar leaves a tenth of the vocabulary. Given tokens: half of them
    likely ones."""
    g = torch.Generator(DEV).manual_seed(seed + 1)
    r, v = c["rows"], c["vocab"]
    x = _normal(g, r, v) * 2.5
    peak = torch.randint(v, (r, 1), generator=g, device=DEV)
    x.scatter_add_(1, peak, (torch.rand(r, 1, generator=g, device=DEV) < 0.5) * 15.0)
    if c["masked"]:
        off = torch.rand(v, generator=g, device=DEV) < 0.9
        off[:64] = False
        x.masked_fill_(off[None] & (torch.arange(v, device=DEV)[None] != peak), -math.inf)
        ids = torch.randint(64, (r, c["ids"]), generator=g, device=DEV)
    else:
        ids = torch.randint(v, (r, c["ids"]), generator=g, device=DEV)
    ids[:, ::2] = peak
    return x, ids.to(torch.int32)


def _prep_logprobs(c, seed):
    x, ids = _logits(c, seed)
    r, k = c["rows"], c["top"]
    s = dict(c=c, x=x, ids=ids)
    if own:
        from lgml_amd import hip
        ws = hip.lib().lgmlh_log_probs_workspace(r, c["vocab"], k)
        s.update(lp=torch.empty(r, c["ids"], device=DEV), ent=torch.empty(r, device=DEV),
                 top=torch.empty(r, k, dtype=torch.int32, device=DEV), top_lp=torch.empty(r, k, device=DEV),
                 ws=torch.empty(max(ws, 1), dtype=torch.uint8, device=DEV))
    return s


def _run_logprobs(s):
    c, x, ids = s["c"], s["x"], s["ids"]
    if own:
        from lgml_amd import hip
        hip.check(hip.lib().lgmlh_log_probs(x.data_ptr(), c["rows"], c["vocab"], ids.data_ptr(), c["ids"],
                                            s["lp"].data_ptr(), s["ent"].data_ptr(), c["top"],
                                            s["top"].data_ptr(), s["top_lp"].data_ptr(), s["ws"].data_ptr(),
                                            s["ws"].numel(), hip.stream()))
        return dict(lp=s["lp"], entropy=s["ent"], top=s["top"], top_lp=s["top_lp"])
    d = x.double()  # 64 bits: near a certain token, log Z is what is left of 1 + a little
    d = d - d.amax(1, keepdim=True)
    e = d.exp()
    z = e.sum(1, keepdim=True)
    lp = d - z.log()
    ent = z.log()[:, 0] - torch.where(e > 0, e * d, 0.0).sum(1) / z[:, 0]
    top = x.sort(dim=1, descending=True, stable=True).indices[:, :c["top"]]
    return dict(lp=lp.gather(1, ids.long()).float(), entropy=ent.float(), top=top.to(torch.int32),
                top_lp=lp.gather(1, top).float())


_PREPARE = dict(cache=_prep_cache, move=_prep_move, attention=_prep_attention, logprobs=_prep_logprobs)
_RUN = dict(cache=_run_cache, move=_run_move, attention=_run_attention, logprobs=_run_logprobs)


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
            return dict(bytes=n * (1.0625 + out), flops=n)
        return dict(bytes=n * (4 + 1.0625 + out), flops=4.0 * n)
    if kind == "move":
        n = 2.0 * c["layers"] * c["seqs"] * c["accept"] * c["kv"] * c["dim"]
        return dict(bytes=2 * n * (2.0 if c["pool"] == "f16" else 1.0625), flops=0.0)
    if kind == "attention":
        mean, n = (c["lo"] + c["hi"]) / 2, c["nodes"]
        size = 2.0 if c["pool"] == "f16" else 1.0625
        return dict(bytes=c["seqs"] * (2 * (mean + n) * c["kv"] * c["dim"] * size + 8.0 * n * c["heads"] * c["dim"]),
                    flops=4.0 * c["seqs"] * n * (mean + n / 2) * c["heads"] * c["dim"])
    r, v = c["rows"], c["vocab"]
    return dict(bytes=4.0 * r * (v + 2 * c["ids"] + 1 + 2 * c["top"]), flops=4.0 * r * v)


# ---- the definitions in 64 bits ------------------------------------------------
def _quantised(x):
    """The values that 8 bits keep of x (n, kv, D): its steps are the format's
    definition, d and 1 / d and x / d rounded to 32 bits, d kept in 16."""
    n, kv, d = x.shape
    g = x.double().view(n, kv, d // 32, 32)
    big = (g.abs().max(3).values / 127).float()
    inv = torch.where(big > 0, (1 / big.double()).float(), 0.0)
    y = (g * inv.double()[..., None]).float().double()
    return (y.sign() * (y.abs() + 0.5).floor() * big.half().double()[..., None]).view(n, kv, d)


def _held(pool, d, which, cells):
    """What cells of a Q8_0 pool stand for, (n, kv, D), by each value's place in its tile."""
    x = torch.arange(d, device=DEV)
    cell = (cells % 64)[:, None]
    if which == 0:
        at = ((x // 64 * 64 + cell) * 4 + x % 32 // 8) * 16 + x % 64 // 32 * 8 + x % 8
    else:
        at = x * 64 + cell % 32 // 8 * 16 + cell // 32 * 8 + cell % 8
    scale = 64 * d + 2 * (x // 32 * 64 + cell)
    n, kv = len(cells), pool.shape[1]
    t = pool[cells // 64].to(torch.int64)                                              # (n, kv, 68 D)
    byte = lambda i: t.gather(2, i[:, None].expand(n, kv, d))
    q = byte(at)
    bits = (byte(scale) + 256 * byte(scale + 1)).to(torch.int32)
    bits = torch.where(bits > 32767, bits - 65536, bits).to(torch.int16)
    return torch.where(q > 127, q - 256, q).double() * bits.view(torch.float16).double()


def _exact_cache(c, seed):
    _, _, k, v = _cache_inputs(c, seed)
    dt = torch.float64 if c["out"] == "f32" else torch.float16
    return [_quantised(x).flatten(1).to(dt).double() for x in (k, v)]


def _exact_move(c, seed):
    src, dst, blocks = _move_inputs(c, seed)
    pools = _move_pools(c, seed, blocks)
    kv, d = c["kv"], c["dim"]
    if c["pool"] == "q8":
        at = torch.from_numpy(src).to(DEV)
        return torch.stack([_held(pools[p], d, p % 2, at).flatten(1) for p in range(len(pools))])
    new = pools.clone()
    for a, b in zip(src.tolist(), dst.tolist()):
        k0, k1 = pools[0::2].view(-1, blocks, kv, 64, d), new[0::2].view(-1, blocks, kv, 64, d)
        v0, v1 = pools[1::2].view(-1, blocks, kv, d, 64), new[1::2].view(-1, blocks, kv, d, 64)
        k1[:, b // 64, :, b % 64] = k0[:, a // 64, :, a % 64]
        v1[:, b // 64, :, :, b % 64] = v0[:, a // 64, :, :, a % 64]
    return new.double()


def _exact_attention(c, seed):
    past, tab, blocks, q, k, v = _attention_inputs(c, seed)
    h, kv, d, n = c["heads"], c["kv"], c["dim"], c["nodes"]
    out = torch.empty(len(q), h, d, dtype=torch.float64, device=DEV)
    for i, (p, par) in enumerate(zip(past, _parents(c, seed))):
        cells = torch.from_numpy(_cells([0], [p + n], tab[i:i + 1])).to(DEV)
        if c["pool"] == "f16":
            ks = k.view(blocks, kv, 64, d)[cells // 64, :, cells % 64].double()
            vs = v.view(blocks, kv, d, 64)[cells // 64, :, :, cells % 64].double()
        else:
            ks, vs = (torch.cat([_held(x, d, w, part) for part in cells.split(1024)]) for w, x in ((0, k), (1, v)))
        ks, vs = ks.permute(1, 2, 0).contiguous(), vs.permute(1, 0, 2).contiguous()
        for j in range(n):
            far = torch.zeros(p + n, dtype=torch.float64, device=DEV)
            line, at = [], j
            while at >= 0:
                line.append(p + at)
                at = par[at]
            far[p:] = -math.inf
            far[torch.tensor(line, device=DEV)] = 0.0
            x = torch.bmm(q[i * n + j].double().view(kv, h // kv, d), ks) * d ** -0.5 + far
            out[i * n + j] = torch.bmm(torch.softmax(x, 2), vs).view(h, d)
    return out


def _exact_logprobs(c, seed):
    x, ids = _logits(c, seed)
    x = x.double()
    lp = x - torch.logsumexp(x, 1, keepdim=True)
    at = torch.arange(c["vocab"], device=DEV)
    left, top = x.clone(), []
    for _ in range(c["top"]):
        best = torch.where(left == left.amax(1, keepdim=True), at, c["vocab"]).amin(1, keepdim=True)
        top.append(best)
        left.scatter_(1, best, -math.inf)
    top = torch.cat(top, 1)
    ent = -torch.where(lp > -1e4, lp.exp() * lp, 0.0).sum(1)
    return dict(lp=lp.gather(1, ids.long()), entropy=ent, top=top.to(torch.int32), top_lp=lp.gather(1, top))


def exact(case, seed):
    return dict(cache=_exact_cache, move=_exact_move, attention=_exact_attention,
                logprobs=_exact_logprobs)[case["kind"]](case, seed)
