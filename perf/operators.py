"""Cases that time the paged 4-bit cache operators and check what they compute.

The operators serve sequences of different lengths from one pool of pages:
rows are appended to a 4-bit key/value cache (and read back), attention reads
it with a sliding window and first tokens that stay visible, pages are forked,
freed and compacted, and drafted tokens are verified against the target's
probabilities. With ``own`` false every case runs in its plain form,
elementary torch operations; with ``own`` true it runs through needle_b200.

A tile of the cache holds 16 positions of one kv head: key codes [16][dk / 2]
bytes, value codes [16][dv / 2], the keys' f16 (scale, minimum) pairs, the
values' pairs; two codes a byte, the lower dimension in the low nibble. A page
holds its heads one after another, each page / 16 tiles; value = minimum +
scale * code.
"""

import math
import os
import sys

import numpy as np
import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "needle-rs_b200")
_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}

# Head layouts: the Needle 3 model's (12 query heads on 2 kv heads, keys of 48
# and values of 64), and two generic ones.
_HEADS = {"needle": (12, 2, 48, 64), "small": (8, 8, 64, 64), "wide": (32, 8, 128, 128)}


def _nb():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import needle_b200

    return needle_b200


def listed():
    return [
        # one session's next token early in its first turn: the smallest call
        dict(name="attend one session", op="attend", heads="needle", dtype="f32", S=1, T=1, L=40, page=16, window=0,
             sink=0, ragged=False, mix=0),
        # the agent workload's decode step: 1024 sequences of up to 256 positions
        dict(name="attend agent decode", op="attend", heads="needle", dtype="f32", S=1024, T=1, L=256, page=16,
             window=0, sink=0, ragged=True, mix=1),
        # few sequences with a long history: the cache streams from HBM
        dict(name="attend long decode", op="attend", heads="wide", dtype="bf16", S=8, T=1, L=32768, page=64, window=0,
             sink=0, ragged=True, mix=2),
        # a draft of four and the token before it, inside the model's window of
        # 1024 with a static prefix that stays visible
        dict(name="attend draft in window", op="attend", heads="needle", dtype="f16", S=256, T=5, L=3456, page=32,
             window=1024, sink=118, ragged=True, mix=3),
        # chunks of prompts over what the sequences hold already
        dict(name="attend prompt chunk", op="attend", heads="wide", dtype="bf16", S=4, T=512, L=4096, page=64,
             window=0, sink=0, ragged=True, mix=4),
        # every sequence's new token into the cache, and the rows as it keeps them
        dict(name="append a token each", op="append", heads="needle", dtype="f32", S=1024, T=1, L=256, page=16,
             ragged=True, mix=5),
        # whole prompts into the cache
        dict(name="append prompts", op="append", heads="wide", dtype="bf16", S=16, T=1024, L=2048, page=64,
             ragged=True, mix=6),
        # one search of four beams: a step's reordering
        dict(name="fork four beams", op="fork", B=1, W=4, prompt=118, tail=45, page=16, elems=512, layers=1, mix=7),
        # 64 searches of 16 beams over a pool that holds several layers
        dict(name="fork many beams", op="fork", B=64, W=16, prompt=700, tail=90, page=16, elems=4096, layers=4, mix=8),
        # a pool half empty after sequences ended: live pages to the front
        dict(name="compact a pool", op="compact", S=256, L=1000, page=16, N=24576, elems=4096, layers=1, mix=9),
        # one session's four drafted tokens
        dict(name="verify one session", op="verify", dtype="f32", S=1, T=4, V=16384, q=True, ragged=False, mix=10),
        # a batch's drafts
        dict(name="verify a batch", op="verify", dtype="f32", S=256, T=7, V=16384, q=True, ragged=True, mix=11),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    while True:
        op = rng.choice(["attend", "attend", "attend", "append", "fork", "compact", "verify"])
        mix = rng.randrange(1 << 20)
        if op in ("attend", "append"):
            heads = rng.choice(["needle", "small", "wide"])
            c = dict(op=op, heads=heads, dtype=rng.choice(["f32", "bf16", "f16"]), S=_log(rng, 1, 1024),
                     T=rng.choice([1, 1, rng.randint(2, 8), _log(rng, 9, 512 if op == "attend" else 1024)]), L=0,
                     page=rng.choice([16, 32, 64, 128]), ragged=rng.random() < 0.7, mix=mix)
            c["L"] = _log(rng, c["T"], 32768)
            if op == "attend":
                c["window"] = rng.choice([0, 0, _log(rng, 1, 4096)])
                c["sink"] = rng.choice([0, rng.randint(1, 200)]) if c["window"] else 0
            hq, h, dk, dv = _HEADS[heads]
            cells = c["S"] * c["L"] * h * (dk + dv)
            scores = c["S"] * c["T"] * hq * c["L"]
            if cells > 5.4e8 or (op == "attend" and (scores > 2.7e8 or c["S"] * c["T"] > 8192)) or c["S"] * c["T"] > 16384:
                continue
        elif op == "fork":
            c = dict(op=op, B=_log(rng, 1, 64), W=rng.randint(1, 16), prompt=_log(rng, 1, 1500), tail=_log(rng, 1, 200),
                     page=rng.choice([16, 32, 64]), elems=8 * _log(rng, 8, 1024), layers=rng.choice([1, 2, 4]), mix=mix)
        elif op == "compact":
            S, L, page = _log(rng, 1, 256), _log(rng, 10, 2000), rng.choice([16, 32, 64])
            c = dict(op=op, S=S, L=L, page=page, N=int(S * -(-L // page) * rng.uniform(1.02, 3)) + rng.randint(1, 9),
                     elems=8 * _log(rng, 8, 512), layers=rng.choice([1, 2]), mix=mix)
        else:
            c = dict(op=op, dtype=rng.choice(["f32", "f32", "bf16", "f16"]), S=_log(rng, 1, 256), T=rng.randint(1, 10),
                     V=_log(rng, 500, 130000), q=rng.random() < 0.7, ragged=rng.random() < 0.7, mix=mix)
            if c["S"] * (c["T"] + 1) * c["V"] > 256 * 8 * 16384:
                continue
        if op in ("fork", "compact") and _pool_pages(c) * c["elems"] * c["layers"] > 1.6e8:
            continue
        return c


# ------------------------------------------------------------------ inputs


def _spans(c):
    """(lens, n): positions held and new rows of each sequence."""
    r = np.random.RandomState(1000 + c["mix"])
    S, T, L = c["S"], c["T"], c["L"]
    if not c["ragged"]:
        return np.full(S, L), np.full(S, T)
    n = np.full(S, T) if T == 1 else r.randint(max(1, T // 2), T + 1, S)
    if S > 2:
        n[1] = 0  # a sequence that gets nothing this time
    lens = np.maximum(r.randint(max(1, L // 2), L + 1, S), n)
    lens[0], n[0] = L, T
    if S > 3:
        lens[2] = n[2]  # a new sequence: its rows are all it holds
    return lens, n


def _visible(c, lens, n):
    """(row, key) pairs that attention computes, and positions it reads."""
    w, sink = c["window"], c["sink"]
    pairs = cells = 0
    for length, rows in zip(lens.tolist(), n.tolist()):
        if not rows:
            continue
        pos = np.arange(length - rows, length)
        lo = np.maximum(pos - w + 1, 0) if w else np.zeros_like(pos)
        pairs += int((pos + 1 - lo + np.minimum(sink, lo)).sum())
        cells += length - int(lo[0]) + min(sink, int(lo[0]))
    return pairs, cells


def _pool_pages(c):
    if c["op"] == "compact":
        return c["N"]
    D, cols, full = c["B"] * c["W"], -(-(c["prompt"] + c["tail"]) // c["page"]) + 1, c["prompt"] // c["page"]
    return (c["B"] * full + D * (cols - full)) * 5 // 4 + D


def _values(g, *shape):
    """Keys or values as projections give them: normal, with a few channels that stand out."""
    x = torch.randn(shape, device="cuda", generator=g)
    return x * (1 + 4 * (torch.arange(shape[-1], device="cuda") % 17 == 3)) + 0.3


def _codes(x):
    """The cache's f32 arithmetic: rows of x to (codes, scales, minima)."""
    lo, hi = x.amin(-1), x.amax(-1)
    s = ((hi - lo) / torch.full_like(lo, 15.0)).clamp(max=65504.0).half()
    m = lo.clamp(-65504.0, 65504.0).half()
    sf, mf = s.float()[..., None], m.float()[..., None]
    c = torch.where(sf > 0, ((x - mf) / sf).round().clamp(0, 15), torch.zeros_like(x))
    return c.to(torch.uint8), s, m


def _bytes_of(x):
    """(code bytes, (scale, minimum) bytes) of rows of x."""
    c, s, m = _codes(x.float())
    return c[..., 0::2] | (c[..., 1::2] << 4), torch.stack((s, m), -1).contiguous().view(torch.uint8)


def _tile(dk, dv):
    return 16 * (dk // 2 + dv // 2 + 8)


def _paged(c, g, dev="cuda"):
    """(pool, table, lens, start, rows): a pool of random bytes with pages in
    random order; what the sequences hold is written in."""
    hq, h, dk, dv = _HEADS[c["heads"]]
    lens, n = _spans(c)
    P = -(-c["L"] // c["page"])
    used = -(-lens // c["page"])
    N = int(used.sum()) + 3
    pool = torch.randint(0, 256, (N, h, c["page"] // 16, _tile(dk, dv)), device=dev, dtype=torch.uint8, generator=g)
    ids = torch.randperm(N, device=dev, generator=g)
    lens_t = torch.tensor(lens, device=dev, dtype=torch.int32)
    used_t = torch.tensor(used, device=dev)
    col = torch.arange(P, device=dev)
    at = torch.cumsum(used_t, 0)[:, None] - used_t[:, None] + col
    table = torch.where(col < used_t[:, None], ids[at.clamp(max=N - 1)], torch.full_like(at, -1)).int()
    # earlier rows, a few thousand at a time
    seq = torch.repeat_interleave(torch.arange(c["S"], device=dev), lens_t.long())
    pos = torch.arange(seq.numel(), device=dev) - (torch.cumsum(lens_t, 0) - lens_t)[seq]
    for a in range(0, seq.numel(), 1 << 16):
        s, p = seq[a:a + (1 << 16)], pos[a:a + (1 << 16)]
        _plain_append(pool, _values(g, s.numel(), h, dk), _values(g, s.numel(), h, dv), table[s, p // c["page"]].long(),
                      p % c["page"])
    start = torch.tensor(np.concatenate([[0], np.cumsum(n)]), device=dev, dtype=torch.int32)
    return pool, table, lens_t, start, int(n.sum())


def _beams(c):
    """The old set of a beam step and what the new one asks for: lengths,
    parents, positions kept and wanted."""
    r = np.random.RandomState(2000 + c["mix"])
    B, W, D = c["B"], c["W"], c["B"] * c["W"]
    lens = np.repeat(c["prompt"] + r.randint(1, c["tail"] + 1, B), W)
    src = np.repeat(np.arange(B) * W, W) + r.randint(0, W, D)
    drop = np.where(r.rand(D) < 0.25, r.randint(0, 5, D), 0)  # drafted positions that were refused
    keep = np.maximum(lens[np.maximum(src, 0)] - drop, 1)
    need = keep + r.randint(1, 6, D)
    if D > 8:
        src[5] = -1  # a search that ended and one that starts anew
        keep[5], need[5] = 0, c["prompt"]
    return lens, src, keep, need


def _beam_table(c, lens, ids):
    """Prompts' whole pages shared by a group's beams, the rest their own."""
    B, W, page = c["B"], c["W"], c["page"]
    cols, full = -(-(c["prompt"] + c["tail"]) // page) + 1, c["prompt"] // page
    col = np.arange(cols)[None]
    d = np.arange(B * W)[:, None]
    at = np.where(col < full, (d // W) * full + col, B * full + d * (cols - full) + col - full)
    return np.where(col < -(-lens // page)[:, None], ids[at], -1).astype(np.int32)


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    st = dict(c=c)
    if c["op"] in ("attend", "append"):
        hq, h, dk, dv = _HEADS[c["heads"]]
        pool, table, lens, start, rows = _paged(c, g)
        st.update(pool=pool, table=table, lens=lens, start=start, rows=rows)
        t = _TYPES[c["dtype"]]
        if c["op"] == "attend":
            st["q"] = _values(g, rows, hq, dk).to(t)
        else:
            st["k"], st["v"] = _values(g, rows, h, dk).to(t), _values(g, rows, h, dv).to(t)
    elif c["op"] in ("fork", "compact"):
        N = _pool_pages(c)
        ids = np.random.RandomState(seed % (1 << 31)).permutation(N)
        shape = (N, c["elems"]) if c["layers"] == 1 else (c["layers"], N, c["elems"])
        st["pool"] = torch.randn(shape, device="cuda", generator=g, dtype=torch.bfloat16)
        if c["op"] == "fork":
            lens, src, keep, need = _beams(c)
            table = _beam_table(c, lens, ids)
            for name, v in (("src", src), ("keep", keep), ("need", need)):
                st[name] = torch.tensor(v, device="cuda", dtype=torch.int32)
        else:
            r = np.random.RandomState(3000 + c["mix"])
            cols = -(-c["L"] // c["page"])
            used = r.randint(max(1, cols // 2), cols + 1, c["S"])
            table = np.where(np.arange(cols)[None] < used[:, None], ids[: c["S"] * cols].reshape(c["S"], cols), -1)
        st["table"] = torch.tensor(table, device="cuda", dtype=torch.int32)
    else:
        S, T, V = c["S"], c["T"], c["V"]
        logits = torch.randn((S, T + 1, V), device="cuda", generator=g) * 2
        logits[..., : max(1, V // 400)] += 5
        n = np.random.RandomState(4000 + c["mix"]).randint(0, T + 1, S) if c["ragged"] else np.full(S, T)
        n[0] = T
        # every fourth sequence is greedy, the others sample at their own temperature
        temp = torch.rand(S, device="cuda", generator=g) + 0.5
        temp[3::4] = 0
        near = torch.softmax((logits[:, :T] + 0.5 * torch.randn((S, T, V), device="cuda", generator=g))
                             / temp.clamp(min=0.3)[:, None, None], -1)
        st["draft"] = torch.multinomial(near.view(S * T, V), 1, generator=g).view(S, T).int()
        st["q"] = near if c["q"] else None
        st["u"] = torch.rand((S, T + 1), device="cuda", generator=g)
        st["logits"] = logits.to(_TYPES[c["dtype"]])
        st["temp"], st["n"] = temp, torch.tensor(n, device="cuda", dtype=torch.int32)
    return st


# ------------------------------------------------------------- plain forms


def _row_places(st):
    """(sequence, index in its new rows, position) of every new row."""
    start, lens = st["start"].long(), st["lens"].long()
    r = torch.arange(st["rows"], device=start.device)
    seq = torch.bucketize(r, start[1:], right=True)
    i = r - start[seq]
    return seq, i, lens[seq] - (start[seq + 1] - start[seq]) + i


def _plain_append(pool, k, v, page, at):
    """Rows k, v into slot `at` of their page (page ids in range)."""
    h, dk, dv = k.shape[1], k.shape[2], v.shape[2]
    t, j = (at // 16)[:, None, None], (at % 16)[:, None, None]
    head = torch.arange(h, device=k.device)[None, :, None]
    page = page[:, None, None]

    def put(x, d, base, pbase):
        code, par = _bytes_of(x)
        pool[page, head, t, base + j * (d // 2) + torch.arange(d // 2, device=x.device)] = code
        pool[page, head, t, pbase + j * 4 + torch.arange(4, device=x.device)] = par

    put(k, dk, 0, 8 * (dk + dv))
    put(v, dv, 8 * dk, 8 * (dk + dv) + 64)


def _plain_values(tiles, dk, dv):
    """Tiles [..., tile] to keys [..., 16, dk] and values [..., 16, dv]."""
    def one(code, par, d):
        b = code.reshape(*code.shape[:-1], 16, d // 2)
        c = torch.stack((b & 15, b >> 4), -1).flatten(-2).float()
        p = par.contiguous().view(torch.float16).reshape(*par.shape[:-1], 16, 2).float()
        return p[..., 1:] + p[..., :1] * c

    a, b = 8 * dk, 8 * (dk + dv)
    return (one(tiles[..., :a], tiles[..., b:b + 64], dk), one(tiles[..., a:b], tiles[..., b + 64:b + 128], dv))


def _plain_read(st, dk, dv):
    c, pool = st["c"], st["pool"]
    seq, _, pos = _row_places(st)
    page = st["table"].long()[seq, pos // c["page"]]
    tiles = pool[page, :, (pos % c["page"]) // 16]  # [rows, heads, tile]
    k, v = _plain_values(tiles, dk, dv)
    r = torch.arange(st["rows"], device=pool.device)
    return k[r, :, pos % 16], v[r, :, pos % 16]


def _plain_attend(st):
    c, q, pool, lens = st["c"], st["q"], st["pool"], st["lens"].long()
    hq, h, dk, dv = _HEADS[c["heads"]]
    S, T, G = c["S"], c["T"], hq // h
    tiles = pool[st["table"].long().clamp(min=0)]  # [S, P, h, page / 16, tile]
    tiles = tiles.permute(0, 2, 1, 3, 4).reshape(S, h, -1, pool.shape[-1])
    k, v = _plain_values(tiles, dk, dv)
    k, v = k.flatten(2, 3), v.flatten(2, 3)
    L = k.shape[2]
    key = torch.arange(L, device=q.device)
    held = (key < lens[:, None])[:, None, :, None]
    k, v = torch.where(held, k, 0.0), torch.where(held, v, 0.0)
    seq, i, pos = _row_places(st)
    qp = torch.zeros((S, T, hq, dk), device=q.device)
    qp[seq, i] = q.float()
    at = torch.full((S, T), -1, device=q.device, dtype=torch.long)
    at[seq, i] = pos
    qp = qp.view(S, T, h, G, dk).permute(0, 2, 1, 3, 4).reshape(S, h, T * G, dk)
    s = (qp @ k.transpose(2, 3)).view(S, h, T, G, L) * (1.0 / math.sqrt(dk))
    seen = key <= at[..., None]
    if c["window"]:
        seen &= (key > at[..., None] - c["window"]) | (key < c["sink"])
    s = torch.where(seen[:, None, :, None], s, -math.inf)
    m = s.amax(-1, keepdim=True).clamp(min=-1e30)
    e = torch.exp(s - m)
    z = e.sum(-1, keepdim=True)
    o = (e / torch.where(z > 0, z, 1.0)).view(S, h, T * G, L) @ v
    o = o.view(S, h, T, G, dv).permute(0, 2, 1, 3, 4).reshape(S, T, hq, dv)
    return o[seq, i].to(q.dtype)


def _move(pool, src, dst, layers):
    if layers == 1:
        pool[dst] = pool[src]
    else:
        pool[:, dst] = pool[:, src]


def _count(ids, N):
    return torch.bincount(ids, minlength=N)[:N]


def _plain_fork(st):
    c, pool, table = st["c"], st["pool"], st["table"].long()
    page, N = c["page"], _pool_pages(c)
    src, keep, need = st["src"].long(), st["keep"].long(), st["need"].long()
    D, P, dev = src.numel(), table.shape[1], table.device
    has = (src >= 0) & (src < table.shape[0])
    par = table[src.clamp(0, table.shape[0] - 1)]
    keep = torch.where(has, keep.clamp(0, P * page), 0)
    need = torch.maximum(need.clamp(max=P * page), keep)
    nk, nn = (keep + page - 1) // page, (need + page - 1) // page
    col, d = torch.arange(P, device=dev)[None], torch.arange(D, device=dev)[:, None]
    kept = (col < nk[:, None]) & (par >= 0) & (par < N)
    writes = kept & ((keep % page > 0) & (need > keep))[:, None] & (col == nk[:, None] - 1)
    refs, wr = _count(par[kept], N), _count(par[writes], N)
    first = torch.full((N,), D, device=dev).scatter_reduce(0, par[writes], d.expand(D, P)[writes], "amin")
    pc = par.clamp(0, N - 1)
    copy = writes & ~((refs[pc] == 1) | ((refs[pc] == wr[pc]) & (first[pc] == d)))
    fresh = copy | ((col >= nk[:, None]) & (col < nn[:, None]))
    rank = torch.cumsum(fresh.flatten().long(), 0).view(D, P) - 1
    free = torch.nonzero(refs == 0).flatten()
    pad = torch.cat([free, torch.full((D * P,), -1, device=dev)])
    new = torch.where(fresh, pad[rank.clamp(min=0)], torch.where(kept, par, -1))
    made = copy & (new >= 0)
    _move(pool, par[made], new[made], c["layers"])
    refs = _count(new[new >= 0], N)
    given = (fresh & (new >= 0)).sum()
    info = torch.stack([(refs > 0).sum(), given, made.sum(), fresh.sum() - given])
    return dict(table=new.int(), refs=refs.int(), info=info.int(), pool=pool)


def _plain_compact(st):
    c, pool, table = st["c"], st["pool"], st["table"].long()
    N, dev = c["N"], table.device
    ok = (table >= 0) & (table < N)
    live = _count(table[ok], N) > 0
    n, ids = live.sum(), torch.arange(N, device=dev)
    movers, holes = torch.nonzero(live & (ids >= n)).flatten(), torch.nonzero(~live & (ids < n)).flatten()
    to = torch.where(live, ids, -1)
    to[movers] = holes
    _move(pool, movers, holes, c["layers"])
    return dict(table=torch.where(ok, to[table.clamp(0, N - 1)], -1).int(), map=to.int(),
                info=torch.stack([n, (to != ids)[live].sum()]).int(), pool=pool)


def _plain_verify(st):
    c, u, draft, n = st["c"], st["u"].double(), st["draft"].long(), st["n"].long()
    S, T, V = c["S"], c["T"], c["V"]
    lg, temp = st["logits"].double(), st["temp"].double()[:, None, None]
    top = lg.amax(-1, keepdim=True)
    ids = torch.arange(V, device=lg.device)
    first = torch.where(lg == top, ids, V).amin(-1, keepdim=True)
    e = torch.exp((lg - top) / torch.where(temp > 0, temp, 1.0))
    p = torch.where(temp > 0, e / e.sum(-1, keepdim=True), (ids == first).double())
    px = p[:, :T].gather(2, draft[..., None])[..., 0]
    qx = st["q"].gather(2, draft[..., None])[..., 0].double() if st["q"] is not None else torch.ones_like(px)
    ok = (u[:, :T] * qx < px) & (torch.arange(T, device=lg.device) < n[:, None])
    a = torch.cumprod(ok.long(), 1).sum(1)
    s = torch.arange(S, device=lg.device)
    pa = p[s, a]
    if st["q"] is not None:
        qa = st["q"][s, a.clamp(max=T - 1)].double()
    else:
        qa = (ids == draft[s, a.clamp(max=T - 1)][:, None]) * 2.0  # nothing is left of the refused token
    r = torch.where((a < n)[:, None], (pa - qa).clamp(min=0), pa)
    r = torch.where(r.sum(1, keepdim=True) > 0, r, pa)
    cum = torch.cumsum(r, 1)
    j = (cum <= u[:, T:] * cum[:, -1:]).sum(1)
    j = torch.minimum(j, torch.where(r > 0, ids, 0).amax(1))
    at = torch.arange(T + 1, device=lg.device)
    d1 = torch.cat([draft, draft[:, :1]], 1)
    p1 = torch.cat([px, px[:, :1]], 1)
    tok = torch.where(at < a[:, None], d1, torch.where(at == a[:, None], j[:, None], -1))
    pr = torch.where(at < a[:, None], p1, torch.where(at == a[:, None], pa.gather(1, j[:, None]), 0.0))
    return dict(tokens=tok.int(), accepted=a.int(), probs=pr.float())


def run(state):
    st, c = state, state["c"]
    if own:
        return _own(st)
    if c["op"] == "attend":
        return dict(out=_plain_attend(st))
    if c["op"] == "append":
        hq, h, dk, dv = _HEADS[c["heads"]]
        seq, _, pos = _row_places(st)
        _plain_append(st["pool"], st["k"], st["v"], st["table"].long()[seq, pos // c["page"]], pos % c["page"])
        k, v = _plain_read(st, dk, dv)
        return dict(k=k.to(st["k"].dtype), v=v.to(st["v"].dtype))
    if c["op"] == "fork":
        return _plain_fork(st)
    if c["op"] == "compact":
        return _plain_compact(st)
    return _plain_verify(st)


def _own(st):
    nb, c = _nb(), st["c"]
    if c["op"] in ("attend", "append"):
        if "kv" not in st:  # the handle a program keeps beside its pool
            hq, h, dk, dv = _HEADS[c["heads"]]
            st["kv"] = nb.KV4Pool(st["pool"], dk, dv)
        kv = st["kv"]
        if c["op"] == "attend":
            return dict(out=nb.op_kv4_attend(kv, st["q"], st["table"], st["lens"], st["start"], window=c["window"],
                                             sink=c["sink"]))
        nb.op_kv4_append(kv, st["k"], st["v"], st["table"], st["lens"], st["start"])
        k, v = nb.op_kv4_read(kv, st["table"], st["lens"], st["start"], rows=st["rows"], dtype=st["k"].dtype)
        return dict(k=k, v=v)
    axis = 0 if c.get("layers", 1) == 1 else 1
    if c["op"] == "fork":
        table, refs, info = nb.op_pages_fork(st["pool"], st["table"], st["src"], st["keep"], st["need"], c["page"],
                                             axis=axis)
        return dict(table=table, refs=refs, info=info, pool=st["pool"])
    if c["op"] == "compact":
        table, to, info = nb.op_pages_compact(st["pool"], st["table"], axis=axis)
        return dict(table=table, map=to, info=info, pool=st["pool"])
    tokens, accepted, probs = nb.op_verify(st["logits"], st["draft"], st["u"], st["temp"], q=st["q"], counts=st["n"])
    return dict(tokens=tokens, accepted=accepted, probs=probs)


# ------------------------------------------------------------- work, exact


def work(case):
    c = case
    if c["op"] in ("attend", "append"):
        hq, h, dk, dv = _HEADS[c["heads"]]
        lens, n = _spans(c)
        rows, row = int(n.sum()), h * (dk // 2 + dv // 2 + 8)
        if c["op"] == "append":  # rows in, codes out; codes in, rows out
            return dict(bytes=2.0 * rows * (h * (dk + dv) * _SIZE[c["dtype"]] + row), flops=4.0 * rows * h * (dk + dv))
        pairs, cells = _visible(c, lens, n)
        return dict(bytes=float(cells * row + rows * hq * (dk + dv) * _SIZE[c["dtype"]] + 4 * cells // c["page"]),
                    flops=2.0 * pairs * hq * (dk + dv))
    if c["op"] == "fork":
        lens, src, keep, need = _beams(c)
        N, D = _pool_pages(c), len(src)
        table = _beam_table(c, lens, np.arange(N))
        copies = _copies(table, src, keep, need, c["page"])
        small = 4 * (2 * table.size + 3 * D + N)
        return dict(bytes=float(small + 2 * copies * c["layers"] * c["elems"] * 2), flops=0.0)
    if c["op"] == "compact":
        r = np.random.RandomState(3000 + c["mix"])
        cols = -(-c["L"] // c["page"])
        n = int(r.randint(max(1, cols // 2), cols + 1, c["S"]).sum())
        moved = n * (1 - n / c["N"])  # pages lie at random: that share of them is past the n-th place
        return dict(bytes=float(4 * (2 * c["S"] * cols + c["N"]) + 2 * moved * c["layers"] * c["elems"] * 2), flops=0.0)
    S, T, V = c["S"], c["T"], c["V"]
    n = np.random.RandomState(4000 + c["mix"]).randint(0, T + 1, S) if c["ragged"] else np.full(S, T)
    n[0] = T
    rows = int(n.sum()) + S
    return dict(bytes=float(rows * V * _SIZE[c["dtype"]] + (S * V * 4 if c["q"] else 0)), flops=4.0 * rows * V)


def _copies(table, src, keep, need, page):
    """Pages a fork copies, counted page by page."""
    users, writers = {}, {}
    for d in range(len(src)):
        if src[d] < 0:
            continue
        k = -(-int(keep[d]) // page)
        for p in table[src[d], :k].tolist():
            users[p] = users.get(p, 0) + 1
        if keep[d] % page and need[d] > keep[d]:
            p = int(table[src[d], k - 1])
            writers[p] = writers.get(p, 0) + 1
    return sum(w - (w == users[p]) for p, w in writers.items())


def exact(case, seed):
    st = prepare(case, seed)
    c = case
    if c["op"] == "append":
        return _exact_append(st)
    if c["op"] == "attend":
        return _exact_attend(st)
    if c["op"] == "verify":
        return _exact_verify(st)
    return None  # whole numbers and moved bytes: nothing is rounded


def _f32(x):
    return x.float().double()


def _exact_append(st):
    """The format's definition: each step in 64 bits, rounded where the format says it is."""
    def one(x):
        y = x.double()
        lo, hi = y.min(-1).values, y.max(-1).values
        s = torch.clamp(_f32(_f32(hi - lo) / 15), max=65504.0).float().half().double().unsqueeze(-1)
        m = lo.clamp(-65504.0, 65504.0).float().half().double().unsqueeze(-1)
        code = torch.round(_f32(_f32(y - m) / s)).clamp(0, 15)
        return (m + s * torch.nan_to_num(code)).to(torch.float32).to(x.dtype)

    return dict(k=one(st["k"]), v=one(st["v"]))


def _exact_attend(st):
    c = st["c"]
    hq, h, dk, dv = _HEADS[c["heads"]]
    page, G = c["page"], hq // h
    lens, start = st["lens"].tolist(), st["start"].tolist()
    out = torch.zeros((st["rows"], hq, dv), device="cuda", dtype=torch.float64)
    nib = 4 * torch.arange(2, device="cuda", dtype=torch.uint8)
    for s in range(c["S"]):
        a, b, L = start[s], start[s + 1], lens[s]
        if a == b:
            continue
        first = max(0, L - (b - a) - c["window"] + 1) // 16 * 16 if c["window"] and not c["sink"] else 0
        at = torch.arange(first, L, device="cuda")
        t = st["pool"][st["table"][s].long()[at // page], :, (at % page) // 16]  # [L, h, tile]
        rows = torch.arange(at.numel(), device="cuda"), slice(None), at % 16

        def vals(lo, d, plo):
            code = t[..., lo:lo + 8 * d].reshape(-1, h, 16, d // 2)[rows]
            code = ((code[..., None] >> nib) & 15).reshape(-1, h, d).double()
            par = t[..., plo:plo + 64].contiguous().view(torch.float16).view(-1, h, 16, 2)[rows].double()
            return par[..., 1:2] + par[..., 0:1] * code

        k, v = vals(0, dk, 8 * (dk + dv)), vals(8 * dk, dv, 8 * (dk + dv) + 64)
        pos = torch.arange(L - (b - a), L, device="cuda")[:, None]
        seen = at <= pos
        if c["window"]:
            seen = seen & ((at > pos - c["window"]) | (at < c["sink"]))
        q = st["q"][a:b].double().view(b - a, h, G, dk)
        for lo in range(0, b - a, 64):  # some rows at a time: the scores are large
            x = torch.einsum("thgd,lhd->hgtl", q[lo:lo + 64], k) / math.sqrt(dk)
            x = x.masked_fill(~seen[lo:lo + 64], -math.inf)
            out[a + lo:min(b, a + lo + 64)] = torch.einsum("hgtl,lhd->thgd", torch.softmax(x, -1), v).reshape(-1, hq, dv)
    return dict(out=out)


def _exact_verify(st):
    c = st["c"]
    S, T, V = c["S"], c["T"], c["V"]
    tokens, probs = np.full((S, T + 1), -1), np.zeros((S, T + 1))
    accepted = np.zeros(S, np.int64)
    for s in range(S):
        lg = st["logits"][s].double().cpu().numpy()
        q = st["q"][s].double().cpu().numpy() if st["q"] is not None else None
        x, u = st["draft"][s].tolist(), st["u"][s].double().tolist()
        temp, n = float(st["temp"][s].double()), int(st["n"][s])
        for i in range(n + 1):
            if temp > 0:
                w = np.exp((lg[i] - lg[i].max()) / temp)
                p = w / w.sum()
            else:
                p = np.zeros(V)
                p[int(np.argmax(lg[i]))] = 1.0
            if i < n and u[i] * (q[i][x[i]] if q is not None else 1.0) < p[x[i]]:
                tokens[s, i], probs[s, i] = x[i], p[x[i]]
                continue
            r = p.copy()
            if i < n:
                r = np.maximum(p - q[i], 0.0) if q is not None else np.where(np.arange(V) == x[i], 0.0, p)
            if not r.sum() > 0:
                r = p
            cum = np.cumsum(r)
            j = int(np.searchsorted(cum, u[T] * cum[-1], side="right"))
            j = min(j, int(np.nonzero(r)[0][-1]))
            tokens[s, i], probs[s, i], accepted[s] = j, p[j], i
            break
    return dict(tokens=torch.tensor(tokens).int(), accepted=torch.tensor(accepted).int(), probs=torch.tensor(probs))
