"""Forking and compacting pages (nd_op_pages_fork, nd_op_pages_compact)
against a restatement over Python lists. Everything is whole numbers and moved
bytes: results have to be equal."""

import ctypes as C

import numpy as np
import pytest


def ref_fork(pool, table, src, keep, need, page, pages, pinned):
    """pool: list of layers, each a list of page contents."""
    seqs, cols = table.shape
    n = len(src)
    kept, nn, writer = [], [], []
    for d in range(n):
        has = 0 <= src[d] < seqs
        k = min(max(int(keep[d]), 0), cols * page) if has else 0
        w = max(min(int(need[d]), cols * page), k)
        row = [int(p) if 0 <= p < pages else -1 for p in table[src[d], : -(-k // page)]] if has else []
        kept.append(row)
        nn.append(-(-w // page))
        writer.append(row[-1] if k % page and w > k and row[-1] >= 0 else None)
    users = {}
    for row in kept:
        for p in row:
            if p >= 0:
                users[p] = users.get(p, 0) + 1
    writers = {}
    for d, p in enumerate(writer):
        if p is not None:
            writers.setdefault(p, []).append(d)
    free = [p for p in range(pages) if p not in users and not pinned[p]]
    wanted = given = copies = 0
    new = np.full((n, cols), -1, np.int64)
    pool = [list(layer) for layer in pool]
    old = [list(layer) for layer in pool]

    def take():
        nonlocal wanted, given
        wanted += 1
        if free:
            given += 1
            return free.pop(0)
        return -1

    for d in range(n):
        row = list(kept[d])
        p = writer[d]
        if p is not None:
            alone = users[p] == 1 or (users[p] == len(writers[p]) and writers[p][0] == d)
            if pinned[p] or not alone:
                row[-1] = take()
                if row[-1] >= 0:
                    copies += 1
                    for layer, was in zip(pool, old):
                        layer[row[-1]] = was[p]
        while len(row) < nn[d]:
            row.append(take())
        new[d, : len(row)] = row
    refs = np.bincount(new[new >= 0], minlength=pages)
    used = int(((refs > 0) | np.array(pinned, bool)).sum())
    return new, refs, [used, given, copies, wanted - given], pool


def ref_compact(pool, table, pages, pinned):
    live = {int(p) for p in table.ravel() if 0 <= p < pages} | {p for p in range(pages) if pinned[p]}
    n = len(live)
    holes = [p for p in range(n) if p not in live]
    to = {p: p for p in live}
    pool = [list(layer) for layer in pool]
    moved = 0
    for p in sorted(live):
        if p >= n and not pinned[p]:
            to[p] = holes.pop(0)
            moved += 1
            for layer in pool:
                layer[to[p]] = layer[p]
    new = np.array([[to[int(p)] if 0 <= p < pages else -1 for p in row] for row in table])
    return new, np.array([to.get(p, -1) for p in range(pages)]), [n, moved], pool


def _dev(a):
    import torch

    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()


def _pool(pages, elems, layers, dtype="int16", seed=0):
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)
    shape = (pages, elems) if layers == 1 else (layers, pages, elems)
    return torch.randint(-30000, 30000, shape, device="cuda", generator=g, dtype=getattr(torch, dtype))


def _pages(pool, layers):
    return [[p for p in layer] for layer in (pool[None] if layers == 1 else pool).cpu().numpy()]


def check_fork(table, src, keep, need, page, pages, pinned=None, layers=1, elems=24, seed=0):
    import needle_b200 as nb
    import torch

    pin = np.zeros(pages, bool) if pinned is None else pinned
    pool = _pool(pages, elems, layers, seed=seed)
    want = ref_fork(_pages(pool, layers), table, src, keep, need, page, pages, pin)
    pt = None if pinned is None else torch.from_numpy(pin).cuda()
    axis = 0 if layers == 1 else 1
    for _ in range(2):  # repeating the call changes nothing
        got = nb.op_pages_fork(pool, _dev(table), _dev(src), _dev(keep), _dev(need), page, pinned=pt, axis=axis)
        assert np.array_equal(got[0].cpu().numpy(), want[0]), "table"
        assert np.array_equal(got[1].cpu().numpy(), want[1]), "references"
        assert got[2].tolist() == want[2], "info"
        assert np.array_equal(np.array(_pages(pool, layers)), np.array(want[3])), "pool"
    return want


@pytest.mark.gpu
def test_fork_of_one_sequence(cuda_device):
    table = np.array([[5, 2, 7, -1]])
    # a beam of three from a partly filled page: two copies, the first stays
    w = check_fork(table, [0, 0, 0], [40, 40, 40], [41, 41, 41], 16, 9)
    assert w[2][2] == 2
    # nobody writes: all shared
    assert check_fork(table, [0, 0], [40, 40], [40, 40], 16, 9)[2][2] == 0
    # one holds the page whole, one writes into it
    assert check_fork(table, [0, 0], [48, 40], [48, 44], 16, 9)[2][2] == 1
    # a border: nothing partly filled
    assert check_fork(table, [0, 0], [32, 32], [33, 33], 16, 9)[2][2] == 0
    # truncating, growing past the columns, an ended and a new sequence
    check_fork(table, [0, -1, 0], [3, 99, 40], [64, 20, 4000], 16, 30)
    check_fork(table, [-1], [0], [0], 16, 9)


@pytest.mark.gpu
def test_fork_when_pages_run_out(cuda_device):
    table = np.array([[0, 1, 2], [3, 4, -1]])
    w = check_fork(table, [0, 0, 1, 1], [40, 40, 20, 20], [41, 41, 48, 48], 16, 6)
    assert w[2][3] > 0
    check_fork(table, [0, 0, 0, 0], [47, 47, 47, 47], [48, 48, 48, 48], 16, 5)


@pytest.mark.gpu
def test_fork_bad_entries_and_values(cuda_device):
    table = np.array([[0, -3, 2, 99], [2 ** 31 - 1, 4, 1, -1]])
    check_fork(table, [0, 1, 7, -2 ** 31, 0], [50, 2 ** 31 - 1, 5, 5, -7], [60, 2 ** 31 - 1, 9, -4, 17], 16, 12)
    check_fork(table, [1, 0], [10, 30], [11, 31], 16, 12)  # the page to be written does not exist


@pytest.mark.gpu
def test_fork_pinned_pages(cuda_device):
    table = np.array([[5, 2, 7, -1], [5, 3, -1, -1]])
    pinned = np.zeros(12, bool)
    pinned[[5, 7, 0, 1]] = True
    w = check_fork(table, [0, 1], [40, 20], [41, 40], 16, 12, pinned=pinned)
    assert w[2][2] == 1  # 7 is pinned: written on a copy
    check_fork(table, [-1], [0], [64], 16, 12, pinned=np.ones(12, bool))


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(12))
def test_fork_drawn(cuda_device, seed):
    r = np.random.default_rng(seed)
    page, cols = int(r.choice([1, 16, 33])), int(r.integers(1, 70))
    seqs, n = int(r.integers(1, 40)), int(r.choice([1, 3, 50, 1500]))
    pages = int(r.choice([seqs * cols + 5, 5000]))
    shared = r.integers(0, pages, (1, cols))
    table = np.where(r.random((seqs, cols)) < 0.5, shared, r.integers(-2, pages + 2, (seqs, cols)))
    table = np.stack([np.array(list(dict.fromkeys(row.tolist()))[:cols] + [-1] * cols)[:cols] for row in table])
    src = r.integers(-1, seqs, n)
    keep = r.integers(0, cols * page + 2, n)
    need = keep + r.integers(-3, 2 * page + 3, n)
    pinned = r.random(pages) < 0.1 if seed % 2 else None
    check_fork(table, src, keep, need, page, pages, pinned, layers=1 + seed % 3, elems=8 * int(r.integers(1, 40)), seed=seed)


@pytest.mark.gpu
@pytest.mark.parametrize("seqs,cols,n,pages", [(300, 400, 500, 140000), (40, 20, 9000, 2000), (700, 300, 20, 70000)])
def test_large_sets(cuda_device, seqs, cols, n, pages):
    """Past what one cluster takes: pages, entries of the new and of the old table."""
    r = np.random.default_rng(seqs)
    table = np.full(seqs * cols, -1)
    some = r.permutation(pages)[: seqs * cols // 3]
    table[: len(some)] = some
    table = table.reshape(seqs, cols)
    src = r.integers(0, seqs // 4 + 1, n)
    keep = r.integers(0, 16 * cols, n)
    check_fork(table, src, keep, keep + r.integers(0, 40, n), 16, pages, elems=8)
    check_compact(table, pages, elems=8)


def check_compact(table, pages, pinned=None, layers=1, elems=24, seed=0):
    import needle_b200 as nb
    import torch

    pin = np.zeros(pages, bool) if pinned is None else pinned
    pool = _pool(pages, elems, layers, seed=seed)
    want = ref_compact(_pages(pool, layers), table, pages, pin)
    pt = None if pinned is None else torch.from_numpy(pin.astype(np.uint8)).cuda()
    for _ in range(2):
        got = nb.op_pages_compact(pool, _dev(table), pinned=pt, axis=0 if layers == 1 else 1)
        assert np.array_equal(got[0].cpu().numpy(), want[0]), "table"
        assert np.array_equal(got[1].cpu().numpy(), want[1]), "map"
        assert got[2].tolist() == want[2], "info"
        assert np.array_equal(np.array(_pages(pool, layers)), np.array(want[3])), "pool"


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(8))
def test_compact_drawn(cuda_device, seed):
    r = np.random.default_rng(100 + seed)
    pages = int(r.choice([7, 1024, 1025, 5000]))
    cols = int(r.integers(1, 40))
    seqs = max(1, int(pages * r.uniform(0.1, 0.9)) // cols)
    ids = r.permutation(pages)[: min(pages, seqs * cols)]
    flat = np.full(seqs * cols, -1)
    flat[: len(ids)] = ids
    table = flat.reshape(seqs, cols)
    table[r.random(table.shape) < 0.2] = -1
    if seed % 2:
        table[0, :] = table[-1, :]  # shared pages
        table[-1, -1] = pages + 4
    pinned = r.random(pages) < 0.2 if seed % 3 == 0 else None
    check_compact(table, pages, pinned, layers=1 + seed % 2, elems=8 * int(r.integers(1, 30)), seed=seed)


@pytest.mark.gpu
def test_compact_edges(cuda_device):
    check_compact(np.full((2, 3), -1), 5)                                # nothing live
    check_compact(np.arange(6).reshape(2, 3), 6)                          # all live
    check_compact(np.array([[2047, 1024]]), 2048)                        # the last pages of two blocks
    check_compact(np.array([[3]]), 4, pinned=np.array([0, 0, 1, 0], bool))
    check_compact(np.array([[0]]), 1)


@pytest.mark.gpu
def test_fork_then_compact_in_a_graph(cuda_device):
    """Captured and replayed with other tables; a kv4 pool's layers move."""
    import needle_b200 as nb
    import torch

    pages, page, layers = 64, 16, 2
    data = torch.randint(0, 256, (layers, pages, 2, 1, nb.KV4Pool.tile_bytes(48, 64)), dtype=torch.uint8, device="cuda")
    table = _dev(np.array([[1, 2, 3, 40], [50, 51, 52, 53], [-1, -1, -1, -1]]))
    src, keep, need = _dev([0, 0, 1]), _dev([50, 50, 60]), _dev([52, 52, 64])

    def step():
        t, refs, info = nb.op_pages_fork(data, table, src, keep, need, page, axis=1)
        return (t, info) + nb.op_pages_compact(data, t, axis=1)

    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        t, info, t2, to, moved = step()
    for s in ([0, 0, 1], [1, 1, 1], [2, 0, -1]):
        src.copy_(_dev(s))
        before = _pages(data.view(layers, pages, -1), layers)
        g.replay()
        torch.cuda.synchronize()
        w = ref_fork(before, table.cpu().numpy(), s, [50, 50, 60], [52, 52, 64], page, pages, np.zeros(pages, bool))
        assert np.array_equal(t.cpu().numpy(), w[0]) and info.tolist() == w[2]
        w2 = ref_compact(w[3], w[0], pages, np.zeros(pages, bool))
        assert np.array_equal(t2.cpu().numpy(), w2[0]) and np.array_equal(to.cpu().numpy(), w2[1]) and moved.tolist() == w2[2]
        assert np.array_equal(np.array(_pages(data.view(layers, pages, -1), layers)), np.array(w2[3]))


@pytest.mark.gpu
def test_refusals(cuda_device):
    import needle_b200 as nb
    import torch

    pool, table = _pool(8, 24, 1), _dev([[0, 1]])
    one = _dev([0])
    for call in (
        lambda: nb.op_pages_fork(pool.cpu(), table, one, one, one, 16),
        lambda: nb.op_pages_fork(pool, table.long(), one, one, one, 16),
        lambda: nb.op_pages_fork(pool, table, one, _dev([0, 1]), one, 16),
        lambda: nb.op_pages_fork(pool, table, one, one, one[:0], 16),
        lambda: nb.op_pages_fork(pool, table, one[:0], one[:0], one[:0], 16),
        lambda: nb.op_pages_fork(pool[:, ::2], table, one, one, one, 16),
        lambda: nb.op_pages_fork(pool, table, one, one, one, 16, pinned=torch.zeros(7, dtype=torch.uint8, device="cuda")),
        lambda: nb.op_pages_compact(pool, table[0]),
        lambda: nb.op_pages_compact(pool, table, axis=2),
    ):
        with pytest.raises(ValueError):
            call()
    for call in (
        lambda: nb.op_pages_fork(pool, table, one, one, one, 0),
        lambda: nb.op_pages_fork(_pool(8, 23, 1), table, one, one, one, 16),
        lambda: nb.op_pages_compact(pool[:1].expand(8, 24), table),
    ):
        with pytest.raises(RuntimeError):
            call()


def test_entry_points_refuse_without_a_gpu():
    import needle_b200 as nb
    from needle_b200._abi import PAGES

    lib = nb.lib()
    good = dict(device=0, pool=4096, page_stride=64, layer_stride=0, page_bytes=64, num_pages=8, layers=1)

    def fork(stride=2, seqs=1, cols=2, page=16, src=4096, n=1, out=8192, ws=4096, nbytes=1 << 20, table=4096, **bad):
        p = PAGES(**{**good, **bad})
        return lib.nd_op_pages_fork(C.byref(p), table, stride, seqs, cols, page, src, 4096, 4096, n, None, out, 4096, 4096, ws,
                                    nbytes, None)

    for bad, message in ((dict(page_bytes=60), b"aligned"), (dict(page_stride=48), b"overlap"), (dict(pool=4100), b"aligned"),
                         (dict(num_pages=0), b"positive"), (dict(layers=2), b"overlap"), (dict(num_pages=1 << 29), b"2^28"),
                         (dict(stride=1), b"overlap"), (dict(seqs=0), b"sequences"), (dict(page=0), b"page"),
                         (dict(n=0), b"n must"), (dict(src=None), b"null"), (dict(out=4096), b"old one"),
                         (dict(ws=None), b"workspace"), (dict(nbytes=8), b"workspace"), (dict(table=None), b"null"),
                         (dict(cols=1 << 30, stride=1 << 30), b"2^31")):
        assert fork(**bad) == -1 and message in lib.nd_last_error(), (bad, lib.nd_last_error())
    assert lib.nd_op_pages_compact(None, 4096, 2, 1, 2, None, 8192, 4096, 4096, 4096, 1 << 20, None) == -1
    assert lib.nd_op_pages_fork_ws(0, 1) == 0 and lib.nd_op_pages_compact_ws(-1) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("pages", [131072, 131071, 131073, 32, 33, 128, 129])
@pytest.mark.parametrize("dense,pins", [(0.02, False), (0.98, True), (0.5, True)])
def test_compact_whole_words_and_all_a_plan_takes(cuda_device, pages, dense, pins):
    r = np.random.default_rng(pages)
    some = r.permutation(pages)[: max(1, int(dense * pages))]
    cols = 7
    table = np.full(-(-len(some) // cols) * cols, -1)
    table[: len(some)] = some
    pinned = r.random(pages) < 0.01 if pins else None
    check_compact(table.reshape(-1, cols), pages, pinned, elems=8)
