"""The paged 4-bit cache (nd_op_kv4_append, nd_op_kv4_read) and attention
over it (nd_op_kv4_attend) against a plain numpy restatement.

Codes, scales and minima are defined by single f32 operations, so what the
cache holds has to be equal. Attention's tolerance, per value: half a step of
the output's type, plus 2 d + w times the values' magnitude, where d is how
far a score can be off and w a weight (a relative change of every weight by at
most d moves the quotient by at most 2 d times the values' magnitude):
 d: the tensor cores add up to 16 products' groups, each sum truncated by at
    most 2^-22 of the terms' magnitude B (16 * 2^-22 = 2^-18), the two f16
    terms of an f32 query leave 2^-22, three roundings of 2^-24; exp2 2^-22
    of the weight; together below 2^-17 B + 2^-20;
 w: 2^-11 for the one f16 term of a weight of bf16 rows (half a step, doubled
    for codes being summed before their minimum is taken off), 2^-21 for two
    terms, and one truncation of 2^-22 for each 16 keys.
"""

import ctypes as C

import numpy as np
import pytest

import kv4_ref

HEADS = {"needle": (12, 2, 48, 64), "small": (4, 4, 64, 64), "wide": (8, 2, 128, 128)}


def _torch_type(name):
    import torch

    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def _np(t):
    return t.float().cpu().numpy()


class Setup:
    """A pool with pages in random order, filled for `lens` positions a
    sequence; the last n[s] rows of each are the call's."""

    def __init__(self, heads, dtype, lens, n, page, seed=0, extra_rows=0, gap=0, table_cols=None, qscale=1.0):
        import torch

        import needle_b200 as nb

        self.hq, self.h, self.dk, self.dv = HEADS[heads]
        rng = np.random.default_rng(seed)
        S, self.page = len(lens), page
        cols = table_cols or max(1, -(-max(lens) // page))
        used = [min(cols, -(-int(x) // page)) for x in lens]
        N = sum(used) + 2
        ids = rng.permutation(N)
        self.table = np.full((S, cols), -1, np.int32)
        at = 0
        for s in range(S):
            self.table[s, : used[s]] = ids[at: at + used[s]]
            at += used[s]
        tiles, tile = page // 16, kv4_ref.tile_bytes(self.dk, self.dv)
        # the pool starts as 0xff bytes: scales and minima that are NaN
        data = torch.full((N, self.h + gap, tiles, tile), 255, dtype=torch.uint8, device="cuda")
        self.kv = nb.KV4Pool(data[:, : self.h], self.dk, self.dv)
        self.ref = kv4_ref.Cache(N, self.h, page, self.dk, self.dv)
        self.t = _torch_type(dtype)
        self.lens, self.n = np.array(lens, np.int32), np.array(n, np.int32)
        full = np.concatenate([[0], np.cumsum(self.lens)]).astype(np.int32)
        k = torch.from_numpy(rng.standard_normal((int(full[-1]), self.h, self.dk)).astype(np.float32) * 1.5 + 0.25)
        v = torch.from_numpy(rng.standard_normal((int(full[-1]), self.h, self.dv)).astype(np.float32) * 0.5 - 0.1)
        self.k, self.v = k.to("cuda", self.t), v.to("cuda", self.t)
        self.full = full
        self.start = np.concatenate([[0], np.cumsum(self.n)]).astype(np.int32)
        self.rows = int(self.start[-1]) + extra_rows
        q = rng.standard_normal((self.rows, self.hq, self.dk)).astype(np.float32) * qscale
        self.q = torch.from_numpy(q).to("cuda", self.t)

    def dev(self, a):
        import torch

        return torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()

    def append(self):
        import needle_b200 as nb

        nb.op_kv4_append(self.kv, self.k, self.v, self.dev(self.table), self.dev(self.lens), self.dev(self.full))
        self.ref.append(_np(self.k), _np(self.v), self.table, self.lens, self.full)
        return self


def _tol(dtype, out, b, top, keys):
    half = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[dtype]
    w = (2.0 ** -11 if dtype == "bf16" else 2.0 ** -21) + keys / 16 * 2.0 ** -22
    floor = 2.0 ** -25 if dtype == "f16" else 0.0  # half a subnormal step
    return half * np.abs(out) * (1 + 2.0 ** -7) + floor + (2 * (2.0 ** -17 * b + 2.0 ** -20) + w) * top


def _check(st, dtype, got, window=0, sink=0, scale=None):
    scale = 1 / np.sqrt(st.dk) if scale is None else scale
    want, b, top = st.ref.attend(_np(st.q), st.table, st.lens, st.start, scale, window, sink)
    n = int(st.start[-1])
    err = np.abs(_np(got)[:n] - want[:n])
    tol = _tol(dtype, want[:n], b[:n], top[:n], max(st.lens))
    bad = ~(err <= tol)
    assert not bad.any(), f"{bad.sum()} values off, worst {np.nanmax(err / tol):.3g} of the tolerance at {np.argwhere(bad)[0]}"


# ------------------------------------------------------------------ append


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads", list(HEADS))
@pytest.mark.parametrize("page", [16, 48, 128])
def test_append_holds_the_formats_values(cuda_device, heads, dtype, page):
    import needle_b200 as nb

    lens = [1, 0, 15, 16, 17, 130, 33]
    st = Setup(heads, dtype, lens, lens, page, seed=page).append()
    k, v = nb.op_kv4_read(st.kv, st.dev(st.table), st.dev(st.lens), st.dev(st.full), rows=int(st.full[-1]))
    wk, wv = st.ref.read(st.table, st.lens, st.full, int(st.full[-1]))
    assert np.array_equal(_np(k), wk.astype(np.float32)) and np.array_equal(_np(v), wv.astype(np.float32))
    kt, vt = nb.op_kv4_read(st.kv, st.dev(st.table), st.dev(st.lens), st.dev(st.full), rows=int(st.full[-1]), dtype=st.t)
    import torch

    assert torch.equal(kt, k.to(st.t)) and torch.equal(vt, v.to(st.t))


@pytest.mark.gpu
def test_append_extreme_rows(cuda_device):
    """Constant rows, rows of zeros, subnormal and huge ranges, NaN, infinities."""
    import needle_b200 as nb
    import torch

    st = Setup("small", "f32", [12], [12], 16)
    k = st.k
    k[0] = 0.0
    k[1] = -3.14159
    k[2] *= 1e-7
    k[3] *= 1e-30
    k[4] *= 1e6
    k[5] *= 1e38
    k[6, 0, 3] = float("nan")
    k[7, 1, 63] = float("inf")
    k[8, 2, 0] = float("-inf")
    k[9] = torch.linspace(0, 15, 64, device="cuda")
    st.append()
    got, _ = nb.op_kv4_read(st.kv, st.dev(st.table), st.dev(st.lens), st.dev(st.full), rows=12)
    want, _ = st.ref.read(st.table, st.lens, st.full, 12)
    assert np.array_equal(_np(got), want.astype(np.float32), equal_nan=True)
    assert np.isnan(_np(got)[6, 0]).all() and np.isfinite(_np(got)[6, 1]).all()


@pytest.mark.gpu
def test_append_leaves_the_rest_alone(cuda_device):
    """Rows without a place (a page id outside the pool, positions before 0
    or past the table), rows behind the last sequence, other slots and other
    pages' bytes."""
    import needle_b200 as nb

    st = Setup("needle", "bf16", [40, 40, 70, 20], [40, 40, 70, 20], 16, gap=1, table_cols=4)
    st.table[0, 1] = -1
    st.table[1, 2] = st.kv.num_pages
    st.table[3, 0] = 2 ** 31 - 1
    st.lens[1] = 35  # five rows before position 0
    data = st.kv.data._base
    before = data.clone()
    start = st.full.copy()
    start[-1] -= 4  # the last four rows belong to nobody
    nb.op_kv4_append(st.kv, st.k, st.v, st.dev(st.table), st.dev(st.lens), st.dev(start))
    st.ref.append(_np(st.k), _np(st.v), st.table, st.lens, start)
    held = ~np.isnan(st.ref.k).any(-1)  # [pages, heads, page]
    tile = 16 * (24 + 32 + 8)
    changed = (data != before).cpu().numpy()
    assert not changed[:, 2:].any()
    by_page = changed[:, :2].any((1, 2, 3))
    assert np.array_equal(by_page, held.any((1, 2)))
    codes = changed[:, :2].reshape(data.shape[0], 2, 1, tile)[..., : 16 * 24].reshape(data.shape[0], 2, 16, 24).any(-1)
    assert not (codes & ~held).any()
    k, v = nb.op_kv4_read(st.kv, st.dev(st.table), st.dev(st.lens), st.dev(start), rows=int(st.full[-1]))
    wk, wv = st.ref.read(st.table, st.lens, start, int(st.full[-1]))
    assert np.array_equal(_np(k), wk.astype(np.float32)) and np.array_equal(_np(v), wv.astype(np.float32))


@pytest.mark.gpu
def test_strided_rows_of_a_projection(cuda_device):
    """k and q as views of the row op_rope rotates (12 query and 2 key heads
    of 48 in 672 values), v of an odd stride that no 16-byte load fits."""
    import needle_b200 as nb
    import torch

    st = Setup("needle", "f32", [20, 9], [20, 9], 16)
    x = nb.op_rope(torch.randn((29, 672), device="cuda"))
    st.q, st.k = x[:, :576].view(29, 12, 48), x[:, 576:].view(29, 2, 48)
    w = torch.randn((29, 131), device="cuda")
    st.v = w[:, 1:129].view(29, 2, 64)
    st.append()
    k, v = nb.op_kv4_read(st.kv, st.dev(st.table), st.dev(st.lens), st.dev(st.full), rows=29)
    wk, wv = st.ref.read(st.table, st.lens, st.full, 29)
    assert np.array_equal(_np(k), wk.astype(np.float32)) and np.array_equal(_np(v), wv.astype(np.float32))
    base = torch.full((29, 12, 67), 7.0, device="cuda")
    out = nb.op_kv4_attend(st.kv, st.q, st.dev(st.table), st.dev(st.lens), st.dev(st.start), out=base[:, :, 2:66])
    _check(st, "f32", out)
    assert (base[:, :, :2] == 7).all() and (base[:, :, 66:] == 7).all()


# ------------------------------------------------------------------ attend


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads", list(HEADS))
@pytest.mark.parametrize("window,sink", [(0, 0), (1, 0), (33, 0), (20, 5), (64, 40)])
def test_attend_one_token_each(cuda_device, heads, dtype, window, sink):
    import needle_b200 as nb

    lens = [1, 2, 15, 16, 17, 64, 100, 257, 300]
    st = Setup(heads, dtype, lens, [1] * len(lens), 32, seed=window).append()
    got = nb.op_kv4_attend(st.kv, st.q, st.dev(st.table), st.dev(st.lens), window=window, sink=sink)
    _check(st, dtype, got, window, sink)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads", list(HEADS))
@pytest.mark.parametrize("n", [[2, 3, 1], [5, 0, 4], [9, 1, 0], [37, 20, 64]])
@pytest.mark.parametrize("window,sink", [(0, 0), (17, 3)])
def test_attend_ragged_rows(cuda_device, heads, dtype, n, window, sink):
    """Drafts and prompt chunks: every number of rows a block, sequences
    that bring none, one whose rows are all it holds."""
    import needle_b200 as nb
    import torch

    lens = [max(90, n[0]), max(70, n[1]), n[2]]
    st = Setup(heads, dtype, lens, n, 16, seed=sum(n), extra_rows=2).append()
    out = torch.full((st.rows, st.hq, st.dv), 5.0, dtype=st.t, device="cuda")
    got = nb.op_kv4_attend(st.kv, st.q, st.dev(st.table), st.dev(st.lens), st.dev(st.start), window=window, sink=sink, out=out)
    assert got is out and (out[-2:] == 5).all()
    _check(st, dtype, got, window, sink)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("heads", list(HEADS))
@pytest.mark.parametrize("n,lens", [([200], [200]), ([64, 70, 0], [300, 70, 40]), ([100, 257], [900, 1000])])
@pytest.mark.parametrize("window,sink", [(0, 0), (90, 20)])
def test_attend_many_rows(cuda_device, heads, dtype, n, lens, window, sink):
    """Prompts: several blocks of rows, the last partly filled, keys cut
    between CTAs, a bad page, rows behind the last sequence."""
    import needle_b200 as nb
    import torch

    st = Setup(heads, dtype, lens, n, 32, seed=sum(n), extra_rows=3).append()
    out = torch.full((st.rows, st.hq, st.dv), 5.0, dtype=st.t, device="cuda")
    nb.op_kv4_attend(st.kv, st.q, st.dev(st.table), st.dev(st.lens), st.dev(st.start), window=window, sink=sink, out=out)
    assert (out[-3:] == 5).all()
    _check(st, dtype, out, window, sink)
    st.table[0, 3] = -1
    got = nb.op_kv4_attend(st.kv, st.q, st.dev(st.table), st.dev(st.lens), st.dev(st.start), window=window, sink=sink)
    assert (got[-3:] == 0).all()
    _check(st, dtype, got, window, sink)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_attend_many_rows_odd_values(cuda_device, dtype):
    """In the kernel for many rows: values of very small and large scale,
    constant values, wide scores, NaN rows of keys and queries, scale 0 and
    below."""
    import needle_b200 as nb
    import torch

    for heads, factor in (("wide", 1e-4), ("small", 1e4), ("needle", 0.0)):
        st = Setup(heads, dtype, [300, 230], [250, 210], 32, seed=7)
        st.v *= factor
        if factor == 0.0:
            st.v += 1.5
        st.append()
        _check(st, dtype, nb.op_kv4_attend(st.kv, st.q, st.dev(st.table), st.dev(st.lens), st.dev(st.start)))
    st = Setup("wide", dtype, [280, 200], [260, 200], 32, seed=8, qscale=30.0).append()
    args = (st.kv, st.q, st.dev(st.table), st.dev(st.lens), st.dev(st.start))
    for scale in (None, 0.0, -0.01):
        _check(st, dtype, nb.op_kv4_attend(*args, scale=scale), scale=scale)
    st = Setup("small", dtype, [300], [250], 16, seed=9)
    st.k[100, 1] = float("nan")
    st.v[200, 2] = float("inf")
    st.append()
    st.q[7, 0, 3] = float("nan")
    st.q[40, 3, 1] = float("inf")
    got = _np(nb.op_kv4_attend(st.kv, st.q, st.dev(st.table), st.dev(st.lens), st.dev(st.start)))
    nan = np.zeros((250, 4), bool)
    pos = np.arange(50, 300)
    nan[pos >= 100, 1] = True
    nan[pos >= 200, 2] = True
    nan[7, 0] = nan[40, 3] = True
    assert np.array_equal(np.isnan(got).any(-1), nan) and np.array_equal(np.isnan(got).all(-1), nan)
    got = _np(nb.op_kv4_attend(st.kv, st.q, st.dev(st.table), st.dev(st.lens), st.dev(st.start), window=30))
    nan[pos >= 130, 1] = False
    nan[pos >= 230, 2] = False
    assert np.array_equal(np.isnan(got).any(-1), nan)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads", ["needle", "wide"])
def test_attend_split_over_warps(cuda_device, heads, dtype):
    """A long sequence beside short ones: units cut across warps and joined."""
    import needle_b200 as nb

    st = Setup(heads, dtype, [3000, 5, 700, 40], [1, 1, 1, 1], 64, seed=3).append()
    got = nb.op_kv4_attend(st.kv, st.q, st.dev(st.table), st.dev(st.lens))
    _check(st, dtype, got)
    again = nb.op_kv4_attend(st.kv, st.q, st.dev(st.table), st.dev(st.lens))
    assert (again == got).all()
    got = nb.op_kv4_attend(st.kv, st.q, st.dev(st.table), st.dev(st.lens), window=2000, sink=70)
    _check(st, dtype, got, 2000, 70)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_attend_rows_that_see_nothing(cuda_device, dtype):
    """Lengths of zero, rows before position 0, sequences whose pages are all
    bad: zeros. A bad page in the middle is skipped; NaN in slots past the
    end and in pages outside the window is not touched."""
    import needle_b200 as nb

    st = Setup("needle", dtype, [60, 40, 50, 33], [1, 1, 1, 1], 16).append()
    st.n = np.array([1, 1, 3, 2], np.int32)
    st.start = np.concatenate([[0], np.cumsum(st.n)]).astype(np.int32)
    st.rows = 7
    import torch

    st.q = torch.randn((7, 12, 48), device="cuda").to(st.t)
    st.lens[:] = [60, 0, 2, 33]
    st.table[0, 2] = -5
    st.table[3] = st.kv.num_pages + 3
    got = nb.op_kv4_attend(st.kv, st.q, st.dev(st.table), st.dev(st.lens), st.dev(st.start))
    assert (got[1:3] == 0).all() and (got[5:] == 0).all() and (got[3:5] != 0).any()
    _check(st, dtype, got)


@pytest.mark.gpu
def test_attend_nan_stays_where_it_is_seen(cuda_device):
    import needle_b200 as nb

    st = Setup("small", "f32", [50, 50], [3, 3], 16)
    st.k[20, 1] = float("nan")      # sequence 0, head 1
    st.v[50 + 48, 2] = float("inf")  # sequence 1, head 2, seen by its last two rows
    st.append()
    st.q[1, 3, 5] = float("nan")
    st.q[4, 0, 0] = float("inf")
    got = _np(nb.op_kv4_attend(st.kv, st.q, st.dev(st.table), st.dev(st.lens), st.dev(st.start)))
    nan = np.zeros((6, 4), bool)
    nan[:3, 1] = True
    nan[1, 3] = nan[4, 0] = True
    nan[4:, 2] = True
    assert np.array_equal(np.isnan(got).all(-1), nan) and np.array_equal(np.isnan(got).any(-1), nan)
    windowed = _np(nb.op_kv4_attend(st.kv, st.q, st.dev(st.table), st.dev(st.lens), st.dev(st.start), window=20))
    nan[:3, 1] = False  # position 20 is before the window
    assert np.array_equal(np.isnan(windowed).any(-1), nan)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_attend_scales_of_values_and_scores(cuda_device, dtype):
    """Values of very large and small magnitude, constant values (scale 0),
    and scores spread widely enough that one key takes nearly all weight."""
    import needle_b200 as nb

    for factor in (1e-4, 1e4, 0.0):
        st = Setup("wide", dtype, [80, 200], [2, 2], 32, seed=7)
        st.v *= factor
        if factor == 0.0:
            st.v += 1.5
        st.append()
        _check(st, dtype, nb.op_kv4_attend(st.kv, st.q, st.dev(st.table), st.dev(st.lens), st.dev(st.start)))
    st = Setup("wide", dtype, [80, 200], [2, 2], 32, seed=8, qscale=30.0).append()
    _check(st, dtype, nb.op_kv4_attend(st.kv, st.q, st.dev(st.table), st.dev(st.lens), st.dev(st.start)))
    _check(st, dtype, nb.op_kv4_attend(st.kv, st.q, st.dev(st.table), st.dev(st.lens), st.dev(st.start), scale=0.0), scale=0.0)
    _check(st, dtype, nb.op_kv4_attend(st.kv, st.q, st.dev(st.table), st.dev(st.lens), st.dev(st.start), scale=-0.01), scale=-0.01)


@pytest.mark.gpu
def test_captured_steps_follow_lengths_and_pages(cuda_device):
    """Append and attend in two graphs, replayed in turn with other lengths,
    pages and rows in the same buffers."""
    import needle_b200 as nb
    import torch

    a, b = Setup("needle", "bf16", [90, 30, 64], [1, 1, 1], 16, seed=1).append(), Setup("wide", "f32", [700, 20], [1, 1], 16, seed=2).append()
    graphs = []
    for st in (a, b):
        st.tt, st.lt = st.dev(st.table), st.dev(st.lens)
        st.kn, st.vn = st.k[:len(st.lens)].clone(), st.v[:len(st.lens)].clone()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            nb.op_kv4_append(st.kv, st.kn, st.vn, st.tt, st.lt)
            st.out = nb.op_kv4_attend(st.kv, st.q, st.tt, st.lt)
        graphs.append(g)
    for rep in range(2):
        for st in (a, b):
            st.lens = st.lens - rep * 9
            st.lt.copy_(st.dev(st.lens))
            st.q.copy_(torch.randn_like(st.q))
            one = np.arange(len(st.lens) + 1)
            st.ref.append(_np(st.kn), _np(st.vn), st.table, st.lens, one)
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        _check(a, "bf16", a.out)
        _check(b, "f32", b.out)


@pytest.mark.gpu
def test_other_stream(cuda_device):
    import needle_b200 as nb
    import torch

    st = Setup("wide", "f16", [300, 41], [4, 4], 16, seed=5).append()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = nb.op_kv4_attend(st.kv, st.q, st.dev(st.table), st.dev(st.lens))
    torch.cuda.current_stream().wait_stream(side)
    _check(st, "f16", got)


@pytest.mark.gpu
def test_empty_calls_and_refusals(cuda_device):
    import needle_b200 as nb
    import torch

    st = Setup("needle", "f32", [20, 9], [1, 1], 16).append()
    t, l = st.dev(st.table), st.dev(st.lens)
    none = st.q[:0]
    assert nb.op_kv4_attend(st.kv, none, t, l).shape == (0, 12, 64)
    nb.op_kv4_append(st.kv, st.k[:0], st.v[:0], t, l)
    assert nb.op_kv4_read(st.kv, t, l, rows=0)[0].shape == (0, 2, 48)
    for call in (
        lambda: nb.op_kv4_attend(st.kv, st.q.double(), t, l),
        lambda: nb.op_kv4_attend(st.kv, st.q[:, :, :47], t, l),
        lambda: nb.op_kv4_attend(st.kv, st.q[:, :11], t, l),
        lambda: nb.op_kv4_attend(st.kv, st.q, t.long(), l),
        lambda: nb.op_kv4_attend(st.kv, st.q, t, l[:1]),
        lambda: nb.op_kv4_attend(st.kv, st.q, t, l, st.dev([0, 1])),
        lambda: nb.op_kv4_attend(st.kv, st.q.cpu(), t, l),
        lambda: nb.op_kv4_attend(st.kv, st.q, t, l, out=torch.empty((2, 12, 64), device="cuda").half()),
        lambda: nb.op_kv4_append(st.kv, st.k, st.v.half(), t, l),
        lambda: nb.op_kv4_read(st.kv, t, l, st.dev([0, 1, 2])),
        lambda: nb.KV4Pool(st.kv.data, 64, 64),
        lambda: nb.KV4Pool(st.kv.data.float(), 48, 64),
    ):
        with pytest.raises(ValueError):
            call()
    for call in (
        lambda: nb.op_kv4_attend(st.kv, st.q, t, l, window=-1),
        lambda: nb.op_kv4_attend(st.kv, st.q, t, l, scale=float("nan")),
        lambda: nb.op_kv4_attend(st.kv, torch.zeros((3, 12, 48), device="cuda"), t, l),
        lambda: nb.op_kv4_attend(st.kv, st.q, t, l, out=torch.zeros((2, 1, 64), device="cuda").expand(2, 12, 64)),
        lambda: nb.op_kv4_attend(st.kv, torch.zeros((2, 130, 48), device="cuda"), t, l),
    ):
        with pytest.raises(RuntimeError):
            call()


def test_entry_points_refuse_without_a_gpu():
    """The C entries check their arguments before they touch a device."""
    import needle_b200 as nb
    from needle_b200._abi import KV4

    lib = nb.lib()
    good = dict(device=0, pool=4096, page_stride=2 * 1024, num_pages=4, page=16, heads=2, dk=48, dv=64, table=4096,
                table_stride=2, max_pages=2, seqs=1, lens=4096, start=None, rows=1)

    def attend(row=576, heads=12, type=0, window=0, ws=4096, nbytes=0, q=4096, o_row=768, **bad):
        a = KV4(**{**good, **bad})
        return lib.nd_op_kv4_attend(C.byref(a), type, q, row, 48, heads, 0.1, window, 0, 4096, o_row, 64, ws, nbytes, 0, None)

    for bad, message in ((dict(page=20), b"multiple of 16"), (dict(dk=50), b"(dk, dv)"), (dict(pool=4100), b"aligned"),
                         (dict(page_stride=1024), b"overlap"), (dict(table_stride=1), b"overlap"), (dict(seqs=0), b"positive"),
                         (dict(lens=None), b"null"), (dict(seqs=2), b"multiple of the sequences"),
                         (dict(max_pages=2 ** 30, table_stride=2 ** 30), b"2^31"), (dict(heads=12, type=7), b"type"),
                         (dict(q=4098), b"aligned"), (dict(row=-1), b"negative"), (dict(window=-1), b"negative"),
                         (dict(ws=4100), b"workspace"), (dict(o_row=10, rows=2), b"overlap"), (dict(rows=-1), b"positive")):
        heads = bad.pop("heads", 12)
        assert attend(heads=heads, **bad) == -1, bad
        assert message in lib.nd_last_error(), (bad, lib.nd_last_error())
    assert attend(heads=13) == -1 and b"multiple of heads" in lib.nd_last_error()
    assert lib.nd_op_kv4_attend(None, 0, 4096, 576, 48, 12, 0.1, 0, 0, 4096, 768, 64, 4096, 0, 0, None) == -1
    a = KV4(**good)
    assert lib.nd_op_kv4_append(C.byref(a), 0, None, 96, 48, 4096, 128, 64, None) == -1 and b"null" in lib.nd_last_error()
    assert lib.nd_op_kv4_read(C.byref(a), 0, 4096, 96, 0, 4096, 128, 64, 0, None) == -1 and b"overlap" in lib.nd_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [[1, 1, 1], [3, 1, 7], [40, 0, 5]])
def test_attend_many_heads_on_one(cuda_device, dtype, n):
    """64 query heads on one kv head, the most there may be."""
    import needle_b200 as nb

    HEADS["mqa"] = (64, 1, 64, 64)
    st = Setup("mqa", dtype, [100, 33, 300], n, 16, seed=4).append()
    got = nb.op_kv4_attend(st.kv, st.q, st.dev(st.table), st.dev(st.lens), st.dev(st.start), window=50, sink=7)
    _check(st, dtype, got, 50, 7)


@pytest.mark.gpu
def test_offsets_past_32_bits(cuda_device):
    """Pages that lie more than 4 GB into a pool, and copies between them."""
    import needle_b200 as nb
    import torch

    pages, heads = 34000, 8
    kv = nb.KV4Pool(torch.empty((pages, heads, 8, nb.KV4Pool.tile_bytes(128, 128)), dtype=torch.uint8, device="cuda"), 128, 128)
    assert kv.data.numel() > 1.08 * 2 ** 32
    ids = [pages - 1, 5, pages - 2, 31000, pages - 4]
    table = torch.tensor([ids[:2], ids[2:4]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([250, 140], dtype=torch.int32, device="cuda")
    start = torch.tensor([0, 250, 390], dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(0)
    k, v = (torch.randn((390, heads, 128), device="cuda", generator=g) for _ in range(2))
    nb.op_kv4_append(kv, k, v, table, lens, start)
    low = nb.KV4Pool.new(4, heads, 128, 128, page=128)
    low_table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device="cuda")
    nb.op_kv4_append(low, k, v, low_table, lens, start)
    for q in (torch.randn((2, 32, 128), device="cuda", generator=g), torch.randn((200, 32, 128), device="cuda", generator=g).bfloat16()):
        n = q.shape[0] // 2
        first = torch.tensor([0, n, 2 * n], dtype=torch.int32, device="cuda")
        assert torch.equal(nb.op_kv4_attend(kv, q, table, lens, first), nb.op_kv4_attend(low, q, low_table, lens, first))
    a, b = nb.op_kv4_read(kv, table, lens, start, rows=390), nb.op_kv4_read(low, low_table, lens, start, rows=390)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    # a copy: the second sequence forked, everything below the high pages taken
    pinned = torch.ones(pages, dtype=torch.bool, device="cuda")
    pinned[ids] = False
    src = torch.tensor([1, 1], dtype=torch.int32, device="cuda")
    keep = torch.tensor([140, 140], dtype=torch.int32, device="cuda")
    t2, _, info = nb.op_pages_fork(kv.data, table, src, keep, keep + 1, 128, pinned=pinned)
    assert info[2] == 1 and t2.tolist() == [[pages - 2, 31000], [pages - 2, 5]]
    assert torch.equal(kv.data[5], kv.data[31000])


@pytest.mark.gpu
def test_calls_side_by_side(cuda_device):
    """Attention of three kinds on three streams at once, then replayed from
    three graphs at once: as one after another."""
    import needle_b200 as nb
    import torch

    sets = [Setup("wide", "bf16", [900, 1000], [200, 257], 32, seed=1).append(), Setup("wide", "bf16", [3000, 700], [1, 1], 64, seed=2).append(),
            Setup("needle", "f32", [60, 200, 31], [1, 1, 1], 16, seed=3).append()]
    args = [(st.kv, st.q, st.dev(st.table), st.dev(st.lens), st.dev(st.start)) for st in sets]
    want = [nb.op_kv4_attend(*a) for a in args]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for s, a in zip(streams, args):
            with torch.cuda.stream(s):
                got.append(nb.op_kv4_attend(*a))
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))
    graphs, outs = [], []
    for s, a in zip(streams, args):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(nb.op_kv4_attend(*a))
        graphs.append(g)
    for _ in range(5):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(outs, want))


@pytest.mark.gpu
def test_prompts_replayed_with_other_lengths(cuda_device):
    import needle_b200 as nb
    import torch

    st = Setup("wide", "bf16", [400, 300], [150, 140], 32, seed=6).append()
    t, lens, start = st.dev(st.table), st.dev(st.lens), st.dev(st.start)
    nb.op_kv4_attend(st.kv, st.q, t, lens, start)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = nb.op_kv4_attend(st.kv, st.q, t, lens, start)
    for new_lens, n in (([400, 300], [150, 140]), ([250, 290], [10, 280]), ([0, 5], [0, 290])):
        st.lens, st.start = np.array(new_lens, np.int32), np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
        lens.copy_(st.dev(st.lens))
        start.copy_(st.dev(st.start))
        g.replay()
        torch.cuda.synchronize()
        _check(st, "bf16", out)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_queries_of_nan_that_see_nothing(cuda_device, dtype):
    """Rows before position 0 are zeros whatever their queries hold."""
    import needle_b200 as nb

    st = Setup("small", dtype, [60, 60], [60, 60], 16).append()
    st.n = np.array([200, 200], np.int32)  # rows 0 .. 139 of each lie before position 0
    st.start = np.array([0, 200, 400], np.int32)
    st.rows = 400
    import torch

    st.q = torch.randn((400, st.hq, st.dk), device="cuda").to(st.t)
    st.q[5, 0, 3] = st.q[150, 1, 0] = float("nan")
    st.q[250, 2, 7] = float("inf")
    got = _np(nb.op_kv4_attend(st.kv, st.q, st.dev(st.table), st.dev(st.lens), st.dev(st.start)))
    assert (got[:140] == 0).all() and (got[200:340] == 0).all()
    nan = np.zeros((400, st.hq), bool)
    nan[150, 1] = True
    assert np.array_equal(np.isnan(got).any(-1), nan)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,cols", [(60, 1), (60, 40), (4000, 1), (4000, 40)])
def test_offsets_that_do_not_ascend(cuda_device, dtype, rows, cols):
    """What such a call writes is not specified; it stays among its rows."""
    import needle_b200 as nb
    import torch

    rng = np.random.default_rng(rows)
    S = 12
    kv = nb.KV4Pool.new(S * cols, 2, 48, 64, page=16)
    table = torch.arange(S * cols, dtype=torch.int32, device="cuda").view(S, cols)
    lens = torch.full((S,), 16 * cols, dtype=torch.int32, device="cuda")
    room = torch.full((rows + 200, 12, 64), 7.0, device="cuda").to(_torch_type(dtype))
    k, v = torch.randn((rows, 2, 48), device="cuda"), torch.randn((rows, 2, 64), device="cuda")
    q = torch.randn((rows, 12, 48), device="cuda").to(room.dtype)
    for start in ([0, rows] * 6 + [0], rng.integers(-5, rows + 9, S + 1), rng.integers(-2 ** 31, 2 ** 31, S + 1), [rows] * (S + 1)):
        start = torch.tensor(np.asarray(start), dtype=torch.int32, device="cuda")
        nb.op_kv4_append(kv, k, v, table, lens, start)
        nb.op_kv4_attend(kv, q, table, lens, start, out=room[100:-100])
        nb.op_kv4_read(kv, table, lens, start, rows=rows)
    torch.cuda.synchronize()
    assert (room[:100] == 7).all() and (room[-100:] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("heads,dtype,seqs,most", [("needle", "f32", 700, 600), ("needle", "bf16", 400, 900), ("wide", "f16", 750, 500),
                                                   ("small", "f32", 450, 760)])
def test_attend_many_short_sequences(cuda_device, heads, dtype, seqs, most):
    """Units taken whole, a warp or four each, over more tiles than one round of the GPU."""
    import needle_b200 as nb

    lens = np.random.default_rng(seqs).integers(1, most + 1, seqs)
    lens[:2] = 1, most
    st = Setup(heads, dtype, lens, [1] * seqs, 16).append()
    for window, sink in ((0, 0), (300, 20)):
        got = nb.op_kv4_attend(st.kv, st.q, st.dev(st.table), st.dev(st.lens), window=window, sink=sink)
        _check(st, dtype, got, window=window, sink=sink)


# The many-row kernel is chosen by what the table could hold, so the tests
# above reach it with tables that have columns to spare.
@pytest.fixture
def wide_tables(monkeypatch):
    init = Setup.__init__

    def wide(self, *a, **k):
        init(self, *a, **k)
        self.table = np.pad(self.table, ((0, 0), (0, 40000)), constant_values=-1)

    monkeypatch.setattr(Setup, "__init__", wide)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads", list(HEADS))
@pytest.mark.parametrize("n,lens", [([200], [200]), ([64, 70, 0], [300, 70, 40]), ([100, 257], [900, 1000])])
@pytest.mark.parametrize("window,sink", [(0, 0), (200000, 0), (90, 20)])
def test_many_rows_wide_table(cuda_device, wide_tables, heads, dtype, n, lens, window, sink):
    test_attend_many_rows(cuda_device, heads, dtype, n, lens, window, sink)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_odd_values_wide_table(cuda_device, wide_tables, dtype):
    test_attend_many_rows_odd_values(cuda_device, dtype)
    test_queries_of_nan_that_see_nothing(cuda_device, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("n", [[40, 0, 5], [3, 90, 7]])
def test_many_heads_wide_table(cuda_device, wide_tables, dtype, n):
    test_attend_many_heads_on_one(cuda_device, dtype, n)


@pytest.mark.gpu
def test_prompts_replayed_wide_table(cuda_device, wide_tables):
    test_prompts_replayed_with_other_lengths(cuda_device)


@pytest.mark.gpu
def test_calls_side_by_side_wide_table(cuda_device, wide_tables):
    test_calls_side_by_side(cuda_device)


@pytest.mark.gpu
@pytest.mark.parametrize("heads", list(HEADS))
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("window,sink", [(0, 0), (900, 40)])
def test_attend_long_prompts(cuda_device, heads, dtype, window, sink):
    import needle_b200 as nb

    st = Setup(heads, dtype, [1500, 900, 3, 700], [700, 500, 0, 150], 64).append()
    got = nb.op_kv4_attend(st.kv, st.q, st.dev(st.table), st.dev(st.lens), st.dev(st.start), window=window, sink=sink)
    _check(st, dtype, got, window=window, sink=sink)
