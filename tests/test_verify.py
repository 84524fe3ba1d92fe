"""The check of drafted tokens (nd_op_verify) against numpy in 64 bits. Tokens
and counts have to be equal; a probability is one f32 rounding (2^-24) of a
value whose sum of exponentials may come from the f32 pass: each ex2 is off by
at most 2^-22, an argument by 2^-23 of itself (weighted by 2^-x at most 2^-23
of the sum), a thread's running f32 sum by 2^-24 for each of its terms."""

import numpy as np
import pytest


def ref_verify(logits, draft, u, temp, q, counts):
    S, T1, V = logits.shape
    T = T1 - 1
    tokens, probs, acc = np.full((S, T1), -1), np.zeros((S, T1)), np.zeros(S, np.int64)
    for s in range(S):
        n = min(max(int(counts[s]), 0), T)
        for i in range(n + 1):
            l, t = logits[s, i].astype(np.float64), float(temp[s])
            greedy = not t > 0
            bad = np.isnan(l).any() or l.max() == -np.inf or (not greedy and l.max() == np.inf)
            if bad:
                acc[s] = i
                break
            if greedy:
                p = np.zeros(V)
                p[np.argmax(l)] = 1
            else:
                p = np.exp((l - l.max()) / t)
                p /= p.sum()
            x = int(draft[s, i]) if i < n else -1
            known = 0 <= x < V
            if i < n and known and float(u[s, i]) * (float(q[s, i, x]) if q is not None else 1.0) < p[x]:
                tokens[s, i], probs[s, i] = x, p[x]
                continue
            r = p.copy()
            if i < n and q is not None:
                r = np.maximum(p - q[s, i].astype(np.float64), 0)
            elif i < n and known:
                r[x] = 0
            if not r.sum() > 0:
                r = p
            cum = np.cumsum(r)
            j = min(int(np.searchsorted(cum, float(u[s, T]) * cum[-1], side="right")), int(np.nonzero(r)[0][-1]))
            tokens[s, i], probs[s, i], acc[s] = j, p[j], i
            break
    return tokens, acc, probs


def _dev(a):
    import torch

    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def run(logits, draft, u, temp, q=None, counts=None, dtype="float32"):
    import needle_b200 as nb
    import torch

    lt = logits if torch.is_tensor(logits) else _dev(logits.astype(np.float32)).to(getattr(torch, dtype))
    got = nb.op_verify(lt, _dev(draft.astype(np.int32)), _dev(u.astype(np.float32)), _dev(np.asarray(temp, np.float32)),
                       q=None if q is None else (q if torch.is_tensor(q) else _dev(q.astype(np.float32))),
                       counts=None if counts is None else _dev(np.asarray(counts, np.int32)))
    S, T1 = u.shape
    want = ref_verify(lt.float().cpu().numpy(), draft, u.astype(np.float32), np.asarray(temp, np.float32),
                      None if q is None else (q.cpu().numpy() if torch.is_tensor(q) else q.astype(np.float32)),
                      np.full(S, T1 - 1) if counts is None else counts)
    assert np.array_equal(got[0].cpu().numpy(), want[0]), (got[0].cpu().numpy(), want[0])
    assert np.array_equal(got[1].cpu().numpy(), want[1])
    tol = 2.0 ** -21 + (logits.shape[-1] / 512 + 2) * 2.0 ** -24
    assert (np.abs(got[2].cpu().numpy() - want[2]) <= tol * want[2]).all()
    return want


def case(S, T, V, seed, spread=3.0):
    r = np.random.default_rng(seed)
    logits = r.standard_normal((S, T + 1, V)) * spread
    near = logits[:, :T] + r.standard_normal((S, T, V)) * 0.7
    q = np.exp(near - near.max(-1, keepdims=True)) if T else np.zeros((S, 0, V))
    q /= q.sum(-1, keepdims=True)
    draft = np.array([[r.choice(V, p=q[s, i]) for i in range(T)] for s in range(S)]).reshape(S, T)
    return logits, draft, r.random((S, T + 1)), r.uniform(0.4, 1.5, S), q


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("S,T,V", [(1, 1, 1), (3, 2, 5), (2, 4, 1000), (40, 3, 1027), (9, 10, 16384), (2, 64, 333), (3, 0, 700),
                                   (1, 5, 50021)])
@pytest.mark.parametrize("with_q", [True, False])
def test_matches_reference(cuda_device, dtype, S, T, V, with_q):
    logits, draft, u, temp, q = case(S, T, V, S * 100 + T)
    temp[::3] = 0
    run(logits, draft, u, temp, q if with_q and T else None, dtype=dtype)
    counts = np.random.default_rng(1).integers(-1, T + 3, S)
    run(logits, draft, u, temp, q if with_q and T else None, counts, dtype=dtype)


@pytest.mark.gpu
def test_every_draft_accepted_or_refused(cuda_device):
    logits, draft, u, temp, q = case(6, 5, 2000, 3)
    u[:, :5] = 0.0  # any token with a probability stands
    assert (run(logits, draft, u, temp, q)[1] == 5).all()
    draft[:] = logits[:, :5].argmin(-1)
    u[:, :5] = 0.999999
    assert (run(logits, draft, u, temp)[1] == 0).all()
    draft[2, 1], draft[3, 0], draft[4, 2] = -1, 2000, 2 ** 31 - 1
    u[:, :5] = 0.0
    assert run(logits, draft, u, temp, q)[1].tolist() == [5, 5, 1, 0, 2, 5]
    run(logits, draft, u, temp)


@pytest.mark.gpu
def test_greedy_ties_and_lowest_index(cuda_device):
    logits = np.zeros((4, 3, 600))
    logits[0, :, [7, 300, 511, 512]] = 2.0  # ties: the first
    logits[1] = -1e30
    logits[2, :, 599] = 1.0
    draft = np.array([[7, 300], [0, 0], [599, 599], [0, 1]])
    u = np.full((4, 3), 0.5)
    w = run(logits, draft, u, np.zeros(4))
    assert w[1].tolist() == [1, 2, 2, 1] and w[0][0].tolist() == [7, 7, -1] and w[0][1].tolist() == [0, 0, 0]
    run(logits, draft, u, np.full(4, -1.0))
    run(logits, draft, u, np.full(4, np.nan))


@pytest.mark.gpu
def test_draws_at_the_ends(cuda_device):
    logits, draft, u, temp, q = case(8, 2, 4099, 9)
    logits[:, :, :10] = -np.inf
    logits[:, :, -20:] = -np.inf
    u[::2, 2] = 0.0
    u[1::2, 2] = 1.0  # past the allowed range: the last that could be drawn
    u[:4, 0] = 1.0
    w = run(logits, draft, u, temp, q)
    t = w[0][np.arange(8), w[1]]
    assert (t >= 10).all() and (t < 4079).all()
    run(logits, draft, u, temp)


@pytest.mark.gpu
def test_draft_equal_to_target(cuda_device):
    """p = q up to rounding: all accepted for u < 1; where u is 1 the residual
    is rounding noise or zero and something with a probability is drawn."""
    V = 512
    logits = np.zeros((2, 2, V))  # p = 1 / 512 exactly
    q = np.full((2, 1, V), 1 / V)
    u = np.array([[0.99, 0.25], [1.0, 0.25]])
    w = run(logits, np.array([[3], [3]]), u, np.ones(2), q)
    assert w[1].tolist() == [1, 0] and w[0][1, 0] == 128  # the residual is zero: p itself


@pytest.mark.gpu
def test_rows_that_are_no_distribution(cuda_device):
    """NaN, +infinity, nothing above -infinity, NaN in q: nothing accepted at
    that row, -1 drawn with probability 0; other sequences are not touched."""
    import needle_b200 as nb

    logits, draft, u, temp, q = case(7, 3, 900, 4)
    u[:, :3] = 0.0
    logits[0, 1, 5] = np.nan
    logits[1, 0, 899] = np.inf
    logits[2, 2] = -np.inf
    logits[3, 3, 0] = np.nan
    temp[4] = 0
    logits[4, 1, 3] = np.nan
    w = run(logits, draft, u, temp, q)
    assert w[1][:4].tolist() == [1, 0, 2, 3] and w[0][0].tolist()[1:] == [-1, -1, -1]
    q[6, 0, 17] = np.nan
    draft[6, 0] = -1
    got = nb.op_verify(_dev(logits.astype(np.float32)), _dev(draft.astype(np.int32)), _dev(u.astype(np.float32)),
                       _dev(temp.astype(np.float32)), q=_dev(q.astype(np.float32)))
    assert got[0][6].tolist() == [-1] * 4 and got[1][6] == 0 and got[2][6].tolist() == [0.0] * 4


@pytest.mark.gpu
def test_strided_logits_and_replay(cuda_device):
    """Rows of a wider buffer (17 logits a row are padding), unaligned rows,
    and a captured call that follows its inputs."""
    import needle_b200 as nb
    import torch

    logits, draft, u, temp, q = case(5, 3, 1003, 11)
    wide = torch.full((5, 5, 1020), float("nan"), device="cuda")
    wide[:, 1:, 1:1004] = _dev(logits.astype(np.float32))
    qw = torch.full((3, 5, 1010), float("nan"), device="cuda")
    qw[:, :, 3:1006] = _dev(q.astype(np.float32)).transpose(0, 1)
    run(wide[:, 1:, 1:1004], draft, u, temp, qw[:, :, 3:1006].transpose(0, 1))
    lt, dt, ut, tt = _dev(logits.astype(np.float32)), _dev(draft.astype(np.int32)), _dev(u.astype(np.float32)), _dev(temp.astype(np.float32))
    nb.op_verify(lt, dt, ut, tt)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = nb.op_verify(lt, dt, ut, tt)
    for seed in (1, 2):
        logits, draft, u, temp, _ = case(5, 3, 1003, seed)
        for d, h in ((lt, logits), (dt, draft), (ut, u), (tt, temp)):
            d.copy_(torch.from_numpy(h))
        g.replay()
        torch.cuda.synchronize()
        w = ref_verify(lt.cpu().numpy(), draft, ut.cpu().numpy(), tt.cpu().numpy(), None, np.full(5, 3))
        assert np.array_equal(got[0].cpu().numpy(), w[0]) and np.array_equal(got[1].cpu().numpy(), w[1])


@pytest.mark.gpu
def test_draws_follow_the_distribution(cuda_device):
    """Over many sequences with one distribution the tokens come out as the
    target has them, whatever the draft: within five standard deviations."""
    import needle_b200 as nb
    import torch

    S, V = 20000, 6
    g = torch.Generator(device="cuda").manual_seed(5)
    logits = torch.tensor([0.1, 1.2, -0.7, 0.5, -2.0, 0.9], device="cuda").expand(S, 2, V)
    q = torch.tensor([0.3, 0.1, 0.2, 0.1, 0.1, 0.2], device="cuda")
    draft = torch.multinomial(q.expand(S, V), 1, generator=g).int()
    u = torch.rand((S, 2), device="cuda", generator=g)
    tok, acc, _ = nb.op_verify(logits, draft, u, torch.ones(S, device="cuda"), q=q.expand(S, 1, V))
    p = torch.softmax(logits[0, 0].double(), 0)
    first = torch.bincount(tok[:, 0].long(), minlength=V).double() / S
    assert ((first - p).abs() < 5 * (p * (1 - p) / S).sqrt()).all()
    expect = torch.minimum(p, q.double()).sum()
    assert (acc.double().mean() - expect).abs() < 5 * (expect * (1 - expect) / S).sqrt()


@pytest.mark.gpu
def test_refusals(cuda_device):
    import needle_b200 as nb

    logits, draft, u, temp, q = case(2, 2, 50, 0)
    l, d, ut, t, qt = _dev(logits.astype(np.float32)), _dev(draft.astype(np.int32)), _dev(u.astype(np.float32)), _dev(temp.astype(np.float32)), _dev(q.astype(np.float32))
    for call in (
        lambda: nb.op_verify(l.double(), d, ut, t),
        lambda: nb.op_verify(l, d.long(), ut, t),
        lambda: nb.op_verify(l, d[:, :1], ut, t),
        lambda: nb.op_verify(l, d, ut[:, :2], t),
        lambda: nb.op_verify(l, d, ut, t[:1]),
        lambda: nb.op_verify(l, d, ut, t, q=qt[:, :1]),
        lambda: nb.op_verify(l, d, ut, t, q=qt.half()),
        lambda: nb.op_verify(l, d, ut, t, counts=d[0, :1]),
        lambda: nb.op_verify(l.cpu(), d, ut, t),
        lambda: nb.op_verify(l[:, :, ::2], d, ut, t),
    ):
        with pytest.raises(ValueError):
            call()


def test_entry_point_refuses_without_a_gpu():
    import needle_b200 as nb

    lib = nb.lib()

    def verify(type=0, logits=4096, row=50, draft=4096, q=None, seqs=1, T=2, V=50, tokens=4096, ws=4096, nbytes=1 << 20):
        return lib.nd_op_verify(0, type, logits, 150, row, draft, None, 4096, 4096, q, 100, 50, seqs, T, V, tokens, 4096, 4096, ws,
                                nbytes, None)

    for bad, message in ((dict(type=3), b"type"), (dict(logits=None), b"null"), (dict(logits=4098), b"aligned"), (dict(q=4097), b"aligned"),
                         (dict(row=-1), b"negative"), (dict(draft=None), b"null"), (dict(seqs=0), b"sequences"),
                         (dict(T=65), b"64"), (dict(T=-1), b"64"), (dict(V=0), b"1 <= V"), (dict(tokens=None), b"null"), (dict(ws=None), b"workspace"), (dict(nbytes=8), b"workspace")):
        assert verify(**bad) == -1 and message in lib.nd_last_error(), bad


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("S,T,V", [(3, 2, 100003), (2, 1, 130001), (1, 1, 300007), (40, 1, 130001), (300, 0, 8200)])
def test_long_rows(cuda_device, dtype, S, T, V):
    """Runs that a warp keeps with two CTAs an SM, alone on one, and not at all."""
    test_matches_reference(cuda_device, dtype, S, T, V, True)


@pytest.mark.gpu
@pytest.mark.parametrize("below,off", [(0.4875, 4e-4), (0.6125, -5e-4)])
def test_sums_of_very_long_flat_rows(cuda_device, below, off):
    """16.8 million logits, all alike but for the first 4096, and drafts whose u
    lies 4e-4 or 5e-4 of p from their border. Equal terms round the same way, so a
    running f32 sum of 65,536 of them is off by twice that (these two by -8e-4
    and +1e-3); the header promises f64's decisions. Probabilities within 5e-6,
    the bound that the kernel states for its first sum."""
    import needle_b200 as nb
    import torch

    S, V = 160, 1 << 24  # 320 rows: a CTA takes a whole one
    row = torch.full((V,), -below, device="cuda")
    row[:4096] = 0.0
    l = row.double().cpu().numpy()
    e = np.exp(l)
    p = e / e.sum()
    draft = np.full((S, 1), 77, np.int32)
    u = np.random.default_rng(3).random((S, 2)).astype(np.float32)
    u[:, 0] = p[77] * (1 + off)
    tokens, accepted, probs = nb.op_verify(row.expand(S, 2, V), _dev(draft), _dev(u), torch.ones(S, device="cuda"))
    stands = int(off < 0)
    assert (accepted.cpu().numpy() == stands).all()
    if not stands:
        e[77] = 0.0
    cum = np.cumsum(e)
    drawn = np.searchsorted(cum, u[:, 1].astype(np.float64) * cum[-1], side="right")
    tokens, probs = tokens.cpu().numpy(), probs.cpu().numpy()
    assert np.array_equal(tokens[:, stands], drawn) and (tokens[:, 1 - stands] == (77 if stands else -1)).all()
    assert (np.abs(probs[:, stands] - p[drawn]) <= 2.0 ** -23 * p[drawn]).all()
    if stands:
        assert (np.abs(probs[:, 0] - p[77]) <= 5e-6 * p[77]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("T,V", [(3, 50), (2, 20011)])
def test_temperatures_below_the_normal_numbers(cuda_device, T, V):
    """Above 0 is above 0: of tied logits each is drawn, also where 1 /
    temperature is no f32, and differences as small as the temperature count."""
    r = np.random.default_rng(V)
    temp = np.array([1e-39, 1.4e-45, 3e-40, 4.2e-39, 1.2e-38, 1e-41, 0.0])
    S = len(temp)
    logits = r.integers(0, 3, (S, T + 1, V)).astype(np.float64)
    logits[5] = r.integers(0, 2000, (T + 1, V)) * 1e-44
    draft = logits[:, :T].argmax(-1)
    q = np.full((S, T, V), 1 / V)
    u = r.random((S, T + 1))
    w = run(logits, draft, u, temp, q)
    assert len({int(t) for t in w[0][np.arange(S), w[1]]}) > 3
    run(logits, draft, u, temp)
    run(np.maximum(logits, 1.0), draft, u, temp, dtype="bfloat16")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("S,T,V", [(2, 2, 9), (5, 3, 20011), (1, 1, 130001)])
def test_infinite_temperatures(cuda_device, dtype, S, T, V):
    """The limit of ever larger ones: all tokens alike, but those at -infinity."""
    logits, draft, u, temp, q = case(S, T, V, 17)
    w = run(logits, draft, u, np.full(S, np.inf), q, dtype=dtype)
    assert (w[0][np.arange(S), w[1]] >= 0).all()
    run(logits, draft, u, np.full(S, 3e38), dtype=dtype)
    logits[:, :, 1::2] = -np.inf
    import needle_b200 as nb
    import torch

    lt = _dev(logits.astype(np.float32)).to(getattr(torch, dtype))
    got = nb.op_verify(lt, _dev(draft.astype(np.int32)), _dev(u.astype(np.float32)), _dev(np.full(S, np.inf, np.float32)))
    want = ref_verify(lt.float().cpu().numpy(), draft, u.astype(np.float32), np.full(S, 3e38, np.float32), None, np.full(S, T))
    assert np.array_equal(got[0].cpu().numpy(), want[0]) and np.array_equal(got[1].cpu().numpy(), want[1])
