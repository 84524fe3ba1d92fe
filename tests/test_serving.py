"""The serving ops together, as a speculative server would run them: sequences
of different lengths grow by drafts over one pool of pages. Each step forks
the set (accepted positions kept, refused ones freed, room for the next
draft), appends the drafts' rows, attends, scores and verifies. Every op's
result is checked against its restatement on the same inputs, and at the end
the pool is compacted and answers as before."""

import numpy as np
import pytest

import kv4_ref
from test_kv4 import _np, _tol
from test_pages import ref_fork
from test_verify import ref_verify


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,heads,kv_heads,dk,dv", [("f32", 12, 2, 48, 64), ("bf16", 8, 2, 128, 128)])
def test_speculative_steps(cuda_device, dtype, heads, kv_heads, dk, dv):
    import needle_b200 as nb
    import torch

    dt = {"f32": torch.float32, "bf16": torch.bfloat16}[dtype]
    g = torch.Generator(device="cuda").manual_seed(3)
    V, D, S, T, page, pages, cols = 300, 64, 5, 4, 16, 60, 10

    def rand(*shape, scale=1.0):
        return torch.randn(shape, device="cuda", generator=g) * scale

    emb = rand(V, D)
    wq, wk, wv, wo = rand(D, heads * dk, scale=0.2), rand(D, kv_heads * dk, scale=0.2), rand(D, kv_heads * dv, scale=0.2), rand(heads * dv, V, scale=0.3)
    kv = nb.KV4Pool.new(pages, kv_heads, dk, dv, page=page)
    ref = kv4_ref.Cache(pages, kv_heads, page, dk, dv)
    table = torch.full((S, cols), -1, dtype=torch.int32, device="cuda")
    held = torch.zeros(S, dtype=torch.int32, device="cuda")  # positions of accepted tokens in the cache
    rng = np.random.default_rng(0)
    tokens = [list(rng.integers(0, V, n)) for n in (3, 17, 1, 30, 16)]
    pending = [list(t) for t in tokens]  # tokens whose rows the cache does not hold
    nobody = np.zeros(pages, bool)

    def dev(a):
        return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")

    for step in range(6):
        draft = torch.randint(0, V, (S, T), device="cuda", generator=g, dtype=torch.int32)
        if step % 2:  # likely tokens, so that some stand
            draft = torch.topk(emb[[t[-1] for t in tokens]] @ emb.T, T).indices.int()
        counts = rng.integers(0, T + 1, S)
        feed = [p + draft[s, : counts[s]].tolist() for s, p in enumerate(pending)]
        n = np.array([len(f) for f in feed])
        src = list(range(S))
        if step == 3:  # a sequence is abandoned for a copy of another
            src[0] = 3
            tokens[0], pending[0] = list(tokens[3]), list(pending[3])
            feed[0] = pending[0] + draft[0, : counts[0]].tolist()
            n[0] = len(feed[0])
        keep = held[src]
        need = keep + dev(n)
        old = (_np(table), keep.cpu().numpy(), need.cpu().numpy())
        data_before = [[p for p in kv.data.view(pages, -1).cpu().numpy()]]
        new_table, refs, info = nb.op_pages_fork(kv.data, table, dev(src), keep, need, page)
        w = ref_fork(data_before, old[0].astype(np.int64), src, old[1], old[2], page, pages, nobody)
        assert np.array_equal(new_table.cpu().numpy(), w[0]) and info.tolist() == w[2] and w[2][3] == 0
        assert np.array_equal(kv.data.view(pages, -1).cpu().numpy(), np.array(w[3][0]))
        k_ref, v_ref = ref.k.copy(), ref.v.copy()  # the copies in the restatement
        for s in range(S):
            for c in range(cols):
                a, b = (int(old[0][src[s], c]) if c * page < old[1][s] else -1), int(w[0][s, c])
                if a >= 0 and b != a:
                    ref.k[b], ref.v[b] = k_ref[a], v_ref[a]
        table, lens = new_table, need
        start = dev(np.concatenate([[0], np.cumsum(n)]))
        x = emb[torch.tensor(sum(feed, []), device="cuda")]
        k, v, q = ((x @ m).to(dt) for m in (wk, wv, wq))
        k, v, q = k.view(-1, kv_heads, dk), v.view(-1, kv_heads, dv), q.view(-1, heads, dk)
        nb.op_kv4_append(kv, k, v, table, lens, start)
        args = (table.cpu().numpy(), lens.cpu().numpy(), start.cpu().numpy())
        ref.append(_np(k), _np(v), *args)
        out = nb.op_kv4_attend(kv, q, table, lens, start, window=24, sink=3)
        want, b, top = ref.attend(_np(q), *args, 1 / np.sqrt(dk), 24, 3)
        assert (np.abs(_np(out) - want) <= _tol(dtype, want, b, top, int(lens.max()))).all()
        # the last counts + 1 rows of each sequence predict its drafts and what follows
        logits = out.float().reshape(-1, heads * dv) @ wo
        ends = np.cumsum(n)
        at = np.array([[min(ends[s] - 1 - counts[s] + i, ends[s] - 1) for i in range(T + 1)] for s in range(S)])
        rows = logits[torch.from_numpy(at).cuda()]
        u = torch.rand((S, T + 1), device="cuda", generator=g)
        temp = torch.tensor([0.0, 1.0, 3.0, 0.0, 2.0], device="cuda")
        qd = torch.softmax(rand(S, T, V), -1)
        got = nb.op_verify(rows, draft, u, temp, q=qd, counts=dev(counts))
        wv_ = ref_verify(_np(rows), draft.cpu().numpy(), _np(u), _np(temp), _np(qd), counts)
        assert np.array_equal(got[0].cpu().numpy(), wv_[0]) and np.array_equal(got[1].cpu().numpy(), wv_[1])
        # the refused drafts' rows are dropped: the next fork keeps the rest
        held = lens - dev(counts) + got[1]
        for s in range(S):
            a = int(wv_[1][s])
            tokens[s] += [int(t) for t in wv_[0][s, : a + 1]]
            pending[s] = tokens[s][-1:]
            assert len(tokens[s]) == int(held[s]) + 1

    one = torch.randn((S, heads, dk), device="cuda", generator=g).to(dt)
    before = nb.op_kv4_attend(kv, one, table, held)
    moved, to, info = nb.op_pages_compact(kv.data, table)
    assert int(moved.max()) + 1 == int(info[0])
    assert torch.equal(nb.op_kv4_attend(kv, one, moved, held), before)
