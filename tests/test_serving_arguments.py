"""Arguments of the serving calls that C's types would change, or that would
be written while they are read: refused before anything is queued."""

import numpy as np
import pytest


def test_integers_beyond_a_c_int():
    from needle_b200 import serving

    for x in (0, -1, 2 ** 31 - 1, -2 ** 31):
        assert serving._int(x, "x") == x
    for x in (2 ** 31, -2 ** 31 - 1, 2 ** 32, 2 ** 32 + 10):
        with pytest.raises(ValueError):
            serving._int(x, "x")


@pytest.mark.gpu
def test_calls_refuse_integers_beyond_a_c_int(cuda_device):
    """As 32 bits each of these would be another call: a window of 10, no
    window, no first tokens, one row, pages of 16 positions, one sequence, one page."""
    import needle_b200 as nb
    import torch

    kv = nb.KV4Pool.new(4, 2, 48, 64, page=16)
    table = torch.zeros((1, 2), dtype=torch.int32, device="cuda")
    one = torch.ones(1, dtype=torch.int32, device="cuda")
    q = torch.randn((1, 12, 48), device="cuda")
    for call in (
        lambda: nb.op_kv4_attend(kv, q, table, one, window=2 ** 32 + 10),
        lambda: nb.op_kv4_attend(kv, q, table, one, window=2 ** 32),
        lambda: nb.op_kv4_attend(kv, q, table, one, window=16, sink=2 ** 32),
        lambda: nb.op_kv4_attend(kv, q.expand(2 ** 32 + 1, 12, 48), table, one, out=q.new_empty((1, 12, 64)).expand(2 ** 32 + 1, 12, 64)),
        lambda: nb.op_kv4_attend(kv, q[:, :1].expand(1, 2 ** 32 + 12, 48), table, one, out=q.new_empty((1, 1, 64)).expand(1, 2 ** 32 + 12, 64)),
        lambda: nb.op_kv4_read(kv, table, one, rows=2 ** 32 + 1),
        lambda: nb.KV4Pool(kv.data[:1].expand(2 ** 32 + 1, 2, 1, nb.KV4Pool.tile_bytes(48, 64)), 48, 64),
        lambda: nb.op_pages_fork(kv.data, table, one, one, one, 2 ** 32 + 16),
        lambda: nb.op_pages_fork(kv.data, table, one.expand(2 ** 32 + 1), one, one, 16),
        lambda: nb.op_pages_compact(kv.data[:1].expand(2 ** 32 + 1, 2, 1, nb.KV4Pool.tile_bytes(48, 64)), table),
        lambda: nb.op_verify(torch.zeros((1, 1, 4), device="cuda").expand(1, 2 ** 32 + 1, 4), one.view(1, 1)[:, :0],
                             torch.zeros((1, 1), device="cuda"), torch.zeros(1, device="cuda")),
    ):
        with pytest.raises(ValueError, match="32 bits"):
            call()


def _touched(x, base):
    """The bytes of base that x's values lie on."""
    size, at = x.element_size(), x.data_ptr() - base
    i = [np.arange(n) * s * size for n, s in zip(x.shape, x.stride())]
    first = (at + i[0][:, None, None] + i[1][:, None] + i[2]).reshape(-1, 1) + np.arange(size)
    return set(first.ravel().tolist())


def test_overlap_is_exact():
    """Views of one buffer against the sets of their bytes: side by side within
    a head, a row, whole blocks, shifted by rows, and drawn at random."""
    import torch
    from needle_b200.serving import _overlap

    buf = torch.zeros(40000, dtype=torch.bfloat16)
    at = lambda off, rows, heads, d, r, h: buf.as_strided((rows, heads, d), (r, h, 1), off)
    cases = [(at(0, 9, 4, 8, 64, 16), at(8, 9, 4, 8, 64, 16)),          # q and out of each head side by side
             (at(0, 9, 4, 8, 64, 16), at(9, 9, 4, 8, 64, 16)),          # one value short
             (at(0, 9, 4, 8, 96, 8), at(32, 9, 4, 16, 96, 16)),          # of each row side by side
             (at(0, 9, 4, 8, 96, 8), at(96 + 32, 9, 4, 16, 96, 16)),
             (at(0, 9, 4, 8, 96, 8), at(31, 9, 4, 16, 96, 16)),
             (at(0, 9, 4, 8, 32, 8), at(288, 9, 4, 8, 32, 8)),           # one behind the other
             (at(0, 9, 4, 8, 32, 8), at(287, 9, 4, 8, 32, 8)),
             (at(0, 9, 4, 8, 0, 0), at(8, 9, 4, 8, 32, 8)),              # one query for all rows
             (at(64, 9, 4, 8, 32, 8), at(0, 9, 4, 8, 32, 8))]
    r = np.random.default_rng(0)
    for _ in range(300):
        d, e = r.integers(1, 9, 2)
        cases.append((at(int(r.integers(0, 200)), *(int(x) for x in r.integers(1, 6, 2)), int(d), int(r.integers(0, 90)), int(r.integers(0, 20))),
                      at(int(r.integers(0, 200)), *(int(x) for x in r.integers(1, 6, 2)), int(e), int(r.integers(0, 90)), int(r.integers(0, 20)))))
    seen = {False: 0, True: 0}
    for a, b in cases:
        want = bool(_touched(a, buf.data_ptr()) & _touched(b, buf.data_ptr()))
        assert _overlap(a, b) == want and _overlap(b, a) == want, (a.stride(), b.stride(), a.shape, b.shape)
        seen[want] += 1
    assert min(seen.values()) > 50
    assert not _overlap(buf[:0].view(0, 4, 8), at(0, 2, 4, 8, 32, 8))


@pytest.mark.gpu
def test_out_over_other_rows_queries(cuda_device):
    """An out that lies over rows of q which are still to be read is refused;
    one between q's heads in the same buffer is as good as another."""
    import needle_b200 as nb
    import torch

    kv = nb.KV4Pool.new(8, 2, 64, 64, page=16)
    table = torch.arange(8, dtype=torch.int32, device="cuda").view(4, 2)
    lens = torch.full((4,), 30, dtype=torch.int32, device="cuda")
    nb.op_kv4_append(kv, torch.randn((120, 2, 64), device="cuda"), torch.randn((120, 2, 64), device="cuda"), table, lens,
                     torch.arange(0, 121, 30, dtype=torch.int32, device="cuda"))
    buf = torch.randn((6, 8, 128), device="cuda")
    q = buf[:4, :, :64]
    want = nb.op_kv4_attend(kv, q.contiguous(), table, lens)
    for out in (q, buf[1:5, :, :64], buf[:4, :, 32:96], buf.view(-1)[512:2560].view(4, 8, 64)):
        before = buf.clone()
        with pytest.raises(ValueError, match="overlap"):
            nb.op_kv4_attend(kv, q, table, lens, out=out)
        assert torch.equal(buf, before)
    assert torch.equal(nb.op_kv4_attend(kv, q, table, lens, out=buf[:4, :, 64:]), want)
