"""Arguments of the serving calls that C's types would change: refused before
anything is queued."""

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
