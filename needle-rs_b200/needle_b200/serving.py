"""Serving from one pool of pages (include/needle_engine.h, "Serving from one
pool of pages"): a 4-bit key/value cache that sequences of different lengths
share, and attention over it.

Tensors are CUDA tensors of one device; work is queued on that device's
current torch stream. Tables, lengths and offsets are int32 and read on the
device, so calls can be captured into a CUDA graph and replayed as they
change. Bad arguments raise ValueError before anything is queued.
"""

import ctypes as C
import math

import torch

from . import _err, lib
from ._abi import KV4 as _KV4

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_TILE = 16  # positions a tile


def _need(ok, what):
    if not ok:
        raise ValueError(what)


def _stream(device):
    return torch.cuda.current_stream(device).cuda_stream


def _int32(t, shape, device, name):
    _need(t.dtype == torch.int32 and t.device == device and tuple(t.shape) == shape and t.is_contiguous(),
          f"{name} must be a contiguous int32 tensor {list(shape)} on {device}")
    return t.data_ptr()


class KV4Pool:
    """A pool of pages of 4-bit keys and values. ``data`` is a uint8 CUDA
    tensor [pages, heads, page / 16, tile] as the header lays it out (a page's
    part contiguous; pages may lie further apart, as in a slice of a pool of
    several layers). ``KV4Pool.new`` makes one."""

    def __init__(self, data, dk, dv):
        _need(data.dtype == torch.uint8 and data.dim() == 4 and data.is_cuda, "data must be a 4-D uint8 CUDA tensor")
        n, h, tiles, tile = data.shape
        _need(min(n, h, tiles) > 0 and tile == self.tile_bytes(dk, dv),
              f"a tile of ({dk}, {dv}) holds {self.tile_bytes(dk, dv)} bytes, got {list(data.shape)}")
        _need(data.stride(3) == 1 and data.stride(2) == tile and (data.stride(1) == tiles * tile or h == 1),
              "a page's heads and tiles must be contiguous")
        self.data, self.dk, self.dv = data, dk, dv
        self.num_pages, self.heads, self.page = n, h, tiles * _TILE
        self.device = data.device

    @staticmethod
    def tile_bytes(dk, dv):
        return _TILE * (dk // 2 + dv // 2 + 8)

    @classmethod
    def new(cls, num_pages, heads, dk, dv, page=64, device="cuda"):
        _need(page > 0 and page % _TILE == 0, "page must be a multiple of 16 positions")
        return cls(torch.zeros((num_pages, heads, page // _TILE, cls.tile_bytes(dk, dv)), dtype=torch.uint8,
                               device=device), dk, dv)

    def _args(self, table, lens, start, rows):
        """The C view of a call; its tensors must outlive the call."""
        dev = self.device
        _need(table.dtype == torch.int32 and table.dim() == 2 and table.device == dev and table.stride(1) == 1
              and table.shape[0] > 0 and table.shape[1] > 0, f"table must be an int32 tensor [seqs, pages] on {dev}")
        s, p = table.shape
        stride = table.stride(0) if s > 1 else max(table.stride(0), p)
        return _KV4(dev.index, self.data.data_ptr(), self.data.stride(0), self.num_pages, self.page, self.heads, self.dk,
                    self.dv, table.data_ptr(), stride, p, s, _int32(lens, (s,), dev, "lens"),
                    None if start is None else _int32(start, (s + 1,), dev, "start"), rows)

    def _rows(self, x, heads, d, name):
        _need(x.dtype in _TYPES and x.dim() == 3 and x.device == self.device and x.shape[1] == heads and x.shape[2] == d
              and (x.stride(2) == 1 or not x.numel()),
              f"{name} must be a float32, float16 or bfloat16 tensor [rows, {heads}, {d}] on {self.device}")
        return x.data_ptr(), x.stride(0), x.stride(1)


def op_kv4_append(kv, k, v, table, lens, start=None):
    """Quantize rows k [rows, heads, dk] and v [rows, heads, dv] into the
    pages of ``kv`` (nd_op_kv4_append). ``table`` [seqs, pages] holds page
    ids, ``lens`` [seqs] the positions each sequence holds with these rows,
    ``start`` [seqs + 1] the rows' offsets (None: as many rows for each)."""
    _need(k.dtype == v.dtype and k.shape[0] == v.shape[0], "k and v must have one type and as many rows")
    a = kv._args(table, lens, start, k.shape[0])
    if lib().nd_op_kv4_append(C.byref(a), _TYPES.get(k.dtype, -1), *kv._rows(k, kv.heads, kv.dk, "k"),
                              *kv._rows(v, kv.heads, kv.dv, "v"), _stream(kv.device)) != 0:
        raise _err()


def op_kv4_read(kv, table, lens, start=None, rows=None, dtype=torch.float32):
    """The values the cache holds for those rows: (k [rows, heads, dk],
    v [rows, heads, dv]) (nd_op_kv4_read). Rows behind the last sequence are
    zeros. ``rows`` is needed with ``start``; without it the default is one
    row a sequence."""
    _need(rows is not None or start is None, "rows must be given with start")
    _need(dtype in _TYPES, "dtype must be float32, float16 or bfloat16")
    rows = table.shape[0] if rows is None else rows
    a = kv._args(table, lens, start, rows)
    make = torch.empty if start is None else torch.zeros
    k = make((rows, kv.heads, kv.dk), dtype=dtype, device=kv.device)
    v = make((rows, kv.heads, kv.dv), dtype=dtype, device=kv.device)
    if lib().nd_op_kv4_read(C.byref(a), _TYPES[dtype], *kv._rows(k, kv.heads, kv.dk, "k"),
                            *kv._rows(v, kv.heads, kv.dv, "v"), _stream(kv.device)) != 0:
        raise _err()
    return k, v


def op_kv4_attend(kv, q, table, lens, start=None, scale=None, window=0, sink=0, out=None):
    """Attention of rows q [rows, q_heads, dk] over the cache, their own keys
    appended before (nd_op_kv4_attend); returns out [rows, q_heads, dv] of q's
    type. A row sees the positions up to its own, with ``window`` the last
    ``window`` of them and the first ``sink``. ``scale`` defaults to
    1 / sqrt(dk). Rows behind the last sequence are left as they were in a
    given ``out`` and are zeros in a new one."""
    _need(q.dim() == 3, "q must be [rows, q_heads, dk]")
    rows, hq = q.shape[0], q.shape[1]
    _need(hq > 0 and hq % kv.heads == 0, f"q_heads must be a multiple of the {kv.heads} kv heads")
    qa = kv._rows(q, hq, kv.dk, "q")
    a = kv._args(table, lens, start, rows)
    if out is None:
        make = torch.empty if start is None else torch.zeros
        out = make((rows, hq, kv.dv), dtype=q.dtype, device=kv.device)
    _need(out.dtype == q.dtype and out.shape[0] == rows, "out must have q's type and rows")
    n = lib().nd_op_kv4_attend_ws(C.byref(a), hq)
    ws = torch.empty(n, dtype=torch.uint8, device=kv.device)
    if lib().nd_op_kv4_attend(C.byref(a), _TYPES[q.dtype], *qa, hq, 1 / math.sqrt(kv.dk) if scale is None else scale,
                              window, sink, *kv._rows(out, hq, kv.dv, "out"), ws.data_ptr(), n, _stream(kv.device)) != 0:
        raise _err()
    return out
