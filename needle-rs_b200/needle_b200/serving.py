"""Serving from one pool of pages (include/needle_engine.h, "Serving from one
pool of pages"): a 4-bit key/value cache that sequences of different lengths
share, attention over it, forking and compacting of pages, and the check of
drafted tokens.

Tensors are CUDA tensors of one device; work is queued on that device's
current torch stream. Tables, lengths and offsets are int32 and read on the
device, so calls can be captured into a CUDA graph and replayed as they
change. Bad arguments raise ValueError, or RuntimeError where the C entry
refuses them, before anything is queued.
"""

import ctypes as C
import math

import torch

from . import _err, lib
from ._abi import KV4 as _KV4
from ._abi import PAGES as _PAGES

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_TILE = 16  # positions a tile
_ZERO_REST = 2


def _stream(device):
    """The address of the device's current stream (without the object that
    torch.cuda.current_stream makes of it, 2 us)."""
    return torch._C._cuda_getCurrentRawStream(device.index)


def _int(x, name):
    """x, where a C int holds it: ctypes drops the bits above without a word."""
    if not -2147483648 <= x <= 2147483647:
        raise ValueError(f"{name} is beyond 32 bits: {x}")
    return x


def _int32(t, n, device, name):
    """The address of a contiguous int32 vector of n."""
    if t.dtype is not torch.int32 or t.shape != (n,) or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor [{n}] on {device}")
    return t.data_ptr()


def _overlap(a, b):
    """Whether a value of a and one of b [rows, heads, d] (one type, d
    contiguous, strides not negative) share memory."""
    if not a.numel() or not b.numel():
        return False
    size, (n, h, da), db = a.element_size(), a.shape, b.shape[2]
    off = b.data_ptr() - a.data_ptr()
    if off % size:  # values that lie across one another: by bytes
        (ra, ha), (rb, hb), da, db = [s * size for s in a.stride()[:2]], [s * size for s in b.stride()[:2]], da * size, db * size
    else:
        (ra, ha), (rb, hb), off = a.stride()[:2], b.stride()[:2], off // size
    heads = b.shape[1]
    if off >= (n - 1) * ra + (h - 1) * ha + da or -off >= (b.shape[0] - 1) * rb + (heads - 1) * hb + db:
        return False
    # parts of one buffer that repeats by heads, or by rows
    if ha == hb > 0 and ra % ha == 0 and rb % ha == 0 and off % ha >= da and off % ha + db <= ha:
        return False
    if ra == rb > 0 and off % ra >= (h - 1) * ha + da and off % ra + (heads - 1) * hb + db <= ra:
        return False
    runs = lambda n, r, h, s: (torch.arange(n, device="cpu")[:, None] * r + torch.arange(h, device="cpu") * s).flatten()
    first, other = runs(n, ra, h, ha).sort().values, runs(b.shape[0], rb, heads, hb) + off
    at = torch.searchsorted(first, other + db) - 1  # the last run of a that begins before the one of b ends
    return bool(((at >= 0) & (first[at.clamp(min=0)] + da > other)).any())


class KV4Pool:
    """A pool of pages of 4-bit keys and values. ``data`` is a uint8 CUDA
    tensor [pages, heads, page / 16, tile] as the header lays it out (a page's
    part contiguous; pages may lie further apart, as in a slice of a pool of
    several layers). ``KV4Pool.new`` makes one."""

    def __init__(self, data, dk, dv):
        if data.dtype is not torch.uint8 or data.dim() != 4 or not data.is_cuda:
            raise ValueError("data must be a 4-D uint8 CUDA tensor")
        n, h, tiles, tile = data.shape
        if min(n, h, tiles) < 1 or tile != self.tile_bytes(dk, dv):
            raise ValueError(f"a tile of ({dk}, {dv}) holds {self.tile_bytes(dk, dv)} bytes, got {list(data.shape)}")
        if data.stride(3) != 1 or (tiles > 1 and data.stride(2) != tile) or (h > 1 and data.stride(1) != tiles * tile):
            raise ValueError("a page's heads and tiles must be contiguous")
        _int(max(n, h, tiles * _TILE), "a size of the pool")
        self.data, self.dk, self.dv = data, dk, dv
        self.num_pages, self.heads, self.page = n, h, tiles * _TILE
        self.device = data.device
        self._fixed = bytes(_KV4(data.device.index, data.data_ptr(), data.stride(0) if n > 1 else h * tiles * tile, n,
                                 self.page, h, dk, dv))

    @staticmethod
    def tile_bytes(dk, dv):
        return _TILE * (dk // 2 + dv // 2 + 8)

    @classmethod
    def new(cls, num_pages, heads, dk, dv, page=64, device="cuda"):
        if page < 1 or page % _TILE:
            raise ValueError("page must be a multiple of 16 positions")
        return cls(torch.zeros((num_pages, heads, page // _TILE, cls.tile_bytes(dk, dv)), dtype=torch.uint8,
                               device=device), dk, dv)

    def _args(self, table, lens, start, rows):
        """The C view of a call; its tensors must outlive the call."""
        dev = self.device
        s, a = table.shape[0], _KV4.from_buffer_copy(self._fixed)
        a.seqs, a.max_pages, a.table_stride = _table(table, dev)
        a.table, a.lens, a.rows = table.data_ptr(), _int32(lens, s, dev, "lens"), _int(rows, "rows")
        if start is not None:
            a.start = _int32(start, s + 1, dev, "start")
        return C.byref(a)

    def _rows(self, x, heads, d, name):
        shape, stride = x.shape, x.stride()
        if len(shape) != 3 or shape[1] != heads or shape[2] != d or stride[2] != 1 or x.dtype not in _TYPES or x.device != self.device:
            raise ValueError(f"{name} must be a float32, float16 or bfloat16 tensor [rows, {heads}, {d}] on {self.device}, "
                             "its last dimension contiguous")
        return x.data_ptr(), stride[0], stride[1]


def op_kv4_append(kv, k, v, table, lens, start=None):
    """Quantize rows k [rows, heads, dk] and v [rows, heads, dv] into the
    pages of ``kv`` (nd_op_kv4_append). ``table`` [seqs, pages] holds page
    ids, ``lens`` [seqs] the positions each sequence holds with these rows,
    ``start`` [seqs + 1] the rows' offsets (None: as many rows for each)."""
    if k.dtype is not v.dtype or k.shape[:1] != v.shape[:1]:
        raise ValueError("k and v must have one type and as many rows")
    ka, va = kv._rows(k, kv.heads, kv.dk, "k"), kv._rows(v, kv.heads, kv.dv, "v")
    a = kv._args(table, lens, start, k.shape[0])
    if lib().nd_op_kv4_append(a, _TYPES[k.dtype], *ka, *va, _stream(kv.device)) != 0:
        raise _err()


def op_kv4_read(kv, table, lens, start=None, rows=None, dtype=torch.float32):
    """The values the cache holds for those rows: (k [rows, heads, dk],
    v [rows, heads, dv]) (nd_op_kv4_read). Rows behind the last sequence are
    zeros. ``rows`` is needed with ``start``; without it the default is one
    row a sequence."""
    if rows is None and start is not None:
        raise ValueError("rows must be given with start")
    if dtype not in _TYPES:
        raise ValueError("dtype must be float32, float16 or bfloat16")
    rows = table.shape[0] if rows is None else rows
    a = kv._args(table, lens, start, rows)
    k = kv.data.new_empty((rows, kv.heads, kv.dk), dtype=dtype)
    v = kv.data.new_empty((rows, kv.heads, kv.dv), dtype=dtype)
    hk, hv = kv.heads * kv.dk, kv.heads * kv.dv
    if lib().nd_op_kv4_read(a, _TYPES[dtype], k.data_ptr(), hk, kv.dk, v.data_ptr(), hv, kv.dv, _ZERO_REST,
                            _stream(kv.device)) != 0:
        raise _err()
    return k, v


def op_kv4_attend(kv, q, table, lens, start=None, scale=None, window=0, sink=0, out=None):
    """Attention of rows q [rows, q_heads, dk] over the cache, their own keys
    appended before (nd_op_kv4_attend); returns out [rows, q_heads, dv] of q's
    type. A row sees the positions up to its own, with ``window`` the last
    ``window`` of them and the first ``sink``. ``scale`` defaults to
    1 / sqrt(dk). Rows behind the last sequence are left as they were in a
    given ``out``, which must not overlap ``q``, and are zeros in a new one."""
    shape = q.shape
    if len(shape) != 3 or not shape[1] or shape[1] % kv.heads:
        raise ValueError(f"q must be [rows, q_heads, dk] with a multiple of {kv.heads} heads")
    rows, hq = shape[0], shape[1]
    qa = kv._rows(q, hq, kv.dk, "q")
    a = kv._args(table, lens, start, rows)
    new = out is None
    if new:
        out = q.new_empty((rows, hq, kv.dv))
        oa = out.data_ptr(), hq * kv.dv, kv.dv
    else:
        if out.dtype is not q.dtype or out.shape[:1] != q.shape[:1]:
            raise ValueError("out must have q's type and rows")
        oa = kv._rows(out, hq, kv.dv, "out")
        if _overlap(q, out):
            raise ValueError("out must not overlap q")
    L = lib()
    _int(hq, "q_heads"), _int(window, "window"), _int(sink, "sink")
    n = L.nd_op_kv4_attend_ws(a, _TYPES[q.dtype], hq, window, sink)
    ws = kv.data.new_empty(n) if n else None
    if L.nd_op_kv4_attend(a, _TYPES[q.dtype], *qa, hq, 1 / math.sqrt(kv.dk) if scale is None else scale, window, sink, *oa,
                          ws.data_ptr() if n else None, n, _ZERO_REST if new else 0, _stream(kv.device)) != 0:
        raise _err()
    return out


def _pages(pool, axis):
    """The C view of a pool whose pages lie along `axis` (0: [pages, ..], 1:
    [layers, pages, ..])."""
    if not pool.is_cuda or axis not in (0, 1) or pool.dim() <= axis or not pool.numel():
        raise ValueError("pool must be a CUDA tensor [pages, ..], or [layers, pages, ..] with axis=1")
    n, layers = _int(pool.shape[axis], "pages"), _int(pool.shape[0], "layers") if axis else 1
    size = pool.element_size()
    inner = 1
    for d in range(pool.dim() - 1, axis, -1):
        if pool.stride(d) != inner and pool.shape[d] != 1:
            raise ValueError("a page must be contiguous")
        inner *= pool.shape[d]
    nbytes = inner * size
    return C.byref(_PAGES(pool.device.index, pool.data_ptr(), pool.stride(axis) * size if n > 1 else nbytes,
                          pool.stride(0) * size if axis and layers > 1 else 0, nbytes, n, layers)), n


def _table(table, device):
    if table.dtype is not torch.int32 or table.dim() != 2 or table.device != device:
        raise ValueError(f"table must be an int32 tensor [seqs, pages] on {device}")
    (s, p), (stride, inner) = table.shape, table.stride()
    if not s or not p or (inner != 1 and p > 1):
        raise ValueError("table must have sequences and columns, each row contiguous")
    _int(max(s, p, stride), "a size of the table")
    return s, p, stride if s > 1 else p


def _pinned(pinned, n, device):
    if pinned is None:
        return None
    if (pinned.dtype not in (torch.uint8, torch.bool) or pinned.device != device or pinned.shape != (n,)
            or not pinned.is_contiguous()):
        raise ValueError(f"pinned must be a contiguous uint8 or bool tensor [{n}] on {device}")
    return pinned.data_ptr()


def op_pages_fork(pool, table, src, keep, need, page, pinned=None, axis=0):
    """A new set of sequences from the old ones' pages (nd_op_pages_fork):
    sequence d keeps ``keep[d]`` positions of old sequence ``src[d]`` (-1: of
    none) and gets pages for ``need[d]``, ``page`` positions a page. Whole
    pages are shared, a partly filled one that will be written is copied in
    ``pool`` (any type; [pages, ..], or [layers, pages, ..] with axis=1), pages
    nothing refers to are free. Returns (table [n, columns], refs [pages],
    info [4]: pages in use, given, copied, wanted but not had)."""
    dev = pool.device
    pv, n_pages = _pages(pool, axis)
    s, p, stride = _table(table, dev)
    n = _int(src.shape[0], "src's length") if src.dim() else 0
    if not n:
        raise ValueError("src must name at least one sequence")
    out, refs = table.new_empty((n, p)), table.new_empty(n_pages)
    _int(page, "page")
    L = lib()
    size = L.nd_op_pages_fork_ws(n_pages, n)
    ws = table.new_empty(4 + (size + 3) // 4)
    info = ws[:4]
    if L.nd_op_pages_fork(pv, table.data_ptr(), stride, s, p, page, _int32(src, n, dev, "src"), _int32(keep, n, dev, "keep"),
                          _int32(need, n, dev, "need"), n, _pinned(pinned, n_pages, dev), out.data_ptr(), refs.data_ptr(),
                          ws.data_ptr(), ws.data_ptr() + 16, size, _stream(dev)) != 0:
        raise _err()
    return out, refs, info


def op_pages_compact(pool, table, pinned=None, axis=0):
    """Live pages to the front of the pool (nd_op_pages_compact). Returns
    (table, map [pages]: each live page's new id or -1, info [2]: live pages,
    pages moved)."""
    dev = pool.device
    pv, n_pages = _pages(pool, axis)
    s, p, stride = _table(table, dev)
    out, to = table.new_empty((s, p)), table.new_empty(n_pages)
    L = lib()
    size = L.nd_op_pages_compact_ws(n_pages)
    ws = table.new_empty(4 + (size + 3) // 4)
    info = ws[:2]
    if L.nd_op_pages_compact(pv, table.data_ptr(), stride, s, p, _pinned(pinned, n_pages, dev), out.data_ptr(), to.data_ptr(),
                             ws.data_ptr(), ws.data_ptr() + 16, size, _stream(dev)) != 0:
        raise _err()
    return out, to, info


def op_verify(logits, draft, u, temperature, q=None, counts=None):
    """Check drafted tokens and draw the next (nd_op_verify): logits
    [seqs, T + 1, V] float32, float16 or bfloat16, draft [seqs, T] int32,
    u [seqs, T + 1] float32 in [0, 1), temperature [seqs] float32 (not above
    0: greedy), q [seqs, T, V] float32 the draft's probabilities (None: it was
    certain), counts [seqs] int32 how many drafts there are (None: T). Returns
    (tokens [seqs, T + 1]: accepted drafts, the drawn token, then -1;
    accepted [seqs]; probs [seqs, T + 1])."""
    dev = logits.device
    if logits.dtype not in _TYPES or logits.dim() != 3 or not logits.is_cuda or logits.stride(2) != 1 or not logits.numel():
        raise ValueError("logits must be a float32, float16 or bfloat16 CUDA tensor [seqs, T + 1, V], rows contiguous")
    s, t1, v = logits.shape
    _int(max(s, t1, v), "a size of logits")
    t = t1 - 1
    if draft.dtype is not torch.int32 or draft.shape != (s, t) or draft.device != dev or not draft.is_contiguous():
        raise ValueError(f"draft must be a contiguous int32 tensor [{s}, {t}] on {dev}")
    if u.dtype is not torch.float32 or u.shape != (s, t1) or u.device != dev or not u.is_contiguous():
        raise ValueError(f"u must be a contiguous float32 tensor [{s}, {t1}] on {dev}")
    if temperature.dtype is not torch.float32 or temperature.shape != (s,) or temperature.device != dev or not temperature.is_contiguous():
        raise ValueError(f"temperature must be a contiguous float32 tensor [{s}] on {dev}")
    if q is not None and (q.dtype is not torch.float32 or q.shape != (s, t, v) or q.device != dev
                          or (t and q.stride(2) != 1 and v > 1)):
        raise ValueError(f"q must be a float32 tensor [{s}, {t}, {v}] on {dev}, rows contiguous")
    c = None if counts is None else _int32(counts, s, dev, "counts")
    tokens, accepted, probs = draft.new_empty((s, t1)), draft.new_empty(s), u.new_empty((s, t1))
    qa = (None, 0, 0) if q is None or not t else (q.data_ptr(), q.stride(0), q.stride(1))
    L = lib()
    size = L.nd_op_verify_ws(s, t, v)
    ws = u.new_empty(size // 4)
    if L.nd_op_verify(dev.index, _TYPES[logits.dtype], logits.data_ptr(), logits.stride(0), logits.stride(1),
                      draft.data_ptr(), c, u.data_ptr(), temperature.data_ptr(), *qa, s, t, v, tokens.data_ptr(),
                      accepted.data_ptr(), probs.data_ptr(), ws.data_ptr(), size, _stream(dev)) != 0:
        raise _err()
    return tokens, accepted, probs
