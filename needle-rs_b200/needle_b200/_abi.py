"""The serving ops' part of the C ABI (include/needle_engine.h)."""

import ctypes as C


class KV4(C.Structure):
    _fields_ = [("device", C.c_int), ("pool", C.c_void_p), ("page_stride", C.c_longlong), ("num_pages", C.c_int),
                ("page", C.c_int), ("heads", C.c_int), ("dk", C.c_int), ("dv", C.c_int), ("table", C.c_void_p),
                ("table_stride", C.c_int), ("max_pages", C.c_int), ("seqs", C.c_int), ("lens", C.c_void_p),
                ("start", C.c_void_p), ("rows", C.c_int)]


class PAGES(C.Structure):
    _fields_ = [("device", C.c_int), ("pool", C.c_void_p), ("page_stride", C.c_longlong), ("layer_stride", C.c_longlong),
                ("page_bytes", C.c_longlong), ("num_pages", C.c_int), ("layers", C.c_int)]


_P, _I, _L, _U = C.c_void_p, C.c_int, C.c_longlong, C.c_ulonglong

SIGNATURES = {
    "nd_op_pages_fork_ws": (_U, [_I, _I]),
    "nd_op_pages_fork": (_I, [_P, _P, _I, _I, _I, _I, _P, _P, _P, _I, _P, _P, _P, _P, _P, _U, _P]),
    "nd_op_pages_compact_ws": (_U, [_I]),
    "nd_op_pages_compact": (_I, [_P, _P, _I, _I, _I, _P, _P, _P, _P, _P, _U, _P]),
    "nd_op_verify_ws": (_U, [_I, _I, _I]),
    "nd_op_verify": (_I, [_I, _I, _P, _L, _L, _P, _P, _P, _P, _P, _L, _L, _I, _I, _I, _P, _P, _P, _P, _U, _P]),
    "nd_op_kv4_append": (_I, [_P, _I, _P, _L, _L, _P, _L, _L, _P]),
    "nd_op_kv4_read": (_I, [_P, _I, _P, _L, _L, _P, _L, _L, _I, _P]),
    "nd_op_kv4_attend_ws": (_U, [_P, _I, _I, _I, _I]),
    "nd_op_kv4_attend_wait_rounds": (C.c_uint, [C.c_uint]),
    "nd_op_kv4_attend": (_I, [_P, _I, _P, _L, _L, _I, C.c_float, _I, _I, _P, _L, _L, _P, _U, _I, _P]),
}
