"""The serving ops' part of the C ABI (include/needle_engine.h)."""

import ctypes as C


class KV4(C.Structure):
    _fields_ = [("device", C.c_int), ("pool", C.c_void_p), ("page_stride", C.c_longlong), ("num_pages", C.c_int),
                ("page", C.c_int), ("heads", C.c_int), ("dk", C.c_int), ("dv", C.c_int), ("table", C.c_void_p),
                ("table_stride", C.c_int), ("max_pages", C.c_int), ("seqs", C.c_int), ("lens", C.c_void_p),
                ("start", C.c_void_p), ("rows", C.c_int)]


SIGNATURES = {
    "nd_op_kv4_append": (C.c_int, [C.c_void_p, C.c_int, C.c_void_p, C.c_longlong, C.c_longlong, C.c_void_p,
                                   C.c_longlong, C.c_longlong, C.c_void_p]),
    "nd_op_kv4_read": (C.c_int, [C.c_void_p, C.c_int, C.c_void_p, C.c_longlong, C.c_longlong, C.c_void_p,
                                 C.c_longlong, C.c_longlong, C.c_int, C.c_void_p]),
    "nd_op_kv4_attend_ws": (C.c_ulonglong, [C.c_void_p, C.c_int, C.c_int, C.c_int]),
    "nd_op_kv4_attend": (C.c_int, [C.c_void_p, C.c_int, C.c_void_p, C.c_longlong, C.c_longlong, C.c_int, C.c_float,
                                   C.c_int, C.c_int, C.c_void_p, C.c_longlong, C.c_longlong, C.c_void_p, C.c_ulonglong,
                                   C.c_int, C.c_void_p]),
}
