"""The many-row attention kernel (prompts of 16-bit rows): 64 query heads on
one kv head, windows that hide keys with NaN among them. Each test asserts that
its call goes to that kernel, by the size of the workspace it asks for.
"""

import numpy as np
import pytest

from test_kv4 import HEADS, Setup, _check, _np

TYPES = {"f32": 0, "f16": 1, "bf16": 2}


def uses_many_row_kernel(kv, q, table, lens, start=None, window=0, sink=0):
    import needle_b200 as nb
    import torch

    name = {torch.float32: "f32", torch.float16: "f16", torch.bfloat16: "bf16"}[q.dtype]
    n = nb.lib().nd_op_kv4_attend_ws(kv._args(table, lens, start, q.shape[0]), TYPES[name], q.shape[1], window, sink)
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    return n == sms * (16 + 2 * 4 * 256 * (kv.dv + 2))  # a join and two parts of 256 rows a CTA


def attend(st, window=0, sink=0, scale=None):
    import needle_b200 as nb

    t, lens, start = st.dev(st.table), st.dev(st.lens), st.dev(st.start)
    assert uses_many_row_kernel(st.kv, st.q, t, lens, start, window, sink)
    return nb.op_kv4_attend(st.kv, st.q, t, lens, start, window=window, sink=sink, scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("window,sink", [(0, 0), (900, 40)])
def test_many_heads_on_one(cuda_device, dtype, window, sink):
    HEADS["mqa"] = (64, 1, 64, 64)
    try:
        st = Setup("mqa", dtype, [1500, 40, 1000], [70, 0, 20], 64, seed=4).append()
        _check(st, dtype, attend(st, window, sink), window, sink)
    finally:
        del HEADS["mqa"]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads", list(HEADS))
@pytest.mark.parametrize("window,sink", [(800, 0), (830, 70)])
def test_windows_that_hide_keys(cuda_device, heads, dtype, window, sink):
    rows = {"needle": 300, "small": 700, "wide": 700}[heads]
    st = Setup(heads, dtype, [1500, 1400], [rows, rows - 100], 64, seed=window).append()
    _check(st, dtype, attend(st, window, sink), window, sink)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_nan_behind_a_window(cuda_device, dtype):
    st = Setup("small", dtype, [1500], [1300], 64, seed=9)
    st.k[300, 1] = float("nan")
    st.v[400, 2] = float("inf")
    st.v[5, 0] = float("nan")  # a first token that stays visible
    st.append()
    st.q[7, 3, 3] = float("nan")
    pos = np.arange(200, 1500)
    for sink in (0, 8):
        got = _np(attend(st, 900, sink))
        nan = np.zeros((1300, 4), bool)
        nan[(pos >= 300) & (pos < 1200), 1] = True
        nan[(pos >= 400) & (pos < 1300), 2] = True
        nan[pos < 905, 0] = True
        if sink:
            nan[:, 0] = True
        nan[7, 3] = True
        assert np.array_equal(np.isnan(got).any(-1), nan) and np.array_equal(np.isnan(got).all(-1), nan)
