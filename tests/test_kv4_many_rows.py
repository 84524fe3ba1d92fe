"""The many-row attention kernel (prompts of 16-bit rows): values whose scales
lie far apart, 64 query heads on one kv head, windows that hide keys with NaN
among them. Each test asserts that its call goes to that kernel, by the size of
the workspace it asks for. (test_kv4's tests on wide tables reach it where no
window, or one of more than 48 tiles, is given: smaller ones make units short.)
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


def widen(st):
    """Columns to spare: the call's plan follows what a table could hold."""
    st.table = np.pad(st.table, ((0, 0), (0, 40000)), constant_values=-1)
    return st


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads", list(HEADS))
@pytest.mark.parametrize("at", [100, 288, 319, 330])
def test_a_large_value_that_rows_cannot_see(cuda_device, heads, dtype, at):
    """One position's values 2^20 times the others': rows before it answer
    as if it were not there, with the tolerance of what they see."""
    st = Setup(heads, dtype, [400, 60], [380, 40], 32, seed=at)
    st.v *= 2.0 ** -8
    st.v[at] *= 2.0 ** 20
    widen(st.append())
    _check(st, dtype, attend(st))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads", list(HEADS))
def test_a_large_value_of_small_weight(cuda_device, heads, dtype):
    """The same where every later row sees it, with a score some 40 nats
    below the others. Tolerance: errors follow the weighted magnitude
    sum p_j max |v_j| of what is seen, not the largest value: (2 d + w) of it
    with test_kv4's d and w, f16's last step for each key (2^-25 against 2^11
    and codes to 8), and the truncated sums, keys / 16 of 2^-22."""
    st = Setup(heads, dtype, [400], [380], 32, seed=5)
    st.q = (st.q * 0.25 + 1).to(st.t)
    st.v *= 2.0 ** -8
    st.v[50] *= 2.0 ** 20
    st.k *= 0.5
    st.k[50] = -320.0 / st.dk
    widen(st.append())
    scale = 0.125
    got = _np(attend(st, scale=scale))
    pages = st.table[0, np.arange(400) // 32]
    kk, vv = st.ref.k[pages, :, np.arange(400) % 32], st.ref.v[pages, :, np.arange(400) % 32]  # [keys, heads, d]
    group = st.hq // st.h
    half = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}[dtype]
    for g in range(st.hq):
        x = _np(st.q)[:, g].astype(np.float64) @ kk[:, g // group].T * scale
        x[np.arange(400)[None] > np.arange(20, 400)[:, None]] = -np.inf
        p = np.exp(x - x.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        want = p @ vv[:, g // group]
        mag = (p @ np.abs(vv[:, g // group]).max(1))[:, None]
        assert (p[31:, 50] < 1e-13).all()
        b = scale * np.abs(_np(st.q)[:, g]).sum(1, keepdims=True) * 2 * np.abs(kk).max()
        tol = half * np.abs(want) * (1 + 2.0 ** -7) + 2.0 ** -25 + mag * (
            2 * (2.0 ** -17 * b + 2.0 ** -20) + (2.0 ** -11 if dtype == "bf16" else 2.0 ** -21) + 400 * 2.0 ** -33 + 400 / 16 * 2.0 ** -22)
        err = np.abs(got[:, g] - want)
        assert (err <= tol).all(), f"head {g}: {np.nanmax(err / tol):.3g} of the tolerance"


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


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads", list(HEADS))
def test_waits_that_run_out(cuda_device, heads, dtype):
    """With hardly a round for its waits the kernel gives rows up: what it
    returns is NaN or right, it ends, and the next call is right. (Nothing that
    follows a wait takes an address from what was waited for, the barriers among
    warps are passed either way, and products under way are drained.)"""
    import needle_b200 as nb
    import torch

    st = widen(Setup(heads, dtype, [900, 600, 300], [250, 200, 300], 32, seed=2, extra_rows=2).append())
    want = attend(st)
    for rounds in (0, 1, 2, 4):
        was = nb.lib().nd_op_kv4_attend_wait_rounds(rounds)
        try:
            got = attend(st)
            torch.cuda.synchronize()
        finally:
            assert nb.lib().nd_op_kv4_attend_wait_rounds(was) == rounds
        gone = torch.isnan(got)
        assert (gone | (got == want)).all() and (got[-2:] == 0).all()
        assert rounds or gone[:-2].all()
    assert torch.equal(attend(st), want)
