"""Attention over the paged 4-bit cache where one key takes nearly all weight
of a long row: what tens of thousands of small weights add up to must not be
lost beside it.

The first key's score lies `gap` nats above those of all others, which are
equal (keys of one value each, so that scores are exact but for roundings),
and the background's values repeat a page. So with n background keys

    out = (e^gap v_0 + sum_{1 .. n} v_j) / (e^gap + n)

in 64 bits, from the values as the format holds them. Every sequence reads the
same two pages, and there are as many sequences as warps (or CTAs of the
many-row kernel), so that each takes a whole row in one run.

Tolerance, relative to the largest value that a row sees (top):
 - half a step of the output type;
 - the scores: scale, product, sum with the running reference, 2^-24 each of
   |score| <= gap, and 2^-22 for the exponential: d = gap 2^-22 + 2^-22,
   which moves the result by at most share (1 - share) d |v_0 - v_j|, where
   share is the background's part of the weight and |v_0 - v_j| <= 2 top;
 - weights: 2^-22 of themselves in two f16 terms (bf16 rows: 2^-12 in one),
   never more than top in all; and half of f16's last step, 2^-25, for each key
   where the largest weight is 2^11 or more: codes to 8, top at least 7 of
   the value's steps: n 2^-25 2^-11 8 / 7;
 - sums: f32 rows add 16 rounds in f32 (2^-24 each) to sums in f64, with the
   codes' part and the middles' part of at most 2 top each; 16-bit rows add
   64 products a term that are truncated at 2^-23 each, and such sums, of
   1024 keys, in f32; the many-row kernel has 256 products a term, and sums of 4096
   keys (64 additions) in f32.
"""

import numpy as np
import pytest

import kv4_ref
from test_kv4 import _np, _torch_type
from test_kv4_many_rows import uses_many_row_kernel

HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
PAGE = 128


def tolerance(dtype, n, gap, share, top, want, many_rows):
    d = (gap + 1) * 2.0 ** -22
    weights = (2.0 ** -12 if dtype == "bf16" else 2.0 ** -22) + n * 2.0 ** -36 * 8 / 7
    terms = 1 if dtype == "bf16" else 2
    if many_rows:
        sums = 2 * (256 * 2.0 ** -23 * terms + (n / 4096 + 64) * 2.0 ** -24)
    elif dtype == "f32":
        sums = 2 * 16 * 2.0 ** -24 + 2.0 ** -21
    else:
        sums = 2 * (64 * 2.0 ** -23 * terms + (n / 1024 + 32) * 2.0 ** -24)
    floor = 2.0 ** -25 if dtype == "f16" else 0.0
    return HALF[dtype] * np.abs(want) * (1 + 2.0 ** -7) + floor + (2 * share * (1 - share) * d + weights + sums) * top


def run(dtype, dk, dv, keys, rows, seqs, gap, flat, many_rows=False, factor=1.0):
    import needle_b200 as nb
    import torch

    t = _torch_type(dtype)
    r = np.random.default_rng(int(gap))
    kv = nb.KV4Pool.new(2, 1, dk, dv, page=PAGE)
    pages = -(-keys // PAGE)
    k = np.zeros((2 * PAGE, 1, dk), np.float32)
    k[0] = 1.0
    v = r.standard_normal((2 * PAGE, 1, dv)).astype(np.float32) * factor
    v[PAGE:] = v[:PAGE]  # the background's page, and the first one with its first key's value
    if flat:
        v[:] = v[1]
    v[0] = r.standard_normal((1, dv)).astype(np.float32) * factor
    k, v = torch.from_numpy(k).cuda().to(t), torch.from_numpy(v).cuda().to(t)
    nb.op_kv4_append(kv, k, v, torch.tensor([[0, 1]], dtype=torch.int32, device="cuda"),
                     torch.tensor([2 * PAGE], dtype=torch.int32, device="cuda"))
    table = torch.ones((1, pages), dtype=torch.int32, device="cuda")
    table[0, 0] = 0
    table = table.repeat(seqs, 1)
    lens = torch.full((seqs,), keys, dtype=torch.int32, device="cuda")
    q = torch.full((seqs * rows, 1, dk), gap / dk, device="cuda", dtype=t)
    assert float(q[0, 0, 0]) * dk == gap
    if many_rows:
        assert uses_many_row_kernel(kv, q, table, lens)
    got = _np(nb.op_kv4_attend(kv, q, table, lens, scale=1.0).view(seqs, rows, dv))
    c, s, m = kv4_ref.quantize(_np(v))
    val = (m.astype(np.float64)[..., None] + s.astype(np.float64)[..., None] * c)[:, 0]
    pos = np.arange(keys - rows, keys)
    whole, part = np.divmod(pos + 1, PAGE)  # background keys of the repeated page, less the first key's slot
    cum = np.concatenate([np.zeros((1, dv)), np.cumsum(val[PAGE:], 0)])
    background = whole[:, None] * cum[-1] + cum[part] - val[PAGE]
    e = np.exp(float(gap))
    want = (e * val[0] + background) / (e + pos[:, None])
    share = (pos / (e + pos))[:, None]
    top = np.abs(val).max()
    err = np.abs(got - want)
    tol = tolerance(dtype, keys, gap, share, top, want, many_rows)
    assert (err <= tol).all(), f"{err.max() / top:.3g} of the values, {(err / tol).max():.3g} of the tolerance"


def _sms():
    import torch

    return torch.cuda.get_device_properties(0).multi_processor_count


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dk,dv", [(64, 64), (128, 128)])
@pytest.mark.parametrize("gap", [10, 14, 18])
@pytest.mark.parametrize("flat", [True, False])
def test_one_key_ahead_of_a_long_row(cuda_device, dtype, dk, dv, gap, flat):
    run(dtype, dk, dv, 32768, 1, _sms() * (16 if dv == 64 else 12), gap, flat)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,gap", [("f32", 18), ("f32", 20), ("f16", 18), ("f16", 16)])
def test_one_key_ahead_of_a_million(cuda_device, dtype, gap):
    run(dtype, 64, 64, 1 << 20, 1, _sms() * 16, gap, True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dk,dv", [("f32", 64, 64), ("f32", 128, 128)])
@pytest.mark.parametrize("gap", [12, 18])
def test_blocks_of_sixteen_rows(cuda_device, dtype, dk, dv, gap):
    """f32 prompts: sixteen rows a unit, a warp's run a whole unit."""
    run(dtype, dk, dv, 16384, 272, _sms() * 12 // 17, gap, True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dk,dv", [(64, 64), (128, 128)])
@pytest.mark.parametrize("gap,keys", [(10, 4096), (14, 16384), (18, 16384), (17.5, 1 << 18)])
def test_prompts(cuda_device, dtype, dk, dv, gap, keys):
    run(dtype, dk, dv, keys, 256, _sms(), gap, True, many_rows=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("factor", [1e-4, 1000.0])
def test_values_of_other_magnitudes(cuda_device, dtype, factor):
    run(dtype, 64, 64, 8192, 1, _sms() * 16, 14, False, factor=factor)
