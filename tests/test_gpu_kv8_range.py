"""GPU: attention over the 8-bit KV cache where queries and value scales are far from 1 or from one another, in both
of its kernels (which one a call took is asserted).

Tolerances, per row with weights w_j, largest weight w, keys k, values v, T the largest value that a key's block can
hold (127 * its scale), n keys in view:
  scores   e = 2^-20 * scale * sum |q k| (sums in f32 or exacter) + 2^-30 * scale * max|q| * sum |k| (a query's
           elements are held to 2^-30 of its largest or exacter).  Each moves a weight by twice that, relative.
  weights  their exponentials and sums 2^-18.  Few rows: fixed point relative to the largest weight * scale of a pair
           of pages, to 2^-16 of it for 16-bit rows, 2^-30 for f32 ones: 32 keys a pair, 2 * 32 * (a page's largest
           w_j T_j) summed over pages bounds it for either pairing.  Many rows: f16 (2^-11, twice: numerator and sum),
           or for f32 rows f16 and what that left over; the largest w_j T_j of a row is at 2^6 or above, so f16's
           subnormal step (half of 2^-24) is worth 2^-31 of it, for each of n keys.
  zeros    weights below 2^-126 of the largest are zero.
  result   its type's half step, and the type's smallest number.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

import kv8_util as ku
import s2k
from test_gpu_kv8 import DT, GRAIN, HALF_STEP, Call

pytestmark = pytest.mark.gpu

FEW, MANY = 1, 2
LEAST = {"f32": 2.0**-149, "f16": 2.0**-24, "bf16": 2.0**-133}
# a few rows; and enough for the other kernel, the last 104 of a 256-row tile's (row, head) pairs among them
ROWS = {FEW: 2, MANY: 730}
PAST, H, HKV = 70, 8, 2


def make(kernel, typ, D, seed):
    return Call([ROWS[kernel]], [PAST], H, HKV, D, typ, seed=seed)


def check(c, kernel, q, **kw):
    """attend, and its result for some rows against 64 bits."""
    c.upload()
    out = c.cache.attend(c.layer, q, *c.args, **kw)
    assert s2k.lib().s2k_debug_kv8_attend_kernel() == kernel
    T, scale = ROWS[kernel], c.D ** -0.5
    k = ku.values(c.kq, c.ks, c.layer, c.table[0], PAST + T, False)
    v = ku.values(c.vq, c.vs, c.layer, c.table[0], PAST + T, True)
    top = np.repeat(c.vs[c.table[0, : (PAST + T + 15) // 16], c.layer].astype(np.float64), 16, 0) * 127
    qn, on = q.double().cpu().numpy(), out.double().cpu().numpy()
    assert np.isfinite(on).all()
    worst = 0.0
    for i in sorted({0, T - 1} | set(range(5, T, 61))):
        n = PAST + i + 1
        for h in range(H):
            kk, vv, t, x = k[:n, h // (H // HKV)], v[:n, h // (H // HKV)], top[:, h // (H // HKV)], qn[i, h]
            s = kk @ x * scale
            e = scale * (2.0**-20 * (np.abs(kk) @ np.abs(x)).max() + 2.0**-30 * np.abs(x).max() * np.abs(kk).sum(1).max())
            w = np.exp(s - s.max())
            w /= w.sum()
            want, mag = w @ vv, w @ np.abs(vv)
            wt = np.zeros(len(t))
            wt[:n] = w * t[:n]
            if kernel == FEW:
                tol = GRAIN[c.typ] * 64 * wt.reshape(-1, 16).max(1).sum() + mag * (2 * e + 2.0**-18)
            else:
                tol = 2.0**-31 * n * wt.max() + mag * (2 * e + 2.0**-18 + (0 if c.typ == "f32" else 2 * 2.0**-11))
            tol = tol + n * 2.0**-126 * w.max() * t[:n].max() + np.abs(want) * HALF_STEP[c.typ] * 1.01 + LEAST[c.typ]
            worst = max(worst, (np.abs(on[i, h] - want) / tol).max())
    assert worst <= 1, f"{worst} times the tolerance"
    return out


KERNELS = pytest.mark.parametrize("kernel", [FEW, MANY])


@KERNELS
@pytest.mark.parametrize("typ", ["f32", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
def test_queries_up_to_the_largest_number(D, typ, kernel):
    """Elements around 5e37 and up to 3.3e38, keys so small that the scores are of a usual size."""
    c = make(kernel, typ, D, 1)
    c.ks = (c.ks / 0.01 * 1e-39).astype(np.float32)
    q = c.rng.standard_normal((c.n, H, D)) * 5e37
    q[:, ::3, 7] = 3.3e38 * np.sign(q[:, ::3, 7])
    q[:, 1] *= 1e-3  # a head of smaller ones beside them
    check(c, kernel, torch.from_numpy(np.clip(q, -3.3e38, 3.3e38)).to(DT[typ]).cuda())


@KERNELS
@pytest.mark.parametrize("typ", ["f16", "bf16"])
@pytest.mark.parametrize("outlier", [300.0, 3000.0])
def test_one_large_query_element(outlier, typ, kernel):
    """A dimension that no key uses must not cost the others their bits."""
    c = make(kernel, typ, 128, 2)
    c.kq[..., 5] = 0
    q = c.heads(H, 1.5)
    q[:, :, 5] = outlier
    check(c, kernel, q)


@KERNELS
@pytest.mark.parametrize("typ", ["f32", "bf16"])
@pytest.mark.parametrize("size", [1e-30, 1e-18])
def test_small_queries(size, typ, kernel):
    """Under keys as much larger."""
    c = make(kernel, typ, 128, 5)
    c.ks = (c.ks / size).astype(np.float32)
    q = c.rng.standard_normal((c.n, H, 128)) * 1.5 * size
    check(c, kernel, torch.from_numpy(q).to(DT[typ]).cuda())


def spread(c, kind):
    r = c.rng.random(c.vs.shape)
    if kind == "tiny":
        return 1e-30 * (0.5 + r)
    if kind == "subnormal":
        return 10.0 ** (-41 + 3 * r)
    if kind == "huge":
        return 2.6e36 * (0.3 + 0.7 * r)
    if kind == "all":
        return 10.0 ** (-38 + 74 * r)
    return np.where(r < 0.5, 0.0, 0.01 * r)  # zeros


@KERNELS
@pytest.mark.parametrize("typ", ["f32", "bf16"])
@pytest.mark.parametrize("kind", ["tiny", "subnormal", "huge", "all", "zeros"])
@pytest.mark.parametrize("D", [64, 128])
def test_value_scales(D, kind, typ, kernel):
    c = make(kernel, typ, D, 3)
    c.vs = spread(c, kind).astype(np.float32)
    if kind == "zeros":  # the block of the largest scores among them
        q = c.heads(H, 0.3)
        c.kq[c.table[0, 2], c.layer] = 90
        c.vs[c.table[0, 2], c.layer] = 0.0
        q += 0.2
    else:
        q = c.heads(H, 1.5)
    check(c, kernel, q)


@KERNELS
@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("ratio", [1e4, 1e6, 1e8])
def test_large_value_scales_of_small_weights(ratio, typ, kernel):
    """Every third page has values `ratio` times the others' and scores ~20 below them: it must not cost the others'
    weights their bits."""
    c = make(kernel, typ, 128, 4)
    sign = np.where(c.rng.random(128) < 0.5, -1, 1)
    for pg in c.table[0, : (PAST + ROWS[kernel] + 15) // 16][1::3]:
        c.kq[pg, c.layer] = (-60 * sign).astype(np.int8)
        c.ks[pg, c.layer] = 0.01
        c.vs[pg, c.layer] *= ratio if typ != "f16" else min(ratio, 1e6)
    q = torch.from_numpy(c.rng.standard_normal((c.n, H, 128)) * 0.3 + 3.0 * sign).to(DT[typ]).cuda()
    check(c, kernel, q)


@KERNELS
@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("size", [1e4, 1e8])
def test_sure_rows_beside_large_value_scales(size, typ, kernel):
    """One key whose score is ahead by `size` and more: the result is its value, whatever the other pages hold."""
    c = make(kernel, typ, 128, 6)
    n = PAST + ROWS[kernel]
    key = 21  # in the third page of 16
    c.kq[:, c.layer] = 0
    c.ks[:, c.layer] = 1.0
    for pg in c.table[0, : (n + 15) // 16]:
        c.kq[pg, c.layer, :, :, 0] = c.rng.integers(-100, 60, (HKV, 16))
        c.vs[pg, c.layer] *= 1e6
    at = c.table[0, key // 16]
    c.kq[at, c.layer, :, key % 16, 0] = 127
    c.vs[at, c.layer] /= 1e6
    q = torch.zeros(c.n, H, 128, dtype=DT[typ], device="cuda")
    q[:, :, 0] = size if typ != "f16" else min(size, 3e4)
    c.upload()
    out = c.cache.attend(c.layer, q, *c.args).double().cpu().numpy()
    assert s2k.lib().s2k_debug_kv8_attend_kernel() == kernel
    # the other weights are below e^-5000; the value is off by the weight's rounding in numerator and result
    want = ku.values(c.vq, c.vs, c.layer, c.table[0], n, True)[key].repeat(H // HKV, 0)
    step = {"f32": 2.0**-20, "f16": 2.0**-11, "bf16": 2.0**-8}[typ] + (0 if typ == "f32" else 2 * 2.0**-11)
    top = c.vs[at, c.layer].max() * 127
    # few rows: fixed point relative to the largest weight * scale, here the key's own
    assert np.all(np.abs(out - want) <= step * np.abs(want) + GRAIN[typ] * top + LEAST[typ])



@KERNELS
@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
def test_rows_do_not_change_with_their_neighbours(typ, kernel):
    """A row of very large finite scores, and an infinite one, beside others: their bits stay."""
    c = make(kernel, typ, 128, 7)
    q = c.heads(H, 1.5)
    want = c.cache.attend(c.layer, q, *c.args)
    odd = q.clone()
    odd[0, 0] *= 3e4
    odd[0, 3] = float("inf")
    odd[1, 2] *= -3e4
    got = c.cache.attend(c.layer, odd, *c.args)
    assert s2k.lib().s2k_debug_kv8_attend_kernel() == kernel
    for r, h in ((0, 0), (0, 3), (1, 2)):  # f16 has no number for some of them
        assert (torch.isfinite if torch.isfinite(odd[r, h]).all() else torch.isnan)(got[r, h]).all()
        got[r, h] = want[r, h]
    assert torch.equal(got, want)


@KERNELS
@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
def test_hidden_blocks_of_any_scale(typ, kernel):
    """A window before which blocks hold infinities, NaN and the largest scales; behind the rows as well."""
    T = 2 if kernel == FEW else 2400
    c = Call([T], [PAST], H, HKV, 64, typ, seed=8)
    q = c.heads(H, 1.5)
    want = c.cache.attend(c.layer, q, *c.args, window=20, sinks=3)
    keep = [int(p) for p in c.table[0, [0]]] + [int(p) for p in c.table[0, (PAST - 20) // 16:(PAST + T + 15) // 16]]
    gone = np.setdiff1d(np.arange(c.kq.shape[0]), keep)
    for scale in (np.inf, np.nan, 2e36):
        c.vs[gone] = c.ks[gone] = scale
        c.upload()
        assert torch.equal(c.cache.attend(c.layer, q, *c.args, window=20, sinks=3), want)
        assert s2k.lib().s2k_debug_kv8_attend_kernel() == kernel
