"""GPU: the 8-bit KV cache's operators (append, read, attend) against plain
64-bit forms, at the sizes, masks and layouts where they can go wrong.

Tolerances.  append / read: the stored integers are defined exactly (the
quotient correctly rounded), so integers and scales must be equal.  attend:
the score's size is e = scale * sum |q k|.  f32 rows: a score is off by at most
2^-20 e (sums in f32 or exacter), which moves each weight by twice that,
relative; the weights' exponentials and sums add 2^-18; both scale the summed
|w v|.  16-bit rows: a query's elements are held to 2^-16 of its largest, which
moves a score by up to 2^-16 * scale * max|q| * sum |k|, and a weight by twice
that; the weights' rounding to f16 in the prompt kernel adds 2^-11 twice
(numerator and sum), the result its own half step (f16 2^-11, bf16 2^-8).
Weights are held in fixed point relative to the largest of their pair of pages
(32 keys): to 2^-16 of it for 16-bit rows, 2^-30 for f32 ones, whatever their
own size; for the 32 keys together 32 * that * (the pair's largest weight times
value scale) * 127, which `grain` sums over all pairs (of either parity).  The
prompt kernel's weights are f16 (f32 rows: and what that left over) with the
largest weight times the largest value scale at 2^7 or up to twice above: f16's
unit below 2^-14 is 2^-24, so a weight is off by up to 2^-25 / 2^6 of that,
2^-31 times `coarse` for all keys together.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

import kv8_util as ku
import s2k

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF_STEP = {"f32": 2.0**-24, "f16": 2.0**-11, "bf16": 2.0**-8}
GRAIN = {"f32": 2.0**-30, "f16": 2.0**-16, "bf16": 2.0**-16}
QUERY = {"f32": 0.0, "f16": 2.0**-16, "bf16": 2.0**-16}
EXTRA = {"f32": 2.0**-18, "f16": 2.0**-18 + 2 * 2.0**-11, "bf16": 2.0**-18 + 2 * 2.0**-11}


def dev(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Call:
    """A cache filled with random blocks and a ragged call over it."""

    def __init__(self, rows, past, H, Hkv, D, typ, seed=0, layers=2, spare=3, pad=0, ld_extra=0):
        rng = self.rng = np.random.default_rng(seed)
        self.rows, self.past, self.H, self.Hkv, self.D, self.typ = rows, past, H, Hkv, D, typ
        P = sum(ku.pages_for(rows, past)) + spare
        self.table = ku.make_table(rng, rows, past, P, max(max(ku.pages_for(rows, past)), 1) + ld_extra)
        self.kq = rng.integers(-127, 128, (P, layers, Hkv, 16, D), dtype=np.int8)
        self.vq = rng.integers(-127, 128, (P, layers, Hkv, D, 16), dtype=np.int8)
        self.ks = (rng.random((P, layers, Hkv), dtype=np.float32) * 0.02 + 0.003)
        self.vs = (rng.random((P, layers, Hkv), dtype=np.float32) * 0.02 + 0.003)
        self.start = [sum(rows[:b]) for b in range(len(rows) + 1)]
        self.n = self.start[-1] + pad
        self.layer = layers - 1
        used = set(int(p) for b, n in enumerate(ku.pages_for(rows, past)) for p in self.table[b, :n])
        free = [p for p in range(P) if p not in used]
        self.ks[free] = np.nan  # a page of no sequence reaches nothing
        self.vs[free] = np.nan
        self.kw = dict(row_start=i32(self.start), max_rows=max(rows) if rows else 0)
        self.upload()

    def upload(self):
        self.cache = s2k.KV8Cache(dev(self.kq), dev(self.vq), dev(self.ks), dev(self.vs))
        self.args = (i32(self.past), dev(self.table))

    def heads(self, n_heads, std=1.0):
        x = torch.from_numpy(self.rng.standard_normal((self.n, n_heads, self.D)) * std).to(DT[self.typ])
        return x.cuda()

    def check_attend(self, q, out, scale=None, window=0, sinks=0, skip=()):
        scale = self.D ** -0.5 if scale is None else scale
        qn, on = q.double().cpu().numpy(), out.double().cpu().numpy()
        for b, (t, p) in enumerate(zip(self.rows, self.past)):
            if b in skip or t == 0:
                continue
            k = ku.values(self.kq, self.ks, self.layer, self.table[b], p + t, False)
            v = ku.values(self.vq, self.vs, self.layer, self.table[b], p + t, True)
            sl = slice(self.start[b], self.start[b + 1])
            vtop = np.repeat(self.vs[self.table[b, : (p + t + 15) // 16], self.layer].astype(np.float64), 16, 0)[: p + t] * 127
            want, mag, size, reach, grain, coarse = ku.attend(k, v, qn[sl], p, scale, window, sinks, vtop)
            score = 2.0**-20 * size + QUERY[self.typ] * reach
            tol = (GRAIN[self.typ] * grain + 2.0**-31 * coarse)[..., None] + mag * (2 * score[..., None] + EXTRA[self.typ]) + np.abs(want) * HALF_STEP[self.typ] * 1.01 + 1e-30
            d = np.abs(on[sl] - want)
            assert np.all(d <= tol), f"sequence {b}: {np.nanmax(d / tol)} times the tolerance"


# --------------------------------------------------------------------------- append / read
@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("D,Hkv", [(128, 8), (64, 3)])
@pytest.mark.parametrize("rows,past", [([1], [0]), ([1], [15]), ([1], [512]), ([1, 0, 40, 17, 2], [3, 9, 0, 31, 16]),
                                       ([129, 16, 33], [7, 0, 1000])])
def test_append_is_exact(rows, past, D, Hkv, typ):
    c = Call(rows, past, Hkv, Hkv, D, typ, seed=sum(rows), pad=3)
    k, v = c.heads(Hkv, 1.4), c.heads(Hkv, 0.7)
    k[0] *= 4  # the page of an earlier token must take a larger scale
    c.cache.append(c.layer, k, v, *c.args, **c.kw)
    ku.append(c.kq, c.ks, c.layer, k.double().cpu().numpy(), c.start, c.past, c.table, False)
    ku.append(c.vq, c.vs, c.layer, v.double().cpu().numpy(), c.start, c.past, c.table, True)
    assert np.array_equal(c.cache.k_scale.cpu().numpy(), c.ks, equal_nan=True)
    assert np.array_equal(c.cache.v_scale.cpu().numpy(), c.vs, equal_nan=True)
    # every slot, those behind a sequence's last token too: they stay as they were
    assert np.array_equal(c.cache.k.cpu().numpy(), c.kq)
    assert np.array_equal(c.cache.v.cpu().numpy(), c.vq)
    kb, vb = torch.full_like(k, 7.0), torch.full_like(v, 7.0)
    c.cache.read(c.layer, c.n, *c.args, out=(kb, vb), **c.kw)
    for b, (t, p) in enumerate(zip(rows, past)):
        for got, q, s, tr in ((kb, c.kq, c.ks, False), (vb, c.vq, c.vs, True)):
            want = ku.values(q, s, c.layer, c.table[b], p + t, tr)[p:]
            want = torch.from_numpy(want.astype(np.float32)).to(DT[typ])
            assert torch.equal(got[c.start[b]:c.start[b + 1]].cpu(), want)
    assert torch.all(kb[c.start[-1]:] == 7.0) and torch.all(vb[c.start[-1]:] == 7.0)


def test_append_ties_extremes_and_not_a_number():
    """Quotients at halves, blocks of zeros, the smallest and largest numbers, NaN and infinity."""
    D, n = 64, 16
    x = np.zeros((6 * n, 1, D), np.float32)
    x[:n, 0] = (np.arange(n * D).reshape(n, D) % 255 - 127) * 0.5  # scale 0.5: every other value is a tie of scale 1
    x[0, 0, 0] = 127.0
    x[2 * n:3 * n, 0] = 1e-45 * (np.arange(n * D).reshape(n, D) % 300)  # subnormal: amax / 127 is subnormal
    x[3 * n:4 * n, 0] = 3.0e38 * np.sin(np.arange(n * D).reshape(n, D))
    x[4 * n + 3, 0, 5] = np.nan
    x[5 * n + 9, 0, 63] = -np.inf
    c = Call([6 * n], [0], 1, 1, D, "f32", layers=1)
    t = dev(x)
    c.cache.append(0, t, t, *c.args, **c.kw)
    ku.append(c.kq, c.ks, 0, x, c.start, c.past, c.table, False)
    assert np.array_equal(c.cache.k_scale.cpu().numpy(), c.ks, equal_nan=True)
    assert np.array_equal(c.cache.k.cpu().numpy(), c.kq)
    kb, _ = c.cache.read(0, 6 * n, *c.args, **c.kw)
    kb = kb.cpu().numpy()
    assert np.isnan(kb[4 * n:]).all() and np.isfinite(kb[:4 * n]).all()
    # the block stays NaN until its page is entered at slot 0 again
    one = torch.ones((1, 1, D), device="cuda")
    last = i32([c.past[0] + 6 * n - 1])
    c.cache.append(0, one, one, last, c.args[1])
    assert torch.isnan(c.cache.read(0, 1, last, c.args[1])[0]).all()
    c.cache.append(0, one, one, i32([5 * n]), c.args[1])
    assert torch.equal(c.cache.read(0, 1, i32([5 * n]), c.args[1])[0], one)


def test_append_one_by_one_and_strided_rows():
    """Single tokens from a fused QKV row (row stride beyond the heads, an odd offset) into a filling page."""
    D, Hkv, T = 128, 4, 37
    c = Call([T], [0], Hkv, Hkv, D, "f32")
    for off in (0, 1):  # 1: rows that no 16-byte access fits
        fused = torch.randn(T, 3 * Hkv * D + 5, device="cuda")
        k = fused[:, off:off + Hkv * D].unflatten(1, (Hkv, D))
        v = fused[:, off + Hkv * D:off + 2 * Hkv * D].unflatten(1, (Hkv, D))
        for i in range(T):
            c.cache.append(c.layer, k[i:i + 1], v[i:i + 1], i32([i]), c.args[1])
            ku.append(c.kq, c.ks, c.layer, k[i:i + 1].cpu().numpy(), [0, 1], [i], c.table, False)
            ku.append(c.vq, c.vs, c.layer, v[i:i + 1].cpu().numpy(), [0, 1], [i], c.table, True)
        assert np.array_equal(c.cache.k.cpu().numpy(), c.kq) and np.array_equal(c.cache.v.cpu().numpy(), c.vq)
        assert np.array_equal(c.cache.k_scale.cpu().numpy(), c.ks, equal_nan=True)


# --------------------------------------------------------------------------- attend
STEPS = [  # rows, past, H, Hkv, D
    ([1], [0], 4, 1, 128), ([1], [512], 32, 8, 128), ([1, 1, 1], [0, 15, 1000], 8, 2, 64),
    ([3, 0, 1, 2], [40, 5, 0, 333], 14, 2, 128), ([1, 1], [2000, 17], 16, 1, 128), ([2, 1], [70, 900], 5, 5, 64),
    ([9, 4], [31, 0], 8, 2, 128),
]
PROMPTS = [([130], [0], 4, 2, 128), ([64, 1, 0, 257], [0, 40, 3, 100], 8, 2, 64), ([200], [77], 7, 1, 128),
           ([33, 140], [500, 0], 8, 8, 128), ([300, 20], [5, 600], 8, 1, 64)]


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (50, 0), (37, 5), (16, 40), (100000, 3)])
@pytest.mark.parametrize("rows,past,H,Hkv,D", STEPS + PROMPTS)
def test_attend(rows, past, H, Hkv, D, window, sinks, typ):
    c = Call(rows, past, H, Hkv, D, typ, seed=len(rows) + H, pad=2, ld_extra=3)
    q = c.heads(H, 1.5)
    out = torch.full_like(q, 9.0)
    got = c.cache.attend(c.layer, q, *c.args, window=window, sinks=sinks, out=out, **c.kw)
    assert got is out
    c.check_attend(q, out, window=window, sinks=sinks)
    assert torch.all(out[c.start[-1]:] == 9.0)


@pytest.mark.parametrize("rows", [[1], [70]])
@pytest.mark.parametrize("typ", ["f32", "bf16"])
def test_attend_strides_scale_and_in_place(rows, typ):
    H, Hkv, D = 8, 2, 128
    c = Call(rows, [45], H, Hkv, D, typ)
    fused = torch.randn(rows[0], (H + 2 * Hkv) * D + 3, device="cuda").to(DT[typ])
    q = fused[:, 1:1 + H * D].unflatten(1, (H, D))  # element-aligned only
    want = c.cache.attend(c.layer, q, *c.args, scale=0.05, **c.kw)
    c.check_attend(q, want, scale=0.05)
    by_head = torch.empty(H, rows[0], D, device="cuda", dtype=DT[typ]).transpose(0, 1)  # [heads][rows][dim] in memory
    assert torch.equal(c.cache.attend(c.layer, q, *c.args, scale=0.05, out=by_head, **c.kw), want)
    copy = q.clone()
    keep = fused.clone()
    assert torch.equal(c.cache.attend(c.layer, q, *c.args, scale=0.05, out=q, **c.kw), want)
    fused[:, 1:1 + H * D] = copy.flatten(1)
    assert torch.equal(fused, keep)  # nothing beside the rows was written


@pytest.mark.parametrize("rows,past", [([1], [700]), ([100], [300])])
@pytest.mark.parametrize("typ", ["f32", "f16"])
def test_attend_hidden_blocks_may_hold_anything(rows, past, typ):
    """NaN scales in pages outside every row's view, and behind the last token, reach nothing; inside it they do."""
    c = Call(rows, past, 8, 2, 128, typ)
    hidden = [int(p) for p in c.table[0, 2:(past[0] - 64) // 16]]
    c.ks[hidden] = np.nan
    c.vs[hidden] = np.nan
    c.upload()
    q = c.heads(8)
    out = c.cache.attend(c.layer, q, *c.args, window=64, sinks=20, **c.kw)
    c.check_attend(q, out, window=64, sinks=20)
    c.vs[int(c.table[0, 1])] = np.nan  # slots 16..19 are sinks
    c.upload()
    assert torch.isnan(c.cache.attend(c.layer, q, *c.args, window=64, sinks=20, **c.kw)).all()


@pytest.mark.parametrize("rows", [[2], [90]])
@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
def test_attend_negative_scale_and_odd_queries(rows, typ):
    """A scale below 0; rows whose scores are all -inf, +inf or NaN are NaN, their neighbours sound."""
    c = Call(rows, [150], 8, 2, 64, typ)
    q = c.heads(8)
    c.check_attend(q, c.cache.attend(c.layer, q, *c.args, scale=-0.2, **c.kw), scale=-0.2)
    good = c.cache.attend(c.layer, q, *c.args, **c.kw)
    c.cache.k[:, c.layer, :, :, 5] = 3  # one dim of one sign
    same = c.cache.attend(c.layer, q, *c.args, **c.kw)
    odd = q.clone()
    odd[0, 0, 5], odd[0, 1, 5], odd[1, 2, 5] = float("inf"), -float("inf"), float("nan")
    out = c.cache.attend(c.layer, odd, *c.args, **c.kw)
    for r, h in ((0, 0), (0, 1), (1, 2)):
        assert torch.isnan(out[r, h]).all()
        out[r, h] = same[r, h]
    assert torch.equal(out, same) and not torch.equal(good, same)


@pytest.mark.parametrize("rows", [1, 90])
def test_attend_far_scores_scales_and_not_a_number(rows):
    """Queries and blocks of very different size, a row of zeros, a NaN and an infinite row beside sound ones."""
    c = Call([rows, rows], [200, 33], 8, 2, 128, "f32")
    c.ks *= (10.0 ** c.rng.integers(-3, 2, c.ks.shape)).astype(np.float32)
    c.vs *= (10.0 ** c.rng.integers(-6, 4, c.vs.shape)).astype(np.float32)
    c.upload()
    q = c.heads(8)
    q[0, 1] *= 1e-6
    q[0, 2] *= 30.0
    q[0, 3] = 0.0
    good = c.cache.attend(c.layer, q, *c.args, **c.kw)
    c.check_attend(q, good)
    q2 = q.clone()
    q2[0, 4, 7] = float("nan")
    q2[rows, 5, 0] = float("inf")
    bad = c.cache.attend(c.layer, q2, *c.args, **c.kw)
    assert torch.isnan(bad[0, 4]).all() and torch.isnan(bad[rows, 5]).all()
    good[0, 4] = bad[0, 4] = 0
    good[rows, 5] = bad[rows, 5] = 0
    assert torch.equal(good, bad)


@pytest.mark.parametrize("rows", [1, 80])
def test_bad_entries_are_skipped_and_told(rows):
    """Sequences and pages that do not fit the call leave its other rows right and set the error word."""
    c = Call([rows] * 4, [100, 50, 20, 60], 8, 2, 128, "f32")
    q = c.heads(8)
    err = i32([0])
    out = torch.full_like(q, 3.0)
    past = i32([100, -1, 10 ** 6, 60])
    c.cache.attend(c.layer, q, past, c.args[1], err=err, out=out, **c.kw)
    assert err.item() == 8
    c.check_attend(q, out, skip=(1, 2))
    assert torch.all(out[rows:3 * rows] == 3.0)
    # a start that runs backwards, and more rows than max_rows
    for start in ([0, rows, 0, 3 * rows, 4 * rows], [0, rows, rows, 3 * rows + 1, 4 * rows]):
        err.zero_()
        c.cache.attend(c.layer, q, c.args[0], c.args[1], row_start=i32(start), max_rows=rows, err=err)
        assert err.item() == 8
    # every page of sequence 0 out of range: its rows see nothing
    err.zero_()
    t = c.args[1].clone()
    t[0] = -5
    out = c.cache.attend(c.layer, q, c.args[0], t, err=err, **c.kw)
    assert err.item() == 8 and torch.all(out[:rows] == 0)
    c.check_attend(q, out, skip=(0,))
    before = (c.cache.k.clone(), c.cache.v.clone())
    c.cache.append(c.layer, q[:, :2], q[:, :2], past, t, err=err, **c.kw)
    kq, vq = c.kq.copy(), c.vq.copy()
    x = q[:, :2].double().cpu().numpy()
    one = [0, 0, 0, 0, rows]
    ku.append(kq, c.ks, c.layer, np.concatenate([x[3 * rows:]]), one, [0, 0, 0, 60], c.table, False)
    assert np.array_equal(c.cache.k.cpu().numpy(), kq)
    del before, vq


def test_no_rows_and_no_sequences():
    c = Call([0, 0], [5, 0], 8, 2, 128, "f32")
    q = c.heads(8)
    assert c.cache.attend(c.layer, q, *c.args, row_start=c.kw["row_start"], max_rows=0).shape == (0, 8, 128)
    none = i32([]), torch.empty((0, 4), dtype=torch.int32, device="cuda")
    c.cache.append(c.layer, q[:, :2], q[:, :2], *none, row_start=i32([0]), max_rows=0)


def test_far_pages_pass_32_bit_offsets():
    """Blocks beyond 4 GiB of the pool: 2^21 + 8 pages of 2 KB."""
    P, D = (1 << 21) + 8, 128
    cache = s2k.KV8Cache.empty(P, 1, 1, D)
    table = i32([[P - 1, P - 3, 1 << 20]])
    x = torch.randn(40, 1, D, device="cuda")
    y = torch.randn(40, 1, D, device="cuda")
    cache.append(0, x, y, i32([0]), table)
    kb, vb = cache.read(0, 40, i32([0]), table)
    assert (kb - x).abs().max() <= x.abs().max() / 127 * 0.51 and (vb - y).abs().max() <= y.abs().max() / 127 * 0.51
    q = torch.randn(40, 4, D, device="cuda")
    out = cache.attend(0, q, i32([0]), table)
    one = cache.attend(0, q[39:], i32([39]), table)
    want, mag, size, _, _, _ = ku.attend(kb.double().cpu().numpy(), vb.double().cpu().numpy(), q.double().cpu().numpy(), 0, D ** -0.5)
    tol = mag * (2 * 2.0**-20 * size[..., None] + EXTRA["f32"]) + np.abs(want) * 2.0**-24 * 2
    assert np.all(np.abs(out.double().cpu().numpy() - want) <= tol)
    assert np.all(np.abs(one[0].double().cpu().numpy() - want[39]) <= tol[39])
    del cache
    torch.cuda.empty_cache()


def test_captured_replayed_and_on_another_stream():
    """A decode step captured once, replayed over changing lengths, rows and streams."""
    c = Call([1, 1, 1], [14, 700, 31], 32, 8, 128, "bf16", ld_extra=2)
    c.table[:, -2:] = np.arange(6).reshape(3, 2) % 3 + (c.kq.shape[0] - 3)
    for b in range(3):  # two more pages each, of their own
        n = ku.pages_for([1], [c.past[b]])[0]
        c.table[b, n:n + 1] = c.kq.shape[0] - 3 + b
    c.ks[-3:] = 0.01
    c.vs[-3:] = 0.01
    c.upload()
    past, table = c.args
    k, v, q = c.heads(8), c.heads(8), c.heads(32)
    ref = s2k.KV8Cache(*[t.clone() for t in (c.cache.k, c.cache.v, c.cache.k_scale, c.cache.v_scale)])
    out = torch.empty_like(q)

    def step(cache, out):
        cache.append(c.layer, k, v, past, table)
        cache.attend(c.layer, q, past, table, out=out)

    g = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    with torch.cuda.graph(g, stream=side):
        step(c.cache, out)
    for i in range(4):
        for t in (k, v, q):
            t.copy_(torch.randn_like(t))
        torch.cuda.synchronize()
        if i % 2:
            with torch.cuda.stream(side):
                g.replay()
        else:
            g.replay()
        torch.cuda.synchronize()
        want = torch.empty_like(q)
        step(ref, want)
        assert torch.equal(out, want) and torch.equal(c.cache.k, ref.k) and torch.equal(c.cache.v, ref.v)
        past += 1


def test_two_streams_at_once():
    cs = [Call([1], [900], 32, 8, 128, "f32", seed=s) for s in (1, 2)]
    qs = [c.heads(32) for c in cs]
    want = [c.cache.attend(c.layer, q, *c.args) for c, q in zip(cs, qs)]
    streams = [torch.cuda.Stream() for _ in cs]
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        for c, q, s in zip(cs, qs, streams):
            got.append(c.cache.attend(c.layer, q, *c.args, stream=s))
    torch.cuda.synchronize()
    for i, o in enumerate(got):
        assert torch.equal(o, want[i % 2])


def test_binding_refusals():
    c = Call([2], [10], 8, 2, 128, "f32")
    q = c.heads(8)
    past, table = c.args
    ok = dict(row_start=c.kw["row_start"], max_rows=2)
    for bad in (lambda: c.cache.attend(2, q, past, table, **ok), lambda: c.cache.attend(0, q[:, :3], past, table, **ok),
                lambda: c.cache.attend(0, q.double(), past, table, **ok), lambda: c.cache.attend(0, q.cpu(), past, table, **ok),
                lambda: c.cache.attend(0, q, past.long(), table, **ok), lambda: c.cache.attend(0, q, past, table[0], **ok),
                lambda: c.cache.attend(0, q.transpose(0, 2), past, table, **ok),
                lambda: c.cache.attend(0, q, past, table, row_start=c.kw["row_start"]),
                lambda: c.cache.attend(0, q, past, table, window=-1, **ok),
                lambda: c.cache.attend(0, q, past, table, out=q[:1], **ok),
                lambda: c.cache.attend(0, q, past, table, out=q.half(), **ok),
                lambda: c.cache.append(0, q[:, :2], q[:, :3], past, table, **ok),
                lambda: c.cache.append(0, q, q, past, table, **ok),
                lambda: s2k.KV8Cache(c.cache.k, c.cache.k, c.cache.k_scale, c.cache.v_scale),
                lambda: s2k.KV8Cache(c.cache.k.cpu(), c.cache.v, c.cache.k_scale, c.cache.v_scale)):
        with pytest.raises(s2k.S2KError):
            bad()


def test_results_belong_to_the_stream_that_writes_them():
    """Memory that the current stream gave back, and may still be using, is not handed to another stream's call."""
    c = Call([1], [40], 8, 2, 128, "f32")
    q = c.heads(8)
    side = torch.cuda.Stream()
    x = torch.randn(1, 1000, device="cuda")

    def results(stream):
        k, v = c.cache.read(c.layer, 1, *c.args, stream=stream)
        ids = s2k.logprobs(x, torch.zeros(1, dtype=torch.int32, device="cuda"), 4, stream=stream)
        return [c.cache.attend(c.layer, q, *c.args, stream=stream), k, v, *ids]

    torch.cuda.synchronize()
    kept = results(None)
    want = [t.clone() for t in kept]
    torch.cuda.synchronize()
    ours = {t.untyped_storage().data_ptr() for t in kept}
    del kept
    for stream in (side, side.cuda_stream):
        got = results(stream)
        torch.cuda.synchronize()
        assert not ours & {t.untyped_storage().data_ptr() for t in got}
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        del got


# Which kernel a call takes depends on how much there is to do per SM: the calls above are small, these are the same
# cases at sizes that the prompt kernel gets (many sequences, most of them without rows, or more rows).
@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (50, 0), (37, 5), (16, 40), (100000, 3)])
@pytest.mark.parametrize("rows,past,H,Hkv,D", PROMPTS)
def test_attend_of_a_crowd(rows, past, H, Hkv, D, window, sinks, typ):
    test_attend(rows + [0] * 200, past + [0] * 200, H, Hkv, D, window, sinks, typ)


@pytest.mark.parametrize("typ", ["f32", "bf16"])
def test_attend_strides_scale_and_in_place_of_many_rows(typ):
    test_attend_strides_scale_and_in_place([900], typ)


@pytest.mark.parametrize("typ", ["f32", "f16"])
def test_attend_hidden_blocks_of_many_rows(typ):
    test_attend_hidden_blocks_may_hold_anything([1500], [300], typ)


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
def test_attend_negative_scale_and_odd_queries_of_many_rows(typ):
    test_attend_negative_scale_and_odd_queries([1000], typ)


def test_attend_far_scores_of_many_rows():
    test_attend_far_scores_scales_and_not_a_number(400)


def test_bad_entries_of_many_rows():
    test_bad_entries_are_skipped_and_told(400)


@pytest.mark.parametrize("bits", [1, 2, 4, 7])
@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
def test_append_of_few_mantissa_bits(typ, bits):
    """Values and maxima of few bits, whose quotients are halves or next to one nearly everywhere, from the smallest
    magnitudes of the type to large ones; page by page in one call, then in parts."""
    rows, D, Hkv = [16 * 24], 128, 2
    rng = np.random.default_rng(bits)
    lo, hi = {"f32": (-149, 100), "f16": (-24, 14), "bf16": (-133, 100)}[typ]
    c = Call(rows, [0], 4, Hkv, D, typ)
    m = rng.integers(-(2 ** bits), 2 ** bits + 1, (rows[0], Hkv, D)).astype(np.float64)
    e = np.repeat(rng.integers(lo, hi - bits, (24, Hkv, 1)), 16, 0)
    k = torch.from_numpy(np.ldexp(m, e)).to(DT[typ]).cuda()
    v = k.flip(2).contiguous()
    assert torch.isfinite(k).all()
    for parts in ([rows[0]], [5, 16, 1, 6, rows[0] - 28]):
        at = 0
        for n in parts:
            past = i32([at])
            x, y = k[at:at + n].contiguous(), v[at:at + n].contiguous()
            c.cache.append(c.layer, x, y, past, c.args[1])
            ku.append(c.kq, c.ks, c.layer, x.double().cpu().numpy(), [0, n], [at], c.table, False)
            ku.append(c.vq, c.vs, c.layer, y.double().cpu().numpy(), [0, n], [at], c.table, True)
            at += n
        assert np.array_equal(c.cache.k_scale.cpu().numpy(), c.ks, equal_nan=True)
        assert np.array_equal(c.cache.v_scale.cpu().numpy(), c.vs, equal_nan=True)
        assert np.array_equal(c.cache.k.cpu().numpy(), c.kq) and np.array_equal(c.cache.v.cpu().numpy(), c.vq)
