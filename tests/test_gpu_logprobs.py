"""GPU: s2k_logprobs against a plain 64-bit form.

Tolerances: x - M is rounded once (2^-24 relative to it, and it is at most
`span`), so a log probability is off by span * 2^-24 from that, its own
rounding and as much from log S, whose terms' errors are relative to S:
together 2^-21 * (1 + span).  The entropy is a mean of such terms.  Rows that
are nearly sure are checked relative to their small entropy."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import s2k

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def plain(x, targets, k):
    x = x.double().cpu().numpy()
    m = x.max(1, keepdims=True)
    m0 = np.where(np.isinf(m), 0, m)
    with np.errstate(divide="ignore", invalid="ignore"):
        e = np.exp(x - m0)
        top = x == m
        cnt = np.where(np.isinf(m[:, 0]), 0, top.sum(1))
        rest = np.where(top & ~np.isinf(m), 0, e).sum(1)
        ls = np.log(cnt) + np.log1p(rest / cnt)
        z = x - m0 - ls[:, None]
        none = np.isinf(m[:, 0])
        z[none] = -np.inf
        ent = np.where(none, 0, -np.where(e > 0, np.exp(z) * z, 0).sum(1))
    ids = np.argsort(-x, axis=1, kind="stable")[:, :k]
    lp = z[np.arange(len(x)), targets]
    return lp, ent, ids, np.take_along_axis(z, ids, 1), np.where(np.isinf(x), 0, np.abs(x - m0)).max(1)


def check(x, targets, k):
    t = torch.tensor(targets, dtype=torch.int32, device="cuda")
    lp, ent, ids, top = s2k.logprobs(x, t, n_top=k)
    wl, we, wi, wt, span = plain(x, targets, k)
    tol = 2.0**-21 * (1 + span)
    for got, want in ((lp, wl), (ent, we)):
        got = got.double().cpu().numpy()
        with np.errstate(invalid="ignore"):
            assert np.all((got == want) | (np.abs(got - want) <= tol)), np.abs(got - want).max()
    if k:
        assert np.array_equal(ids.cpu().numpy(), wi)
        got = top.double().cpu().numpy()
        with np.errstate(invalid="ignore"):
            assert np.all((got == wt) | (np.abs(got - wt) <= tol[:, None]))
    else:
        assert ids is None and top is None


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,n", [(1, 1), (3, 2), (2, 31), (5, 33), (7, 1000), (1, 4096), (2, 19457), (1, 155648),
                                    (65, 5001), (1, 400003)])
def test_against_plain(rows, n, typ):
    g = torch.Generator().manual_seed(rows * n)
    x = (torch.randn(rows, n, generator=g) * 3).to(DT[typ]).cuda()
    check(x, [(r * 7919) % n for r in range(rows)], min(n, 20))


@pytest.mark.parametrize("k", [0, 1, 7, 32])
def test_top_counts_and_strided_rows(k):
    big = torch.randn(6, 3001, device="cuda") * 2
    for off in (0, 1, 3):  # rows on every alignment
        check(big[:, off:off + 2900], [0, 1, 2, 3, 2899, 5], k)
    check(big[1::2, :2999], [5, 6, 7], k)


@pytest.mark.parametrize("n", [40, 4096, 155648])
def test_ties_masks_and_empty_rows(n):
    x = torch.zeros(8, n)
    x[1] = torch.arange(n) // 3 * 1.0  # ties in threes, ascending
    x[2] = -torch.arange(n) * 1.0
    x[3] = -np.inf
    x[3, n - 5:] = torch.tensor([1.0, 2.0, 2.0, -1.0, 0.5])  # all but five tokens masked
    x[4] = -np.inf  # every token masked
    x[5] = -1e30
    x[5, n // 2] = 1e30
    x[6, ::2] = -0.0  # equal to +0
    x[7] = torch.where(torch.arange(n) % 512 == 17, 5.0, -3.0)
    check(x.cuda(), [0, n - 1, 3, n - 4, 2, n // 2, 1, 17], 32)


def test_nearly_sure_rows_keep_their_small_entropy():
    n = 20000
    x = torch.full((4, n), 0.0)
    for r, top in enumerate((18.0, 25.0, 32.0, 60.0)):
        x[r, 777] = top
    x = x.cuda()
    lp, ent, _, _ = s2k.logprobs(x, torch.full((4,), 777, dtype=torch.int32, device="cuda"))
    wl, we, _, _, _ = plain(x, [777] * 4, 1)
    assert np.all(np.abs(lp.double().cpu().numpy() - wl) <= 2e-5 * np.abs(wl))
    assert np.all(np.abs(ent.double().cpu().numpy() - we) <= 2e-5 * np.abs(we))


def test_not_a_number_infinity_and_targets_outside():
    x = torch.randn(5, 3000, device="cuda")
    x[1, 2000] = float("nan")
    x[2, 100] = float("inf")
    x[4] = float("nan")
    t = torch.tensor([-1, 3, 3, 3000, 0], dtype=torch.int32, device="cuda")
    lp, ent, ids, top = s2k.logprobs(x, t, n_top=3)
    assert torch.isnan(lp).all()
    assert torch.equal(torch.isnan(ent).cpu(), torch.tensor([False, True, True, False, True]))
    want = x[1].nan_to_num(-1e9).topk(3).indices
    assert torch.equal(ids[1].long(), want) and torch.isnan(top[1]).all()
    assert ids[2, 0] == 100 and ids[4].tolist() == [0, 1, 2]
    lp, ent, _, _ = s2k.logprobs(x[:1])
    assert lp is None and torch.isfinite(ent).all()


def test_no_rows_captured_and_streams():
    lp, ent, ids, top = s2k.logprobs(torch.empty(0, 10, device="cuda"), torch.empty(0, dtype=torch.int32, device="cuda"), n_top=2)
    assert lp.shape == (0,) and ids.shape == (0, 2)
    x = torch.randn(3, 155648, device="cuda")
    t = torch.tensor([1, 2, 3], dtype=torch.int32, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = s2k.logprobs(x, t, n_top=5)
    for _ in range(3):
        x.copy_(torch.randn_like(x))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        want = s2k.logprobs(x, t, n_top=5, stream=side)
        side.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)


def test_refusals():
    x = torch.randn(2, 50, device="cuda")
    t = torch.zeros(2, dtype=torch.int32, device="cuda")
    for bad in (lambda: s2k.logprobs(x[0]), lambda: s2k.logprobs(x.T), lambda: s2k.logprobs(x.double()),
                lambda: s2k.logprobs(x, t.long()), lambda: s2k.logprobs(x, t[:1]), lambda: s2k.logprobs(x, t, n_top=33),
                lambda: s2k.logprobs(x[:, :3], t, n_top=4), lambda: s2k.logprobs(x.cpu(), t),
                lambda: s2k.logprobs(x, t.cpu())):
        with pytest.raises(s2k.S2KError):
            bad()
