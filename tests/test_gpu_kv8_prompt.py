"""GPU: calls that the 8-bit KV cache's kernel of many rows takes, each with the assertion that it did: the model's
prompts, blocks beyond 4 GiB, captured and concurrent calls, and so many rows that their division by the heads leaves
f32.  Tolerances as in test_gpu_kv8.py."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import kv8_util as ku
import s2k
import synthetic
from test_gpu_kv8 import DT, EXTRA, Call, i32
from test_gpu_kv8_model import LastLayer

pytestmark = pytest.mark.gpu

FEW, MANY = 1, 2


def taken():
    return s2k.lib().s2k_debug_kv8_attend_kernel()


@pytest.fixture(scope="module")
def small_gpu(small_model_data):
    hp, tensors = small_model_data
    m = s2k.SlowARModel(hp)
    m.load_tensors(tensors)
    yield m
    m.close()


@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 20)])
def test_a_models_prompt(small_gpu, small_model_data, window, sinks):
    """A prompt of 600 tokens, a second part behind it, and steps, over one cache; twice the same."""
    hp, _ = small_model_data
    m = small_gpu
    p = synthetic.text_prompt(hp, 1142, seed=3).T.copy()
    first = None
    for again in range(2):
        m.init_kv8_cache(1160, window, sinks)
        layer = LastLayer(hp, 1160, window, sinks)
        at, last = 0, []
        for T, kernel in ((600, MANY), (540, MANY), (1, FEW), (1, FEW)):
            h, lg = m.prefill_fast(p[at:at + T].reshape(-1), T)
            assert taken() == kernel
            if not again:
                layer.check(m, T)
            at += T
            assert m.n_past == at
            last.append((h, lg))
        if first is None:
            first = last
    for a, b in zip(first, last):
        assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])


def test_far_pages():
    """Blocks beyond 4 GiB of the pool: 2^21 + 8 pages of 2 KB."""
    P, D = (1 << 21) + 8, 128
    cache = s2k.KV8Cache.empty(P, 1, 1, D)
    table = i32([[P - 1, P - 3, 1 << 20]])
    x, y = torch.randn(2, 40, 1, D, device="cuda")
    cache.append(0, x, y, i32([0]), table)
    kb, vb = (t.double().cpu().numpy() for t in cache.read(0, 40, i32([0]), table))
    q = torch.randn(40, 128, D, device="cuda")
    out = cache.attend(0, q, i32([0]), table).double().cpu().numpy()
    assert taken() == MANY
    want, mag, size, _, _, _ = ku.attend(kb, vb, q.double().cpu().numpy(), 0, D ** -0.5)
    tol = mag * (2 * 2.0**-20 * size[..., None] + EXTRA["f32"]) + np.abs(want) * 2.0**-24 * 2
    assert np.all(np.abs(out - want) <= tol)
    del cache
    torch.cuda.empty_cache()


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
def test_captured_replayed_and_on_another_stream(typ):
    """A prompt's part stored and attended, captured once, replayed over changing positions, rows and streams."""
    c = Call([600], [45], 32, 8, 128, typ, ld_extra=2)
    c.table[0, -2:] = np.setdiff1d(np.arange(c.kq.shape[0]), c.table[0, :-2])[:2]  # two more pages of its own
    c.ks[c.table[0, -2:]] = c.vs[c.table[0, -2:]] = 0.01
    c.upload()
    past, table = c.args
    k, v, q = c.heads(8), c.heads(8), c.heads(32)
    ref = s2k.KV8Cache(*[t.clone() for t in (c.cache.k, c.cache.v, c.cache.k_scale, c.cache.v_scale)])
    out = torch.empty_like(q)

    def part(cache, out):
        cache.append(c.layer, k, v, past, table)
        cache.attend(c.layer, q, past, table, out=out)
        assert taken() == MANY

    g, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(g, stream=side):
        part(c.cache, out)
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
        part(ref, want)
        assert torch.equal(out, want) and torch.equal(c.cache.k, ref.k) and torch.equal(c.cache.v, ref.v)
        past += 9


@pytest.mark.parametrize("typ", ["f32", "bf16"])
def test_two_streams_at_once(typ):
    cs = [Call([700], [90], 32, 8, 128, typ, seed=s) for s in (1, 2)]
    qs = [c.heads(32) for c in cs]
    want = [c.cache.attend(c.layer, q, *c.args) for c, q in zip(cs, qs)]
    assert taken() == MANY
    streams = [torch.cuda.Stream() for _ in cs]
    torch.cuda.synchronize()
    got = []
    for _ in range(8):
        for c, q, s in zip(cs, qs, streams):
            got.append(c.cache.attend(c.layer, q, *c.args, stream=s))
    torch.cuda.synchronize()
    for i, o in enumerate(got):
        assert torch.equal(o, want[i % 2])


@pytest.mark.parametrize("typ", ["f32", "f16"])
def test_rows_beyond_two_to_the_twenty(typ):
    """257 rows of 4099 query heads on one kv head: 1,053,443 (row, head) pairs."""
    rows, past, H, D = 257, 30, 4099, 64
    c = Call([rows], [past], H, 1, D, typ, layers=1)
    q = torch.randn(rows, H, D, device="cuda", generator=torch.Generator("cuda").manual_seed(5)).to(DT[typ])
    out = c.cache.attend(0, q, *c.args, window=50, sinks=3)
    assert taken() == MANY
    for r in (0, 1, 128, 255, 256):  # of these rows the first heads, some in the middle and the last ones
        heads = [0, 1, 2, 2047, 2048, 4000, 4096, 4097, 4098]
        part = Call([1], [past + r], len(heads), 1, D, typ, layers=1)
        part.kq, part.vq, part.ks, part.vs, part.table = c.kq, c.vq, c.ks, c.vs, c.table
        part.check_attend(q[r:r + 1, heads], out[r:r + 1, heads], window=50, sinks=3)
