"""GPU: the model's paths over an 8-bit KV cache and its token log
probabilities.

The last layer's buffers of a call (rotated queries, this call's keys and
values, the attention's output) are read back, and the attention is checked
against the plain 64-bit form over a cache that the same keys and values were
stored into by the definition: the tolerance is test_gpu_kv8.py's for f32 rows.
"""
from __future__ import annotations

import numpy as np
import pytest

import kv8_util as ku
import s2k
import synthetic

pytestmark = pytest.mark.gpu

ARG, KV_FULL, UNSUPPORTED = -1, -4, -7


@pytest.fixture(scope="module")
def small_gpu(small_model_data):
    hp, tensors = small_model_data
    m = s2k.SlowARModel(hp)
    m.load_tensors(tensors)
    yield m
    m.close()


class LastLayer:
    """The last layer's cache, kept by the definition from what each call stores."""

    def __init__(self, hp, max_seq_len, window=0, sinks=0):
        self.hp, self.window, self.sinks, self.n = hp, window, sinks, 0
        P = (max_seq_len + 15) // 16
        H, D = hp.head_count_kv, hp.head_dim
        self.table = np.arange(P, dtype=np.int32)[None]
        self.kq, self.vq = np.zeros((P, 1, H, 16, D), np.int8), np.zeros((P, 1, H, D, 16), np.int8)
        self.ks, self.vs = np.zeros((2, P, 1, H), np.float32)

    def store(self, k, v):
        T = k.shape[0]
        ku.append(self.kq, self.ks, 0, k, [0, T], [self.n], self.table, False)
        ku.append(self.vq, self.vs, 0, v, [0, T], [self.n], self.table, True)
        self.n += T

    def check(self, m, T):
        hp = self.hp
        H, Hkv, D = hp.head_count, hp.head_count_kv, hp.head_dim
        rows = (H + 2 * Hkv) * D
        q = m.debug_buffer("qkv")[: T * rows].reshape(T, rows)[:, : H * D].reshape(T, H, D).astype(np.float64)
        k = m.debug_buffer("kcur")[: T * Hkv * D].reshape(T, Hkv, D)
        v = m.debug_buffer("vcur")[: T * Hkv * D].reshape(T, Hkv, D)
        out = m.debug_buffer("attn")[: T * H * D].reshape(T, H, D)
        past = self.n
        self.store(k, v)
        kk = ku.values(self.kq, self.ks, 0, self.table[0], self.n, False)
        vv = ku.values(self.vq, self.vs, 0, self.table[0], self.n, True)
        vtop = np.repeat(self.vs[:, 0].astype(np.float64), 16, 0)[: self.n] * 127
        want, mag, size, _, grain, coarse = ku.attend(kk, vv, q, past, D ** -0.5, self.window, self.sinks, vtop)
        tol = (2.0**-30 * grain + 2.0**-31 * coarse)[..., None] + mag * (2.0**-19 * size[..., None] + 2.0**-18) + 1e-30
        assert np.all(np.abs(out - want) <= tol + np.abs(want) * 2.0**-23)


@pytest.mark.parametrize("window,sinks", [(0, 0), (20, 3)])
def test_eval_over_an_8_bit_cache(small_gpu, small_model_data, window, sinks):
    """A prompt on the prompt kernel, parts of a few tokens and single steps."""
    hp, _ = small_model_data
    m = small_gpu
    m.init_kv8_cache(130, window, sinks)
    layer = LastLayer(hp, 130, window, sinks)
    p = synthetic.text_prompt(hp, 120, seed=3).T.copy()
    at = 0
    for T in (70, 3, 1, 1, 17, 1, 2):
        h, lg = m.prefill_fast(p[at:at + T].reshape(-1), T)
        assert np.isfinite(lg).all() and np.isfinite(h).all()
        layer.check(m, T)
        at += T
        assert m.n_past == at
    with pytest.raises(s2k.S2KError) as e:
        m.prefill_fast(np.zeros(60 * p.shape[1], np.int32), 60)
    assert e.value.status == KV_FULL
    # after a reset its pages start afresh
    m.reset()
    layer = LastLayer(hp, 130, window, sinks)
    m.step(p[0])
    layer.check(m, 1)


def test_restored_cache(small_gpu, small_model_data):
    hp, _ = small_model_data
    m = small_gpu
    n = 37
    rng = np.random.default_rng(5)
    shape = (hp.block_count, n, hp.head_count_kv, hp.head_dim)
    k, v = rng.standard_normal(shape).astype(np.float16), rng.standard_normal(shape).astype(np.float16)
    m.init_kv8_cache(64)
    layer = LastLayer(hp, 64)
    m.load_kv(k, v)
    layer.store(k[-1].astype(np.float64), v[-1].astype(np.float64))
    assert m.n_past == n
    p = synthetic.text_prompt(hp, 2, seed=8).T.copy()
    for i in range(2):
        m.step(p[i])
        layer.check(m, 1)


def test_generate_over_an_8_bit_cache(small_gpu, small_model_data):
    """Frames come out the same twice; the cache they leave is the one that the same calls leave one by one."""
    hp, _ = small_model_data
    m = small_gpu
    p = synthetic.text_prompt(hp, 30, seed=9)
    m.init_kv8_cache(64, 24, 4)
    codes = m.generate(p, 9, temperature=0.0, seed=1)
    n = codes.shape[1]
    assert n > 0
    end = synthetic.text_prompt(hp, 1, seed=2).T.copy()[0]
    past = m.n_past
    assert past == 30 + n
    _, after = m.step(end)
    m.init_kv8_cache(64, 24, 4)
    assert np.array_equal(m.generate(p, 9, temperature=0.0, seed=1), codes)
    m.init_kv8_cache(64, 24, 4)
    m.prefill_fast(p.T.reshape(-1).copy(), 30)
    for f in range(n):
        m.step(np.concatenate([[codes[0, f] + hp.semantic_begin_id], codes[:, f]]).astype(np.int32))
    assert m.n_past == past
    _, again = m.step(end)
    assert np.array_equal(after, again)
    # a longer request makes a larger cache of the same kind
    m.generate(p, 60, temperature=0.7, seed=3)
    assert m._kv8 == (24, 4) and m._max_seq_len == 90


def test_an_8_bit_cache_is_half_as_large(small_gpu, small_model_data):
    hp, _ = small_model_data
    m = small_gpu
    m.clear_kv_cache()
    base = m.device_bytes()
    m.init_kv_cache(4096)
    f16 = m.device_bytes() - base
    m.init_kv8_cache(4096)
    kv8 = m.device_bytes() - base
    values = 2 * hp.block_count * hp.head_count_kv * hp.head_dim * 4096
    assert f16 - kv8 == values - values // (16 * hp.head_dim) * 4
    m.clear_kv_cache()
    assert m.device_bytes() == base


def test_eval_logprobs(small_gpu, small_model_data):
    """Against the softmax, in 64 bits, of the logits that s2k_eval gives for every prefix."""
    hp, _ = small_model_data
    m = small_gpu
    T = 75  # two chunks of rows, the second one ragged
    p = synthetic.text_prompt(hp, T, seed=4).T.copy()
    m.init_kv_cache(128)
    lp, ent, ids, top = m.eval_logprobs(p.reshape(-1), T, n_top=5)
    assert lp.shape == (T - 1,) and m.n_past == T
    for t in list(range(0, T, 9)) + [63, 64, T - 1]:
        m.reset()
        _, x = m.prefill_fast(p[: t + 1].reshape(-1), t + 1)
        x = x.astype(np.float64)
        z = x - x.max()
        z -= np.log(np.exp(z).sum())
        tol = 2.0**-21 * (1 + x.max() - x.min())
        if t + 1 < T:
            assert abs(lp[t] - z[p[t + 1, 0]]) <= tol
        assert abs(ent[t] + (np.exp(z) * z).sum()) <= tol
        order = np.argsort(-x, kind="stable")[:5]
        assert np.array_equal(ids[t], order) and np.all(np.abs(top[t] - z[order]) <= tol)
    # in parts, without alternatives, over an 8-bit cache
    m.init_kv8_cache(128)
    a = m.eval_logprobs(p[:40].reshape(-1), 40)
    b = m.eval_logprobs(p[40:].reshape(-1), T - 40)
    assert a[2] is None and b[0].shape == (T - 41,) and m.n_past == T
    # rounding keys and values to 8 bits moves them a little, not beyond recognition
    assert np.corrcoef(np.concatenate([a[0], b[0]]), np.delete(lp, 39))[0, 1] > 0.99


def test_refusals(small_gpu, small_model_data):
    hp, _ = small_model_data
    m = small_gpu
    for bad in ((0, 0, 0), (64, -1, 0), (64, 8, -1), (hp.context_length + 1, 0, 0)):
        with pytest.raises(s2k.S2KError) as e:
            m.init_kv8_cache(*bad)
        assert e.value.status == ARG
    m.init_kv8_cache(64)
    p = synthetic.text_prompt(hp, 4, seed=6)
    gp = s2k._GenParams(4, 0.0, 0.8, 30, 0, -1, 0, 0)
    import ctypes
    tm = np.ascontiguousarray(p, np.int32)
    assert s2k.lib().s2k_seq_begin(m.handle, m.seq_handle, tm.ctypes.data, 4, ctypes.byref(gp)) == UNSUPPORTED
    arr = (ctypes.c_void_p * 1)(m.seq_handle)
    assert s2k.lib().s2k_batch_frame(m.handle, arr, 1, None) == UNSUPPORTED
    for n_top in (-1, 33):
        with pytest.raises(s2k.S2KError) as e:
            m.eval_logprobs(p.T.reshape(-1).copy(), 4, n_top=n_top)
        assert e.value.status == ARG


def test_a_failed_restore_leaves_the_sequence_as_it_was(small_gpu, small_model_data):
    """No memory for the rows: the device's position must not part from the host's."""
    hp, _ = small_model_data
    m = small_gpu
    p = synthetic.text_prompt(hp, 4, seed=9).T.copy()
    shape = (hp.block_count, 20, hp.head_count_kv, hp.head_dim)
    k = np.ones(shape, np.float16)
    got = []
    for fail in (False, True):
        m.init_kv8_cache(64)
        m.prefill(p[:3].reshape(-1).copy(), 3)
        if fail:
            m.fail_alloc(0)
            with pytest.raises(s2k.S2KError):
                m.load_kv(k, k)
            m.fail_alloc(-1)
        assert m.n_past == 3
        got.append(m.step(p[3]))
    for a, b in zip(*got):
        assert np.array_equal(a, b)
