"""CPU: the operators' argument checks (they come before any device call), the
binding's structs against the header, and the plain form's own properties."""
from __future__ import annotations

import ctypes
import os
import re

import numpy as np
import pytest

import kv8_util as ku
import s2k

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ARG, UNSUPPORTED, NO_DEVICE = -1, -7, -8
A = 1 << 20  # an aligned address that no check dereferences


def cache(**kw):
    f = dict(k=A, v=A, k_scale=A, v_scale=A, device=0, n_pages=8, n_layers=2, n_kv_heads=2, head_dim=128)
    f.update(kw)
    return s2k._KV8(**f)


def rows(**kw):
    f = dict(n_seqs=2, n_rows=6, max_rows=3, table_ld=4, past=A, row_start=None, block_table=A, err=None)
    f.update(kw)
    return s2k._KV8Rows(**f)


def heads(h=2, d=128, **kw):
    f = dict(data=A, row_stride=h * d, head_stride=d, type=0)
    f.update(kw)
    return s2k._Heads(**f)


def call(c=None, layer=0, r=None, k=None, v=None, fn="s2k_kv8_append"):
    c, r, k, v = c or cache(), r or rows(), k or heads(), v or heads()
    return getattr(s2k.lib(), fn)(ctypes.byref(c), layer, ctypes.byref(r), ctypes.byref(k), ctypes.byref(v), None)


def attend(c=None, layer=0, r=None, q=None, out=None, n_heads=4, scale=0.1, window=0, sinks=0):
    c, r, q, out = c or cache(), r or rows(), q or heads(4), out or heads(4)
    return s2k.lib().s2k_kv8_attend(ctypes.byref(c), layer, ctypes.byref(r), ctypes.byref(q), ctypes.byref(out),
                                    n_heads, scale, window, sinks, None)


BAD = [
    (dict(c=dict(head_dim=96)), UNSUPPORTED), (dict(c=dict(n_pages=0)), ARG), (dict(c=dict(n_layers=-1)), ARG),
    (dict(c=dict(k=None)), ARG), (dict(c=dict(v=A + 8)), ARG), (dict(c=dict(v_scale=A + 2)), ARG),
    (dict(layer=2), ARG), (dict(layer=-1), ARG),
    (dict(r=dict(n_seqs=-1)), ARG), (dict(r=dict(max_rows=7)), ARG), (dict(r=dict(n_seqs=3)), ARG),
    (dict(r=dict(table_ld=0)), ARG), (dict(r=dict(table_ld=1 << 27)), ARG), (dict(r=dict(past=None)), ARG),
    (dict(r=dict(block_table=None)), ARG),
    (dict(r=dict(n_seqs=1 << 20, n_rows=1 << 30, max_rows=1 << 14, row_start=A)), ARG),
    (dict(k=dict(type=8)), UNSUPPORTED), (dict(k=dict(data=None)), ARG), (dict(k=dict(data=A + 2)), ARG),
    (dict(k=dict(row_stride=-256)), ARG),
]


@pytest.mark.skipif(s2k.device_count() > 0, reason="fake addresses: only where nothing can be launched")
@pytest.mark.parametrize("kw,status", BAD)
def test_kv8_refusals(kw, status):
    mk = dict(c=cache, r=rows, k=heads)
    args = {n: mk[n](**v) if n in mk else v for n, v in kw.items()}
    assert call(**args) == status
    assert s2k.lib().s2k_last_error()
    assert call(fn="s2k_kv8_read", **args) == status
    if "k" in args:
        args["q"] = heads(4, **kw["k"])
        del args["k"]
    assert attend(**args) == status


@pytest.mark.skipif(s2k.device_count() > 0, reason="fake addresses: only where nothing can be launched")
def test_kv8_refusals_of_pairs_and_masks():
    assert call() == attend() == NO_DEVICE
    assert call(v=heads(type=1)) == ARG
    assert attend(out=heads(4, type=1)) == ARG
    assert attend(n_heads=3) == ARG and attend(n_heads=0) == ARG
    assert attend(scale=float("nan")) == ARG and attend(scale=float("inf")) == ARG
    assert attend(window=-1) == ARG and attend(sinks=-1) == ARG
    # outputs whose rows overlap; inputs may
    assert call(k=heads(row_stride=0)) == NO_DEVICE
    assert call(fn="s2k_kv8_read", k=heads(row_stride=128)) == ARG
    assert attend(out=heads(4, row_stride=128)) == ARG
    assert attend(out=heads(4, row_stride=128, head_stride=6 * 128)) == NO_DEVICE  # [heads][rows][dim]
    # no rows: nothing to point at
    empty = rows(n_seqs=0, n_rows=0, max_rows=0, past=None, block_table=None)
    assert call(r=empty, k=heads(data=None), v=heads(data=None)) == NO_DEVICE


@pytest.mark.skipif(s2k.device_count() > 0, reason="fake addresses: only where nothing can be launched")
def test_logprobs_refusals():
    def lp(x=A, type=0, rows=2, n=100, ld=100, tgt=A, top=4, lp=A, ent=A, ids=A, tlp=A):
        return s2k.lib().s2k_logprobs(0, x, type, rows, n, ld, tgt, top, lp, ent, ids, tlp, None)
    assert lp() == NO_DEVICE and lp(top=0, ids=None, tlp=None) == NO_DEVICE and lp(tgt=None, lp=None) == NO_DEVICE
    assert lp(type=14) == UNSUPPORTED
    for kw in (dict(x=None), dict(x=A + 2), dict(rows=-1), dict(n=0), dict(ld=-1), dict(tgt=None), dict(top=33),
               dict(top=-1), dict(n=3, ld=3), dict(ids=None), dict(tlp=None)):
        assert lp(**kw) == ARG, kw


def test_structs_match_header():
    txt = open(os.path.join(ROOT, "include", "s2k.h")).read()
    for name, cls in (("s2k_kv8", s2k._KV8), ("s2k_kv8_rows", s2k._KV8Rows), ("s2k_heads", s2k._Heads)):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), txt, flags=re.S).group(1)
        body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
        names = [n.strip().lstrip("*") for d in body.split(";") if d.strip() for n in d.strip().split(None, 1)[1].split(",")]
        names = [n.split()[-1].lstrip("*") for n in names]
        assert names == [f for f, _ in cls._fields_]
    # the packed forms that the binding passes
    for pack, s in ((s2k._PACK_KV8, cache(device=3)), (s2k._PACK_ROWS, rows(row_start=A + 64, err=A + 128)),
                    (s2k._PACK_HEADS, heads(type=30))):
        assert pack(*[getattr(s, f) or 0 for f, _ in s._fields_]) == bytes(s)


def test_plain_append_by_steps_stays_near_one_call():
    """Tokens stored one by one end within the roundings that the scale's growth adds."""
    rng = np.random.default_rng(0)
    x = rng.standard_normal((16, 1, 64)).astype(np.float32)
    t = np.zeros((1, 1), np.int32)
    one, steps = np.zeros((2, 1, 1, 1, 16, 64), np.int8)
    s1, s2 = np.zeros((2, 1, 1, 1), np.float32)
    ku.append(one, s1, 0, x, [0, 16], [0], t, False)
    grew, last = 0, 0.0
    for i in range(16):
        ku.append(steps, s2, 0, x[i:i + 1], [0, 1], [i], t, False)
        grew += s2[0, 0, 0] > last
        last = s2[0, 0, 0]
    assert s1[0, 0, 0] == s2[0, 0, 0]
    d = np.abs(ku.values(steps, s2, 0, t[0], 16, False) - x)
    assert d.max() <= s2[0, 0, 0] * (0.5 * grew + 0.01)


@pytest.mark.skipif(s2k.device_count() > 0, reason="fake addresses: only where nothing can be launched")
def test_strides_whose_extents_pass_64_bits():
    far = 1 << 62
    many = rows(n_seqs=1, n_rows=9, max_rows=9)
    for bad in (heads(row_stride=far), heads(head_stride=far)):
        assert call(r=many, k=bad) == call(r=many, k=bad, fn="s2k_kv8_read") == ARG
    assert attend(r=many, out=heads(4, row_stride=128, head_stride=far)) == ARG
    assert attend(r=many, out=heads(4, row_stride=far, head_stride=128)) == ARG
    assert call(k=heads(row_stride=1 << 30)) == NO_DEVICE
    assert call(k=heads(row_stride=128, head_stride=1 << 34)) == NO_DEVICE  # [heads][rows][dim] of many rows


def test_numbers_beyond_32_bits_are_not_cut():
    """ctypes would pass 2^32 + 5 as 5."""
    torch = pytest.importorskip("torch")
    c = object.__new__(s2k.KV8Cache)
    s2k._torch_module()
    c.device, c.n_pages, c.n_layers, c.n_kv_heads, c.head_dim, c._c = 0, 1, 1, 1, 64, b""
    c.k_scale = torch.zeros(1)
    q, past, table = torch.zeros(1, 1, 64), torch.zeros(1, dtype=torch.int32), torch.zeros(1, 1, dtype=torch.int32)
    big = (1 << 32) + 5
    for f in (lambda: c.append(big, q, q, past, table), lambda: c.read(big, 1, past, table),
              lambda: c.read(0, big, past, table),
              lambda: c.attend(big, q, past, table), lambda: c.attend(0, q, past, table, window=big),
              lambda: c.attend(0, q, past, table, sinks=big), lambda: c._rows(1, past, table, past, big, None),
              lambda: s2k.logprobs(torch.zeros(1, 64), n_top=big),
              lambda: s2k.logprobs(torch.zeros(1, 1).expand(big, 1))):
        with pytest.raises(s2k.S2KError, match="out of range"):
            f()


@pytest.mark.skipif(s2k.device_count() > 0, reason="fake addresses: only where nothing can be launched")
def test_logprobs_row_strides_whose_extents_pass_64_bits():
    def lp(rows, ld):
        return s2k.lib().s2k_logprobs(0, A, 0, rows, 100, ld, A, 4, A, A, A, A, None)
    for rows, ld in ((9, 1 << 62), (2, 1 << 60), (1 << 30, 1 << 34), (3, 1 << 40)):
        assert lp(rows, ld) == ARG, (rows, ld)
    assert lp(1, 1 << 62) == NO_DEVICE  # one row: its stride leads nowhere
    assert lp(9, 1 << 30) == lp(1 << 20, 155648) == lp(9, 0) == NO_DEVICE


@pytest.mark.skipif(s2k.device_count() > 0, reason="fake addresses: only where nothing can be launched")
def test_row_counts_next_to_32_bits():
    """Sums of the largest row counts with a page's size must not wrap."""
    for n in ((1 << 31) - 1, (1 << 31) - 3, (1 << 31) - 16):
        r = rows(n_seqs=1, n_rows=n, max_rows=n)
        assert call(r=r) == call(r=r, fn="s2k_kv8_read") == attend(r=r) == ARG, n
    r = rows(n_seqs=1, n_rows=1 << 30, max_rows=1 << 30)
    assert call(r=r) == NO_DEVICE
