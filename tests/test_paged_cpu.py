"""The paged cache's C entries without a device: bounds, alignment and types are refused before anything is launched;
and the 64-bit definitions that the GPU tests compare with, against the formulas written another way."""
import ctypes
import math

import numpy as np
import pytest

from __graft_entry__ import load_package
from oracle import paged as orc

sv = load_package()
MEM = ctypes.create_string_buffer(4096)
P = (ctypes.addressof(MEM) + 255) & ~255            # aligned; never followed: every call here is refused


def _step(**kw):
    s = sv._PagedStep(4, 64, 16, 8, 8, 2, 128, 32, 100)
    for n in ("n_past", "n_new", "table", "q_start", "kv_len", "tok_req", "tok_pos", "tok_slot", "work"):
        setattr(s, n, P)
    s.work_bytes = 1 << 40
    for k, v in kw.items():
        setattr(s, k, v)
    return s


def _store(**kw):
    s = sv._Paged(P, P, P, P, 100, 2, 32, 128, None)
    for k, v in kw.items():
        setattr(s, k, v)
    return s


def _refused(rc):
    assert rc < 0 and rc != -3, rc                  # refused by a check, not by CUDA
    return rc


@pytest.mark.parametrize("kw", [dict(n_req=0), dict(n_req=4097), dict(n_tokens=0), dict(n_tokens=-5), dict(max_new=0),
                                dict(head_dim=96), dict(head_dim=512), dict(page_size=8), dict(page_size=48), dict(n_head=7),
                                dict(n_head=0), dict(n_kv_head=0), dict(n_pages=0), dict(page_size=0)])
def test_bounds_that_have_no_step(kw):
    assert sv.lib().sv_paged_step_bytes(ctypes.byref(_step())) > 0
    s = _step(**kw)
    assert sv.lib().sv_paged_step_bytes(ctypes.byref(s)) == 0
    _refused(sv.lib().sv_paged_plan(ctypes.byref(s), P, P, P + 4, None))
    assert sv.lib().sv_paged_step_bytes(None) == 0


def test_step_bytes_do_not_depend_on_pointers_and_grow_with_the_bounds():
    size = lambda **kw: sv.lib().sv_paged_step_bytes(ctypes.byref(_step(**kw)))  # noqa: E731
    assert size() == size(n_past=None, work=None, max_blocks=77)
    assert size() <= size(n_tokens=128) <= size(n_tokens=128, max_new=128)
    assert size(n_req=8) >= size()


@pytest.mark.parametrize("kw", [dict(n_past=None), dict(n_new=None), dict(table=None), dict(q_start=None), dict(kv_len=None),
                                dict(tok_req=None), dict(tok_pos=None), dict(tok_slot=None), dict(work=None),
                                dict(max_blocks=0), dict(work=P + 16), dict(work_bytes=64)])
def test_plan_refusals(kw):
    _refused(sv.lib().sv_paged_plan(ctypes.byref(_step(**kw)), P, P, P + 4, None))


def test_plan_refuses_missing_lists():
    L, s = sv.lib(), ctypes.byref(_step())
    for free, n, out in ((None, P, P + 4), (P, None, P + 4), (P, P, None), (P, P, P)):
        _refused(L.sv_paged_plan(s, free, n, out, None))
    _refused(L.sv_paged_plan(None, P, P, P + 4, None))


@pytest.mark.parametrize("kw", [dict(k=None), dict(v=None), dict(k_scale=None), dict(v_scale=None), dict(k=P + 8),
                                dict(v_scale=P + 2), dict(n_pages=0), dict(n_pages=99), dict(n_kv_head=4), dict(page_size=16),
                                dict(page_size=20), dict(head_dim=64), dict(head_dim=80), dict(n_pages=2 ** 30)])
def test_store_refusals(kw):
    L, kv, s = sv.lib(), ctypes.byref(_store(**kw)), ctypes.byref(_step())
    _refused(L.sv_paged_attn(kv, s, P, sv.TYPE_F16, 2048, 0.1, 0, P, sv.TYPE_F16, None))
    rows = ctypes.create_string_buffer(sv._ROWS.pack(P, P, P, sv.TYPE_F16, 2048, 512, 512, 0, 0, 1e-6, 0, 0, P, sv.TYPE_F16))
    _refused(L.sv_paged_append(kv, s, rows, None))


@pytest.mark.parametrize("bad", [dict(q=None), dict(q=P + 8), dict(qt=8), dict(nb=2040), dict(nb=2000), dict(nb=1024), dict(out=None),
                                 dict(ot=8), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf),
                                 dict(q=P, qt=0)])
def test_attention_refusals(bad):
    a = dict(q=P, qt=sv.TYPE_F16, nb=2048, scale=0.1, out=P, ot=sv.TYPE_F16)
    a.update(bad)                                   # (f32 rows of 8 x 128 need 4096 bytes)
    _refused(sv.lib().sv_paged_attn(ctypes.byref(_store()), ctypes.byref(_step()), a["q"], a["qt"], a["nb"], a["scale"], 0,
                                    a["out"], a["ot"], None))


@pytest.mark.parametrize("i,value", [(0, 0), (1, 0), (2, 0), (12, 0), (0, P + 4), (2, P + 8), (3, 8), (13, 8), (4, 2040), (4, 1024),
                                     (5, 256), (6, 500), (9, -1e-6), (9, math.nan)])
def test_append_refusals(i, value):
    args = [P, P, P, sv.TYPE_F16, 2048, 512, 512, 0, 0, 1e-6, 0, 0, P, sv.TYPE_F16]
    args[i] = value
    rows = ctypes.create_string_buffer(sv._ROWS.pack(*args))
    _refused(sv.lib().sv_paged_append(ctypes.byref(_store()), ctypes.byref(_step()), rows, None))


def test_append_in_place_needs_the_same_type_and_packed_rows():
    for qt, nb, ot in ((sv.TYPE_F16, 2048, sv.TYPE_F32), (sv.TYPE_F32, 4096, sv.TYPE_F16), (sv.TYPE_F16, 3072 + 1024, sv.TYPE_F16)):
        rows = ctypes.create_string_buffer(sv._ROWS.pack(P, P, P, qt, nb, 1024, 1024, 0, 0, 1e-6, 0, 0, P, ot))
        _refused(sv.lib().sv_paged_append(ctypes.byref(_store()), ctypes.byref(_step()), rows, None))


def test_read_and_release_refusals():
    L, kv = sv.lib(), ctypes.byref(_store())
    for slots, n, k, v, t in ((None, 4, P, P, 1), (P, -1, P, P, 1), (P, 4, None, P, 1), (P, 4, P, None, 1), (P, 4, P + 4, P, 1),
                              (P, 4, P, P, 8)):
        _refused(L.sv_paged_read(kv, slots, n, k, v, t, None))
    ok = [P, 4, 8, 32, 100, P, 2, P, P, P, None]
    for i, x in ((0, None), (1, 0), (2, 0), (3, 24), (4, 0), (5, None), (6, -1), (6, 5), (7, None), (8, None), (9, None)):
        args = list(ok)
        args[i] = x
        _refused(L.sv_paged_release(*args, None))
    ok[6] = 0
    assert L.sv_paged_release(*ok, None) == 0       # nothing to give back


@pytest.mark.parametrize("kw", [dict(mode=99), dict(n_dims=0), dict(n_dims=7), dict(n_dims=300), dict(freq_base=0.0),
                                dict(freq_base=math.inf), dict(freq_scale=0.0), dict(ext_factor=-1.0), dict(ext_factor=1.0),
                                dict(attn_factor=math.nan), dict(freq_scale=math.inf), dict(freq_base=math.nan)])
def test_rope_table_refusals(kw):
    p = sv._RopeParams(sv.ROPE_NORM, 64, (ctypes.c_int * 4)(0, 0, 0, 0), 10000.0, 1.0, 0.0, 1.0, 32.0, 1.0, 0, None)
    for k, v in kw.items():
        setattr(p, k, v)
    out = ctypes.c_void_p()
    _refused(sv.lib().sv_rope_table_create(0, ctypes.byref(p), ctypes.byref(out)))
    assert not out.value


def test_rope_table_refuses_negative_sections_and_factors():
    out = ctypes.c_void_p()
    p = sv._RopeParams(sv.ROPE_IMROPE, 64, (ctypes.c_int * 4)(24, -1, 20, 0), 10000.0, 1.0, 0.0, 1.0, 32.0, 1.0, 0, None)
    _refused(sv.lib().sv_rope_table_create(0, ctypes.byref(p), ctypes.byref(out)))
    bad = np.ones(32, np.float32)
    bad[7] = 0
    p = sv._RopeParams(sv.ROPE_NORM, 64, (ctypes.c_int * 4)(), 10000.0, 1.0, 0.0, 1.0, 32.0, 1.0, 0, bad.ctypes.data)
    _refused(sv.lib().sv_rope_table_create(0, ctypes.byref(p), ctypes.byref(out)))
    assert not out.value


# ------------------------------------------------------------------ the definitions
def test_plan_definition_covers_every_token_once():
    rng = np.random.default_rng(1)
    past, new = rng.integers(0, 200, 30).tolist(), rng.integers(0, 50, 30).tolist()
    table = np.full((30, 20), -1)
    pages = rng.permutation(1000)
    at = 0
    for r, p in enumerate(past):
        held = -(-p // 16)
        table[r, :held] = pages[at:at + held]
        at += held
    free = pages[at:]
    qs, kl, req, pos, slot, out, left = orc.plan(past, new, table, free, len(free), 16)
    assert kl == [p + n for p, n in zip(past, new)] and qs == np.concatenate([[0], np.cumsum(new)]).tolist()
    assert len(set(slot)) == len(slot) == sum(new)
    taken = sum(-(-k // 16) for k in kl) - sum(-(-p // 16) for p in past)
    assert left == len(free) - taken
    flat = out[out >= 0]
    assert len(np.unique(flat)) == len(flat)
    assert all(out[r, p // 16] * 16 + p % 16 == s for r, p, s in zip(req, pos, slot))


def test_quantise_definition_keeps_values_to_half_a_step():
    rng = np.random.default_rng(2)
    a, b = rng.standard_normal((7, 64)), 5 * rng.standard_normal((4, 64))
    c, s = orc.quantise(a, np.zeros((0, 64)), 0.0)
    assert np.abs(c * float(s) - a).max() <= 0.5001 * s and np.abs(c).max() == 127
    c2, s2 = orc.quantise(b, c, s)
    assert s2 > s and np.abs(c2[:7] * float(s2) - a).max() <= 0.5001 * (s + s2)
    assert np.abs(c2[7:] * float(s2) - b).max() <= 0.5001 * s2
    c3, s3 = orc.quantise(a * 0.01, c, s)
    assert s3 == s and np.array_equal(c3[:7], c)
    assert orc.quantise(np.zeros((2, 64)), np.zeros((0, 64)), 3.0)[1] == 0


@pytest.mark.parametrize("pairs", [False, True])
def test_rotate_definition_is_a_rotation_by_the_distance(pairs):
    rng = np.random.default_rng(3)
    q, k = rng.standard_normal((2, 1, 1, 64))
    f, mag = orc.frequencies(32, 10000.0)
    assert mag == 1.0
    dot = [float((orc.rotate(q, np.array([f * m]), 1.0, pairs) * orc.rotate(k, np.array([f * n]), 1.0, pairs)).sum())
           for m, n in ((5, 3), (1005, 1003), (2, 0))]
    assert abs(dot[0] - dot[1]) < 1e-9 and abs(dot[0] - dot[2]) < 1e-9
    assert np.array_equal(orc.rotate(q, np.array([f * 9]), 1.0, pairs)[..., 32:], q[..., 32:])


def test_frequencies_between_kept_and_stretched():
    f0, _ = orc.frequencies(128, 1e6)
    f1, mag = orc.frequencies(128, 1e6, freq_scale=0.25, ext_factor=1.0, n_ctx_orig=8192)
    r = f1 / f0
    assert r[0] == 1 and abs(r[-1] - 0.25) < 1e-12 and np.all(np.diff(r) <= 1e-12)
    assert abs(mag - (1 + 0.1 * math.log(4))) < 1e-12


def test_attention_definition_against_a_dense_product():
    rng = np.random.default_rng(4)
    k, v = rng.integers(-127, 128, (2, 6, 2, 16, 64))
    ks, vs = np.exp(rng.standard_normal((2, 6, 2))) / 100
    table = np.array([[4, 1, -1], [0, 5, 2]])
    past, new, kv_len = [20, 40], [3, 4], [23, 44]
    q = rng.standard_normal((7, 4, 64))
    for window in (0, 10):
        got = orc.attention(q, k, v, ks, vs, table, past, new, kv_len, 0.1, window)
        t = 0
        for r in range(2):
            n = kv_len[r]
            pages = table[r][np.arange(n) // 16]
            for i in range(new[r]):
                d = past[r] + i - np.arange(n)
                seen = (d >= 0) & ((d < window) if window else True)
                for h in range(4):
                    x = np.einsum("d,jd->j", q[t, h], k[pages, h // 2, np.arange(n) % 16] * ks[pages, h // 2][:, None]) * 0.1
                    w = np.where(seen, np.exp(x - x[seen].max()), 0)
                    want = np.einsum("j,jd->d", w / w.sum(), v[pages, h // 2, np.arange(n) % 16] * vs[pages, h // 2][:, None])
                    assert np.abs(got[t, h] - want).max() < 1e-12
                t += 1
