"""The paged 8-bit cache (sv_paged_*) against the oracle's 64-bit definitions.

Tolerances.  Plan: integers, equal.  Codes and scales of unrotated rows: the f32 steps are fixed, equal bit for
bit.  Rotated f32 values: the norm's sum and root cost ~10 units of 2^-24, the sine and cosine and the
angle (2^-24 turns = 2 pi 2^-24 rad) ~8, the two products and the norm weights ~4: under 2^-19 of the row's
largest magnitude.  f16 outputs add half a unit, 2^-11.  A rotated row's code stands for the value to half a
step plus that.  Attention: each softmax weight may be rounded to f16 once (2^-11 relative) and the scores'
f32 sums move a weight by less than that again, so an output is off by at most 2^-10 of the largest |v| that
its row sees; an f16 output adds 2^-11 of itself."""
import numpy as np
import pytest
import torch

from __graft_entry__ import load_package
from oracle import paged as orc

sv = load_package()
pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def _i(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)


class Batch:
    """A pool, a table with the past pages, the step planned."""

    def __init__(self, seed, past, new, *, n_head=8, n_kv=2, hd=64, ps=16, n_layer=1, spare=3, free=None, T=None, max_new=None,
                 blocks=None):
        rng = self.rng = np.random.default_rng(seed)
        self.past, self.new, self.ps, self.nh, self.nkv, self.hd = list(past), list(new), ps, n_head, n_kv, hd
        held = [-(-p // ps) for p in past]
        want = [-(-(p + max(c, 0)) // ps) for p, c in zip(past, new)]
        self.n_pages = sum(want) + spare
        perm = rng.permutation(self.n_pages)
        self.table = np.full((len(past), blocks or max(max(want), 1)), -1)
        at = 0
        for r, h in enumerate(held):
            self.table[r, :h] = perm[at:at + h]
            at += h
        self.free = perm[at:]
        self.n_free = len(self.free) if free is None else free
        self.T = T or max(1, sum(new))
        self.kv = sv.PagedKv(n_layer, n_kv, hd, ps, self.n_pages)
        self.step = sv.PagedStep(len(past), self.T, max_new or max(1, max(new)), ps, self.n_pages, n_head, n_kv, hd)
        self.d_past, self.d_new, self.d_table, self.d_free, self.d_nf = (
            _i(self.past), _i(self.new), _i(self.table), _i(self.free), _i([self.n_free]))

    def plan(self, **kw):
        self.step.plan(self.d_past, self.d_new, self.d_table, self.d_free, self.d_nf, **kw)
        return self

    def want(self, **kw):
        return orc.plan(self.past, self.new, self.table, self.free, self.n_free, self.ps, **kw)

    def fill(self, k_spread=0.3, v_spread=0.3):
        """Random codes and scales in every page: (k, v, ks, vs) as numpy."""
        out = []
        for is_v, spread in ((0, k_spread), (1, v_spread)):
            c = np.clip(np.rint(self.rng.standard_normal((self.n_pages, self.nkv, self.ps, self.hd)) * 40), -127, 127)
            s = (np.exp(spread * self.rng.standard_normal((self.n_pages, self.nkv))) / 40).astype(np.float32)
            self.kv.codes(0, is_v).copy_(torch.from_numpy(c.astype(np.int8)))
            self.kv.scales(0, is_v).copy_(torch.from_numpy(s))
            out.append((c, s))
        return out[0][0], out[1][0], out[0][1], out[1][1]


# ------------------------------------------------------------------ plan
def _check_plan(b, **kw):
    qs, kl, req, pos, slot, table, nf = b.want(**kw)
    st, n = b.step, len(req)
    assert st.q_start.tolist() == qs and st.kv_len.tolist() == kl
    assert st.tok_req.tolist() == req + [-1] * (b.T - n)
    assert st.tok_pos.tolist()[:n] == pos
    assert st.tok_slot.tolist() == slot + [-1] * (b.T - n)
    assert np.array_equal(b.d_table.cpu().numpy(), table)
    assert st.n_free.item() == nf


@pytest.mark.parametrize("ps", [16, 32, 64, 128])
@pytest.mark.parametrize("n,hi,past", [(1, 1, 0), (1, 1, 64), (3, 0, 20), (7, 1, 300), (40, 33, 500), (257, 5, 90), (1000, 9, 200),
                                       (2, 3000, 100)])
def test_plan(n, hi, past, ps):
    rng = np.random.default_rng(n * 131 + hi)
    p, c = rng.integers(0, past + 1, n), rng.integers(0, hi + 1, n)
    b = Batch(1, p.tolist(), c.tolist(), ps=ps)
    for _ in range(2):          # planning again changes nothing
        b.plan()
        _check_plan(b)
    assert b.step.error_flags() == 0


def test_plan_padded_rows_and_4096_requests():
    rng = np.random.default_rng(3)
    b = Batch(2, rng.integers(0, 50, 4096).tolist(), rng.integers(0, 3, 4096).tolist(), ps=16, T=9000, max_new=5)
    b.plan()
    _check_plan(b)


@pytest.mark.parametrize("free", [0, 1, 4])
def test_plan_runs_out_of_pages(free):
    b = Batch(4, [0, 30, 16, 5], [40, 3, 0, 20], ps=16, free=free)
    b.plan()
    _check_plan(b)
    assert b.step.error_flags() == sv.DEVERR_PAGES
    assert b.step.error_flags() == 0


def test_plan_table_full_and_lengths_cut():
    b = Batch(5, [30, 0], [40, 8], ps=16, blocks=3).plan()
    _check_plan(b)
    assert b.step.error_flags() == sv.DEVERR_PAGES
    b = Batch(6, [3, 0, 7], [5, 9, 4], ps=16, T=12, max_new=6).plan()
    _check_plan(b, n_tokens=12, max_new=6)
    assert b.step.error_flags() == sv.DEVERR_STEP
    b = Batch(6, [3, 0], [5, 0], ps=16)
    b.d_new[1] = -4
    b.plan()
    _check_plan(b)
    assert b.step.error_flags() == sv.DEVERR_STEP


def test_release_gives_pages_back_in_order():
    b = Batch(7, [100, 0, 33, 16], [10, 5, 1, 0], ps=16).plan()
    table = b.d_table.cpu().numpy()
    kl = b.step.kv_len.cpu().numpy()
    free = torch.full((b.n_pages,), -7, dtype=torch.int32, device=DEV)
    nf = int(b.step.n_free.item())
    free[:nf] = b.d_free[:nf]
    count = b.step.n_free.clone()
    req = [2, 0, 3]
    b.kv.release(b.d_table, _i(req), _i(kl[req]), free, count)
    want = free.cpu().numpy()[:nf].tolist()
    for r in req:
        want += table[r, :-(-kl[r] // 16)].tolist()
        table[r, :-(-kl[r] // 16)] = -1
    assert count.item() == len(want) and free.cpu().numpy()[:len(want)].tolist() == want
    assert np.array_equal(b.d_table.cpu().numpy(), table) and b.kv.error_flags() == 0
    b.kv.release(b.d_table, _i([9]), _i([16]), free, count)      # no such request
    assert b.kv.error_flags() == sv.DEVERR_STEP and count.item() == len(want)


# ------------------------------------------------------------------ append and read
def _rows(b, dtype, spread=1.0, packed=True):
    x = b.rng.standard_normal((b.T, b.nh + 2 * b.nkv, b.hd)) * spread
    t = torch.from_numpy(x).to(DEV, dtype)
    q, k, v = t[:, :b.nh], t[:, b.nh:b.nh + b.nkv], t[:, b.nh + b.nkv:]
    return (q, k, v) if packed else (q.contiguous(), k.contiguous(), v.contiguous())


def _np(t):
    return t.double().cpu().numpy()


def _append(b, q, k, v, *, rope=None, angle=None, mag=1.0, pairs=False, qn=None, kn=None, pos=None, q_out=None):
    """Appends and checks every output; returns q_out."""
    old_c = [b.kv.codes(0, i).cpu().numpy().copy() for i in (0, 1)]
    old_s = [b.kv.scales(0, i).cpu().numpy().copy() for i in (0, 1)]
    eq, ek = (orc.norm(_np(x), None if w is None else _np(w), 1e-6) for x, w in ((q, qn), (k, kn)))
    vn = v.float().cpu().numpy()
    if angle is not None:
        eq, ek = orc.rotate(eq, angle, mag, pairs), orc.rotate(ek, angle, mag, pairs)
    exact_k = rope is None and kn is None
    out = b.kv.rope_append(0, b.step, q, k, v, rope=rope, q_norm=qn, k_norm=kn, pos=pos, q_out=q_out)
    big = np.abs(eq).max(-1, keepdims=True)
    live = sum(b.new)
    tol = 2.0 ** -19 * big + (2.0 ** -11 * np.abs(eq) + 2.0 ** -24 if out.dtype == torch.float16 else 0)
    assert np.all(np.abs(_np(out) - eq)[:live] <= tol[:live])
    _, kv_len, _, _, _, table, _ = b.want()
    codes = [b.kv.codes(0, i).cpu().numpy() for i in (0, 1)]
    scales = [b.kv.scales(0, i).cpu().numpy() for i in (0, 1)]
    touched = set()
    t = 0
    for r, (p, c) in enumerate(zip(b.past, b.new)):
        i = p
        while i < p + c:
            page, o = table[r, i // b.ps], i % b.ps
            m = min(p + c - i, b.ps - o)
            touched.add(page)
            for h in range(b.nkv):
                want, s = orc.quantise(vn[t:t + m, h], old_c[1][page, h, :o], old_s[1][page, h])
                assert scales[1][page, h] == s
                assert np.array_equal(codes[1][page, h, :o + m], want)
                x, got, gs = ek[t:t + m, h], codes[0][page, h], scales[0][page, h]
                if exact_k:
                    want, s = orc.quantise(x, old_c[0][page, h, :o], old_s[0][page, h])
                    assert gs == s and np.array_equal(got[:o + m], want)
                else:
                    near = 2.0 ** -19 * np.abs(x).max()
                    old = old_s[0][page, h] if o else 0.0
                    assert abs(gs - max(old, np.abs(x).max() / 127)) <= 2.0 ** -18 * gs
                    assert np.all(np.abs(got[o:o + m] * float(gs) - x) <= gs * 0.5001 + near)
                    if o:
                        f = np.float32(old) * (np.float32(1) / gs)
                        kept = np.rint(old_c[0][page, h, :o].astype(np.float32) * f) if gs > old else old_c[0][page, h, :o]
                        assert np.array_equal(got[:o], kept)
            i, t = i + m, t + m
    rest = [x for x in range(b.n_pages) if x not in touched]
    for is_v in (0, 1):
        assert np.array_equal(codes[is_v][rest], old_c[is_v][rest]) and np.array_equal(scales[is_v][rest], old_s[is_v][rest])
    assert b.kv.error_flags() == 0
    return out


LENS = [([0], [1]), ([15], [1]), ([17], [40]), ([0, 100, 31, 64, 5], [130, 1, 0, 70, 3])]


@pytest.mark.parametrize("past,new", LENS)
@pytest.mark.parametrize("hd,ps", [(64, 16), (64, 128), (128, 32), (128, 128), (256, 16), (256, 64), (256, 128)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_append_unrotated_bit_exact(past, new, hd, ps, dtype):
    b = Batch(11, past, new, hd=hd, ps=ps, n_head=6, n_kv=2).plan()
    b.fill()
    _append(b, *_rows(b, dtype, 1.7))


@pytest.mark.parametrize("mode,n_dims,hd", [("half", 128, 128), ("pairs", 128, 128), ("half", 64, 128), ("pairs", 32, 128),
                                            ("half", 24, 64), ("pairs", 24, 64), ("half", 2, 64), ("pairs", 254, 256),
                                            ("half", 256, 256), ("half", 250, 256), ("half", 64, 64)])
@pytest.mark.parametrize("normed", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_append_rotated(mode, n_dims, hd, normed, dtype):
    b = Batch(12, [0, 100, 31, 64, 70001], [70, 1, 0, 33, 3], hd=hd, ps=32, n_head=10, n_kv=2).plan()
    b.fill()
    f, _ = orc.frequencies(n_dims, 1e4)
    w = [torch.from_numpy(1 + 0.2 * b.rng.standard_normal(hd)).to(DEV, torch.float32) if normed else None for _ in range(2)]
    pos = np.array(b.want()[3], np.float64)
    rope = sv.Rope(n_dims, mode=sv.ROPE_NEOX if mode == "half" else sv.ROPE_NORM)
    _append(b, *_rows(b, dtype), rope=rope, angle=pos[:, None] * f[None], pairs=mode == "pairs", qn=w[0], kn=w[1],
            q_out=torch.empty((b.T, b.nh, hd), dtype=torch.float32, device=DEV) if dtype == torch.float32 else None)


@pytest.mark.parametrize("long", [dict(freq_scale=0.25), dict(freq_scale=0.25, ext_factor=1.0, n_ctx_orig=8192),
                                  dict(freq_scale=0.125, ext_factor=0.7, n_ctx_orig=4096, attn_factor=0.9, beta_fast=16.0,
                                       beta_slow=2.0),
                                  dict(freq_factors=np.linspace(1, 8, 64).astype(np.float32))])
def test_append_scaled_contexts(long):
    b = Batch(13, [131000, 20000000], [40, 2], hd=128, ps=128, n_head=4, n_kv=1, spare=1).plan()
    f, mag = orc.frequencies(128, 5e5, **long)
    pos = np.array(b.want()[3], np.float64)
    _append(b, *_rows(b, torch.float32), rope=sv.Rope(128, freq_base=5e5, **long), angle=pos[:, None] * f[None], mag=mag,
            q_out=torch.empty((b.T, b.nh, 128), dtype=torch.float32, device=DEV))


def test_append_three_axes():
    """Interleaved multi-axis positions of the framework's IMROPE rule, given as four streams."""
    b = Batch(14, [50, 3], [20, 9], hd=128, ps=16).plan()
    sec = (24, 20, 20, 0)
    pos = np.stack([b.rng.integers(0, 9000, b.T) for _ in range(4)])
    f, _ = orc.frequencies(128, 5e6)
    axis = [1 if j % 3 == 1 and j < 60 else 2 if j % 3 == 2 and j < 60 else 0 if j % 3 == 0 and j < 72 else 3 for j in range(64)]
    _append(b, *_rows(b, torch.float16), rope=sv.Rope(128, mode=sv.ROPE_IMROPE, freq_base=5e6, sections=sec),
            angle=pos[axis].T * f[None], pos=_i(pos))


def test_append_given_positions_and_in_place_queries():
    b = Batch(15, [50, 3], [20, 9], hd=128, ps=16, n_head=5, n_kv=1).plan()
    q, k, v = _rows(b, torch.float16, packed=False)
    pos = b.rng.integers(0, 1000, b.T)
    f, _ = orc.frequencies(128, 1e4)
    want = b.kv.rope_append(0, b.step, q, k, v, rope=sv.Rope(128), pos=_i(pos)).clone()
    b.kv.codes(0, 0).zero_()
    out = _append(b, q, k, v, rope=sv.Rope(128), angle=pos[:, None] * f[None], pos=_i(pos), q_out=q)
    assert out.data_ptr() == q.data_ptr() and torch.equal(q, want)


def test_append_many_tokens():
    """Enough rows for several heads per thread; a head count that the groups do not divide."""
    b = Batch(16, [5, 0, 900], [900, 300, 77], hd=128, ps=64, n_head=20, n_kv=4).plan()
    b.fill()
    f, _ = orc.frequencies(128, 1e6)
    pos = np.array(b.want()[3], np.float64)
    _append(b, *_rows(b, torch.float16), rope=sv.Rope(128, freq_base=1e6), angle=pos[:, None] * f[None])


def test_append_non_finite_zero_and_tiny_rows():
    b = Batch(17, [4, 0, 20], [20, 16, 3], hd=64, ps=16, n_kv=1, n_head=2).plan()
    b.fill()
    q, k, v = _rows(b, torch.float32)
    v[0, 0, :4] = torch.tensor([float("nan"), float("inf"), -float("inf"), 0.0])
    v[20:36] = 0                      # a whole page of zeros
    k[20:36] = 1e-33
    v[36:39] = float("inf")           # no finite value beside the page's earlier rows
    _append(b, q, k, v)
    assert not torch.isnan(b.kv.scales(0, 1)).any()


def test_append_page_grows_token_by_token():
    """One row at a time into one page: codes follow the running scale, and stand for the rows to within half a
    step for each time that the scale grew."""
    b = Batch(18, [0], [1], hd=64, ps=32, n_kv=1, n_head=1, spare=4)
    rows, grew = [], 0
    for t in range(32):
        b.past, b.d_past = [t], _i([t])
        b.plan()
        x = torch.from_numpy(b.rng.standard_normal((1, 1, 64)) * (1 + 0.1 * t)).to(DEV, torch.float32)
        before = float(b.kv.scales(0, 1)[int(b.d_table[0, 0]), 0]) if t else 0.0
        b.kv.rope_append(0, b.step, x, x, x)
        rows.append(_np(x)[0, 0])
        s = float(b.kv.scales(0, 1)[int(b.d_table[0, 0]), 0])
        grew += s > before
        b.table, b.d_nf, b.n_free = b.d_table.cpu().numpy(), b.step.n_free.clone(), int(b.step.n_free.item())
    page = int(b.d_table[0, 0])
    got = b.kv.codes(0, 1)[page, 0].cpu().numpy() * s
    assert grew > 2 and np.abs(got - np.array(rows)).max() <= s * (0.5 + 0.5 * grew)


def test_append_drops_rows_without_a_page():
    b = Batch(19, [16, 0], [20, 30], hd=64, ps=16, free=1).plan()
    b.fill()
    before = [b.kv.codes(0, i).clone() for i in (0, 1)]
    b.kv.rope_append(0, b.step, *_rows(b, torch.float16))
    slots = b.step.tok_slot.cpu().numpy()
    written = {int(s) // 16 for s in slots if s >= 0}
    assert len(written) == 1 and (slots < 0).sum() == 34
    for i in (0, 1):
        rest = [p for p in range(b.n_pages) if p not in written]
        assert torch.equal(b.kv.codes(0, i)[rest], before[i][rest])


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("hd,ps,nkv", [(64, 16, 3), (128, 64, 8), (256, 128, 1)])
def test_read(hd, ps, nkv, dtype):
    b = Batch(20, [100, 40], [1, 1], hd=hd, ps=ps, n_kv=nkv, n_head=nkv).plan()
    k, v, ks, vs = b.fill()
    slots = b.rng.integers(0, b.n_pages * ps, 77)
    shape = (77, nkv, hd)
    ko, vo = b.kv.read(0, _i(slots), *(torch.empty(shape, dtype=dtype, device=DEV) for _ in range(2)))
    for got, c, s in ((ko, k, ks), (vo, v, vs)):
        want = c[slots // ps, :, slots % ps].astype(np.float32) * s[slots // ps][:, :, None]
        assert torch.equal(got.cpu(), torch.from_numpy(want.astype(np.float32)).to(dtype))
    assert b.kv.error_flags() == 0
    ko, vo = b.kv.read(0, _i([-1, 3]))
    assert not ko[0].any() and b.kv.error_flags() == 0
    ko, vo = b.kv.read(0, _i([b.n_pages * ps, 3, -2]))
    assert not ko[0].any() and not vo[2].any() and b.kv.error_flags() == sv.DEVERR_ROW_RANGE
    assert b.kv.read(0, _i([]))[0].shape == (0, nkv, hd)


# ------------------------------------------------------------------ attention
def _attn(b, filled, *, window=0, dtype=torch.float16, out=torch.float16, scale=None, q=None, strided=False):
    k, v, ks, vs = filled
    scale = scale or 1 / np.sqrt(b.hd)
    if q is None:
        q = torch.from_numpy(b.rng.standard_normal((b.T, b.nh * (2 if strided else 1), b.hd))).to(DEV, dtype)[:, :b.nh]
    o = torch.full((b.T, b.nh, b.hd), 7.0, dtype=out, device=DEV)
    b.kv.attn(0, b.step, q, scale, window=window, out=o)
    _, kv_len, _, _, _, table, _ = b.want()
    want = orc.attention(q.half().double().cpu().numpy(), k, v, ks, vs, table, b.past, b.new, kv_len, scale, window)
    got, live = _np(o), sum(b.new)
    big = max(np.abs(v[p]).max() * vs[p].max() for p in range(b.n_pages))
    tol = 2.0 ** -10 * big + (2.0 ** -11 * np.abs(want[:live]) if out == torch.float16 else 0)
    assert np.all(np.isfinite(got))
    assert np.all(np.abs(got[:live] - want[:live]) <= tol), np.abs(got[:live] - want[:live]).max() / big
    assert np.all(got[live:] == 7.0)
    assert b.kv.error_flags() == 0
    return o


@pytest.mark.parametrize("past,new", [([0], [1]), ([1], [1]), ([62], [2]), ([63], [1]), ([64], [1]), ([3000], [1]), ([0, 5, 700, 64], [1, 0, 1, 2]),
                                      ([90, 2000, 17, 0, 1, 333, 128], [1, 1, 2, 1, 0, 1, 1])])
@pytest.mark.parametrize("hd,ps,nh,nkv", [(64, 16, 8, 2), (64, 64, 3, 3), (128, 16, 32, 8), (128, 64, 8, 1), (128, 128, 10, 2),
                                          (256, 32, 16, 4), (256, 128, 6, 2)])
def test_attn_few_rows(past, new, hd, ps, nh, nkv):
    b = Batch(21, past, new, hd=hd, ps=ps, n_head=nh, n_kv=nkv).plan()
    _attn(b, b.fill())


@pytest.mark.parametrize("past,new", [([0], [128]), ([0], [129]), ([5], [33]), ([300], [65]), ([1000], [300]), ([0, 40, 200], [100, 1, 257]),
                                      ([100, 7, 0, 900], [1, 50, 0, 1])])
@pytest.mark.parametrize("hd,ps,nh,nkv", [(64, 32, 8, 2), (64, 16, 2, 2), (128, 16, 8, 2), (128, 64, 5, 1), (128, 128, 12, 4),
                                          (256, 16, 8, 2), (256, 64, 3, 1)])
def test_attn_many_rows(past, new, hd, ps, nh, nkv):
    b = Batch(22, past, new, hd=hd, ps=ps, n_head=nh, n_kv=nkv).plan()
    _attn(b, b.fill())


@pytest.mark.parametrize("window", [1, 2, 16, 63, 64, 65, 100, 1000])
@pytest.mark.parametrize("hd,nh,nkv", [(64, 8, 2), (128, 8, 2), (256, 4, 1)])
def test_attn_window(window, hd, nh, nkv):
    b = Batch(23, [500, 0, 130, 63], [1, 90, 2, 200], hd=hd, ps=32, n_head=nh, n_kv=nkv).plan()
    _attn(b, b.fill(), window=window)


@pytest.mark.parametrize("g", [1, 3, 7, 8, 9, 16, 17, 40])
def test_attn_group_sizes(g):
    b = Batch(24, [300, 20, 0], [1, 3, 40], hd=64, ps=16, n_head=2 * g, n_kv=2).plan()
    _attn(b, b.fill())


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("out", [torch.float16, torch.float32])
def test_attn_types_and_strides(dtype, out):
    for hd in (64, 128, 256):
        b = Batch(25, [300, 20, 0], [1, 3, 70], hd=hd, ps=16, n_head=8, n_kv=2).plan()
        _attn(b, b.fill(), dtype=dtype, out=out, strided=True)


def test_attn_scales_far_apart_and_empty_pages():
    """Value scales over four orders of magnitude in one request, and pages of zeros with scale 0."""
    for new in ([1, 2], [90, 60]):
        for hd in (64, 128, 256):
            b = Batch(26, [400, 999], new, hd=hd, ps=16, n_head=4, n_kv=1).plan()
            k, v, ks, vs = b.fill(k_spread=1.0, v_spread=2.0)
            for p in range(0, b.n_pages, 3):
                k[p], v[p], ks[p], vs[p] = 0, 0, 0, 0
            for is_v, (c, s) in enumerate(((k, ks), (v, vs))):
                b.kv.codes(0, is_v).copy_(torch.from_numpy(c.astype(np.int8)))
                b.kv.scales(0, is_v).copy_(torch.from_numpy(s))
            _attn(b, (k, v, ks, vs), out=torch.float32)


def test_attn_does_not_read_past_the_end():
    """Rows past a request's end and pages of nobody hold the largest codes and scales that are not numbers."""
    for past, new in (([70, 9], [1, 1]), ([70, 9], [40, 70])):
        for hd in (64, 128, 256):
            b = Batch(27, past, new, hd=hd, ps=32, n_head=4, n_kv=2).plan()
            k, v, ks, vs = b.fill()
            _, kv_len, _, _, _, table, _ = b.want()
            used = set()
            for r, n in enumerate(kv_len):
                for j in range(-(-n // 32)):
                    used.add(int(table[r, j]))
                if n % 32:
                    for i in (0, 1):
                        b.kv.codes(0, i)[int(table[r, n // 32]), :, n % 32:] = 127
            for p in range(b.n_pages):
                if p not in used:
                    for i in (0, 1):
                        b.kv.codes(0, i)[p] = 127
                        b.kv.scales(0, i)[p] = float("nan")
                    v[p] = 0
                    vs[p] = 0
            _attn(b, (k, v, ks, vs))


@pytest.mark.parametrize("new", [[3, 2, 0], [40, 60, 0]])
def test_attn_rows_that_see_no_key(new):
    """No page was free: rows attend to what is held, and a request that holds nothing gets zeros; more
    rows than tokens are left alone."""
    b = Batch(28, [16, 0, 0], new, hd=128, ps=16, n_head=8, n_kv=2, free=0, T=sum(new) + 5, max_new=64).plan()
    assert b.step.error_flags() == sv.DEVERR_PAGES
    o = _attn(b, b.fill())
    assert not o[new[0]:new[0] + new[1]].any()


def test_attn_table_entry_out_of_range_is_skipped():
    for new in ([1], [50]):
        b = Batch(29, [100], new, hd=128, ps=16, n_head=4, n_kv=1).plan()
        filled = b.fill()
        b.d_table[0, 2] = b.n_pages + 5
        o = b.kv.attn(0, b.step, torch.zeros((b.T, 4, 128), dtype=torch.float16, device=DEV), 0.1)
        assert b.kv.error_flags() & sv.DEVERR_PAGES and torch.isfinite(o).all()
        # with equal weights the rest of the keys average as if the page were not there
        k, v, ks, vs = filled
        n = 100 + new[0]
        keep = [j for j in range(n) if j // 16 != 2]
        table = b.d_table.cpu().numpy()
        rows = np.stack([v[table[0, j // 16], 0, j % 16] * vs[table[0, j // 16], 0] for j in keep])
        assert np.abs(_np(o[-1, 0]) - rows.mean(0)).max() <= 2.0 ** -10 * np.abs(rows).max()


def test_attn_large_scores():
    """Scores far apart: the weights of most keys vanish, nothing overflows."""
    for new in ([1], [100]):
        for hd in (64, 128, 256):
            b = Batch(30, [700], new, hd=hd, ps=16, n_head=4, n_kv=2).plan()
            _attn(b, b.fill(), scale=4.0, out=torch.float32)


def test_attn_same_bits_each_time_and_on_another_stream():
    b = Batch(31, [5000, 100, 2500], [1, 200, 2], hd=128, ps=64, n_head=8, n_kv=2).plan()
    filled = b.fill()
    q = torch.from_numpy(b.rng.standard_normal((b.T, 8, 128))).to(DEV, torch.float16)
    first = _attn(b, filled, q=q)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    for i in range(5):
        with torch.cuda.stream(s):
            b.plan()
            o = b.kv.attn(0, b.step, q, 1 / np.sqrt(128))
        s.synchronize()
        assert torch.equal(o, first)


def test_steps_of_a_session_in_a_graph():
    """A captured decode step (plan, append, attend on two layers), replayed while the lengths advance on the
    device, equals the same steps launched one by one."""
    outs = []
    for graph in (False, True):
        b = Batch(32, [30, 0, 127], [1, 1, 1], hd=128, ps=32, n_head=8, n_kv=2, n_layer=2, spare=12, blocks=8)
        b.rng = np.random.default_rng(5)
        for layer in (0, 1):
            for i in (0, 1):
                g = torch.Generator(device=DEV).manual_seed(9 + i)
                b.kv.codes(layer, i).copy_(torch.randint(-127, 128, b.kv.codes(layer, i).shape, generator=g, device=DEV))
                b.kv.scales(layer, i).fill_(0.01)
        x = torch.zeros((3, 12, 128), dtype=torch.float16, device=DEV)
        o = torch.zeros((2, 3, 8, 128), dtype=torch.float16, device=DEV)
        qo = torch.zeros((3, 8, 128), dtype=torch.float16, device=DEV)
        rope = sv.Rope(128)

        def one():
            b.plan()
            for layer in (0, 1):
                b.kv.rope_append(layer, b.step, x[:, :8], x[:, 8:10], x[:, 10:], rope=rope, q_out=qo)
                b.kv.attn(layer, b.step, qo, 0.09, out=o[layer])
            b.d_nf.copy_(b.step.n_free)
            sv.counter_add(b.d_past, 1)

        rows = [torch.from_numpy(b.rng.standard_normal((3, 12, 128))).to(DEV, torch.float16) for _ in range(40)]
        x.copy_(rows[0])
        if graph:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                one()
            s.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                one()
        else:
            one()
        got = [o.clone()]
        for r in rows[1:]:
            x.copy_(r)
            if graph:
                g.replay()
            else:
                one()
            torch.cuda.synchronize()
            got.append(o.clone())
        assert b.step.error_flags() == 0 and b.kv.error_flags() == 0
        outs.append(torch.stack(got))
    assert torch.equal(outs[0], outs[1])


def test_refusals():
    b = Batch(33, [10], [4], hd=128, ps=16, n_head=4, n_kv=2).plan()
    q = torch.zeros((4, 4, 128), dtype=torch.float16, device=DEV)
    kk = torch.zeros((4, 2, 128), dtype=torch.float16, device=DEV)
    with pytest.raises(sv.SvError):
        b.kv.attn(0, b.step, q.bfloat16(), 0.1)
    with pytest.raises(sv.SvError):
        b.kv.attn(0, b.step, q, -0.1)
    with pytest.raises(sv.SvError):
        b.kv.attn(0, b.step, q[:3], 0.1)
    with pytest.raises(sv.SvError):
        b.kv.attn(0, b.step, q.transpose(1, 2).contiguous().transpose(1, 2), 0.1)
    with pytest.raises(sv.SvError):
        b.kv.rope_append(0, b.step, q, kk, kk.float())
    with pytest.raises(sv.SvError):
        b.kv.rope_append(0, b.step, q, kk, kk, rope=sv.Rope(256))
    with pytest.raises(sv.SvError):
        b.kv.rope_append(0, b.step, q, kk, kk, rope=sv.Rope(128, mode=sv.ROPE_IMROPE, sections=(24, 20, 20, 0)))
    with pytest.raises(sv.SvError):
        b.kv.rope_append(0, b.step, torch.zeros((4, 8, 128), dtype=torch.float16, device=DEV)[:, :4, :], kk, kk,
                         q_out=torch.zeros((4, 8, 128), dtype=torch.float16, device=DEV)[:, :4])
    with pytest.raises(sv.SvError):
        b.step.plan(b.d_past, b.d_new, b.d_table, b.d_free, b.step.n_free)     # in and out are one word
    with pytest.raises(sv.SvError):
        b.step.plan(b.d_past.long(), b.d_new, b.d_table, b.d_free, b.d_nf)
    other = sv.PagedKv(1, 2, 128, 32, b.n_pages)
    with pytest.raises(sv.SvError):
        other.attn(0, b.step, q, 0.1)
    for bad in (dict(n_dims=3), dict(n_dims=0), dict(n_dims=258), dict(n_dims=64, mode=7), dict(n_dims=64, freq_base=0.0),
                dict(n_dims=64, freq_scale=0.0), dict(n_dims=64, ext_factor=1.0), dict(n_dims=64, freq_factors=[1.0])):
        with pytest.raises(sv.SvError):
            sv.Rope(**bad)


# ------------------------------------------------------------------ large steps, long pools, rows that are no numbers
@pytest.mark.parametrize("past,new,hd,ps,nh,nkv", [([0], [1100], 64, 16, 8, 2), ([700, 0, 33], [600, 450, 1], 128, 32, 8, 2),
                                                   ([100], [1030], 256, 64, 8, 1), ([40, 5], [129, 900], 128, 128, 9, 3),
                                                   ([0] * 9, [250] * 9, 64, 32, 4, 4)])
@pytest.mark.parametrize("window", [0, 200])
def test_attn_large_steps(past, new, hd, ps, nh, nkv, window):
    """More query rows in the step than the small-step kernels take: the weights go as one f16 each."""
    b = Batch(34, past, new, hd=hd, ps=ps, n_head=nh, n_kv=nkv).plan()
    assert b.T * nh > 8192
    _attn(b, b.fill(), window=window)


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_attn_large_steps_scales_far_apart(hd):
    b = Batch(35, [300, 20], [700, 400], hd=hd, ps=16, n_head=8, n_kv=2).plan()
    _attn(b, b.fill(k_spread=1.0, v_spread=2.0), out=torch.float32)


@pytest.mark.parametrize("past,new", [([3000], [1]), ([300, 20], [3, 5]), ([700, 40], [150, 90]), ([10], [1100])])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_attn_rows_that_are_no_numbers_stay_alone(past, new, hd):
    """A query row with NaN, infinities or values past f16's range changes no other row's bits."""
    b = Batch(36, past, new, hd=hd, ps=16, n_head=8, n_kv=2).plan()
    b.fill()
    q = torch.from_numpy(b.rng.standard_normal((b.T, 8, hd))).to(DEV, torch.float32)
    first = b.kv.attn(0, b.step, q, 0.1)
    bad = q.clone()
    rows = torch.zeros((b.T, 8), dtype=torch.bool, device=DEV)
    for t in range(0, b.T, 37):
        for h, x in ((1, float("nan")), (2, float("inf")), (6, 1e30)):
            bad[t, h, 5] = x
            rows[t, h] = True
    out = b.kv.attn(0, b.step, bad, 0.1)
    # (a row's reference may be taken earlier because of its neighbours, so the weights' rounding differs: twice the
    # tolerance of one output)
    big = max(float(b.kv.scales(0, 1).max()) * 127, 1e-30)
    tol = 2 * (2.0 ** -10 * big + 2.0 ** -11 * first[~rows].double().abs())
    assert ((out[~rows].double() - first[~rows].double()).abs() <= tol).all()
    assert b.kv.error_flags() == 0


@pytest.mark.parametrize("past,new", [([3000], [1]), ([500, 64], [2, 1]), ([600, 31], [200, 161]), ([100], [1100])])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("window", [16, 0])
def test_attn_rows_of_small_values_beside_large_ones(past, new, hd, window):
    """Value scales 2^22 apart from page to page: a row whose window (or whose weights) holds small values alone is as
    exact as any other, against the largest |weight x value| that it sees."""
    b = Batch(38, past, new, hd=hd, ps=16, n_head=8, n_kv=2).plan()
    k, v, ks, vs = b.fill()
    _, kv_len, _, _, _, table, _ = b.want()
    for r, n in enumerate(kv_len):
        for j in range(-(-n // 16)):
            p = int(table[r, j])
            vs[p] *= 2.0 ** -22 if j % 2 else 1.0
            if window == 0:                           # keys of the large values get no weight: 50 binary orders less
                k[p] = -8 if j % 2 == 0 else 8
                ks[p] = 0.05
    for is_v, (c, s) in enumerate(((k, ks), (v, vs))):
        b.kv.codes(0, is_v).copy_(torch.from_numpy(np.ascontiguousarray(c).astype(np.int8)))
        b.kv.scales(0, is_v).copy_(torch.from_numpy(s.astype(np.float32)))
    q = b.rng.standard_normal((b.T, 8, hd)) * 0.01
    if window == 0:
        q = np.abs(q) + 50 * np.log(2) / (2 * 0.4 * hd * 0.5)
    q = torch.from_numpy(q).to(DEV, torch.float16)
    got = _np(b.kv.attn(0, b.step, q, 0.5, window=window, out=torch.empty((b.T, 8, hd), dtype=torch.float32, device=DEV)))
    qd = _np(q)
    want = orc.attention(qd, k, v, ks, vs, table, b.past, b.new, kv_len, 0.5, window)
    # the same with |v| and, per row, the largest weight x scale in place of the sum
    t = 0
    for r, c in enumerate(b.new):
        for i in range(c):
            p = b.past[r] + i
            lo, hi = (max(0, p - window + 1) if window else 0), min(p + 1, kv_len[r])
            pages = np.array([int(table[r, j // 16]) for j in range(lo, hi)])
            at = np.arange(lo, hi) % 16
            for h in (0, 7):
                x = (k[pages, h // 4, at] * ks[pages, h // 4][:, None].astype(np.float64)) @ qd[t, h] * 0.5
                w = np.exp(x - x.max())
                each = w[:, None] * np.abs(v[pages, h // 4, at]) * vs[pages, h // 4][:, None].astype(np.float64) / w.sum()
                tol = 2.0 ** -10 * each.sum(0) + 2.0 ** -20 * each.max()
                assert np.all(np.abs(got[t, h] - want[t, h]) <= tol)
            t += 1
    assert b.kv.error_flags() == 0


@pytest.mark.parametrize("n", [9, 36, 37, 38, 54, 55, 56, 57, 130, 200])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_attn_many_short_requests(n, hd):
    """About as many requests, and pieces of requests, as thread blocks run at once, and more of either."""
    rng = np.random.default_rng(n)
    for hi in (30, 500):
        past, new = rng.integers(0, hi, n).tolist(), rng.integers(0, 3, n).tolist()
        b = Batch(39, past, new, hd=hd, ps=32, n_head=8, n_kv=8).plan()
        _attn(b, b.fill())


def test_pool_past_32_bit_offsets():
    """The pages of a step lie beyond 2^31 bytes and 2^31 elements of the pool: the same bits as in a small pool."""
    hd, nkv, nh, ps, past, new = 256, 8, 16, 128, [300, 70], [1, 200]
    small = Batch(37, [0, 0], [p + n for p, n in zip(past, new)], hd=hd, ps=ps, n_head=nh, n_kv=nkv)
    rows = torch.from_numpy(small.rng.standard_normal((sum(past) + sum(new), nh + 2 * nkv, hd))).to(DEV, torch.float16)
    outs = []
    for n_pages in (small.n_pages, 9000):
        kv = sv.PagedKv(1, nkv, hd, ps, n_pages)
        free = _i(np.arange(n_pages))               # the last are taken first
        table, nf = _i(np.full((2, 4), -1)), _i([n_pages])
        got, rope = [], sv.Rope(hd)
        for had, add, x in (([0, 0], past, rows[:sum(past)]), (past, new, rows[sum(past):])):
            step = sv.PagedStep(2, sum(add), max(add), ps, n_pages, nh, nkv, hd)
            step.plan(_i(had), _i(add), table, free, nf)
            nf = step.n_free.clone()
            q = kv.rope_append(0, step, x[:, :nh], x[:, nh:nh + nkv], x[:, nh + nkv:], rope=rope)
            got += [q, kv.attn(0, step, q, 0.07)]
            k, v = kv.read(0, step.tok_slot)
            got += [k, v]
            assert step.error_flags() == 0 and kv.error_flags() == 0
        if n_pages == 9000:
            assert int(table[table >= 0].min()) * nkv * ps * hd > 2 ** 31
        outs.append(got)
    assert all(torch.equal(x, y) for x, y in zip(*outs))


def test_example_sessions():
    """The example at a small size.  Codes carry values to s / sqrt(12) with s = max / 127 over a page and head (about 3.5
    to 4 standard deviations): 0.9 % of a row, and again each time a page's scale grows; K's part moves the weights by as
    much.  Together below 4 % of the output's norm."""
    from examples.paged_sessions import run
    r = run(seats=5, prompt=150, tokens=12, layers=2, n_head=8, n_kv=2, hd=64, page_size=16)
    assert r["freed"] > 0 and r["rel_err"] < 0.04
