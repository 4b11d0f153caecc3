"""Paged 8-bit cache in numpy, 64 bits: the definitions that include/svkv.h gives, written plainly.

Positions, tables and codes are loops over requests, pages and keys; nothing here is shared with the
library under test."""
import math

import numpy as np


def plan(n_past, n_new, table, free, n_free, ps, n_tokens=None, max_new=None):
    """(q_start, kv_len, tok_req, tok_pos, tok_slot, table, n_free) of a step; -1 slots where no page was left."""
    table = np.array(table, dtype=np.int64)
    q_start, kv_len, req, pos, slot = [0], [], [], [], []
    k = n_free
    for r, (p, c) in enumerate(zip(n_past, n_new)):
        c = max(0, c if max_new is None else min(c, max_new))
        if n_tokens is not None:
            c = min(c, n_tokens - q_start[-1])
        have = -(-p // ps)
        end = p
        for j in range(have, min(-(-(p + c) // ps), table.shape[1])):
            if k > 0:
                k -= 1
                table[r, j] = free[k]
            else:
                table[r, j] = -1
        for i in range(p, p + c):
            j = i // ps
            page = table[r, j] if j < table.shape[1] else -1
            slot.append(page * ps + i % ps if page >= 0 else -1)
            if page >= 0:
                end = i + 1
            req.append(r)
            pos.append(i)
        kv_len.append(end)
        q_start.append(q_start[-1] + c)
    return q_start, kv_len, req, pos, slot, table, k


def frequencies(n_dims, base, freq_scale=1.0, ext_factor=0.0, attn_factor=1.0, beta_fast=32.0, beta_slow=1.0, n_ctx_orig=0,
                freq_factors=None):
    """(radians per position of each pair, factor on cos and sin)"""
    out = []
    for i in range(n_dims // 2):
        f = float(base) ** (-2.0 * i / n_dims) / (1.0 if freq_factors is None else float(freq_factors[i]))
        if ext_factor > 0:
            dim = lambda b: n_dims * math.log(n_ctx_orig / (b * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
            low, high = max(0.0, math.floor(dim(beta_fast))), min(n_dims - 1.0, math.ceil(dim(beta_slow)))
            keep = (1 - min(1.0, max(0.0, (i - low) / max(0.001, high - low)))) * ext_factor
            f = f * freq_scale * (1 - keep) + f * keep
        else:
            f *= freq_scale
        out.append(f)
    return np.array(out), attn_factor * (1 + 0.1 * math.log(1 / freq_scale) if ext_factor > 0 else 1.0)


def norm(x, w, eps):
    x = np.asarray(x, np.float64)
    return x if w is None else x / np.sqrt(np.mean(x * x, -1, keepdims=True) + eps) * np.asarray(w, np.float64)


def rotate(x, angle, mag, pairs):
    """x [T, H, HD], angle [T, n/2]; pairs: (2i, 2i + 1), else (i, i + n/2)"""
    y = x.copy()
    n = 2 * angle.shape[1]
    for i in range(n // 2):
        a, b = (2 * i, 2 * i + 1) if pairs else (i, i + n // 2)
        c, s = mag * np.cos(angle[:, i])[:, None], mag * np.sin(angle[:, i])[:, None]
        y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    return y


def quantise(rows, old_codes, old_scale):
    """One page and head in f32, operation by operation: new rows [n, HD] behind old codes [o, HD].
    Returns (codes [o + n, HD], scale)."""
    f = np.float32
    x = np.asarray(rows, f)
    fin = np.abs(x[np.isfinite(x)])
    amax = fin.max() if fin.size else f(0)
    if amax < f(2.0 ** -100):
        amax = f(0)
    old = f(old_scale) if len(old_codes) else f(0)
    s = max(old, f(amax) / f(127))
    inv = f(1) / s if s > 0 else f(0)
    with np.errstate(invalid="ignore"):
        new = np.clip(np.rint(x * inv), -127, 127)
    new = np.where(np.isnan(x), 0, np.where(np.isposinf(x), 127, np.where(np.isneginf(x), -127, new)))
    kept = np.asarray(old_codes, f)
    if s > old and len(old_codes):
        kept = np.clip(np.rint(kept * (old * inv)), -127, 127)
    return np.concatenate([kept.reshape(-1, x.shape[1]), new]).astype(np.int64), s


def attention(q, k_codes, v_codes, k_scale, v_scale, table, n_past, n_new, kv_len, scale, window=0):
    """q [T, NH, HD]; codes [pages, NKV, ps, HD]; scales [pages, NKV] -> [T, NH, HD] float64"""
    q = np.asarray(q, np.float64)
    nkv, ps = k_codes.shape[1:3]
    g = q.shape[1] // nkv
    out = np.zeros_like(q)
    t = 0
    for r in range(len(n_past)):
        n = kv_len[r]
        pages = [int(table[r][j]) for j in range(-(-n // ps))]
        if n:
            k = (k_codes[pages].astype(np.float64) * k_scale[pages].astype(np.float64)[:, :, None, None])
            v = (v_codes[pages].astype(np.float64) * v_scale[pages].astype(np.float64)[:, :, None, None])
            k = k.transpose(1, 0, 2, 3).reshape(nkv, -1, q.shape[2])[:, :n]
            v = v.transpose(1, 0, 2, 3).reshape(nkv, -1, q.shape[2])[:, :n]
        for i in range(n_new[r]):
            p = n_past[r] + i
            lo, hi = (max(0, p - window + 1) if window > 0 else 0), min(p + 1, n)
            if lo < hi:
                for h in range(q.shape[1]):
                    x = k[h // g, lo:hi] @ q[t, h] * scale
                    w = np.exp(x - x.max())
                    out[t, h] = w @ v[h // g, lo:hi] / w.sum()
            t += 1
    return out
