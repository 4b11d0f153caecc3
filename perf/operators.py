"""The paged 8-bit cache path, as cases that can be run and timed: a step's page plan, rotary
positions with the quantising append, and attention over the paged cache.

    plan    block tables, slot map and positions of a step, from request lengths and a free list
    append  q/k RMSNorm, rotary positions, K/V quantised into 8-bit pages (one scale for each page
            and head); returns the rotated queries and every row of the touched pages, read back
    attn    causal grouped-query attention of the step's tokens over the paged 8-bit cache

`run` computes each in elementary torch operations in 32 bits (own = False) or through the package's
entry points (own = True); `exact` restates the definition in 64 bits.
"""
import importlib.util
import math
import os
import random
import sys

import numpy as np
import torch

own = False
DEV = "cuda:0"
EPS = 1e-6


def _package():
    name = "skyvision_b200"
    if name not in sys.modules:
        at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "skyvision.cpp_b200")
        spec = importlib.util.spec_from_file_location(name, os.path.join(at, "__init__.py"),
                                                      submodule_search_locations=[at])
        sys.modules[name] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules[name])
    return sys.modules[name]


# ------------------------------------------------------------------ cases
def _plan(name, **kw):
    return dict(dict(name=name, op="plan", ps=64, n_req=8, new_lo=1, new_hi=1, past_lo=0, past_hi=4096, chunk=0,
                     lens=1), **kw)


def _append(name, **kw):
    return dict(dict(name=name, op="append", n_head=32, n_kv=8, hd=128, ps=64, n_req=1, new_lo=1, new_hi=1,
                     past_lo=0, past_hi=4096, chunk=0, lens=1, f32=False, norm=True, mode="half", n_dims=128,
                     base=1e6, scaling=1.0), **kw)


def _attn(name, **kw):
    return dict(dict(name=name, op="attn", n_head=32, n_kv=8, hd=128, ps=64, n_req=1, new_lo=1, new_hi=1,
                     past_lo=0, past_hi=4096, chunk=0, lens=1, window=0), **kw)


def listed():
    return [
        # one decode step of eight sessions: a launch's latency, once per token
        _plan("plan_decode_8", n_req=8, past_lo=512, past_hi=8192),
        # a server's full step: a thousand sessions, most decoding, chunks of up to 40 tokens, small pages
        _plan("plan_1000_ragged", n_req=1000, ps=16, new_lo=0, new_hi=40, past_hi=8192, lens=2),
        # the layer step of one decoding session at the 4096-token context, norms and half layout (Qwen3-VL-4B heads)
        _append("append_decode_1", past_lo=4500, past_hi=4500),
        # 200 decoding sessions in fragmented 16-token pages, interleaved pairs on half of the head
        _append("append_decode_200_part", n_req=200, ps=16, past_lo=512, past_hi=32768, mode="pairs", n_dims=64,
                norm=False, base=1e4, lens=3),
        # a 512-token chunk of the 16/4-head, 256-wide layers, f32 projections, a quarter of the head rotated
        _append("append_chunk_512_hd256", n_head=16, n_kv=4, hd=256, new_lo=512, new_hi=512, past_lo=7680,
                past_hi=7680, f32=True, n_dims=64, base=1e7),
        # prompts of five sessions at once, positions scaled by 4 for a long context
        _append("append_prompt_8k_scaled", n_req=5, new_lo=1100, new_hi=2300, past_lo=0, past_hi=100000, ps=32,
                scaling=4.0, lens=4),
        # one decoding session at the splice benchmark's context
        _attn("attn_decode_4481", past_lo=4480, past_hi=4480),
        # one long session
        _attn("attn_decode_131072", past_lo=131071, past_hi=131071, ps=128),
        # 64 sessions of 512 to 32768 tokens: the multi-session decode batch
        _attn("attn_decode_64_ragged", n_req=64, past_lo=511, past_hi=32767, lens=5),
        # the splice tail: 384 new tokens over 4096 cached ones
        _attn("attn_tail_384", new_lo=384, new_hi=384, past_lo=4096, past_hi=4096),
        # a 512-token chunk of the 16/4-head, 256-wide layers behind a 4096-token window
        _attn("attn_chunk_512_hd256", n_head=16, n_kv=4, hd=256, new_lo=512, new_hi=512, past_lo=7680, past_hi=7680,
              window=4096, ps=32),
        # a mixed step: one 8192-token prompt part beside 31 decoding sessions
        _attn("attn_mixed_8192", n_req=32, past_lo=1, past_hi=16384, chunk=8192, lens=6, ps=16),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("plan", "append", "append", "attn", "attn", "attn"))
    c = {"op": op, "ps": rng.choice((16, 32, 64, 128)), "lens": rng.randrange(1 << 20), "chunk": 0}
    if op == "plan":
        n = _log(rng, 1, 1000)
        c.update(n_req=n, new_lo=0 if rng.random() < 0.5 else 1, new_hi=_log(rng, 1, max(2, 16000 // n)), past_lo=0,
                 past_hi=_log(rng, 16, 16384))
        return c
    hd = rng.choice((64, 128, 128, 256))
    nkv = rng.choice((1, 2, 4, 8)) if hd < 256 else rng.choice((1, 2, 4))
    c.update(hd=hd, n_kv=nkv, n_head=nkv * rng.choice((1, 2, 3, 4, 5, 8)))
    if op == "append":
        decode = rng.random() < 0.4
        n = _log(rng, 1, 256) if decode else rng.randint(1, 6)
        hi = 1 if decode else _log(rng, 2, 9000 // n)
        c.update(n_req=n, new_lo=1 if decode else max(1, hi // 2), new_hi=hi, past_lo=0, past_hi=_log(rng, 16, 100000),
                 f32=rng.random() < 0.3, norm=rng.random() < 0.5, mode=rng.choice(("half", "pairs")),
                 n_dims=rng.choice((hd, hd, hd // 2, hd // 4, 24)), base=rng.choice((1e4, 1e6)),
                 scaling=rng.choice((1.0, 1.0, 4.0, 8.0)))
        return c
    c.update(window=rng.choice((0, 0, 0, _log(rng, 16, 4096))))
    kind = rng.random()
    if kind < 0.5:     # decode: one token to a few, single sessions to large batches
        n = _log(rng, 1, 64)
        hi = rng.choice((1, 1, 1, 2, 4))
        c.update(n_req=n, new_lo=rng.choice((0, 1)) if n > 1 else 1, new_hi=hi, past_lo=0,
                 past_hi=_log(rng, 16, min(131072, 1200000 // n)))
    elif kind < 0.85:  # prompts and chunks
        n = rng.randint(1, 5)
        hi = _log(rng, 3, 8000 // n)
        c.update(n_req=n, new_lo=max(1, hi // 3), new_hi=hi, past_lo=0, past_hi=_log(rng, 16, 6000))
    else:              # a prompt part beside decoding sessions
        n = _log(rng, 2, 24)
        c.update(n_req=n, new_lo=1, new_hi=1, past_lo=1, past_hi=_log(rng, 64, 8192), chunk=_log(rng, 32, 4096))
    return c


def _lens(c):
    """(cached, new) token counts of each request: the case's own, not the seed's, so shapes stay."""
    r = random.Random(c["lens"])
    past = [r.randint(c["past_lo"], c["past_hi"]) for _ in range(c["n_req"])]
    new = [r.randint(c["new_lo"], c["new_hi"]) for _ in range(c["n_req"])]
    if c["chunk"]:
        new[c["n_req"] // 2] = c["chunk"]
    if not any(new):
        new[0] = 1
    return past, new


def _up(a, b):
    return -(-a // b)


def _visible(c):
    """(sum over queries of visible keys, keys that any query of their request sees)"""
    w, flops, keys = c["window"], 0, 0
    for p, n in zip(*_lens(c)):
        first = p + 1
        if w <= 0 or p + n <= w:
            flops += n * first + n * (n - 1) // 2
        else:
            flops += sum(min(first + i, w) for i in range(n))
        if n:
            keys += p + n if w <= 0 else min(p + n, w + n - 1)
    return flops, keys


def _rows_back(c):
    """Rows of every page that the step writes to, up to the request's end."""
    return sum(p + n - p // c["ps"] * c["ps"] for p, n in zip(*_lens(c)) if n)


def work(c):
    past, new = _lens(c)
    t, ps = sum(new), c["ps"]
    if c["op"] == "plan":
        held = [_up(p, ps) for p in past]
        fresh = sum(_up(p + n, ps) - h for p, n, h in zip(past, new, held))
        # the table comes back whole: each entry written or kept
        return {"bytes": 8.0 * len(past) + 8.0 * len(past) + 12.0 * t + 8.0 * fresh, "flops": 0}
    nh, nkv, hd = c["n_head"], c["n_kv"], c["hd"]
    if c["op"] == "append":
        es = 4 if c["f32"] else 2
        back = _rows_back(c)
        # projections in, queries out, codes out, rows of the touched pages out
        b = t * (nh + 2 * nkv) * hd * es + t * nh * hd * 2 + t * 2 * nkv * hd + back * 2 * nkv * hd * 2
        return {"bytes": float(b), "flops": float(t * (nh + nkv) * (3 * c["n_dims"] + (4 * hd if c["norm"] else 0)) + 3 * t * 2 * nkv * hd)}
    pairs, keys = _visible(c)
    return {"bytes": float(keys * nkv * hd * 2 + _up(keys, ps) * nkv * 8 + t * nh * hd * 4), "flops": 4.0 * nh * hd * pairs}


# ------------------------------------------------------------------ inputs
def _int(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _freqs(c):
    """Radians per position of each rotated pair, and the factor on cos and sin: base^(-2i/n), and where
    positions are scaled the blend of stretched and kept frequencies by how often a pair turns in the
    original context (Peng et al., YaRN, 2023)."""
    n, s = c["n_dims"], c["scaling"]
    i = np.arange(n // 2, dtype=np.float64)
    f = c["base"] ** (-2.0 * i / n)
    if s == 1.0:
        return f, 1.0
    dim = lambda turns: n * math.log(8192 / (turns * 2 * math.pi)) / (2 * math.log(c["base"]))  # noqa: E731
    low, high = max(0.0, math.floor(dim(32.0))), min(n - 1.0, math.ceil(dim(1.0)))
    keep = 1.0 - np.clip((i - low) / max(0.001, high - low), 0.0, 1.0)
    return f / s * (1.0 - keep) + f * keep, 1.0 + 0.1 * math.log(s)


def prepare(c, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    past, new = _lens(c)
    ps, n = c["ps"], len(past)
    held = [_up(p, ps) for p in past]
    want = [_up(p + k, ps) for p, k in zip(past, new)]
    n_pages = sum(want) + 7
    max_blocks = max(want) + 1
    perm = torch.randperm(n_pages, generator=g, device=DEV).to(torch.int32)   # pages lie anywhere in the pool
    host = perm.cpu().numpy()
    table = np.full((n, max_blocks), -1, dtype=np.int32)
    at = 0
    for r, h in enumerate(held):
        table[r, :h] = host[at:at + h]
        at += h
    free = host[at:].copy()
    if c["op"] == "plan":
        # another seed: other pages, and lengths within the pages held
        r = random.Random(seed)
        past = [p if p % ps == 0 else p - r.randrange(min(2, p % ps)) for p in past]
    s = {"case": c, "T": sum(new), "max_new": max(new), "n_past": _int(past), "n_new": _int(new),
         "table": torch.from_numpy(table).to(DEV), "free": torch.from_numpy(free).to(DEV), "n_free": _int([len(free)])}
    if own:
        sv = _package()
        nh, nkv, hd = c.get("n_head", 32), c.get("n_kv", 8), c.get("hd", 128)
        if c["op"] == "plan":
            s["step"] = sv.PagedStep(n, s["T"], s["max_new"], page_size=ps, n_pages=n_pages, n_head=nh, n_kv_head=nkv,
                                     head_dim=hd, device=0)
    if c["op"] == "plan":
        return s
    full, k = table.copy(), len(free)
    for r in range(n):
        for j in range(held[r], want[r]):
            k -= 1
            full[r, j] = free[k]
    nh, nkv, hd = c["n_head"], c["n_kv"], c["hd"]
    shape = (n_pages, nkv, ps, hd)
    codes, scales = [], []
    for _ in range(2):
        codes.append((torch.randn(shape, generator=g, device=DEV, dtype=torch.float16) * 32).round_().clamp_(-127, 127).to(torch.int8))
        scales.append(torch.exp(0.3 * torch.randn((n_pages, nkv), generator=g, device=DEV)) / 32)
    s.update(k=codes[0], v=codes[1], ks=scales[0], vs=scales[1])
    s["full"] = torch.from_numpy(full).to(DEV)
    if c["op"] == "append":
        dt = torch.float32 if c["f32"] else torch.float16
        # one projection's output: q, k and v heads side by side in each token's row; some k channels are large
        x = torch.randn((s["T"], nh + 2 * nkv, hd), generator=g, device=DEV)
        x[:, nh:nh + nkv] *= torch.exp(0.7 * torch.randn((nkv, hd), generator=g, device=DEV))
        s["qkv"] = x.to(dt)
        s["qn"] = 1 + 0.2 * torch.randn(hd, generator=g, device=DEV) if c["norm"] else None
        s["kn"] = 1 + 0.2 * torch.randn(hd, generator=g, device=DEV) if c["norm"] else None
        pages, first, tok_rank, tok_off, pos, back = [], [], [], [], [], []
        for r in range(n):
            if not new[r]:
                continue
            b0, e = past[r] // ps, past[r] + new[r]
            rank = len(pages)
            for b in range(b0, _up(e, ps)):
                pages.append(int(full[r, b]))
                first.append(max(0, past[r] - b * ps))
            p = np.arange(past[r], e)
            tok_rank.append(rank + p // ps - b0)
            tok_off.append(p % ps)
            pos.append(p)
            q = np.arange(b0 * ps, e)
            back.append(full[r, q // ps].astype(np.int64) * ps + q % ps)
        to = lambda v: torch.from_numpy(np.concatenate(v).astype(np.int64)).to(DEV)  # noqa: E731
        s.update(pages=torch.tensor(pages, device=DEV), first=torch.tensor(first, device=DEV), rank=to(tok_rank),
                 off=to(tok_off), pos=to(pos), back=to(back).to(torch.int32))
        f, s["mag"] = _freqs(c)
        s["freq"] = torch.from_numpy(f).to(DEV)
    else:
        s["q"] = torch.randn((s["T"], nh, hd), generator=g, device=DEV).to(torch.float16)
        few = max(1, 16 * c["n_kv"] // nh)          # requests of few tokens and of many are padded apart
        s["groups"] = []
        start = np.concatenate([[0], np.cumsum(new)])
        for rows in ([r for r in range(n) if 0 < new[r] <= few], [r for r in range(n) if new[r] > few]):
            if not rows:
                continue
            most, t = max(new[r] for r in rows), max(past[r] + new[r] for r in rows)
            tok = np.full((len(rows), most), -1, dtype=np.int64)
            for j, r in enumerate(rows):
                tok[j, :new[r]] = np.arange(start[r], start[r + 1])
            s["groups"].append((torch.from_numpy(tok).to(DEV), torch.from_numpy(full[rows][:, :_up(t, ps)]).long().clamp_(min=0).to(DEV),
                                torch.tensor([past[r] for r in rows], device=DEV)))
    if own:
        s["kv"] = sv.PagedKv(n_layer=1, n_kv_head=nkv, head_dim=hd, page_size=ps, n_pages=n_pages, device=0)
        for is_v, (a, b) in enumerate(((s["k"], s["ks"]), (s["v"], s["vs"]))):
            s["kv"].codes(0, is_v).copy_(a)
            s["kv"].scales(0, is_v).copy_(b)
        del s["k"], s["v"], s["ks"], s["vs"]
        s["step"] = sv.PagedStep(n, s["T"], s["max_new"], page_size=ps, n_pages=n_pages, n_head=nh, n_kv_head=nkv,
                                 head_dim=hd, device=0)
        s["step"].plan(s["n_past"], s["n_new"], s["table"], s["free"], s["n_free"])
        if c["op"] == "append":
            long = {} if c["scaling"] == 1.0 else dict(freq_scale=1 / c["scaling"], ext_factor=1.0, n_ctx_orig=8192)
            s["rope"] = sv.Rope(c["n_dims"], mode=sv.ROPE_NEOX if c["mode"] == "half" else sv.ROPE_NORM,
                                freq_base=c["base"], device=0, **long)
    return s


# ------------------------------------------------------------------ the plain forms
def _plain_plan(s):
    ps = s["case"]["ps"]
    past, new, table, free = s["n_past"], s["n_new"], s["table"], s["free"]
    blocks = torch.arange(table.shape[1], device=DEV, dtype=torch.int32)
    held, want = (past + ps - 1) // ps, ((past + new + ps - 1) // ps).clamp(max=table.shape[1])
    need = (want - held).clamp(min=0)
    before = torch.cumsum(need, 0) - need
    at = s["n_free"] - 1 - (before[:, None] + blocks[None] - held[:, None])
    fresh = (blocks[None] >= held[:, None]) & (blocks[None] < want[:, None])
    table = torch.where(fresh, torch.where(at >= 0, free[at.clamp(0, free.numel() - 1)], -1), table)
    ends = torch.cumsum(new, 0)
    t = torch.arange(s["T"], device=DEV)
    req = torch.searchsorted(ends, t, right=True)
    pos = past[req] + t - (ends - new)[req]
    slot = table[req, pos // ps] * ps + pos % ps
    i32 = torch.int32
    return {"q_start": torch.cat([torch.zeros_like(ends[:1]), ends]).to(i32), "kv_len": past + new, "tok_req": req.to(i32),
            "tok_pos": pos.to(i32), "tok_slot": slot.to(i32), "table": table,
            "n_free": (s["n_free"] - need.sum()).clamp(min=0).to(i32)}


def _norm(x, w):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w


def _turn(x, cos, sin, mode):
    n = 2 * cos.shape[-1]
    cos, sin = cos[:, None], sin[:, None]
    if mode == "half":
        a, b = x[..., :n // 2], x[..., n // 2:n]
        y = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    else:
        a, b = x[..., 0:n:2], x[..., 1:n:2]
        y = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    return torch.cat([y, x[..., n:]], -1)


def _quantise(s, x, codes, scales):
    """The touched pages with the new rows in: the page's scale never shrinks while it fills, and the rows
    that it holds are rounded to the new scale."""
    pages, first, ps = s["pages"], s["first"], s["case"]["ps"]
    rows = torch.zeros((pages.numel(), ps) + x.shape[1:], device=DEV)
    rows[s["rank"], s["off"]] = x
    is_new = torch.zeros((pages.numel(), ps), dtype=torch.bool, device=DEV)
    is_new[s["rank"], s["off"]] = True
    old = torch.where(first[:, None] > 0, scales[pages], 0.0)
    scale = torch.maximum(old, rows.abs().amax((1, 3)) / 127)
    inv = torch.where(scale > 0, 1 / scale, 0.0)
    fresh = (rows * inv[:, None, :, None]).round().clamp(-127, 127)
    kept = (codes[pages].float() * (old * inv)[:, :, None, None]).round().clamp(-127, 127).transpose(1, 2)
    kept = torch.where((scale > old)[:, None, :, None], kept, codes[pages].float().transpose(1, 2))
    out = torch.where(is_new[:, :, None, None], fresh, kept)
    codes[pages] = out.transpose(1, 2).to(torch.int8)
    scales[pages] = scale
    back = s["back"].long()
    page, off = back // ps, back % ps
    return (codes[page, :, off].float() * scales[page][:, :, None]).to(torch.float16)


def _plain_append(s):
    c = s["case"]
    nh, nkv = c["n_head"], c["n_kv"]
    x = s["qkv"].float()
    q, k, v = x[:, :nh], x[:, nh:nh + nkv], x[:, nh + nkv:]
    if c["norm"]:
        q, k = _norm(q, s["qn"]), _norm(k, s["kn"])
    # 24 bits do not hold a long context's angle: the angle alone is taken in 64 bits and brought to one turn
    angle = s["pos"].double()[:, None] * s["freq"][None]
    angle = (angle - 2 * math.pi * torch.round(angle / (2 * math.pi))).float()
    cos, sin = torch.cos(angle) * s["mag"], torch.sin(angle) * s["mag"]
    q, k = _turn(q, cos, sin, c["mode"]), _turn(k, cos, sin, c["mode"])
    return {"q": q.to(torch.float16), "k": _quantise(s, k, s["k"], s["ks"]), "v": _quantise(s, v, s["v"], s["vs"])}


def _plain_group(s, out, tok, table, past):
    """Padded attention of some requests: tok [R, M] token rows (-1: none), table [R, B] pages."""
    c = s["case"]
    nkv, hd, ps, g = c["n_kv"], c["hd"], c["ps"], c["n_head"] // c["n_kv"]
    n, m = tok.shape
    keys = table.shape[1] * ps
    q = s["q"][tok.clamp(min=0)].float().view(n, m, nkv, g, hd).permute(0, 2, 3, 1, 4).reshape(n, nkv, g * m, hd)
    k = (s["k"][table].float() * s["ks"][table][..., None, None]).permute(0, 2, 1, 3, 4).reshape(n, nkv, keys, hd)
    x = torch.matmul(q, k.transpose(2, 3)).view(n, nkv, g, m, keys) * (1 / math.sqrt(hd))
    del k
    at = past[:, None] + torch.arange(m, device=DEV)
    j = torch.arange(keys, device=DEV)
    seen = j[None, None] <= at[:, :, None]
    if c["window"]:
        seen &= j[None, None] > at[:, :, None] - c["window"]
    x = x.masked_fill_(~seen[:, None, None], -math.inf)
    x = x.sub_(x.amax(-1, keepdim=True)).exp_()
    x = x.div_(x.sum(-1, keepdim=True)).view(n, nkv, g * m, keys)
    v = (s["v"][table].float() * s["vs"][table][..., None, None]).permute(0, 2, 1, 3, 4).reshape(n, nkv, keys, hd)
    y = torch.matmul(x, v).view(n, nkv, g, m, hd).permute(0, 3, 1, 2, 4).reshape(n * m, nkv * g, hd)
    out.index_copy_(0, torch.where(tok < 0, s["T"], tok).view(-1), y.to(torch.float16))


def _plain_attn(s):
    c = s["case"]
    out = torch.zeros((s["T"] + 1, c["n_head"], c["hd"]), dtype=torch.float16, device=DEV)   # the last row takes the padding
    for group in s["groups"]:
        _plain_group(s, out, *group)
    return out[:-1]


def run(s):
    c = s["case"]
    if not own:
        return {"plan": _plain_plan, "append": _plain_append, "attn": _plain_attn}[c["op"]](s)
    if c["op"] == "plan":
        t = s["step"]
        t.plan(s["n_past"], s["n_new"], s["table"], s["free"], s["n_free"])
        return {"q_start": t.q_start, "kv_len": t.kv_len, "tok_req": t.tok_req, "tok_pos": t.tok_pos, "tok_slot": t.tok_slot,
                "table": s["table"], "n_free": t.n_free}
    if c["op"] == "append":
        nh, nkv, x = c["n_head"], c["n_kv"], s["qkv"]
        q = s["kv"].rope_append(0, s["step"], x[:, :nh], x[:, nh:nh + nkv], x[:, nh + nkv:], rope=s["rope"], q_norm=s["qn"],
                                k_norm=s["kn"], eps=EPS)
        k, v = s["kv"].read(0, s["back"])
        return {"q": q, "k": k, "v": v}
    return s["kv"].attn(0, s["step"], s["q"], scale=1 / math.sqrt(c["hd"]), window=c["window"])


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(c, seed):
    global own
    if c["op"] == "plan":
        return None
    kept, own = own, False
    try:
        s = prepare(c, seed)
    finally:
        own = kept
    past, new = _lens(c)
    ps, full = c["ps"], s["full"].cpu().numpy()
    nh, nkv, hd = c["n_head"], c["n_kv"], c["hd"]
    if c["op"] == "append":
        freq, mag = _freqs(c)
        x = s["qkv"].cpu().numpy().astype(np.float64)
        q, k, v = x[:, :nh], x[:, nh:nh + nkv], x[:, nh + nkv:]
        if c["norm"]:
            q = q / np.sqrt(np.square(q).mean(-1, keepdims=True) + EPS) * s["qn"].cpu().numpy().astype(np.float64)
            k = k / np.sqrt(np.square(k).mean(-1, keepdims=True) + EPS) * s["kn"].cpu().numpy().astype(np.float64)
        pos = np.concatenate([np.arange(p, p + n) for p, n in zip(past, new)]).astype(np.float64)
        z = np.exp(1j * pos[:, None] * freq[None]) * mag     # a pair turns as a complex number
        h = c["n_dims"] // 2
        first, second = (slice(0, h), slice(h, 2 * h)) if c["mode"] == "half" else (slice(0, 2 * h, 2), slice(1, 2 * h, 2))
        turned = []
        for y in (q, k):
            w = (y[..., first] + 1j * y[..., second]) * z[:, None]
            y = y.copy()
            y[..., first], y[..., second] = w.real, w.imag
            turned.append(y)
        outs = [torch.from_numpy(turned[0])]
        for x, codes, scales in ((turned[1], s["k"], s["ks"]), (v, s["v"], s["vs"])):
            codes, scales = codes.cpu().numpy(), scales.cpu().numpy().astype(np.float64)
            rows, t = [], 0
            for r in range(len(past)):
                p, e = past[r], past[r] + new[r]
                while p < e:
                    page, o = full[r, p // ps], p % ps
                    n = min(e - p, ps - o)
                    part = x[t:t + n]
                    was = scales[page] if o else np.zeros(nkv)
                    scale = np.maximum(was, np.abs(part).max((0, 2)) / 127)
                    by = np.where(scale > 0, scale, 1.0)[None, :, None]
                    old = codes[page][:, :o].transpose(1, 0, 2).astype(np.float64)
                    if o:
                        moved = np.clip(np.rint(old * was[None, :, None] / by), -127, 127)
                        rows.append(np.where((scale > was)[None, :, None], moved, old) * scale[None, :, None])
                    rows.append(np.clip(np.rint(part / by), -127, 127) * scale[None, :, None])
                    p, t = p + n, t + n
            outs.append(torch.from_numpy(np.concatenate(rows)))
        return {"q": outs[0], "k": outs[1], "v": outs[2]}
    if _visible(c)[0] * nh * hd > 4e12:
        return None
    out = torch.zeros((s["T"], nh, hd), dtype=torch.float64, device=DEV)
    t = 0
    for r in range(len(past)):
        if not new[r]:
            continue
        e = past[r] + new[r]
        b = s["full"][r, :_up(e, ps)].long()
        for h in range(nkv):
            k = (s["k"][b, h].double() * s["ks"][b, h].double()[:, None, None]).view(-1, hd)[:e]
            v = (s["v"][b, h].double() * s["vs"][b, h].double()[:, None, None]).view(-1, hd)[:e]
            for i in range(0, new[r], 1024):
                m = min(1024, new[r] - i)
                q = s["q"][t + i:t + i + m, h * (nh // nkv):(h + 1) * (nh // nkv)].double()
                x = torch.einsum("mgd,sd->mgs", q, k) / math.sqrt(hd)
                d = (past[r] + i + torch.arange(m, device=DEV))[:, None] - torch.arange(e, device=DEV)[None]
                dead = (d < 0) | (d >= c["window"]) if c["window"] else d < 0
                x = torch.softmax(x.masked_fill(dead[:, None], -math.inf), -1)
                out[t + i:t + i + m, h * (nh // nkv):(h + 1) * (nh // nkv)] = torch.einsum("mgs,sd->mgd", x, v)
        t += new[r]
    return out
