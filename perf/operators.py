"""Measured operators of a serving step over a paged 4-bit key/value cache.

  norm    add_rmsnorm_q8_K: residual addition, RMS norm and Q8_K quantization
          in one pass, in front of the quantized projections
  append  paged_q4_append: QK norm and rotation of the new rows, keys and values
          stored as 4-bit blocks in their pages (and read back as the values
          that they stand for)
  gather  paged_q4_gather: rows of the cache as linear fp16
  gqa     paged_q4_gqa: attention over the cache: single tokens, a few rows per
          sequence (verify), prompts

Where `own` is false the operators are computed in elementary torch operations.
Head shapes, contexts and batch sizes are those of bench.py and the tests:
16q/8kv and 32q/8kv of head_dim 64, 16q/4kv of head_dim 128 with the output
gate, sliding windows of 256, rows of 2048 values.

The cache: a page holds `page` positions as [kv head][block of 32 positions].
A block of head_dim D is 36 D bytes: 4-bit codes of the keys (16 D), of the
values (16 D), fp16 scales of the keys (2 D) and of the values (2 D), one per
position and 32 dims.  A code c under scale d stands for d * (c - 8).
"""
import math

import numpy as np
import torch

own = False

EPS = 1e-5
BLOCK = 32
D64_SMALL, D64, D128 = dict(nq=16, nkv=8, hd=64), dict(nq=32, nkv=8, hd=64), dict(nq=16, nkv=4, hd=128)


def listed():
    return [
        # the hidden state of one user's next token
        dict(name="norm_n1_2048", kind="norm", rows=1, cols=2048),
        # the rows of several prompts
        dict(name="norm_n6007_2304", kind="norm", rows=6007, cols=2304),
        # one decode step of 64 users
        dict(name="append_b64_32q8kv_ctx8192", kind="append", n_seq=64, rows=1, pos=8191, ragged=True, page=64, **D64),
        # two prompts behind a cached prefix
        dict(name="append_b2_n3001_d128_pos517", kind="append", n_seq=2, rows=3001, pos=517, ragged=False, page=64,
             **D128),
        # one sequence handed to an engine with a linear cache
        dict(name="gather_b1_n1000_16q8kv", kind="gather", n_seq=1, rows=1000, pos=0, ragged=False, page=32,
             **D64_SMALL),
        # a batch of sequences handed over
        dict(name="gather_b32_n4100_d128_ragged", kind="gather", n_seq=32, rows=4100, pos=0, ragged=True, page=128,
             **D128),
        # one user, a short context: latency
        dict(name="gqa_b1_16q8kv_ctx1024", kind="gqa", n_seq=1, rows=1, pos=1023, ragged=False, window=0, gate=False,
             page=64, **D64_SMALL),
        # one user, a very long context
        dict(name="gqa_b1_32q8kv_ctx131072", kind="gqa", n_seq=1, rows=1, pos=131071, ragged=False, window=0,
             gate=False, page=256, **D64),
        # a serving batch of users at different lengths
        dict(name="gqa_b64_32q8kv_ctx8192_ragged", kind="gqa", n_seq=64, rows=1, pos=8191, ragged=True, window=0,
             gate=False, page=64, **D64),
        # long contexts, wide heads, output gate
        dict(name="gqa_b32_d128_ctx32768_gate", kind="gqa", n_seq=32, rows=1, pos=32767, ragged=False, window=0,
             gate=True, page=128, **D128),
        # speculative verify: 8 rows per user
        dict(name="gqa_b16_rows8_32q8kv_ctx4096", kind="gqa", n_seq=16, rows=8, pos=4096, ragged=False, window=0,
             gate=False, page=64, **D64),
        # prompts of different lengths behind a cached prefix
        dict(name="gqa_b4_n1999_32q8kv_pos1023_ragged", kind="gqa", n_seq=4, rows=1999, pos=1023, ragged=True,
             window=0, gate=False, page=64, **D64),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "append", "gather", "gqa", "gqa", "gqa"])
    if kind == "norm":
        return dict(kind=kind, rows=_log(rng, 1, 6007), cols=rng.choice([256, 1024, 1536, 2048, 2304, 4096, 8192]))
    shape = rng.choice([D64_SMALL, D64, D64, D128, D128])
    page = rng.choice([32, 64, 64, 128, 256])
    if kind != "gqa":
        if rng.random() < 0.5:
            n_seq, rows = _log(rng, 1, 128), rng.choice([1, 1, 2, 5, 8])
        else:
            n_seq, rows = rng.randint(1, 4), _log(rng, 16, 3001)
        return dict(kind=kind, n_seq=n_seq, rows=rows, pos=_log(rng, 1, 8192), ragged=rng.random() < 0.6, page=page,
                    **shape)
    form = rng.choice(["one", "one", "few", "prompt"])
    window = rng.choice([0, 256]) if shape is D128 else 0
    if form == "prompt":
        n_seq, rows, pos = rng.randint(1, 4), _log(rng, 16, 1999), _log(rng, 1, 1023)
    else:
        n_seq, rows = _log(rng, 1, 64), 1 if form == "one" else rng.randint(2, 8)
        pos = _log(rng, 1, min(131071, 524288 // n_seq)) if form == "one" else _log(rng, 1, 8192)
    return dict(kind=kind, n_seq=n_seq, rows=rows, pos=pos, ragged=rng.random() < 0.6, window=window,
                gate=shape is D128, page=page, **shape)


# ---- inputs ------------------------------------------------------------------------

def _lengths(case, seed):
    """Per sequence: positions before this call's rows, and its rows.  Ragged:
    uniform from a sixteenth of the longest, which one sequence has.  The seed
    orders them; the work is the case's."""
    n, pos, rows = case["n_seq"], case["pos"], case["rows"]
    if not case["ragged"]:
        return np.full(n, pos, np.int64), np.full(n, rows, np.int64)
    r = np.random.default_rng(n * 65537 + pos * 31 + rows)
    p = r.integers(pos // 16, pos + 1, size=n)
    c = r.integers(max(1, rows // 16), rows + 1, size=n)
    p[0], c[0] = pos, rows
    o = np.random.default_rng(seed).permutation(n)
    return p[o], c[o]


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _cache_rows(g, n, nkv, hd):
    """Keys as after their norm and rotation, with the few strong dims that trained
    models have, and values with a spread of magnitudes per head."""
    k, v = _randn(g, n, nkv, hd), _randn(g, n, nkv, hd)
    k *= 0.5 + 2.0 * torch.rand((nkv, hd), generator=g, device="cuda") ** 4
    v *= 0.1 + torch.rand((nkv, 1), generator=g, device="cuda")
    return k, v


def _pages(g, case, n_pages):
    """Pages filled with cache rows."""
    nkv, hd, page = case["nkv"], case["hd"], case["page"]
    out = torch.empty((n_pages, nkv, page // BLOCK, 36 * hd), device="cuda", dtype=torch.uint8)
    step = max(1, (1 << 25) // (page * nkv * hd))
    for a in range(0, n_pages, step):
        n = min(step, n_pages - a)
        rows = _cache_rows(g, n * page, nkv, hd)
        codes = [_quantize(t) for t in rows]
        blk = [t.reshape(n, page // BLOCK, BLOCK, nkv, -1).permute(0, 3, 1, 2, 4).reshape(-1, BLOCK, t[0, 0].numel())
               for c in codes for t in c]
        out[a:a + n] = _pack(*blk, hd).reshape(n, nkv, page // BLOCK, 36 * hd)
    return out


def _rope(hd, rows):
    f = 1e6 ** (-torch.arange(0, hd, 2, device="cuda", dtype=torch.float64) / hd)
    a = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] * f
    return torch.cos(a).float(), torch.sin(a).float()


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    st = dict(case=dict(case), stream=torch.cuda.current_stream().cuda_stream)
    if case["kind"] == "norm":
        n, cols = case["rows"], case["cols"]
        st["x"], st["res"] = _randn(g, n, cols), 2.0 * _randn(g, n, cols)
        st["w"] = 1.0 + 0.1 * _randn(g, cols)
        st["res_out"] = torch.zeros((n, cols), device="cuda")
        st["xq"] = torch.zeros((n, cols // 256, 292), device="cuda", dtype=torch.uint8)
        return st
    n, rows, nq, nkv, hd, page = (case[k] for k in ("n_seq", "rows", "nq", "nkv", "hd", "page"))
    before, count = _lengths(case, seed)
    used = -(-(before + count) // page)
    stride = int(used.max())
    n_pages = int(used.sum()) + 2
    # pages in any order, -1 behind a sequence's last
    order = np.random.default_rng(seed).permutation(n_pages)[:int(used.sum())]
    table = np.full((n, stride), -1, np.int32)
    table[np.arange(stride)[None] < used[:, None]] = order
    st["pages"], st["n_pages"], st["stride"] = _pages(g, case, n_pages), n_pages, stride
    st["table"] = torch.from_numpy(table).cuda()
    st["pos"] = torch.from_numpy(before.astype(np.int32)).cuda()
    st["count"] = torch.from_numpy(count.astype(np.int32)).cuda()
    st["hint"] = int((before + count).max())
    if case["kind"] != "gqa":
        st["k_out"], st["v_out"] = (torch.zeros((n, rows, nkv, hd), device="cuda", dtype=torch.float16)
                                    for _ in range(2))
        if case["kind"] == "gather":
            return st
        st["k"], st["v"] = _cache_rows(g, n * rows, nkv, hd)
        st["kw"], st["qw"] = (1.0 + 0.1 * _randn(g, hd) for _ in range(2))
        st["cos"], st["sin"] = _rope(hd, st["hint"])
    st["q"] = _randn(g, n, rows, nq, hd)
    st["out"] = torch.zeros((n, rows, nq, hd), device="cuda")
    if case["kind"] == "gqa":
        st["gate"] = _randn(g, n, rows, nq) if case["gate"] else None
    return st


# ---- plain form: blocks of the cache ---------------------------------------------------

def _quantize(x):
    """Codes 0..15 and fp16 scales of groups of 32 dims.  The scale puts the value
    of largest magnitude (the positive one of two) at code 0: d = -m / 8."""
    g = x.reshape(*x.shape[:-1], -1, 32)
    top, low = g.amax(-1), g.amin(-1)
    d = (torch.where(top >= -low, top, low) / -8.0).half()
    f = d.float()[..., None]
    c = torch.where(f == 0, torch.full_like(g, 8.0), torch.floor(g / f + 8.5).clamp(0, 15))
    return c.to(torch.uint8).reshape(x.shape), d


def _words(e):
    """Eight codes e = 0..7 in the last axis as the 4 bytes of a word: code e is nibble e / 2 + 4 (e % 2)."""
    n = e.reshape(*e.shape[:-1], 4, 2).transpose(-1, -2).reshape(*e.shape[:-1], 4, 2)
    return n[..., 0] | (n[..., 1] << 4)


def _codes(b):
    n = torch.stack([b & 15, b >> 4], -1).reshape(*b.shape[:-1], 2, 4)
    return n.transpose(-1, -2).reshape(*b.shape[:-1], 8)


def _pack(kc, kd, vc, vd, hd):
    """Blocks [n, 36 hd] of codes [n, 32, hd] and scales [n, 32, hd / 32]."""
    n, g = kc.shape[0], hd // 32
    k = _words(kc.reshape(n, 2, 16, g, 4, 8))                                   # half, key, group, part, byte
    k = k.permute(0, 4, 2, 1, 3, 5) if hd == 64 else k.permute(0, 1, 4, 2, 3, 5)
    v = vc.reshape(n, 2, 4, 4, hd // 64, 4, 16).permute(0, 4, 2, 6, 5, 1, 3)      # .., token half, token
    v = _words(v.reshape(n, hd // 64, 4, 16, 4, 8))
    s = [d.reshape(n, 2, 4, 4, g).permute(0, 4, 2, 1, 3).contiguous().view(torch.uint8).reshape(n, -1)
         for d in (kd, vd)]
    return torch.cat([k.reshape(n, -1), v.reshape(n, -1)] + s, 1)


def _unpack(blk, hd):
    """Keys and values [n, 32, hd] that blocks stand for, fp32."""
    n, g = blk.shape[0], hd // 32
    k = _codes(blk[:, :16 * hd].reshape(n, *((4, 16, 2, 2, 4) if hd == 64 else (2, 4, 16, 4, 4))))
    k = k.permute(0, 3, 2, 4, 1, 5) if hd == 64 else k.permute(0, 1, 3, 4, 2, 5)
    v = _codes(blk[:, 16 * hd:32 * hd].reshape(n, hd // 64, 4, 16, 4, 4)).reshape(n, hd // 64, 4, 16, 4, 2, 4)
    v = v.permute(0, 5, 2, 6, 1, 4, 3)
    out = []
    for c, s in ((k, blk[:, 32 * hd:34 * hd]), (v, blk[:, 34 * hd:])):
        d = s.contiguous().view(torch.float16).reshape(n, g, 4, 2, 4).permute(0, 3, 2, 4, 1).reshape(n, 32, g, 1)
        out.append(((c.reshape(n, 32, g, 32).float() - 8.0) * d.float()).reshape(n, 32, hd))
    return out


def _rows(st):
    """Keys and values of every position of the sequences' tables [n_seq, positions, nkv, hd], fp32."""
    c = st["case"]
    nkv, hd, page = c["nkv"], c["hd"], c["page"]
    t = st["table"].clamp(min=0).long()
    blk = st["pages"][t].reshape(-1, 36 * hd)
    return [x.reshape(t.shape[0], t.shape[1], nkv, page, hd).permute(0, 1, 3, 2, 4).reshape(t.shape[0], -1, nkv, hd)
            for x in _unpack(blk, hd)]


# ---- plain form: operators ---------------------------------------------------------------

def _plain_norm(st):
    h = st["x"] + st["res"]
    r = 1.0 / torch.sqrt((h.double() * h.double()).mean(-1, keepdim=True) + float(np.float32(EPS)))
    y = (h.double() * r * st["w"].double()).float().reshape(h.shape[0], -1, 256)
    top = y.abs().amax(-1, keepdim=True)
    safe = torch.where(top > 0, top, torch.ones_like(top))
    most = torch.full_like(top, 127.0)  # a tensor: division by a number multiplies by its rounded reciprocal
    q = torch.round(y * (most / safe)).clamp(-128, 127)
    return [h, (q * (top / most)).reshape(h.shape[0], -1, 256)]


def _plain_norm_rope(x, w, cos, sin):
    x = x.double()
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + float(np.float32(EPS))) * w.double()
    lo, hi = x.chunk(2, -1)
    c, s = cos.double(), sin.double()
    return torch.cat([lo * c - hi * s, hi * c + lo * s], -1).float()


def _plain_append(st):
    c = st["case"]
    n, rows, nkv, hd = (c[k] for k in ("n_seq", "rows", "nkv", "hd"))
    r = torch.arange(rows, device="cuda")
    live = (r[None] < st["count"][:, None])[..., None, None]
    at = (st["pos"][:, None].long() + r[None]).clamp(max=st["hint"] - 1)
    cos, sin = st["cos"][at][:, :, None], st["sin"][at][:, :, None]
    q = _plain_norm_rope(st["q"], st["qw"], cos, sin)
    k = _plain_norm_rope(st["k"].reshape(n, rows, nkv, hd), st["kw"], cos, sin)
    kept = []
    for x in (k, st["v"].reshape(n, rows, nkv, hd)):
        code, d = _quantize(x)
        x = (code.float().reshape(*d.shape, 32) - 8.0) * d.float()[..., None]
        kept.append(x.reshape(n, rows, nkv, hd).half())
    zero = torch.zeros((), device="cuda")
    return [torch.where(live, q, zero)] + [torch.where(live, x, zero.half()) for x in kept]


def _plain_gather(st):
    c = st["case"]
    r = torch.arange(c["rows"], device="cuda")
    live = (r[None] < st["count"][:, None])[..., None, None]
    at = (st["pos"][:, None].long() + r[None]).clamp(max=st["stride"] * c["page"] - 1)
    s = torch.arange(c["n_seq"], device="cuda")[:, None]
    zero = torch.zeros((), device="cuda", dtype=torch.float16)
    return [torch.where(live, x[s, at].half(), zero) for x in _rows(st)]


def _plain_gqa(st):
    c = st["case"]
    n, rows, nq, nkv, hd, win = (c[k] for k in ("n_seq", "rows", "nq", "nkv", "hd", "window"))
    mul = nq // nkv
    k, v = (x.permute(0, 2, 1, 3).contiguous() for x in _rows(st))
    t = torch.arange(k.shape[2], device="cuda")
    r = torch.arange(rows, device="cuda")
    p = st["pos"][:, None].long() + r[None]
    live = r[None] < st["count"][:, None]
    see = (t <= p[..., None]) & live[..., None]
    if win:
        see = see & (t > p[..., None] - win)
    see = see.repeat_interleave(mul, 1)[:, None]
    q = st["q"].reshape(n, rows, nkv, mul, hd).permute(0, 2, 1, 3, 4).reshape(n, nkv, rows * mul, hd)
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()) * (1.0 / math.sqrt(hd))
    s = s.masked_fill(~see, -math.inf)
    m = s.amax(-1, keepdim=True)
    s = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
    o = torch.matmul(s, v) / s.sum(-1, keepdim=True).clamp(min=1e-30)
    o = o.reshape(n, nkv, rows, mul, hd).permute(0, 2, 1, 3, 4).reshape(n, rows, nq, hd)
    if st["gate"] is not None:
        o = o * (1.0 / (1.0 + torch.exp(-st["gate"])))[..., None]
    return o


# ---- one pass ----------------------------------------------------------------------

def _a(t):
    return None if t is None else t.data_ptr()


def _own(st):
    import laii_amd as la
    c, s = st["case"], st["stream"]
    if c["kind"] == "norm":
        la.add_rmsnorm_q8_K(_a(st["x"]), _a(st["res"]), _a(st["w"]), EPS, _a(st["res_out"]), None, _a(st["xq"]),
                            c["rows"], c["cols"], s)
        # the 8-bit blocks as the values that they stand for
        d = st["xq"].view(torch.float32)[..., :1]
        return [st["res_out"], st["xq"][..., 4:260].view(torch.int8) * d]
    n, rows, nq, nkv, hd = (c[k] for k in ("n_seq", "rows", "nq", "nkv", "hd"))
    cache = (_a(st["pages"]), st["n_pages"], c["page"], _a(st["table"]), st["stride"])
    if c["kind"] == "append":
        la.paged_q4_append(_a(st["q"]), _a(st["k"]), _a(st["v"]), _a(st["out"]), *cache, _a(st["pos"]),
                           _a(st["count"]), n, rows, nq, nkv, hd, _a(st["qw"]), _a(st["kw"]), EPS, _a(st["cos"]),
                           _a(st["sin"]), st["hint"], s)
    if c["kind"] != "gqa":
        la.paged_q4_gather(_a(st["k_out"]), _a(st["v_out"]), *cache, _a(st["pos"]), _a(st["count"]), n, rows, nkv, hd,
                           s)
        return ([st["out"]] if c["kind"] == "append" else []) + [st["k_out"], st["v_out"]]
    if "scratch" not in st:  # a user's program keeps it beside its cache
        b = la.paged_q4_workspace_bytes(n, rows, st["hint"], nq, nkv, hd, c["page"], st["stride"], c["window"])
        st["scratch"] = torch.empty(b, device="cuda", dtype=torch.uint8)
    la.paged_q4_gqa(_a(st["q"]), _a(st["gate"]), True, *cache, _a(st["pos"]), _a(st["count"]), _a(st["out"]), n, rows,
                    st["hint"], nq, nkv, hd, _a(st["scratch"]), st["scratch"].numel(), c["window"], None, s)
    return st["out"]


def run(st):
    if own:
        return _own(st)
    return {"norm": _plain_norm, "append": _plain_append, "gather": _plain_gather,
            "gqa": _plain_gqa}[st["case"]["kind"]](st)


# ---- what a pass cannot do without ---------------------------------------------------

def work(case):
    if case["kind"] == "norm":
        n = case["rows"] * case["cols"]
        return dict(bytes=12 * n + n // 256 * 292 + 4 * case["cols"], flops=8 * n)
    nq, nkv, hd = case["nq"], case["nkv"], case["hd"]
    before, count = _lengths(case, 0)
    rows, row4 = int(count.sum()), nkv * hd * 9 // 8  # bytes of a position's keys and values: 4.5 bits each
    if case["kind"] == "append":
        new = rows * (nq * hd * 8 + nkv * hd * 8 + row4)
        return dict(bytes=new + rows * hd * 4 + rows * nkv * hd * 4, flops=rows * (nq + 2 * nkv) * hd * 8)
    if case["kind"] == "gather":
        return dict(bytes=rows * (row4 + nkv * hd * 4), flops=rows * nkv * hd * 4)
    win, keys, union = case["window"], 0, 0
    for p, c in zip(before.tolist(), count.tolist()):
        seen = np.arange(p + 1, p + c + 1)
        keys += int((np.minimum(seen, win) if win else seen).sum())
        union += min(p + c, win + c - 1) if win else p + c
    return dict(bytes=union * row4 + rows * nq * hd * 8, flops=4 * hd * nq * keys)


# ---- the same in 64 bits ---------------------------------------------------------------

def _place(hd):
    """Of key and value (position t, dim x) of a block: byte, shift of the code, byte of the scale."""
    t, x = np.arange(32)[:, None], np.arange(hd)[None]
    half, key, part, e = t // 16, t % 16, x % 32 // 8, x % 8
    lane = part * 16 + key
    word = lane * 4 + half * 2 + x // 32 if hd == 64 else half * 256 + lane * 4 + x // 32
    nib = e // 2 + 4 * (e % 2)
    k = 4 * word + nib // 2, 4 * (nib % 2) + 0 * word
    kg, e = t % 16 // 4, t % 4 + 4 * (t // 16)
    word = x // 64 * 256 + (kg * 16 + x % 16) * 4 + x % 64 // 16
    nib = e // 2 + 4 * (e % 2)
    v = 16 * hd + 4 * word + nib // 2, 4 * (nib % 2) + 0 * word
    scale = 32 * hd + x // 32 * 64 + kg * 16 + e * 2
    return [[torch.from_numpy(np.ascontiguousarray(a)).cuda() for a in (*p, scale + 2 * hd * i)]
            for i, p in enumerate((k, v))]


def _sequence64(st, s, length):
    """Keys and values of positions 0 .. length - 1 of a sequence, [length, nkv, hd]."""
    c = st["case"]
    hd, page = c["hd"], c["page"]
    ids = st["table"][s, :-(-length // page)].long()
    blk = st["pages"][ids]                                    # page, head, block, byte
    out = []
    for byte, shift, scale in _place(hd):
        code = (blk[..., byte] >> shift.to(torch.uint8)) & 15
        d = torch.stack([blk[..., scale], blk[..., scale + 1]], -1).view(torch.float16)[..., 0].double()
        x = d * (code.double() - 8.0)                         # page, head, block, position, dim
        out.append(x.permute(0, 2, 3, 1, 4).reshape(-1, c["nkv"], hd)[:length])
    return out


def _norm_rope64(x, w, cos, sin):
    x = x.double()
    x = x * torch.rsqrt(x.square().sum(-1, keepdim=True) / x.shape[-1] + float(np.float32(EPS))) * w.double()
    h = x.shape[-1] // 2
    z = torch.complex(x[..., :h], x[..., h:]) * torch.complex(cos.double(), sin.double())
    return torch.cat([z.real, z.imag], -1)


def _kept64(x):
    """The values that 4-bit groups of 32 hold."""
    g = x.reshape(-1, 32)
    i = torch.where(g.max(-1).values >= g.min(-1).values.abs(), g.max(-1).values, g.min(-1).values)
    d = (-i / 8.0).float().half().double()[:, None]
    c = torch.floor(g / torch.where(d == 0, torch.ones_like(d), d) + 8.5).clamp(0, 15)
    return (d * (c - 8.0)).reshape(x.shape)


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "norm":
        # the residual stream and the norm's result are fp32 by definition, and the
        # blocks' step and its reciprocal too: each is rounded here once, from 64 bits
        h = (st["x"].double() + st["res"].double()).float().double()
        y = h * torch.rsqrt(h.square().sum(-1, keepdim=True) / h.shape[-1] + float(np.float32(EPS)))
        y = (y * st["w"].double()).float().double().reshape(h.shape[0], -1, 256)
        top = y.abs().amax(-1, keepdim=True)
        safe = torch.where(top == 0, torch.ones_like(top), top)
        step, per = (top / 127.0).float().double(), (127.0 / safe).float().double()
        return [h, torch.round((y * per).float().double()) * step]
    n, rows, nq, nkv, hd = (case[k] for k in ("n_seq", "rows", "nq", "nkv", "hd"))
    before, count = _lengths(case, seed)
    outs = [torch.zeros((n, rows, h, hd), device="cuda", dtype=torch.float64) for h in (nq, nkv, nkv)]
    for s in range(n):
        p, c = int(before[s]), int(count[s])
        if case["kind"] == "append":
            cos, sin = st["cos"][p:p + c, None], st["sin"][p:p + c, None]
            outs[0][s, :c] = _norm_rope64(st["q"][s, :c], st["qw"], cos, sin)
            outs[1][s, :c] = _kept64(_norm_rope64(st["k"].reshape(n, rows, nkv, hd)[s, :c], st["kw"], cos, sin))
            outs[2][s, :c] = _kept64(st["v"].reshape(n, rows, nkv, hd)[s, :c].double())
            continue
        k, v = _sequence64(st, s, p + c)
        if case["kind"] == "gather":
            outs[1][s, :c], outs[2][s, :c] = k[p:], v[p:]
            continue
        t, at = torch.arange(p + c, device="cuda"), torch.arange(p, p + c, device="cuda")[:, None]
        hide = (t[None] > at) | ((t[None] <= at - case["window"]) if case["window"] else False)
        for h in range(nq):
            j = h // (nq // nkv)
            a = st["q"][s, :c, h].double() @ k[:, j].t().contiguous() / math.sqrt(hd)
            a = torch.softmax(a.masked_fill(hide, -math.inf), -1)
            outs[0][s, :c, h] = a @ v[:, j].contiguous()
        if st["gate"] is not None:
            outs[0][s] *= torch.sigmoid(st["gate"][s].double())[..., None]
    return {"append": outs, "gather": outs[1:], "gqa": outs[0]}[case["kind"]]
