"""The paged 4-bit cache and the operators around it in numpy, 64 bits, from
their definitions (include/lfm_attn.h)."""
from __future__ import annotations

import numpy as np

BLOCK = 32


def place(hd):
    """Of (position t < 32, dim x): byte of the K word, of the V word, of the K
    scale, of the V scale, and the shifts of the K and V codes in their words."""
    t, x = np.arange(32)[:, None], np.arange(hd)[None]
    g, r = x // 32, x % 32 // 8
    k = 16 * (16 * r + t % 16) + 4 * g + (8 if hd == 64 else 1024) * (t // 16)
    j = t % 16 // 4
    v = 16 * hd + 1024 * (x // 64) + 16 * (16 * j + x % 16) + 4 * (x // 16 % 4)
    e = t % 4 + 4 * (t // 16)
    ks = 32 * hd + 64 * g + 16 * j + 2 * e
    nib = lambda e: 4 * (e // 2 + 4 * (e % 2))  # noqa: E731
    return k, v, ks, ks + 2 * hd, nib(x % 8) + 0 * t, nib(e) + 0 * x


def quantize(x):
    """Codes and fp16 scale bits of groups of 32, with the definition's fp32 steps."""
    g = np.asarray(x, np.float32).reshape(-1, 32)
    top, low = g.max(-1), g.min(-1)
    d = (np.where(top >= -low, top, low) / np.float32(-8)).astype(np.float16)
    d[d == 0] = 0  # no sign on a zero scale
    f = d.astype(np.float32)[:, None]
    with np.errstate(divide="ignore", invalid="ignore"):
        c = np.clip(np.floor(g / f + np.float32(8.5)), 0, 15)
    c = np.where(f == 0, 8, c).astype(np.uint8)
    return c.reshape(x.shape), d.reshape(*x.shape[:-1], x.shape[-1] // 32)


def norm_rope(x, w, eps, cos, sin):
    """fp64 norm (w None: none) and rotation; cos, sin broadcast against [..., hd / 2]."""
    x = np.asarray(x, np.float64)
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + float(np.float32(eps))) * np.asarray(w, np.float64)
    h = x.shape[-1] // 2
    lo, hi = x[..., :h], x[..., h:]
    c, s = np.asarray(cos, np.float64), np.asarray(sin, np.float64)
    return np.concatenate([lo * c - hi * s, hi * c + lo * s], -1)


class Cache:
    """Pages and tables of a layer on the host."""

    def __init__(self, rng, lengths, page, nkv, hd, spare=2, fill=None):
        self.page, self.nkv, self.hd = page, nkv, hd
        used = [-(-int(n) // page) for n in lengths]
        self.stride = max(max(used), 1)
        self.n_pages = sum(used) + spare
        order = rng.permutation(self.n_pages)[:sum(used)]
        self.table = np.full((len(used), self.stride), -1, np.int32)
        at = 0
        for s, u in enumerate(used):
            self.table[s, :u] = order[at:at + u]
            at += u
        shape = (self.n_pages, nkv, page // BLOCK, 36 * hd)
        self.pages = rng.integers(0, 256, shape, dtype=np.uint8) if fill is None else np.full(shape, fill, np.uint8)
        self._place = place(hd)

    def _block(self, s, pos):
        page = int(self.table[s, pos // self.page])
        return None if not 0 <= page < self.n_pages else (page, pos % self.page // BLOCK)

    def store(self, s, pos, k, v):
        """Rows k, v [n, nkv, hd] (fp32) at positions pos .."""
        kb, vb, ksb, vsb, kn, vn = self._place
        for i in range(k.shape[0]):
            at = self._block(s, pos + i)
            if at is None:
                continue
            t = (pos + i) % BLOCK
            for x, byte, scale, nib in ((k[i], kb, ksb, kn), (v[i], vb, vsb, vn)):
                c, d = quantize(x)
                for h in range(self.nkv):
                    blk = self.pages[at[0], h, at[1]]
                    b, n = byte[t] + nib[t] // 8, nib[t] % 8
                    for o in (0, 4):  # two nibbles of a byte, one after the other
                        m = n == o
                        blk[b[m]] = (blk[b[m]] & (0xF0 if o == 0 else 0x0F)) | (c[h][m] << o)
                    db = d[h].view(np.uint8).reshape(-1, 2)
                    for g in range(self.hd // 32):
                        p = scale[t, 32 * g]
                        blk[p:p + 2] = db[g]

    def rows(self, s, length):
        """Values of positions 0 .. length - 1 [length, nkv, hd] in 64 bits; positions without a page: present False."""
        kb, vb, ksb, vsb, kn, vn = self._place
        k = np.zeros((length, self.nkv, self.hd))
        v = np.zeros_like(k)
        there = np.zeros(length, bool)
        for b0 in range(0, length, BLOCK):
            at = self._block(s, b0)
            n = min(BLOCK, length - b0)
            if at is None:
                continue
            there[b0:b0 + n] = True
            blk = self.pages[at[0], :, at[1]]
            for out, byte, scale, nib in ((k, kb, ksb, kn), (v, vb, vsb, vn)):
                c = (blk[:, byte + nib // 8] >> (nib % 8).astype(np.uint8)) & 15
                d = np.stack([blk[:, scale], blk[:, scale + 1]], -1).view(np.float16)[..., 0].astype(np.float64)
                with np.errstate(invalid="ignore"):
                    out[b0:b0 + n] = (d * (c.astype(np.float64) - 8)).transpose(1, 0, 2)[:n]
        return k, v, there


def attend(q, k, v, there, pos, window, scale, gate=None):
    """One sequence: q [rows, nq, hd] at positions pos .., k, v [n, nkv, hd].
    (outputs, magnitudes sum p |v| / l, keys / l * largest |v| per row and head, largest sum |q k| scale) in 64
    bits."""
    rows, nq, hd = q.shape
    nkv = k.shape[1]
    out = np.zeros((rows, nq, hd))
    mag = np.zeros((rows, nq, hd))
    low = np.zeros((rows, nq, 1))
    big = 0.0
    t = np.arange(k.shape[0])
    for r in range(rows):
        p = pos + r
        see = (t <= p) & there
        if window:
            see &= t > p - window
        if not see.any():
            continue
        for h in range(nq):
            j = h // (nq // nkv)
            x = k[see, j] * q[r, h].astype(np.float64)
            s = x.sum(-1) * scale
            big = max(big, float(np.abs(x).sum(-1).max() * scale))
            e = np.exp(s - s.max())
            f = 1.0 / e.sum()
            if gate is not None:
                f = f / (1.0 + np.exp(-float(gate[r, h])))
            out[r, h] = e @ v[see, j] * f
            mag[r, h] = e @ np.abs(v[see, j]) * f
            low[r, h] = see.sum() * np.abs(v[see, j]).max() * f
    return out, mag, low, big


def bound(mag, low, big, keys, hd):
    """How far an fp32 evaluation may be from the 64-bit value.

    Scores: q as fp16 hi + lo is off by at most 2^-23 of the column's largest
    |q| (below 2^-22 of it after the power-of-two scaling), fp32 sums of hd
    products by hd 2^-24 of sum |q k|, and the scaling, the subtraction of m and
    exp2 add a few roundings of the score: within (hd + 16) 2^-24 (1 + big), and
    twice that (numerator and denominator) relative to every weight.
    Values: p d as hi + lo truncated, 2^-20; sums over keys of keys / 8 + 16
    roundings 2^-24 each (the products of 32 keys are summed in at most 4
    roundings).
    Weights too small for fp16: p d is kept below 2^15 by p = exp2(s - m) with
    m <= max s + E - 7, d < 2^E <= 2 max d, and truncated to multiples of 2^-24.
    A key loses at most 2^-24 times |code - 8| <= 8, all n keys n 2^-21, and the
    sum l' of exp2(s - m) is 2^(7 - E) or more times the sum l of exp(s - max s):
    n / l 2^(E - 28) <= n / l max d 2^-27 = n / l max|v| 2^-30, since the largest
    |v| of a group is 8 d."""
    rel = 2 * (hd + 16) * 2.0 ** -24 * (1 + big) + 2.0 ** -20 + (keys / 8 + 16) * 2.0 ** -24
    return mag * rel + low * 2.0 ** -30 + 1e-30
