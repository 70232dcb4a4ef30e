"""GPU parity of the paged 4-bit cache against its definition in 64 bits
(paged_q4_ref.py): pages bit for bit after an append, rows bit for bit from a
gather, attention within a bound derived from its arithmetic."""
import numpy as np
import pytest

import paged_q4_ref as ref

pytestmark = pytest.mark.gpu
EPS = 1e-5
POISON = np.float32(-777.0)


def dev(la, arr):
    return None if arr is None else la.DeviceArray.from_numpy(np.ascontiguousarray(arr))


def rope(hd, n):
    a = np.arange(n)[:, None] * 1e6 ** (-np.arange(0, hd, 2) / hd)
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)


class Layer:
    """A host cache and its device copy."""

    def __init__(self, la, cache):
        self.la, self.c = la, cache
        self.pages, self.table = dev(la, cache.pages), dev(la, cache.table)

    def args(self):
        return self.pages, self.c.n_pages, self.c.page, self.table, self.c.stride

    def append(self, q, k, v, pos, rows=None, qw=None, kw=None, lut=None, in_place=False, stream=None):
        la, c = self.la, self.c
        n_seq, n_rows = k.shape[:2]
        cos, sin = rope(c.hd, lut or int(np.max(pos)) + n_rows + 1)
        qd = dev(la, q)
        qo = None if q is None else qd if in_place else dev(la, np.full(q.shape, POISON))
        la.paged_q4_append(qd, dev(la, k), dev(la, v), qo, *self.args(), dev(la, np.asarray(pos, np.uint32)),
                           None if rows is None else dev(la, np.asarray(rows, np.uint32)), n_seq, n_rows,
                           0 if q is None else q.shape[2], c.nkv, c.hd, dev(la, qw), dev(la, kw), EPS, dev(la, cos),
                           dev(la, sin), cos.shape[0], stream)
        return None if q is None else qo.numpy()

    def gather(self, pos, n_rows, rows=None):
        la, c = self.la, self.c
        out = [dev(la, np.full((len(pos), n_rows, c.nkv, c.hd), -3, np.float16)) for _ in range(2)]
        la.paged_q4_gather(*out, *self.args(), dev(la, np.asarray(pos, np.uint32)),
                           None if rows is None else dev(la, np.asarray(rows, np.uint32)), len(pos), n_rows, c.nkv,
                           c.hd)
        return [o.numpy() for o in out]

    def attend(self, q, pos, rows=None, window=0, gate=None, hint=None, scale=None, logit=True, stream=None):
        la, c = self.la, self.c
        n_seq, n_rows, nq, _ = q.shape
        out = dev(la, np.full(q.shape, POISON))
        hint = int(np.max(pos)) + n_rows if hint is None else hint
        n = la.paged_q4_workspace_bytes(n_seq, n_rows, hint, nq, c.nkv, c.hd, c.page, c.stride, window)
        work = dev(la, np.full(max(n, 16), 0xFF, np.uint8))
        la.paged_q4_gqa(dev(la, q), dev(la, gate), logit, *self.args(), dev(la, np.asarray(pos, np.uint32)),
                        None if rows is None else dev(la, np.asarray(rows, np.uint32)), out, n_seq, n_rows, hint, nq,
                        c.nkv, c.hd, work, n, window, scale, stream)
        return out.numpy()


def check_attend(layer, got, q, pos, rows=None, window=0, gate=None, scale=None):
    c = layer.c
    scale = float(1.0 / np.sqrt(np.float32(c.hd))) if scale is None else scale
    reach = c.stride * c.page
    for s in range(q.shape[0]):
        p = int(pos[s])
        n = q.shape[1] if rows is None else min(int(rows[s]), q.shape[1])
        n = max(0, min(n, reach - p))
        assert np.all(got[s, n:] == POISON), s
        if n == 0:
            continue
        k, v, there = c.rows(s, p + n)
        want, mag, low, big = ref.attend(q[s, :n], k, v, there, p, window, scale, None if gate is None else gate[s])
        off = np.abs(got[s, :n] - want)
        lim = ref.bound(mag, low, big, p + n, c.hd)
        if gate is not None:
            lim = lim + 8 * 2.0 ** -24 * np.abs(want)  # the sigmoid's own roundings
        worst = float((off / lim).max())
        print(f"seq {s}: rows {n} pos {p} worst {worst:.3f} of the bound, rel "
              f"{np.linalg.norm(got[s, :n] - want) / max(np.linalg.norm(want), 1e-30):.2e}", flush=True)
        assert np.all(np.isfinite(got[s, :n])) and worst <= 1.0, (s, worst)


def filled(la, rng, lengths, page, nkv, hd, scale=1.0, **kw):
    """A cache with rows in positions 0 .. length - 1 of every sequence."""
    c = ref.Cache(rng, lengths, page, nkv, hd, **kw)
    for s, n in enumerate(lengths):
        k = rng.standard_normal((n, nkv, hd)).astype(np.float32)
        v = (scale * rng.standard_normal((n, nkv, hd))).astype(np.float32)
        c.store(s, 0, k, v)
    return Layer(la, c)


# ---- append ------------------------------------------------------------------------

@pytest.mark.parametrize("hd,nq,nkv,page,pos,rows,n_rows", [
    (64, 8, 2, 32, [0], None, 1),
    (64, 16, 8, 64, [5, 31, 32, 63], None, 1),
    (128, 16, 4, 128, [0, 100, 127], None, 1),
    (64, 4, 1, 32, [30, 0, 17], [8, 0, 3], 8),
    (64, 6, 2, 64, [3, 70], [100, 33], 100),
    (128, 8, 2, 64, [1, 95], [70, 1], 70),
    (128, 5, 5, 32, [31], [2], 2),
    (64, 3, 3, 256, [250], None, 40)])
def test_append_pages_bit_exact(gpu, hd, nq, nkv, page, pos, rows, n_rows):
    rng = np.random.default_rng(hd + n_rows + len(pos))
    n = len(pos)
    c = ref.Cache(rng, [p + n_rows for p in pos], page, nkv, hd)
    L = Layer(gpu, c)
    q, k, v = (rng.standard_normal((n, n_rows, h, hd)).astype(np.float32) for h in (nq, nkv, nkv))
    v[0, 0, 0, :32] = 0.0                      # a group of zeros
    v[0, 0, 0, 32:34] = [5.0, -5.0]            # two values of the largest magnitude
    qw, kw = ((1 + 0.1 * rng.standard_normal(hd)).astype(np.float32) for _ in range(2))
    got_q = L.append(q, k, v, pos, rows, qw, kw)
    cos, sin = rope(hd, max(pos) + n_rows + 1)
    for s in range(n):
        r = n_rows if rows is None else rows[s]
        a = slice(pos[s], pos[s] + r)
        kr = ref.norm_rope(k[s, :r], kw, EPS, cos[a, None], sin[a, None]).astype(np.float32)
        c.store(s, pos[s], kr, v[s, :r])
        qr = ref.norm_rope(q[s, :r], qw, EPS, cos[a, None], sin[a, None])
        # rounded once, from a value whose own error (of lo c - hi s) is below 2^-48 of the pair
        assert np.all(np.abs(got_q[s, :r] - qr) <= 2.0 ** -24 * np.abs(qr) + 2.0 ** -46)
        assert np.all(got_q[s, r:] == POISON)
    assert np.array_equal(L.pages.numpy(), c.pages)


def test_append_without_norm_in_place_and_without_queries(gpu):
    rng = np.random.default_rng(3)
    pos, n_rows, hd, nkv = [9, 40], 5, 64, 2
    q, k, v = (rng.standard_normal((2, n_rows, h, hd)).astype(np.float32) for h in (4, nkv, nkv))
    cos, sin = rope(hd, 60)
    pages = []
    for q_in, in_place in ((q, False), (q, True), (None, False)):
        r = np.random.default_rng(4)
        c = ref.Cache(r, [p + n_rows for p in pos], 32, nkv, hd)
        L = Layer(gpu, c)
        got = L.append(q_in, k, v, pos, in_place=in_place, lut=60)
        if q_in is not None:
            for s in range(2):
                a = slice(pos[s], pos[s] + n_rows)
                want = ref.norm_rope(q[s], None, EPS, cos[a, None], sin[a, None])
                assert np.all(np.abs(got[s] - want) <= 2.0 ** -24 * np.abs(want) + 2.0 ** -46)
        for s in range(2):
            a = slice(pos[s], pos[s] + n_rows)
            c.store(s, pos[s], ref.norm_rope(k[s], None, EPS, cos[a, None], sin[a, None]).astype(np.float32), v[s])
        assert np.array_equal(L.pages.numpy(), c.pages)


def test_append_skips_what_no_table_reaches(gpu):
    """No page, positions past the table and past the rotation table, huge positions: nothing is stored."""
    rng = np.random.default_rng(5)
    hd, nkv, n_rows = 64, 2, 40
    c = ref.Cache(rng, [128, 128, 128, 128, 128], 32, nkv, hd)
    c.table[0, 1] = -1
    c.table[1, 2] = c.n_pages
    L = Layer(gpu, c)
    pos = [20, 60, 120, 128, 0xFFFFFFF0]
    q, k, v = (rng.standard_normal((5, n_rows, h, hd)).astype(np.float32) for h in (2, nkv, nkv))
    got = L.append(q, k, v, pos, lut=126)
    cos, sin = rope(hd, 126)
    for s, r in enumerate((40, 40, 6, 0, 0)):
        a = slice(pos[s], pos[s] + r)
        if r:
            kr = ref.norm_rope(k[s, :r], None, EPS, cos[a, None], sin[a, None]).astype(np.float32)
            c.store(s, pos[s], kr, v[s, :r])
        assert np.all(got[s, r:] == POISON) and np.all(got[s, :r] != POISON)
    assert np.array_equal(L.pages.numpy(), c.pages)


def test_append_values_that_are_not_finite(gpu):
    """Their groups read back as NaN, no other group changes."""
    rng = np.random.default_rng(6)
    c = ref.Cache(rng, [32], 32, 1, 64)
    L = Layer(gpu, c)
    k, v = (rng.standard_normal((1, 4, 1, 64)).astype(np.float32) for _ in range(2))
    v[0, 0, 0, 3], v[0, 1, 0, 40], v[0, 2, 0, 5], k[0, 3, 0, 7] = np.nan, np.inf, 1e30, np.nan
    L.append(None, k, v, [0])
    gk, gv = L.gather([0], 4)
    bad = np.zeros((4, 64), bool)
    bad[0, :32] = bad[1, 32:] = True
    assert np.array_equal(np.isnan(gv[0, :2, 0]), bad[:2])
    assert np.all(np.isnan(gv[0, 2, 0, :32])) and not np.any(np.isnan(gv[0, 2, 0, 32:]))
    assert not np.any(np.isnan(gv[0, 3])) and not np.any(np.isnan(gk[0, :3])) and np.all(np.isnan(gk[0, 3]))


def test_append_in_pieces_equals_one_append(gpu):
    """Rows stored one, a few and many at a time leave the same pages."""
    rng = np.random.default_rng(7)
    n, hd, nkv = 90, 128, 2
    k, v = (rng.standard_normal((1, n, nkv, hd)).astype(np.float32) for _ in range(2))
    pages = []
    for cuts in ([0, n], [0, 1, 2, 3, 8, 31, 32, 33, 70, n], list(range(n + 1))):
        L = Layer(gpu, ref.Cache(np.random.default_rng(8), [n], 64, nkv, hd))
        for a, b in zip(cuts, cuts[1:]):
            L.append(None, k[:, a:b], v[:, a:b], [a], lut=n)
        pages.append(L.pages.numpy())
    assert np.array_equal(pages[0], pages[1]) and np.array_equal(pages[0], pages[2])


# ---- gather ------------------------------------------------------------------------

@pytest.mark.parametrize("hd,nkv,page,pos,rows,n_rows", [
    (64, 8, 64, [0], None, 1), (64, 2, 32, [5, 31, 0], [60, 0, 33], 60), (128, 4, 128, [0, 77], [130, 5], 130),
    (128, 1, 32, [31], None, 2)])
def test_gather_bit_exact(gpu, hd, nkv, page, pos, rows, n_rows):
    rng = np.random.default_rng(hd + n_rows)
    lengths = [p + n_rows for p in pos]
    L = filled(gpu, rng, lengths, page, nkv, hd)
    gk, gv = L.gather(pos, n_rows, rows)
    for s, p in enumerate(pos):
        r = n_rows if rows is None else rows[s]
        k, v, _ = L.c.rows(s, p + r)
        assert np.array_equal(gk[s, :r], k[p:].astype(np.float32).astype(np.float16))
        assert np.array_equal(gv[s, :r], v[p:].astype(np.float32).astype(np.float16))
        assert np.all(gk[s, r:] == -3) and np.all(gv[s, r:] == -3)


def test_gather_missing_pages_are_zero_and_rows_past_the_table_stay(gpu):
    rng = np.random.default_rng(9)
    L = filled(gpu, rng, [96, 64], 32, 2, 64)
    L.c.table[0, 1] = -1
    L.table.upload(L.c.table)
    gk, gv = L.gather([0, 50], 100)
    k, v, there = L.c.rows(0, 96)
    assert np.array_equal(gk[0, :96], np.where(there[:, None, None], k, 0).astype(np.float32).astype(np.float16))
    assert np.all(gv[0, 32:64] == 0) and np.all(gk[0, 96:] == -3) and np.all(gk[1, 46:] == -3)
    assert np.all(gk[1, 14:46] == 0)  # inside the table, no page: entry -1


# ---- attention ---------------------------------------------------------------------

SHAPES = [(64, 16, 8), (64, 32, 8), (128, 16, 4), (64, 4, 4), (64, 9, 3), (128, 32, 2), (64, 40, 2), (128, 2, 2)]


@pytest.mark.parametrize("hd,nq,nkv", SHAPES)
@pytest.mark.parametrize("page", [32, 128])
def test_decode(gpu, hd, nq, nkv, page):
    """One row per sequence, contexts from one key on."""
    rng = np.random.default_rng(hd + nq + page)
    pos = [0, 1, 15, 31, 32, 63, 64, 200, 517]
    L = filled(gpu, rng, [p + 1 for p in pos], page, nkv, hd)
    q = rng.standard_normal((len(pos), 1, nq, hd)).astype(np.float32)
    check_attend(L, L.attend(q, pos), q, pos)


@pytest.mark.parametrize("hd,nq,nkv", [(64, 32, 8), (128, 16, 4), (64, 16, 8)])
@pytest.mark.parametrize("ctx", [1023, 2500, 5000])
def test_decode_one_sequence(gpu, hd, nq, nkv, ctx):
    rng = np.random.default_rng(ctx)
    L = filled(gpu, rng, [ctx], 64, nkv, hd)
    q = (2 * rng.standard_normal((1, 1, nq, hd))).astype(np.float32)
    check_attend(L, L.attend(q, [ctx - 1]), q, [ctx - 1])


@pytest.mark.parametrize("hd,nq,nkv", [(64, 32, 8), (128, 16, 4), (64, 6, 2), (64, 20, 1)])
@pytest.mark.parametrize("n_rows", [2, 5, 8])
@pytest.mark.parametrize("window", [0, 40])
def test_verify_rows(gpu, hd, nq, nkv, n_rows, window):
    rng = np.random.default_rng(n_rows + window + hd)
    pos, rows = [0, 25, 300, 90, 61], [n_rows, 1, n_rows, 0, n_rows + 5]
    L = filled(gpu, rng, [p + n_rows for p in pos], 32, nkv, hd)
    q = rng.standard_normal((5, n_rows, nq, hd)).astype(np.float32)
    gate = rng.standard_normal((5, n_rows, nq)).astype(np.float32)
    got = L.attend(q, pos, rows, window, gate)
    check_attend(L, got, q, pos, rows, window, gate)


@pytest.mark.parametrize("hd,nq,nkv,n_rows,pos,window", [
    (64, 8, 2, 33, [0, 100], 0), (64, 4, 1, 150, [7], 0), (128, 4, 1, 70, [0, 33], 0), (128, 8, 2, 90, [300], 48),
    (64, 8, 2, 64, [64, 3], 1), (64, 3, 1, 100, [11], 33)])
def test_prompt_rows(gpu, hd, nq, nkv, n_rows, pos, window):
    rng = np.random.default_rng(n_rows + window)
    rows = [n_rows] + [max(1, n_rows // 3)] * (len(pos) - 1)
    L = filled(gpu, rng, [p + n_rows for p in pos], 64, nkv, hd)
    q = rng.standard_normal((len(pos), n_rows, nq, hd)).astype(np.float32)
    check_attend(L, L.attend(q, pos, rows, window), q, pos, rows, window)


@pytest.mark.parametrize("window", [1, 16, 31, 32, 33, 256, 100000])
def test_windows(gpu, window):
    rng = np.random.default_rng(window)
    pos = [0, 14, 32, 255, 256, 700]
    L = filled(gpu, rng, [p + 1 for p in pos], 32, 4, 128)
    q = rng.standard_normal((6, 1, 16, 128)).astype(np.float32)
    gate = rng.standard_normal((6, 1, 16)).astype(np.float32)
    check_attend(L, L.attend(q, pos, None, window, gate), q, pos, None, window, gate)


def test_window_pages_before_it_may_be_gone(gpu):
    """An engine frees the pages that no window reaches any more."""
    rng = np.random.default_rng(12)
    pos, window = [500, 333], 100
    L = filled(gpu, rng, [501, 334], 32, 2, 64)
    for s, p in enumerate(pos):
        L.c.table[s, :(p + 1 - window) // 32] = -1
    L.table.upload(L.c.table)
    q = rng.standard_normal((2, 1, 8, 64)).astype(np.float32)
    check_attend(L, L.attend(q, pos, None, window), q, pos, None, window)


@pytest.mark.parametrize("n_rows", [1, 6, 40])
def test_missing_pages_are_not_attended(gpu, n_rows):
    rng = np.random.default_rng(13)
    pos = [200, 100, 250]
    L = filled(gpu, rng, [p + n_rows for p in pos], 32, 2, 64)
    L.c.table[0, [0, 3]] = [-1, L.c.n_pages]
    L.c.table[1, :] = -7                      # nothing left: zeros
    L.c.table[2, 1:8] = -1
    L.table.upload(L.c.table)
    q = rng.standard_normal((3, n_rows, 8, 64)).astype(np.float32)
    got = L.attend(q, pos)
    assert np.all(got[1] == 0)
    check_attend(L, got, q, pos)


@pytest.mark.parametrize("n_rows", [1, 8, 40])
@pytest.mark.parametrize("hd", [64, 128])
def test_slots_behind_the_last_row_do_not_count(gpu, hd, n_rows):
    """NaN and infinite scales, and huge ones, in positions that no row attends."""
    rng = np.random.default_rng(14)
    pos = [3, 40, 65]
    L = filled(gpu, rng, [p + n_rows for p in pos], 64, 2, hd, scale=0.02)
    _, _, ks, vs, _, _ = ref.place(hd)
    for s, p in enumerate(pos):
        for t in range(p + n_rows, -(-(p + n_rows) // 64) * 64):
            page = L.c.table[s, t // 64]
            for sc in (ks, vs):
                for g in range(hd // 32):
                    at = sc[t % 32, 32 * g]
                    bits = [0x7E00, 0x7C00, 0xFC00, 0x7BFF][(t + g) % 4]
                    L.c.pages[page, :, t % 64 // 32, at:at + 2] = [bits & 255, bits >> 8]
    L.pages.upload(L.c.pages)
    q = rng.standard_normal((3, n_rows, 8, hd)).astype(np.float32)
    check_attend(L, L.attend(q, pos), q, pos)


@pytest.mark.parametrize("n_rows", [1, 5, 40])
def test_not_finite_keys_stay_in_their_sequence(gpu, n_rows):
    rng = np.random.default_rng(15)
    pos = [90, 90]
    L = filled(gpu, rng, [p + n_rows for p in pos], 32, 2, 64)
    _, _, ks, _, _, _ = ref.place(64)
    L.c.pages[L.c.table[0, 1], 0, 0, ks[5, 0]:ks[5, 0] + 2] = [0x00, 0x7E]  # KV head 0 of sequence 0
    L.pages.upload(L.c.pages)
    q = rng.standard_normal((2, n_rows, 8, 64)).astype(np.float32)
    got = L.attend(q, pos)
    assert np.all(np.isnan(got[0, :, :4])) and np.all(np.isfinite(got[0, :, 4:])) and np.all(np.isfinite(got[1]))


@pytest.mark.parametrize("bits", [0x7E00, 0x7C00, 0xFC00])
@pytest.mark.parametrize("hd,nq,n_rows,window,at", [
    (64, 4, 1, 0, 90), (64, 8, 5, 0, 92), (64, 8, 40, 0, 101), (64, 8, 40, 30, 101), (64, 8, 40, 0, 127),
    (64, 8, 9, 7, 91), (128, 8, 1, 0, 90), (128, 16, 40, 0, 101), (128, 16, 40, 20, 96)])
def test_not_finite_values_stay_in_the_rows_that_attend_them(gpu, hd, nq, n_rows, window, at, bits):
    """A V scale that is not finite: NaN in its group of dims, in the rows that attend its position and nowhere else."""
    rng = np.random.default_rng(23)
    p, nkv = 90, 2
    L = filled(gpu, rng, [p + n_rows], 32, nkv, hd)
    k, v, there = L.c.rows(0, p + n_rows)
    _, _, _, vs, _, _ = ref.place(hd)
    where = vs[at % 32, 32]
    L.c.pages[L.c.table[0, at // 32], 0, 0, where:where + 2] = [bits & 255, bits >> 8]
    L.pages.upload(L.c.pages)
    q = rng.standard_normal((1, n_rows, nq, hd)).astype(np.float32)
    got = L.attend(q, [p], None, window)[0]
    t = p + np.arange(n_rows)
    hit = np.zeros((n_rows, nq, hd), bool)
    hit[(t >= at) & ((t < at + window) | (window == 0)), :nq // nkv, 32:64] = True
    assert np.array_equal(np.isnan(got), hit)
    want, mag, low, big = ref.attend(q[0], k, v, there, p, window, float(1.0 / np.sqrt(np.float32(hd))))
    off = np.abs(got - want) / ref.bound(mag, low, big, p + n_rows, hd)
    assert np.all(off[~hit] <= 1.0), float(off[~hit].max())


@pytest.mark.parametrize("n_rows", [1, 5, 40])
@pytest.mark.parametrize("vscale,qscale", [(1e-3, 1.0), (1e4, 1.0), (1.0, 1e-6), (1.0, 60.0), (1e-2, 1e4)])
def test_magnitudes(gpu, n_rows, vscale, qscale):
    """Values near the ends of fp16's range of scales, flat and one-hot softmax."""
    rng = np.random.default_rng(16)
    pos = [150, 31]
    c = ref.Cache(rng, [p + n_rows for p in pos], 32, 2, 64)
    for s, p in enumerate(pos):
        n = p + n_rows
        k = rng.standard_normal((n, 2, 64)).astype(np.float32)
        v = (vscale * rng.standard_normal((n, 2, 64))).astype(np.float32)
        v[n // 2:] *= 8.0
        c.store(s, 0, k, v)
    L = Layer(gpu, c)
    q = (qscale * rng.standard_normal((2, n_rows, 8, 64))).astype(np.float32)
    q[0, 0, 0] = 0.0
    check_attend(L, L.attend(q, pos), q, pos)


@pytest.mark.parametrize("n_rows", [1, 8])
def test_scores_that_rise_or_fall(gpu, n_rows):
    """The running maximum moves at every step, or never after the first."""
    rng = np.random.default_rng(17)
    n = 700
    for sign in (1.0, -1.0):
        c = ref.Cache(rng, [n], 64, 1, 64)
        k = rng.standard_normal((n, 1, 64)).astype(np.float32)
        k[:, 0, :] += (sign * np.linspace(0, 6, n))[:, None].astype(np.float32)
        c.store(0, 0, k, rng.standard_normal((n, 1, 64)).astype(np.float32))
        L = Layer(gpu, c)
        q = (1 + rng.random((1, n_rows, 4, 64))).astype(np.float32)
        check_attend(L, L.attend(q, [n - n_rows]), q, [n - n_rows])


def test_rows_past_the_table_are_left(gpu):
    rng = np.random.default_rng(18)
    L = filled(gpu, rng, [64, 64, 64], 32, 2, 64)
    pos = [60, 64, 0xFFFFFFFF]
    q = rng.standard_normal((3, 8, 4, 64)).astype(np.float32)
    check_attend(L, L.attend(q, pos, hint=64), q, pos)


@pytest.mark.parametrize("hint", [0, 1, 50, 2000, 0xFFFFFFFF])
@pytest.mark.parametrize("n_rows", [1, 8])
def test_keys_hint_only_sizes_the_split(gpu, hint, n_rows):
    rng = np.random.default_rng(19)
    pos = [1500, 3, 700]
    L = filled(gpu, rng, [p + n_rows for p in pos], 64, 2, 64)
    q = rng.standard_normal((3, n_rows, 8, 64)).astype(np.float32)
    check_attend(L, L.attend(q, pos, hint=hint), q, pos)


def test_gate_values_and_logits(gpu):
    rng = np.random.default_rng(20)
    pos = [77, 400]
    L = filled(gpu, rng, [78, 401], 64, 2, 128)
    q = rng.standard_normal((2, 1, 8, 128)).astype(np.float32)
    g = rng.standard_normal((2, 1, 8)).astype(np.float32)
    g[0, 0, :3] = [np.inf, -np.inf, 80.0]
    plain = L.attend(q, pos)
    sig = (1 / (1 + np.exp(-g.astype(np.float64))))[..., None]
    for got, f in ((L.attend(q, pos, gate=g), sig), (L.attend(q, pos, gate=sig[..., 0].astype(np.float32), logit=False),
                                                     sig)):
        assert np.all(np.abs(got - plain * f) <= 2.0 ** -20 * np.abs(plain * f) + 1e-37)


@pytest.mark.parametrize("n_seq", [65, 130, 300])
def test_many_sequences(gpu, n_seq):
    rng = np.random.default_rng(n_seq)
    pos = rng.integers(0, 90, n_seq)
    rows = rng.integers(0, 3, n_seq)
    L = filled(gpu, rng, [int(p) + 2 for p in pos], 32, 1, 64)
    q = rng.standard_normal((n_seq, 2, 2, 64)).astype(np.float32)
    check_attend(L, L.attend(q, pos, rows), q, pos, rows)


def test_shared_prefix_pages(gpu):
    """Two sequences read the same pages."""
    rng = np.random.default_rng(21)
    L = filled(gpu, rng, [200, 200], 32, 2, 64)
    L.c.table[1, :4] = L.c.table[0, :4]
    L.table.upload(L.c.table)
    q = rng.standard_normal((2, 1, 8, 64)).astype(np.float32)
    check_attend(L, L.attend(q, [199, 199]), q, [199, 199])


def test_pages_past_4_gib(gpu):
    """Offsets that pass 32 bits: the last pages of a 4.5 GiB buffer."""
    page, nkv, hd, n = 256, 8, 64, 300
    size = gpu.paged_q4_page_bytes(page, nkv, hd)
    n_pages = (9 << 29) // size
    rng = np.random.default_rng(22)
    c = ref.Cache(rng, [n], page, nkv, hd, spare=0)
    host = c.table.copy()
    big = gpu.DeviceArray((n_pages * size,), np.uint8)
    L = Layer.__new__(Layer)
    L.la, L.c, L.pages = gpu, c, big
    L.table = dev(gpu, np.where(host >= 0, n_pages - 2 + host, -1).astype(np.int32))
    args = (big, n_pages, page, L.table, c.stride)
    L.args = lambda: args
    k, v = (rng.standard_normal((1, n, nkv, hd)).astype(np.float32) for _ in range(2))
    L.append(None, k, v, [0], lut=n)
    cos, sin = rope(hd, n)
    c.store(0, 0, ref.norm_rope(k[0], None, EPS, cos[:, None], sin[:, None]).astype(np.float32), v[0])
    gk, _ = L.gather([0], n)
    assert np.array_equal(gk[0], c.rows(0, n)[0].astype(np.float32).astype(np.float16))
    q = rng.standard_normal((1, 1, 32, hd)).astype(np.float32)
    check_attend(L, L.attend(q, [n - 1]), q, [n - 1])


def test_many_sequences_and_a_long_one(gpu):
    """More sequences than the card has waves for, lengths from none to thousands of keys."""
    rng = np.random.default_rng(24)
    n = 1030
    pos = rng.integers(0, 40, n)
    pos[[0, 511, 1029]] = [3000, 700, 2047]
    rows = np.ones(n, int)
    rows[rng.integers(1, n - 1, 200)] = 0
    L = filled(gpu, rng, [int(p) + 1 for p in pos], 32, 4, 64)
    q = rng.standard_normal((n, 1, 8, 64)).astype(np.float32)
    for hint in (None, 100):
        check_attend(L, L.attend(q, pos, rows, hint=hint), q, pos, rows)


@pytest.mark.parametrize("n_rows", [1, 5, 40])
@pytest.mark.parametrize("scale", [-0.3, 0.0, 1e-20, 2.0])
def test_scales(gpu, n_rows, scale):
    rng = np.random.default_rng(25)
    pos = [130, 7]
    L = filled(gpu, rng, [p + n_rows for p in pos], 32, 2, 64)
    q = rng.standard_normal((2, n_rows, 8, 64)).astype(np.float32)
    check_attend(L, L.attend(q, pos, scale=scale), q, pos, scale=float(np.float32(scale)))


@pytest.mark.parametrize("n_rows", [1, 5, 40])
@pytest.mark.parametrize("hd", [64, 128])
def test_smallest_and_largest_queries(gpu, hd, n_rows):
    """Queries below the normal numbers: all weights alike.  Queries whose scores come near fp32's end or pass it: one
    weight is 1, the others 0, as long as the best score leads by far more than the scores' rounding, so what
    remains is the error of p d as hi + lo, 2^-20 of |v|."""
    rng = np.random.default_rng(26)
    pos = 70
    L = filled(gpu, rng, [pos + n_rows], 32, 2, hd)
    unit = rng.standard_normal((1, n_rows, 8, hd)).astype(np.float32)
    for size in (1e-45, 1e-41, 1e-38, 1e-30):
        q = (size * unit).astype(np.float32)
        check_attend(L, L.attend(q, [pos]), q, [pos])
    k, v, _ = L.c.rows(0, pos + n_rows)
    for size in (1e20, 1e32, 5e37):
        q = (size * unit).astype(np.float32)
        got = L.attend(q, [pos])[0]
        for r in range(n_rows):
            for h in range(8):
                s = k[:pos + r + 1, h // 4] @ q[0, r, h].astype(np.float64)
                first, second = np.argsort(s)[:-3:-1]
                if s[first] - s[second] < 2.0 ** -12 * np.abs(s).max():
                    continue
                want = v[first, h // 4]
                assert np.all(np.abs(got[r, h] - want) <= 2.0 ** -20 * np.abs(want)), (size, r, h)


@pytest.mark.parametrize("n_rows", [1, 5, 40])
@pytest.mark.parametrize("hd", [64, 128])
def test_not_finite_queries_stay_in_their_head(gpu, hd, n_rows):
    rng = np.random.default_rng(27)
    pos = [90, 40]
    L = filled(gpu, rng, [p + n_rows for p in pos], 32, 2, hd)
    q = rng.standard_normal((2, n_rows, 8, hd)).astype(np.float32)
    good = L.attend(q, pos)
    q[0, 0, 1, 5], q[1, n_rows - 1, 7, 40] = np.nan, np.inf
    got = L.attend(q, pos)
    bad = np.zeros(got.shape, bool)
    bad[0, 0, 1] = bad[1, n_rows - 1, 7] = True
    assert np.all(np.isnan(got[bad])) and np.array_equal(got[~bad], good[~bad])


@pytest.mark.parametrize("hint", [1, 700, 20000])
@pytest.mark.parametrize("hd,nq,nkv,n_rows,window", [
    (64, 8, 2, 40, 0), (64, 8, 2, 150, 0), (64, 8, 2, 150, 90), (64, 2, 2, 150, 0), (128, 8, 2, 40, 0),
    (128, 6, 2, 150, 0), (128, 8, 2, 150, 33)])
def test_prompt_rows_in_every_division_of_the_work(gpu, hd, nq, nkv, n_rows, window, hint):
    """The bound of the keys chooses between a wave or workgroup per tile and equal shares; the result may not."""
    rng = np.random.default_rng(28)
    pos, rows = [500, 0, 61, 0], [n_rows, n_rows - 7, n_rows // 2, 0]
    c = ref.Cache(rng, [p + r for p, r in zip(pos, rows)][:3] + [20000], 64, nkv, hd)  # a table of 20000 positions
    for s in range(3):
        k, v = (rng.standard_normal((pos[s] + rows[s], nkv, hd)).astype(np.float32) for _ in range(2))
        c.store(s, 0, k, v)
    L = Layer(gpu, c)
    q = rng.standard_normal((4, n_rows, nq, hd)).astype(np.float32)
    check_attend(L, L.attend(q, pos, rows, window, hint=hint), q, pos, rows, window)


@pytest.mark.parametrize("hd,nq,n_rows", [(64, 4, 40), (128, 4, 20), (64, 1, 3)])
def test_long_windows_in_a_split(gpu, hd, nq, n_rows):
    rng = np.random.default_rng(29)
    pos, window = [3000, 700], 2500
    L = filled(gpu, rng, [p + n_rows for p in pos], 64, 1, hd)
    assert gpu.paged_q4_workspace_bytes(2, n_rows, 3000 + n_rows, nq, 1, hd, 64, L.c.stride, window) > 0
    q = rng.standard_normal((2, n_rows, nq, hd)).astype(np.float32)
    check_attend(L, L.attend(q, pos, None, window), q, pos, None, window)
