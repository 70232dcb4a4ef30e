"""The operators of an attention layer over the paged 4-bit cache as a serving
loop runs them: norm and quantization, fused projections, append, attention,
output projection -- a ragged prompt batch, then decode steps, eager and as a
captured graph that is replayed with new positions; captured graphs of every
launch form; calls on several streams."""
import numpy as np
import pytest

import paged_q4_ref as ref
from helpers import q4k_random
from test_gpu_graph import HipGraphs
from test_gpu_norm_quant import norm64
from test_gpu_paged_q4 import POISON, Layer, check_attend, dev, filled, rope

pytestmark = pytest.mark.gpu
EPS = 1e-5


class Model:
    """One attention layer: weights, cache and the buffers of a call of up to n_rows rows."""

    def __init__(self, la, rng, n_seq, n_rows, hd, nq, nkv, page, room):
        self.la, self.n_seq, self.hd, self.nq, self.nkv = la, n_seq, hd, nq, nkv
        self.n_embd = nq * hd
        self.rows = [nq * hd, nkv * hd, nkv * hd]
        self.w = [q4k_random(rng, r, self.n_embd) for r in self.rows]
        self.wo = q4k_random(rng, self.n_embd, self.n_embd)
        self.norm_w = (1 + 0.1 * rng.standard_normal(self.n_embd)).astype(np.float32)
        self.qw, self.kw = ((1 + 0.1 * rng.standard_normal(hd)).astype(np.float32) for _ in range(2))
        self.L = Layer(la, ref.Cache(rng, [room] * n_seq, page, nkv, hd))
        self.cos, self.sin = rope(hd, room)
        self.room = room
        self.const = [dev(la, a) for a in (*self.w, self.wo, self.norm_w, self.qw, self.kw, self.cos, self.sin)]
        n, z = n_seq * n_rows, la.DeviceArray
        self.x, self.res = z.zeros((n, self.n_embd), np.float32), z.zeros((n, self.n_embd), np.float32)
        self.xq, self.aq = (z.zeros((n, self.n_embd // 256 * 292), np.uint8) for _ in range(2))
        self.q, self.k, self.v = (z.zeros((n, r), np.float32) for r in self.rows)
        self.q_rot, self.att, self.out = (z.zeros((n, self.n_embd), np.float32) for _ in range(3))
        self.pos, self.count = z.zeros(n_seq, np.uint32), z.zeros(n_seq, np.uint32)
        self.n_rows = n_rows
        size = la.paged_q4_workspace_bytes(n_seq, n_rows, room, nq, nkv, hd, page, self.L.c.stride, 0)
        self.work, self.size = z.zeros(max(size, 16), np.uint8), size

    def run(self, stream=None):
        """x (the layer before it) and res in; out: what the layer adds to res."""
        la, n, C = self.la, self.n_seq * self.n_rows, self.n_embd
        wq, wk, wv, wo, nw, qw, kw, cos, sin = self.const
        la.add_rmsnorm_q8_K(self.x, self.res, nw, EPS, self.res, None, self.xq, n, C, stream)
        la.gqa_qkv_fused([self.q, self.k, self.v], [wq, wk, wv], [12, 12, 12], self.rows, C, self.xq, n, stream)
        la.paged_q4_append(self.q, self.k, self.v, self.q_rot, *self.L.args(), self.pos, self.count, self.n_seq,
                           self.n_rows, self.nq, self.nkv, self.hd, qw, kw, EPS, cos, sin, self.room, stream)
        la.paged_q4_gqa(self.q_rot, None, False, *self.L.args(), self.pos, self.count, self.att, self.n_seq,
                        self.n_rows, self.room, self.nq, self.nkv, self.hd, self.work, self.size, 0, None, stream)
        la.quantize_q8_K(self.att, self.aq, n, C, stream)
        la.matmul_q4_K(self.out, wo, C, C, self.aq, n, stream)

    def check(self, orc, x, res, pos, count):
        """Every operator against its definition, from what the one before it left."""
        shape = lambda a, h: a.numpy().reshape(self.n_seq, self.n_rows, h, self.hd)  # noqa: E731
        assert np.array_equal(self.res.numpy(), x + res)
        y = norm64(x + res, self.norm_w)
        xq = self.xq.numpy()
        assert np.array_equal(xq, orc.quantize_q8_K(y.astype(np.float32)))
        for got, w in zip((self.q, self.k, self.v), self.w):
            assert np.array_equal(got.numpy(), orc.matmul_q4_K(w, xq, self.n_embd))
        q, k, v = shape(self.q, self.nq), shape(self.k, self.nkv), shape(self.v, self.nkv)
        rot, c = shape(self.q_rot, self.nq), self.L.c
        for s in range(self.n_seq):
            n = int(count[s])
            a = slice(pos[s], pos[s] + n)
            cs = self.cos[a, None], self.sin[a, None]
            c.store(s, int(pos[s]), ref.norm_rope(k[s, :n], self.kw, EPS, *cs).astype(np.float32), v[s, :n])
            qr = ref.norm_rope(q[s, :n], self.qw, EPS, *cs)
            assert np.all(np.abs(rot[s, :n] - qr) <= 2.0 ** -24 * np.abs(qr) + 2.0 ** -46)
        assert np.array_equal(self.L.pages.numpy(), c.pages)
        check_attend(self.L, shape(self.att, self.nq), rot, pos, count)
        assert np.array_equal(self.aq.numpy(), orc.quantize_q8_K(self.att.numpy()))
        assert np.array_equal(self.out.numpy(), orc.matmul_q4_K(self.wo, self.aq.numpy(), self.n_embd))

    def feed(self, rng, pos, count):
        n = self.n_seq * self.n_rows
        x, res = (rng.standard_normal((n, self.n_embd)).astype(np.float32) for _ in range(2))
        self.x.upload(x), self.res.upload(res)
        self.pos.upload(np.asarray(pos, np.uint32)), self.count.upload(np.asarray(count, np.uint32))
        self.att.upload(np.full(self.att.shape, POISON)), self.q_rot.upload(np.full(self.att.shape, POISON))
        return x, res


@pytest.mark.parametrize("hd,nq,nkv,page", [(64, 8, 2, 64), (128, 8, 4, 32)])
def test_prompt_then_decode_steps(gpu, orc, hd, nq, nkv, page):
    """Prompts of 45, 1 and 0 tokens in one padded call, then decode steps from a graph captured once."""
    la, rng, hg = gpu, np.random.default_rng(31), HipGraphs()
    room, lengths = 128, np.array([45, 1, 0])
    m = Model(la, rng, 3, 45, hd, nq, nkv, page, room)
    x, res = m.feed(rng, [0, 0, 0], lengths)
    m.run()
    la.sync()
    m.check(orc, x, res, [0, 0, 0], lengths)

    d = Model(la, rng, 3, 1, hd, nq, nkv, page, room)  # buffers of one row per sequence, the cache of the prompts
    d.L = m.L
    stream = hg.stream()
    try:
        d.feed(rng, lengths, [0, 0, 0])
        graph, run = hg.capture(stream, lambda: d.run(stream))
        try:
            for step in range(24):  # crosses the ends of blocks and, from 45 on, of a page
                count = [1, 1, 0] if step < 12 else [1, 1, 1]
                x, res = d.feed(rng, lengths, count)
                if step % 5 == 4:  # the loop's own eager calls between the replays
                    d.run()
                    la.sync()
                else:
                    assert hg.lib.hipGraphLaunch(run, stream) == 0
                    assert hg.lib.hipStreamSynchronize(stream) == 0
                d.check(orc, x, res, lengths, count)
                lengths = lengths + count
        finally:
            hg.lib.hipGraphExecDestroy(run)
            hg.lib.hipGraphDestroy(graph)
    finally:
        hg.lib.hipStreamDestroy(stream)


def test_verify_rows_then_rejection(gpu, orc):
    """Draft rows of a step are stored over by the next one from an earlier position."""
    la, rng = gpu, np.random.default_rng(32)
    m = Model(la, rng, 2, 6, 64, 8, 2, 32, 128)
    pos = np.array([0, 0])
    for keep in ([6, 6], [2, 5], [1, 6], [4, 0], [6, 3], [6, 6], [6, 6], [5, 1]):
        x, res = m.feed(rng, pos, [6, 6])
        m.run()
        la.sync()
        m.check(orc, x, res, pos, [6, 6])
        pos = pos + keep


def attend_args(L, q, pos, n_rows, hint, window=0):
    la, c = L.la, L.c
    n_seq, _, nq, _ = q.shape
    size = la.paged_q4_workspace_bytes(n_seq, n_rows, hint, nq, c.nkv, c.hd, c.page, c.stride, window)
    work = la.DeviceArray.from_numpy(np.full(max(size, 16), 0xFF, np.uint8))
    out = la.DeviceArray.from_numpy(np.full(q.shape, POISON))
    keep = dev(la, q), dev(la, np.asarray(pos, np.uint32)), work, out

    def run(stream=None):
        la.paged_q4_gqa(keep[0], None, False, *L.args(), keep[1], None, out, n_seq, n_rows, hint, nq, c.nkv, c.hd,
                        work, size, window, None, stream)

    return run, out, size


# (head_dim, heads, KV heads, rows, positions): a workgroup per unit, a split in few and in many pieces, a wave per unit
FORMS = [(64, 32, 8, 1, [900, 31, 500]), (64, 32, 8, 1, [6000]), (64, 32, 8, 1, [40000, 7]),
         (128, 8, 2, 7, [3000, 12]), (64, 16, 8, 300, [100, 0, 700, 5, 60]), (64, 4, 4, 1, [i % 900 for i in range(1100)])]


@pytest.mark.parametrize("hd,nq,nkv,n_rows,pos", FORMS)
def test_captured_attention_replays(gpu, hd, nq, nkv, n_rows, pos):
    la, rng, hg = gpu, np.random.default_rng(33), HipGraphs()
    small = sum(pos) < 5000
    L = filled(la, rng, [p + n_rows for p in pos], 64, nkv, hd) if small else Layer(
        la, ref.Cache(rng, [p + n_rows for p in pos], 64, nkv, hd, fill=0x35))
    q = rng.standard_normal((len(pos), n_rows, nq, hd)).astype(np.float32)
    run, out, size = attend_args(L, q, pos, n_rows, max(pos) + n_rows)
    run()
    la.sync()
    want = out.numpy()
    assert np.all(np.isfinite(want)) and not np.any(want == POISON)
    if small:
        check_attend(L, want, q, pos)
    stream = hg.stream()
    try:
        graph, ex = hg.capture(stream, lambda: run(stream))
        try:
            for _ in range(4):
                out.upload(np.full(q.shape, POISON))
                assert hg.lib.hipGraphLaunch(ex, stream) == 0
                assert hg.lib.hipStreamSynchronize(stream) == 0
                assert np.array_equal(out.numpy(), want)  # the split has no order of its own: same bits every time
                out.upload(np.full(q.shape, POISON))
                run()
                la.sync()
                assert np.array_equal(out.numpy(), want)
        finally:
            hg.lib.hipGraphExecDestroy(ex)
            hg.lib.hipGraphDestroy(graph)
    finally:
        hg.lib.hipStreamDestroy(stream)


def test_calls_on_several_streams(gpu):
    """Calls that may overlap, with a workspace each, over one cache; graphs with workspaces of their own beside them."""
    la, rng, hg = gpu, np.random.default_rng(34), HipGraphs()
    pos = [3000, 2500, 17, 900]
    L = filled(la, rng, [p + 1 for p in pos], 64, 4, 64)
    calls = []
    for i in range(4):
        q = rng.standard_normal((4, 1, 16, 64)).astype(np.float32)
        run, out, size = attend_args(L, q, pos, 1, 3001, window=0 if i % 2 else 700)
        run()
        la.sync()
        want = out.numpy()
        check_attend(L, want, q, pos, window=0 if i % 2 else 700)
        out.upload(np.full(q.shape, POISON))
        calls.append((run, out, want))
    streams = [hg.stream() for _ in calls]
    made = []
    try:
        made = [hg.capture(s, lambda run=run, s=s: run(s)) for (run, _, _), s in zip(calls[2:], streams[2:])]
        for _ in range(20):
            for (run, _, _), s in zip(calls[:2], streams):
                run(s)
            for (_, ex), s in zip(made, streams[2:]):
                assert hg.lib.hipGraphLaunch(ex, s) == 0
        for s in streams:
            assert hg.lib.hipStreamSynchronize(s) == 0
        for _, out, want in calls:
            assert np.array_equal(out.numpy(), want)
    finally:
        for graph, ex in made:
            hg.lib.hipGraphExecDestroy(ex)
            hg.lib.hipGraphDestroy(graph)
        for s in streams:
            hg.lib.hipStreamDestroy(s)


@pytest.mark.parametrize("hd,nq", [(64, 4), (64, 16), (64, 40), (128, 8), (128, 40)])
def test_groups_of_very_different_scale(gpu, hd, nq):
    """Dims in groups of 32 whose values differ by 2^20: the bound of a row is the largest group's, the small
    groups keep fp16's range below it."""
    rng = np.random.default_rng(35)
    n, nkv = 200, 2
    c = ref.Cache(rng, [n], 32, nkv, hd)
    v = rng.standard_normal((n, nkv, hd)).astype(np.float32)
    v[..., :32] *= 2.0 ** 12
    v[..., 32:64] *= 2.0 ** -8
    c.store(0, 0, rng.standard_normal((n, nkv, hd)).astype(np.float32), v)
    L = Layer(gpu, c)
    q = rng.standard_normal((1, 1, nq, hd)).astype(np.float32)
    check_attend(L, L.attend(q, [n - 1]), q, [n - 1])
