"""Paged 4-bit cache and fused norm, on the CPU: the layout's formulas cover a
block exactly, sizes, and every refusal before a launch."""
import numpy as np
import pytest

import laii_amd as la
import paged_q4_ref as ref

OK, E_INVALID, E_UNSUPPORTED, E_SCRATCH = 0, -1, -3, -7
FAKE = 4096  # never dereferenced: validation rejects the call first
ODD = FAKE + 4


@pytest.mark.parametrize("hd", [64, 128])
def test_layout_covers_a_block_once(hd):
    k, v, ks, vs, kn, vn = ref.place(hd)
    seen = np.zeros(36 * hd * 2, int)  # nibbles
    for byte, nib in ((k, kn), (v, vn)):
        np.add.at(seen, 2 * byte + nib // 4, 1)
    for s in (ks, vs):
        at = s[:, ::32]
        for o in range(4):
            np.add.at(seen, 2 * at + o, 1)
    assert np.all(seen == 1)


def test_page_bytes():
    assert la.paged_q4_page_bytes(64, 8, 64) == 8 * 2 * 36 * 64
    assert la.paged_q4_page_bytes(32, 1, 128) == 36 * 128
    for bad in ((0, 8, 64), (16, 8, 64), (96, 8, 64), (1 << 17, 8, 64), (64, 8, 96), (64, 8, 32)):
        with pytest.raises(la.LfmAttnError) as e:
            la.paged_q4_page_bytes(*bad)
        assert e.value.status == E_UNSUPPORTED
    with pytest.raises(la.LfmAttnError) as e:
        la.paged_q4_page_bytes(64, 0, 64)
    assert e.value.status == E_INVALID


def norm_args(**kw):
    a = dict(x=FAKE, res=FAKE, w=FAKE, eps=1e-5, out=FAKE, y=FAKE, q=FAKE, n=1, cols=256)
    a.update(kw)
    return [*a.values(), None]


@pytest.mark.parametrize("change,status", [
    (dict(n=0), OK), (dict(n=0, cols=3), OK), (dict(x=None), E_INVALID), (dict(out=None, y=None, q=None), E_INVALID),
    (dict(cols=0), E_INVALID), (dict(cols=255), E_UNSUPPORTED), (dict(cols=(1 << 24) + 256), E_UNSUPPORTED),
    (dict(n=1 << 31), E_INVALID), (dict(n=1 << 24), E_UNSUPPORTED), (dict(x=ODD), E_INVALID), (dict(res=ODD), E_INVALID), (dict(w=ODD), E_INVALID),
    (dict(out=ODD), E_INVALID), (dict(y=ODD), E_INVALID), (dict(q=FAKE + 2), E_INVALID)])
def test_norm_refusals(change, status):
    assert la.load().lfm_hip_add_rmsnorm_q8_K(*norm_args(**change)) == status


CACHE = dict(pages=FAKE, n_pages=9, page=64, table=FAKE, stride=4, pos=FAKE, rows=FAKE)
BAD_CACHE = [
    (dict(pages=None), E_INVALID), (dict(pages=FAKE + 8), E_INVALID), (dict(n_pages=0), E_INVALID),
    (dict(n_pages=1 << 31), E_UNSUPPORTED), (dict(page=48), E_UNSUPPORTED), (dict(page=16), E_UNSUPPORTED),
    (dict(table=None), E_INVALID), (dict(table=FAKE + 2), E_INVALID), (dict(stride=0), E_INVALID),
    (dict(stride=1 << 26), E_UNSUPPORTED), (dict(pos=None), E_INVALID), (dict(pos=FAKE + 1), E_INVALID),
    (dict(rows=FAKE + 2), E_INVALID), (dict(n_seq=0), E_INVALID), (dict(n_rows=0), E_INVALID),
    (dict(nkv=0), E_INVALID), (dict(hd=96), E_UNSUPPORTED), (dict(hd=0), E_UNSUPPORTED)]


def append(**kw):
    a = dict(q=FAKE, k=FAKE, v=FAKE, q_out=FAKE, **CACHE, n_seq=2, n_rows=1, nq=8, nkv=2, hd=64, qw=FAKE, kw=FAKE,
             eps=1e-5, cos=FAKE, sin=FAKE, lut=100)
    a.update(kw)
    return la.load().lfm_hip_paged_q4_append(*a.values(), None)


@pytest.mark.parametrize("change,status", BAD_CACHE + [
    (dict(k=None), E_INVALID), (dict(v=None), E_INVALID), (dict(q=None), E_INVALID), (dict(q_out=None), E_INVALID),
    (dict(nq=0), E_INVALID), (dict(cos=None), E_INVALID), (dict(sin=None), E_INVALID), (dict(lut=0), E_INVALID),
    (dict(q=ODD), E_INVALID), (dict(k=ODD), E_INVALID), (dict(v=ODD), E_INVALID), (dict(q_out=ODD), E_INVALID),
    (dict(qw=ODD), E_INVALID), (dict(kw=ODD), E_INVALID), (dict(cos=ODD), E_INVALID), (dict(sin=ODD), E_INVALID),
    (dict(n_seq=1 << 20, n_rows=1 << 20), E_UNSUPPORTED)])
def test_append_refusals(change, status):
    assert append(**change) == status


def gather(**kw):
    a = dict(k=FAKE, v=FAKE, **CACHE, n_seq=2, n_rows=1, nkv=2, hd=64)
    a.update(kw)
    return la.load().lfm_hip_paged_q4_gather(*a.values(), None)


@pytest.mark.parametrize("change,status", BAD_CACHE + [
    (dict(k=None), E_INVALID), (dict(v=None), E_INVALID), (dict(k=FAKE + 2), E_INVALID), (dict(v=ODD), E_INVALID),
    (dict(n_seq=1 << 20, n_rows=1 << 20), E_UNSUPPORTED)])
def test_gather_refusals(change, status):
    assert gather(**change) == status


def gqa(**kw):
    a = dict(q=FAKE, gate=FAKE, logit=1, **CACHE, out=FAKE, n_seq=2, n_rows=1, hint=256, nq=8, nkv=2, hd=64, window=0,
             scale=0.125, work=FAKE, bytes=1 << 40)
    a.update(kw)
    return la.load().lfm_hip_paged_q4_gqa(*a.values(), None)


@pytest.mark.parametrize("change,status", BAD_CACHE + [
    (dict(q=None), E_INVALID), (dict(out=None), E_INVALID), (dict(nq=7), E_INVALID), (dict(nq=0), E_INVALID),
    (dict(q=ODD), E_INVALID), (dict(out=ODD), E_INVALID), (dict(gate=FAKE + 1), E_INVALID),
    (dict(work=FAKE + 8), E_INVALID), (dict(n_seq=1 << 20, n_rows=1 << 20), E_UNSUPPORTED)])
def test_gqa_refusals(change, status):
    assert gqa(**change) == status


def test_workspace_refusals():
    for bad in ((0, 1, 0, 8, 2, 64, 64, 4), (1, 0, 0, 8, 2, 64, 64, 4), (1, 1, 0, 7, 2, 64, 64, 4),
                (1, 1, 0, 8, 0, 64, 64, 4), (1, 1, 0, 8, 2, 64, 64, 0)):
        with pytest.raises(la.LfmAttnError) as e:
            la.paged_q4_workspace_bytes(*bad)
        assert e.value.status == E_INVALID
    for bad in ((1, 1, 0, 8, 2, 96, 64, 4), (1, 1, 0, 8, 2, 64, 48, 4), (1, 1, 0, 8, 2, 64, 64, 1 << 26)):
        with pytest.raises(la.LfmAttnError) as e:
            la.paged_q4_workspace_bytes(*bad)
        assert e.value.status == E_UNSUPPORTED


@pytest.mark.parametrize("n_seq,n_rows,hint,hd,nq,nkv", [(4, 1, 9000, 64, 32, 8), (2, 8, 5000, 128, 16, 4),
                                                         (3, 100, 4000, 64, 8, 2)])
def test_attention_refuses_a_small_workspace(n_seq, n_rows, hint, hd, nq, nkv):
    """A split that needs scratch: one byte less, none, or none given is refused before a launch."""
    need = la.paged_q4_workspace_bytes(n_seq, n_rows, hint, nq, nkv, hd, 64, 200)
    assert need > 0
    for work, size, status in ((FAKE, need - 1, E_SCRATCH), (FAKE, 0, E_SCRATCH), (None, need, E_INVALID),
                               (FAKE + 8, need, E_INVALID)):
        with pytest.raises(la.LfmAttnError) as e:
            la.paged_q4_gqa(FAKE, None, True, FAKE, 10, 64, FAKE, 200, FAKE, None, FAKE, n_seq, n_rows, hint, nq, nkv,
                            hd, work, size)
        assert e.value.status == status, (work, size)


HUGE = [dict(n_seq=0xFFFFFFFF, n_rows=0x7FFFFFFF, nkv=4096), dict(n_rows=0xFFFFFFFF), dict(n_rows=0x80000000),
        dict(n_seq=0xFFFFFFFF, nkv=4096), dict(n_seq=1 << 23, nkv=2), dict(n_seq=1, nkv=1, n_rows=0xFFFFFFE4)]


@pytest.mark.parametrize("change", HUGE)
def test_sizes_whose_products_pass_a_launch(change):
    """Refused, in whatever way the products would wrap."""
    assert append(**change, nq=4096) == E_UNSUPPORTED
    assert gather(**change) == E_UNSUPPORTED
    assert gqa(**change, nq=4096) == E_UNSUPPORTED
    with pytest.raises(la.LfmAttnError) as e:
        la.paged_q4_workspace_bytes(change.get("n_seq", 2), change.get("n_rows", 1), 0, 4096, change.get("nkv", 2), 64,
                                    64, 4)
    assert e.value.status == E_UNSUPPORTED


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), float("-inf")])
def test_scales_that_are_not_finite(scale):
    assert gqa(scale=scale) == E_INVALID
