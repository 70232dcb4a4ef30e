"""lfm_hip_add_rmsnorm_q8_K against its definition: the residual sum in fp32, the
norm in 64 bits rounded once, the blocks bit for bit those that the oracle's
quantizer makes of the norm's own fp32 result."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
EPS = 1e-5


def dev(la, arr):
    return None if arr is None else la.DeviceArray.from_numpy(np.ascontiguousarray(arr))


def norm64(h, w, eps=EPS):
    h = h.astype(np.float64)
    y = h / np.sqrt((h * h).mean(-1, keepdims=True) + float(np.float32(eps)))
    return y if w is None else y * w.astype(np.float64)


def call(la, x, res, w, want=("res", "y", "q"), eps=EPS):
    n, cols = x.shape
    out = dict(res=la.DeviceArray.from_numpy(np.full(x.shape, 7, np.float32)),
               y=la.DeviceArray.from_numpy(np.full(x.shape, 7, np.float32)),
               q=la.DeviceArray.from_numpy(np.full((n, cols // 256 * 292), 7, np.uint8)))
    a = [out[k] if k in want else None for k in ("res", "y", "q")]
    la.add_rmsnorm_q8_K(dev(la, x), dev(la, res), dev(la, w), eps, *a, n, cols)
    return {k: v.numpy() for k, v in out.items()}


def check(orc, got, x, res, w, eps=EPS):
    h = x if res is None else x + res
    assert np.array_equal(got["res"], h)
    want = norm64(h, w, eps)
    # one rounding of a 64-bit value whose own error is far below half a step
    step = np.spacing(np.abs(want).astype(np.float32)).astype(np.float64)
    assert np.all(np.abs(got["y"] - want) <= 0.5001 * step)
    assert np.array_equal(got["q"], orc.quantize_q8_K(got["y"]))


@pytest.mark.parametrize("rows,cols", [(1, 256), (3, 512), (1, 2048), (65, 2304), (7, 4096), (2, 8192), (3, 8448),
                                       (1, 33024), (300, 1024)])
def test_norm_matches_definition(gpu, orc, rows, cols):
    rng = np.random.default_rng(rows * 31 + cols)
    x = rng.standard_normal((rows, cols)).astype(np.float32)
    res = (3 * rng.standard_normal((rows, cols))).astype(np.float32)
    w = (1 + 0.1 * rng.standard_normal(cols)).astype(np.float32)
    check(orc, call(gpu, x, res, w), x, res, w)


@pytest.mark.parametrize("res", [False, True])
@pytest.mark.parametrize("w", [False, True])
@pytest.mark.parametrize("cols", [1536, 8448])
def test_norm_without_residual_or_weight(gpu, orc, res, w, cols):
    rng = np.random.default_rng(5)
    x = rng.standard_normal((5, cols)).astype(np.float32)
    res = rng.standard_normal((5, cols)).astype(np.float32) if res else None
    w = rng.standard_normal(cols).astype(np.float32) if w else None
    check(orc, call(gpu, x, res, w), x, res, w)


@pytest.mark.parametrize("scale", [1e-18, 1e-3, 1e3, 1e15])
def test_norm_magnitudes(gpu, orc, scale):
    """Squares that overflow or vanish in 32 bits; a zero row; a zero block."""
    rng = np.random.default_rng(6)
    x = (scale * rng.standard_normal((4, 2048))).astype(np.float32)
    x[1] = 0.0
    x[2, 256:512] = 0.0
    res = np.zeros_like(x)
    check(orc, call(gpu, x, res, None), x, res, None)


@pytest.mark.parametrize("cols", [512, 8448])
def test_norm_in_place_and_single_outputs(gpu, orc, cols):
    rng = np.random.default_rng(7)
    x, res = (rng.standard_normal((9, cols)).astype(np.float32) for _ in range(2))
    w = rng.standard_normal(cols).astype(np.float32)
    full = call(gpu, x, res, w)
    for want in (("res",), ("y",), ("q",), ("res", "q"), ("y", "q")):
        got = call(gpu, x, res, w, want)
        for k in got:
            assert np.array_equal(got[k], full[k]) if k in want else np.all(got[k] == 7), (want, k)
    for alias in ("x", "res"):
        d = dict(x=dev(gpu, x), res=dev(gpu, res))
        q = gpu.DeviceArray.zeros((9, cols // 256 * 292), np.uint8)
        gpu.add_rmsnorm_q8_K(d["x"], d["res"], dev(gpu, w), EPS, d[alias], None, q, 9, cols)
        assert np.array_equal(d[alias].numpy(), full["res"]) and np.array_equal(q.numpy(), full["q"])


def test_norm_rows_independent_of_batch(gpu):
    rng = np.random.default_rng(8)
    x, res = (rng.standard_normal((40, 2048)).astype(np.float32) for _ in range(2))
    all_ = call(gpu, x, res, None)
    one = call(gpu, x[17:18], res[17:18], None)
    for k in all_:
        assert np.array_equal(all_[k][17:18], one[k])
